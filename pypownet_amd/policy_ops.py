"""Operators of learned policies, as hand-written HIP kernels (include/ppn.h, "operators of learned policies").

A policy that acts on a ``BatchedRunEnv`` sees one observation row per environment and step; these are the parts of it that are
not plain matrix products:

* ``short_conv`` / ``short_conv_step``: short causal convolution over an environment's rows,
* ``selective_scan`` / ``selective_scan_step``: selective state space scan over an environment's rows (its memory),
* ``action_cross_entropy``: cross entropy over a catalogue of switching actions, without keeping the logits.

The window forms take ``[batch, time, ...]`` tensors of recorded rollouts -- any strides, so rollouts recorded step by step are passed as
``recorded.transpose(0, 1)`` -- and are differentiable; ``starts`` marks the first row of an episode, where memory begins empty.  The step
forms take one row of each listed environment and update that environment's state in place; they have no gradient.

Tensors are float32, bfloat16 or float16 on the GPU, all activations of a call of one type; parameters (convolution weights, ``A``, ``D``,
``dt_bias``) and states are float32 -- the convolution's window excepted, which holds rows and has their type.  Kernels are queued on torch's
current stream of the tensors' device; nothing synchronises.  Workspaces come from torch's allocator, so the calls can be captured into a
graph -- a training step as usual with its own leaves: capturing a backward pass of leaves that an eager graph still holds ends in an error of torch's
autograd, here as with any other function.  Arguments the kernels do not take are refused with TypeError / ValueError before anything is
launched; gradients of gradients, forward-mode derivatives and tracing are not available, and refused.
"""
import struct

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version
from torch.jit import is_tracing

from . import _lib
from .engine import EngineError

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_FLOAT = torch.float32
_packers = {name: struct.Struct('%dq' % len(fields)) for name, fields in _lib.POLICY_STRUCTS.items()}
_CONV, _CONV_STEP, _SCAN, _SCAN_STEP, _LOSS = (_packers[n] for n in ('ppn_conv_args', 'ppn_conv_step_args', 'ppn_scan_args', 'ppn_scan_step_args',
                                                                      'ppn_loss_args'))
# The blocks of the window forms in two parts: what the forward pass takes, and what only the backward pass does (from dy on; zeros forward).
_CONV_FRONT, _SCAN_FRONT = (struct.Struct('%dq' % _lib.POLICY_STRUCTS[n].index('dy')) for n in ('ppn_conv_args', 'ppn_scan_args'))
_CONV_BACK, _SCAN_BACK = struct.Struct('%dq' % ((_CONV.size - _CONV_FRONT.size) // 8)), struct.Struct('%dq' % ((_SCAN.size - _SCAN_FRONT.size) // 8))
_CONV_NO_BACK, _SCAN_NO_BACK = bytes(_CONV_BACK.size), bytes(_SCAN_BACK.size)
_library = None


def _load():
    global _library
    if _library is None:
        _library = _lib.load_library()
    return _library


def _call(function, packed, device):
    """Queues one entry point on torch's current stream of `device`."""
    index = device.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(device):
            rc = function(packed, _stream_of(index))
    else:
        rc = function(packed, _stream_of(index))
    if rc != 0:
        _refused(rc)


def _stream_of(index):
    return torch.cuda.current_stream(index).cuda_stream


# the same number without a Stream object around it (a fifth of a short call)
_stream_of = getattr(torch._C, '_cuda_getCurrentRawStream', _stream_of)


def _refused(rc):
    text = _load().ppn_policy_error().decode()
    raise (ValueError if rc == -1 else EngineError)(text)


_LAST_TWO = struct.Struct('2q')


def _with_workspace(size_of, function, packed, device):
    """Queues `function`, which needs as much memory as `size_of` says: the last two of its arguments."""
    size = size_of(packed)
    if size < 0:
        _refused(size)
    if size:
        work = torch.empty((size,), dtype=torch.uint8, device=device)
        packed = packed[:-16] + _LAST_TWO.pack(work.data_ptr(), size)
    _call(function, packed, device)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


# ---- arguments -----------------------------------------------------------------------------------------------------------------------

def _leading(name, x):
    """The tensor that names a call's type and device."""
    if isinstance(x, torch.Tensor) and x.is_cuda and x.dtype in _TYPES:
        return _TYPES[x.dtype]
    if not torch.is_tensor(x):
        raise TypeError('%s must be a torch tensor, got %s' % (name, type(x).__name__))
    if x.dtype not in _TYPES:
        raise TypeError('%s must be float32, bfloat16 or float16, got %s' % (name, x.dtype))
    raise ValueError('%s must live on a GPU: these operators have no CPU form' % name)


def _like(name, t, shape, dtype, device):
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.device == device:
        return
    if not torch.is_tensor(t):
        raise TypeError('%s must be a torch tensor, got %s' % (name, type(t).__name__))
    if t.dtype != dtype:
        raise TypeError('%s must be %s, got %s' % (name, dtype, t.dtype))
    raise ValueError('%s must be %s on %s, got %s on %s' % (name, list(shape), device, list(t.shape), t.device))


def _rows(t):
    """Neighbouring channels next to each other in memory, as the kernels read them; a copy where they are not."""
    return t if t.stride()[-1] == 1 or t.shape[-1] <= 1 else t.contiguous()


def _flags(name, t, shape, device):
    if t is None or isinstance(t, torch.Tensor) and t.dtype in (torch.bool, torch.uint8) and t.shape == shape and t.device == device:
        return t
    if not torch.is_tensor(t):
        raise TypeError('%s must be a torch tensor, got %s' % (name, type(t).__name__))
    if t.dtype not in (torch.bool, torch.uint8):
        raise TypeError('%s must be bool or uint8, got %s' % (name, t.dtype))
    raise ValueError('%s must be %s on %s, got %s on %s' % (name, list(shape), device, list(t.shape), t.device))


def _window_like(x):
    """An output with x's order in memory: time outermost where x has it outermost."""
    b, t, d = x.shape
    if x.is_contiguous():
        return torch.empty_like(x)
    if b > 1 and t > 1 and x.stride(0) < x.stride(1):
        return x.new_empty((t, b, d)).transpose(0, 1)
    return x.new_empty((b, t, d))


def _at(t):
    """Address, batch stride, time stride."""
    if t is None:
        return 0, 0, 0
    strides = t.stride()
    return t.data_ptr(), strides[0], strides[1]


def _wants_grad(*tensors):
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError('forward-mode derivatives are not available')
    if is_tracing():
        raise ValueError('these operators cannot be traced: their kernels are not torch operations')
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _window_rows(x):
    if x.dim() != 3 or x.shape[2] == 0:
        raise ValueError('x must be [batch, time, channels], got %s' % list(x.shape))
    return x.shape


def _step_rows(x):
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError('x must be [rows, channels], got %s' % list(x.shape))
    return x.shape


def _step_state(state, of):
    if not isinstance(state, torch.Tensor):
        raise TypeError('state must be a torch tensor, got %s' % type(state).__name__)
    if state.dim() != 3 or not state.is_contiguous():
        raise ValueError('state must be [environments, %s] and contiguous, got %s' % (of, list(state.shape)))
    return state.shape[0]


def _step_flags(starts, rows, device):
    return None if starts is None else _flags('starts', starts, (rows,), device).contiguous()


def _step_ids(env_ids, rows, environments, device):
    if env_ids is None:
        if rows > environments:
            raise ValueError('there are %d rows and %d environments: env_ids must say whose rows they are' % (rows, environments))
        return None
    if isinstance(env_ids, torch.Tensor) and env_ids.dtype is torch.int32 and env_ids.shape == (rows,) and env_ids.device == device and env_ids.is_contiguous():
        return env_ids
    if not torch.is_tensor(env_ids):
        raise TypeError('env_ids must be a torch tensor, got %s' % type(env_ids).__name__)
    if env_ids.dtype not in (torch.int32, torch.int64):
        raise TypeError('env_ids must be int32 or int64, got %s' % env_ids.dtype)
    if env_ids.device != device or tuple(env_ids.shape) != (rows,):
        raise ValueError('env_ids must be [%d] on %s, got %s on %s' % (rows, device, list(env_ids.shape), env_ids.device))
    if env_ids.dtype == torch.int64:
        # (an id that does not fit stays out of range instead of wrapping round to somebody's)
        env_ids = env_ids.clamp(-1, 2 ** 31 - 1).to(torch.int32)
    return env_ids.contiguous()


# ---- short causal convolution --------------------------------------------------------------------------------------------------------

def _conv_front(x, weight, bias, initial, starts, silu, y, final):
    b, t, d = x.shape
    return _CONV_FRONT.pack(_CONV.size, _TYPES[x.dtype], silu, b, t, d, weight.shape[1], *_at(x), weight.data_ptr(), 0 if bias is None else bias.data_ptr(),
                            0 if initial is None else initial.data_ptr(), *_at(starts), *_at(y), 0 if final is None else final.data_ptr())


def _conv_forward(x, weight, bias, initial, starts, silu, want_final):
    y = _window_like(x)
    final = x.new_empty((x.shape[0], weight.shape[1] - 1, x.shape[2])) if want_final else None
    _call(_load().ppn_conv_forward, _conv_front(x, weight, bias, initial, starts, silu, y, final) + _CONV_NO_BACK, x.device)
    return y, final


class _ShortConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, initial, starts, silu, want_final):
        ctx.set_materialize_grads(False)
        x, weight = _rows(x), weight.contiguous()
        bias, initial = (None if v is None else v.contiguous() for v in (bias, initial))
        ctx.save_for_backward(x, weight, bias, initial, starts)
        ctx.silu = silu
        return _conv_forward(x, weight, bias, initial, starts, silu, want_final)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dfinal):
        x, weight, bias, initial, starts = ctx.saved_tensors
        if dy is None and dfinal is None:
            return (None,) * 7
        dy = torch.zeros_like(x) if dy is None else _rows(dy)
        dfinal = None if dfinal is None else dfinal.contiguous()
        dx, dweight = _window_like(x), torch.empty_like(weight)
        dbias = None if bias is None else torch.empty_like(bias)
        dinitial = None if initial is None else torch.empty_like(initial)
        lib = _load()
        _with_workspace(lib.ppn_conv_backward_workspace, lib.ppn_conv_backward,
                        _conv_front(x, weight, bias, initial, starts, ctx.silu, None, None) +
                        _CONV_BACK.pack(*_at(dy), _ptr(dfinal), *_at(dx), dweight.data_ptr(), _ptr(dbias), _ptr(dinitial), 0, 0), x.device)
        return dx, dweight, dbias, dinitial, None, None, None


def _activation(activation):
    if activation not in (None, 'silu'):
        raise ValueError("activation must be None or 'silu', got %r" % (activation,))
    return 1 if activation else 0


def _conv_parameters(channels, weight, bias, device):
    if not (isinstance(weight, torch.Tensor) and weight.dim() == 2 and 2 <= weight.shape[1] <= 8):
        raise ValueError('weight must be a tensor [channels, taps] with 2 to 8 taps')
    taps = weight.shape[1]
    _like('weight', weight, (channels, taps), torch.float32, device)
    if bias is not None:
        _like('bias', bias, (channels,), torch.float32, device)
    return taps


def short_conv(x, weight, bias=None, activation=None, starts=None, initial_state=None, return_final_state=False):
    """``y[b,t,d] = act(bias[d] + sum_k weight[d,k] x[b, t - taps + 1 + k, d])`` over ``x [batch, time, channels]``; ``weight [channels, taps]``
    (2 to 8 taps) and ``bias [channels]`` in float32; ``activation`` None or 'silu'.

    ``initial_state [batch, taps - 1, channels]`` (x's type) holds the rows in front of the window, zeros when None; ``starts [batch, time]`` (bool /
    uint8) marks first rows of episodes, in front of which every tap is zero.  Returns y, or ``(y, final_state)``: the last ``taps - 1`` rows of the
    episode that is running at the window's end, i.e. the next window's ``initial_state`` and ``short_conv_step``'s state.  Differentiable in
    x, weight, bias and initial_state; the parameters' gradients are summed in a fixed order."""
    try:      # as it is mostly called; the rest is looked at one by one
        b, t, d = x.shape
        taps = weight.shape[1]
        dtype, device = x.dtype, x.device
        usual = (x.is_cuda and dtype in _TYPES and d > 0 and 2 <= taps <= 8 and weight.dtype is _FLOAT and weight.shape == (d, taps) and weight.device == device
                 and (bias is None or bias.dtype is _FLOAT and bias.shape == (d,) and bias.device == device)
                 and (initial_state is None or initial_state.dtype is dtype and initial_state.shape == (b, taps - 1, d) and initial_state.device == device))
    except (AttributeError, ValueError, IndexError):
        usual = False
    if not usual:
        _leading('x', x)
        b, t, d = _window_rows(x)
        device = x.device
        taps = _conv_parameters(d, weight, bias, device)
        if initial_state is not None:
            _like('initial_state', initial_state, (b, taps - 1, d), x.dtype, device)
    silu = _activation(activation)
    if starts is not None:
        starts = _flags('starts', starts, (b, t), device)
    if _wants_grad(x, weight, bias, initial_state):
        y, final = _ShortConv.apply(x, weight, bias, initial_state, starts, silu, bool(return_final_state))
    else:
        y, final = _conv_forward(_rows(x), weight.contiguous(), None if bias is None else bias.contiguous(),
                                 None if initial_state is None else initial_state.contiguous(), starts, silu, return_final_state)
    return (y, final) if return_final_state else y


def short_conv_step(x, state, weight, bias=None, activation=None, env_ids=None, starts=None):
    """One row of each of ``x``'s environments: ``x [rows, channels]``, ``state [environments, taps - 1, channels]`` (x's type, contiguous) moved on in
    place (a window that began with this very tensor cannot be learned from behind that: autograd raises), parameters as for ``short_conv``.  ``env_ids [rows]`` says whose rows they are (``BatchedRunEnv.recv``'s ids; row i is environment i when
    None); a negative id is padding: y = 0 and no state is touched.  An id out of range, or one that an earlier row has, gives NaN and touches no
    state.  ``starts [rows]`` empties the window first.  Returns y [rows, channels]."""
    try:      # as a loop calls it; the rest is looked at one by one
        n, d = x.shape
        environments, before, across = state.shape
        dtype, device = x.dtype, x.device
        usual = (x.is_cuda and dtype in _TYPES and d > 0 and 1 <= before <= 7 and across == d and state.dtype is dtype and state.device == device
                 and weight.dtype is _FLOAT and weight.shape == (d, before + 1) and weight.device == device and x.is_contiguous() and state.is_contiguous()
                 and weight.is_contiguous()
                 and (bias is None or bias.dtype is _FLOAT and bias.shape == (d,) and bias.device == device and bias.is_contiguous()))
    except (AttributeError, ValueError):
        usual = False
    if usual:
        y, row = torch.empty_like(x), d
    else:
        _leading('x', x)
        (n, d), device = _step_rows(x), x.device
        before = _conv_parameters(d, weight, bias, device) - 1
        environments = _step_state(state, 'taps - 1, channels')
        _like('state', state, (environments, before, d), x.dtype, device)
        x, weight, bias = _rows(x), weight.contiguous(), None if bias is None else bias.contiguous()
        y, row = x.new_empty((n, d)), x.stride(0)
    if _wants_grad(x, state, weight, bias):
        raise ValueError('short_conv_step has no gradient: call it under torch.no_grad(), or short_conv on the window')
    if starts is not None:
        starts = _step_flags(starts, n, device)
    if env_ids is not None or n > environments:
        env_ids = _step_ids(env_ids, n, environments, device)
    _call(_load().ppn_conv_step, _CONV_STEP.pack(_CONV_STEP.size, _TYPES[x.dtype], _activation(activation), n, environments, d, before + 1, x.data_ptr(), row,
                                                 weight.data_ptr(), 0 if bias is None else bias.data_ptr(), state.data_ptr(),
                                                 0 if env_ids is None else env_ids.data_ptr(), 0 if starts is None else starts.data_ptr(), y.data_ptr(), d), device)
    increment_version(state)      # (a window that began with this state and is still to be learned from has lost it: autograd says so)
    return y


# ---- selective scan ------------------------------------------------------------------------------------------------------------------

def _scan_front(x, dt, A, B, C, D, z, dt_bias, starts, initial, soft, y, final, marks):
    b, t, d = x.shape
    b_batch, b_time, b_group, _ = B.stride()
    c_batch, c_time, c_group, _ = C.stride()
    return _SCAN_FRONT.pack(_SCAN.size, _TYPES[x.dtype], soft, b, t, d, B.shape[2], A.shape[1], *_at(x), *_at(dt), A.data_ptr(), B.data_ptr(), b_batch,
                            b_time, b_group, C.data_ptr(), c_batch, c_time, c_group, _ptr(D), _ptr(dt_bias), *_at(z), *_at(starts), _ptr(initial), *_at(y),
                            _ptr(final), _ptr(marks))


_CHECKPOINT_ROWS = 8


def _scan_forward(inputs, want_final, train):
    x, A = inputs[0], inputs[2]
    lib = _load()
    y = _window_like(x)
    final = A.new_empty((x.shape[0], *A.shape)) if want_final else None
    marks = None
    if train:      # (ppn_scan_checkpoint_bytes)
        marks = A.new_empty((x.shape[0], -(-x.shape[1] // _CHECKPOINT_ROWS), A.shape[1], A.shape[0]))
    _with_workspace(lib.ppn_scan_forward_workspace, lib.ppn_scan_forward, _scan_front(*inputs, y, final, marks) + _SCAN_NO_BACK, x.device)
    return y, final, marks


def _scan_layout(x, dt, A, B, C, D, z, dt_bias, initial):
    return (_rows(x), _rows(dt), A.contiguous(), _rows(B), _rows(C), None if D is None else D.contiguous(), None if z is None else _rows(z),
            None if dt_bias is None else dt_bias.contiguous(), None if initial is None else initial.contiguous())


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, initial, starts, soft, want_final):
        ctx.set_materialize_grads(False)
        x, dt, A, B, C, D, z, dt_bias, initial = _scan_layout(x, dt, A, B, C, D, z, dt_bias, initial)
        y, final, marks = _scan_forward((x, dt, A, B, C, D, z, dt_bias, starts, initial, soft), want_final, True)
        # (the backward pass restarts from the checkpoints: the initial state itself may have moved on by then)
        ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, starts, marks)
        ctx.soft, ctx.begun = soft, initial is not None
        return y, final

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dfinal):
        x, dt, A, B, C, D, z, dt_bias, starts, marks = ctx.saved_tensors
        if dy is None and dfinal is None:
            return (None,) * 12
        dfinal = None if dfinal is None else dfinal.contiguous()
        dx, ddt, dz = _window_like(x), _window_like(dt), None if z is None else _window_like(z)
        dA, dD = torch.empty_like(A), None if D is None else torch.empty_like(D)
        dbias, dinitial = None if dt_bias is None else torch.empty_like(dt_bias), A.new_empty((x.shape[0], *A.shape)) if ctx.begun else None
        dB, dC = B.new_empty(B.shape), C.new_empty(C.shape)
        if x.shape[0] == 0 or x.shape[1] == 0:          # no rows: the state passes through
            for v in (dA, dD, dbias):
                if v is not None:
                    v.zero_()
            if dinitial is not None:
                dinitial.zero_() if dfinal is None else dinitial.copy_(dfinal)
            return dx, ddt, dA, dB, dC, dD, dz, dbias, dinitial, None, None, None
        dy = torch.zeros_like(x) if dy is None else _rows(dy)
        lib = _load()
        _with_workspace(lib.ppn_scan_backward_workspace, lib.ppn_scan_backward,
                        _scan_front(x, dt, A, B, C, D, z, dt_bias, starts, None, ctx.soft, None, None, marks) +
                        _SCAN_BACK.pack(*_at(dy), _ptr(dfinal), *_at(dx), *_at(ddt), *_at(dz), dB.data_ptr(), dC.data_ptr(), dA.data_ptr(), _ptr(dD), _ptr(dbias),
                                        _ptr(dinitial), 0, 0), x.device)
        return dx, ddt, dA, dB, dC, dD, dz, dbias, dinitial, None, None, None


def _scan_parameters(channels, A, D, dt_bias, device):
    if not (isinstance(A, torch.Tensor) and A.dim() == 2 and 1 <= A.shape[1] <= 64):
        raise ValueError('A must be a tensor [channels, states] with 1 to 64 states')
    states = A.shape[1]
    _like('A', A, (channels, states), torch.float32, device)
    if D is not None:
        _like('D', D, (channels,), torch.float32, device)
    if dt_bias is not None:
        _like('dt_bias', dt_bias, (channels,), torch.float32, device)
    return states


def _groups_of(channels, B, dims):
    if not (isinstance(B, torch.Tensor) and B.dim() == dims):
        raise ValueError('B must be a tensor of %d dimensions: [..., groups, states]' % dims)
    groups = B.shape[-2]
    if groups < 1 or channels % groups:
        raise ValueError('%d channels cannot be shared among %d groups of B and C' % (channels, groups))
    return groups


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, starts=None, initial_state=None, return_final_state=False):
    """Selective state space scan over ``x, dt, z [batch, time, channels]`` and ``B, C [batch, time, groups, states]`` (channel d uses group
    ``d // (channels // groups)``) of one type, with ``A [channels, states]``, ``D, dt_bias [channels]`` in float32, 1 to 64 states:

        delta = dt + dt_bias, then log(1 + e^delta) if dt_softplus
        h[t,d,n] = exp(delta A[d,n]) h[t-1,d,n] + delta B[t,g,n] x[t,d]
        y[t,d] = (sum_n C[t,g,n] h[t,d,n] + D[d] x[t,d]) * silu(z[t,d])           (the last factor only with z)

    ``initial_state [batch, channels, states]`` float32, zeros when None; h is zero in front of a row marked in ``starts [batch, time]``.  Returns y, or
    ``(y, final_state)``, the next window's ``initial_state`` and ``selective_scan_step``'s state.  Differentiable in every tensor but ``starts``; sums
    run in a fixed order, so gradients repeat bit for bit.  A differentiable call keeps the states in front of every 8th row for the backward pass.
    Rows of time may lie at most 2^27 elements apart in memory.  Where an input is infinite, what depends on it is infinite or NaN."""
    _leading('x', x)
    b, t, d = shape = _window_rows(x)
    dtype, device = x.dtype, x.device
    _like('dt', dt, shape, dtype, device)
    if z is not None:
        _like('z', z, shape, dtype, device)
    states, groups = _scan_parameters(d, A, D, dt_bias, device), _groups_of(d, B, 4)
    _like('B', B, (b, t, groups, states), dtype, device)
    _like('C', C, (b, t, groups, states), dtype, device)
    if initial_state is not None:
        _like('initial_state', initial_state, (b, d, states), torch.float32, device)
    if starts is not None:
        starts = _flags('starts', starts, (b, t), device)
    soft = 1 if dt_softplus else 0
    if _wants_grad(x, dt, A, B, C, D, z, dt_bias, initial_state):
        y, final = _SelectiveScan.apply(x, dt, A, B, C, D, z, dt_bias, initial_state, starts, soft, bool(return_final_state))
    else:
        x, dt, A, B, C, D, z, dt_bias, initial_state = _scan_layout(x, dt, A, B, C, D, z, dt_bias, initial_state)
        y, final, _ = _scan_forward((x, dt, A, B, C, D, z, dt_bias, starts, initial_state, soft), return_final_state, False)
    return (y, final) if return_final_state else y


def selective_scan_step(x, dt, A, B, C, state, D=None, z=None, dt_bias=None, dt_softplus=False, env_ids=None, starts=None):
    """One row of each of ``x``'s environments: ``x, dt, z [rows, channels]``, ``B, C [rows, groups, states]``, ``state [environments, channels, states]``
    (float32, contiguous) moved on in place; ``env_ids`` and ``starts`` as in ``short_conv_step``.  Returns y [rows, channels]."""
    try:      # as in short_conv_step
        n, d = rows = x.shape
        groups, states = B.shape[1:]
        environments = state.shape[0]
        dtype, device, cell = x.dtype, x.device, (d, states)
        usual = (x.is_cuda and dtype in _TYPES and d > 0 and groups > 0 and d % groups == 0 and 1 <= states <= 64 and x.is_contiguous()
                 and dt.dtype is dtype and dt.shape == rows and dt.device == device and dt.is_contiguous()
                 and A.dtype is _FLOAT and A.shape == cell and A.device == device and A.is_contiguous()
                 and B.dtype is dtype and B.shape[0] == n and B.device == device and B.stride()[2] == 1
                 and C.dtype is dtype and C.shape == B.shape and C.device == device and C.stride()[2] == 1
                 and state.dtype is _FLOAT and state.shape == (environments, d, states) and state.device == device and state.is_contiguous()
                 and (z is None or z.dtype is dtype and z.shape == rows and z.device == device and z.is_contiguous())
                 and (D is None or D.dtype is _FLOAT and D.shape == (d,) and D.device == device and D.is_contiguous())
                 and (dt_bias is None or dt_bias.dtype is _FLOAT and dt_bias.shape == (d,) and dt_bias.device == device and dt_bias.is_contiguous()))
    except (AttributeError, ValueError, TypeError):
        usual = False
    if usual:
        y, strides, gate = torch.empty_like(x), (d, d), d
    else:
        _leading('x', x)
        (n, d), dtype, device = _step_rows(x), x.dtype, x.device
        _like('dt', dt, (n, d), dtype, device)
        if z is not None:
            _like('z', z, (n, d), dtype, device)
        states, groups = _scan_parameters(d, A, D, dt_bias, device), _groups_of(d, B, 3)
        _like('B', B, (n, groups, states), dtype, device)
        _like('C', C, (n, groups, states), dtype, device)
        environments = _step_state(state, 'channels, states')
        _like('state', state, (environments, d, states), torch.float32, device)
        x, dt, A, B, C, D, z, dt_bias, _ = _scan_layout(x, dt, A, B, C, D, z, dt_bias, None)
        y, strides, gate = x.new_empty((n, d)), (x.stride(0), dt.stride(0)), 0 if z is None else z.stride(0)
    if _wants_grad(x, dt, A, B, C, D, z, dt_bias, state):
        raise ValueError('selective_scan_step has no gradient: call it under torch.no_grad(), or selective_scan on the window')
    if starts is not None:
        starts = _step_flags(starts, n, device)
    if env_ids is not None or n > environments:
        env_ids = _step_ids(env_ids, n, environments, device)
    b_row, b_group, _ = B.stride()
    c_row, c_group, _ = C.stride()
    _call(_load().ppn_scan_step,
          _SCAN_STEP.pack(_SCAN_STEP.size, _TYPES[dtype], 1 if dt_softplus else 0, n, environments, d, groups, states, x.data_ptr(), strides[0], dt.data_ptr(),
                          strides[1], A.data_ptr(), B.data_ptr(), b_row, b_group, C.data_ptr(), c_row, c_group, _ptr(D), _ptr(dt_bias), _ptr(z), gate,
                          state.data_ptr(), _ptr(env_ids), _ptr(starts), y.data_ptr(), d), device)
    increment_version(state)
    return y


# ---- cross entropy over a catalogue of actions -----------------------------------------------------------------------------------------

def _loss_args(hidden, weight, target, allowed, ignore, loss=None, lse=None, dloss=None, dhidden=None, dweight=None):
    return _LOSS.pack(_LOSS.size, _TYPES[hidden.dtype], hidden.shape[0], weight.shape[0], hidden.shape[1], ignore, hidden.data_ptr(), hidden.stride(0),
                      weight.data_ptr(), weight.stride(0), target.data_ptr(), _ptr(allowed), 0 if allowed is None else allowed.stride(0), _ptr(loss),
                      _ptr(lse), _ptr(dloss), _ptr(dhidden), _ptr(dweight), 0, 0)


def _loss_forward(hidden, weight, target, allowed, ignore):
    n, device = hidden.shape[0], hidden.device
    loss = torch.empty((n,), dtype=torch.float32, device=device)
    lse = torch.empty((n,), dtype=torch.float32, device=device)
    lib = _load()
    _with_workspace(lib.ppn_loss_forward_workspace, lib.ppn_loss_forward, _loss_args(hidden, weight, target, allowed, ignore, loss, lse), device)
    return loss, lse


class _ActionCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, target, allowed, ignore):
        hidden, weight = _rows(hidden), _rows(weight)
        loss, lse = _loss_forward(hidden, weight, target, allowed, ignore)
        ctx.save_for_backward(hidden, weight, target, allowed, loss, lse)
        ctx.ignore = ignore
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        hidden, weight, target, allowed, loss, lse = ctx.saved_tensors
        dhidden = hidden.new_empty(hidden.shape) if ctx.needs_input_grad[0] else None
        dweight = weight.new_empty(weight.shape) if ctx.needs_input_grad[1] else None
        if hidden.shape[0] == 0:
            return dhidden, None if dweight is None else dweight.zero_(), None, None, None
        dloss = dloss.contiguous()      # (a name of its own: the copy that sum() and mean() make needed has to outlive the launches)
        lib = _load()
        _with_workspace(lib.ppn_loss_backward_workspace, lib.ppn_loss_backward,
                        _loss_args(hidden, weight, target, allowed, ctx.ignore, loss, lse, dloss, dhidden, dweight), hidden.device)
        return dhidden, dweight, None, None, None


def action_cross_entropy(hidden, weight, target, allowed=None, ignore_index=-100):
    """Cross entropy of every row over a catalogue of actions, ``[rows]`` in float32, without keeping the logits:

        loss[i] = log sum_v exp(hidden[i] . weight[v]) - hidden[i] . weight[target[i]]          over the actions v that ``allowed`` has in row i

    ``hidden [rows, features]`` and ``weight [actions, features]`` of one type, ``target [rows]`` int64.  ``allowed [rows, ceil(actions / 32)]``
    int32 has one bit per action (``pack_allowed``; one row expanded over all is fine), all actions when None.  A row whose target is ``ignore_index``, or that allows nothing, has loss 0
    and no gradient; a target that is not allowed has loss +inf (its gradient is that of the logarithm alone); a target outside 0 .. actions - 1 gives
    NaN, and so does a row whose allowed logits are all -inf.  What a row does not allow is not looked at (behind the loss, a weight row that is not finite still makes NaN of dhidden).  ``-loss`` is the
    log-probability of the action ``target``.  Differentiable in hidden and weight (the result is kept for that: not to be changed in place); sums
    run in a fixed order.  The gradients are products of 16-bit operands where the tensors are 16-bit: the logits' gradient is rounded to that type in
    between (half a step of each entry, about as much again as the results' own rounding; in float16 entries below 2^-28 of
    the largest upstream gradient lose digits).

    Workspace behind the loss: about 0.5 GB, or 2 x 1024 x rows elements where that is more."""
    _leading('hidden', hidden)
    if hidden.dim() != 2 or hidden.shape[1] == 0:
        raise ValueError('hidden must be [rows, features], got %s' % list(hidden.shape))
    n, f = hidden.shape
    if not (isinstance(weight, torch.Tensor) and weight.dim() == 2 and weight.shape[0] > 0):
        raise ValueError('weight must be a tensor [actions, features]')
    v = weight.shape[0]
    _like('weight', weight, (v, f), hidden.dtype, hidden.device)
    _like('target', target, (n,), torch.int64, hidden.device)
    if allowed is not None:
        _like('allowed', allowed, (n, (v + 31) // 32), torch.int32, hidden.device)
        allowed = _rows(allowed)
        if 0 < allowed.stride(0) < allowed.shape[1]:      # (rows that overlap: the entry point takes rows apart, or one for all)
            allowed = allowed.contiguous()
    target = target.contiguous()
    ignore_index = int(ignore_index)
    if _wants_grad(hidden, weight):
        return _ActionCrossEntropy.apply(hidden, weight, target, allowed, ignore_index)
    return _loss_forward(_rows(hidden), _rows(weight), target, allowed, ignore_index)[0]


def pack_allowed(mask):
    """``mask [rows, actions]`` (bool) as the bits ``action_cross_entropy`` takes: int32 ``[rows, ceil(actions / 32)]``, action v in bit v % 32 of word v // 32."""
    if not (torch.is_tensor(mask) and mask.dim() == 2):
        raise ValueError('mask must be a tensor [rows, actions]')
    n, v = mask.shape
    words = (v + 31) // 32
    bits = torch.nn.functional.pad(mask != 0, (0, words * 32 - v)).view(n, words, 4, 8)
    place = torch.tensor([1 << i for i in range(8)], dtype=torch.uint8, device=mask.device)
    octets = (bits * place).sum(-1, dtype=torch.int32).to(torch.uint8)           # little-endian octets of a 32-bit word
    return octets.view(n, words * 4).contiguous().view(torch.int32) if words else octets.view(n, 0).to(torch.int32)
