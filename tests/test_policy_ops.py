"""The policy operators (pypownet_amd.policy_ops) against their definitions in 64 bits on the CPU, and what they refuse.

Tolerances.  A result is computed in 32 bits and rounded once to its type t: half a step of t relative to the value, `half(t)`.  In front of that, every
32-bit operation is off by at most 2^-24 of its result (the hardware's exp, log and reciprocal by at most twice that, plus 2^-24 of the exponential's
argument, which is below 8 in size here).  A result whose longest chain has c such operations, none of whose intermediate sums exceeds `size`, is
therefore within 2 c 2^-24 size; `size` is the same formula over absolute values, in 64 bits, or an upper bound of it."""
import os
import struct
import subprocess
import tempfile

import pytest
import torch

from conftest import ROOT

TYPES = [torch.float32, torch.bfloat16, torch.float16]
STEP = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def close(name, got, want, dtype, chain, size=None):
    got, want = got.detach().double().cpu(), want.detach().double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    if want.numel() == 0:
        return
    size = want.abs().max() if size is None else size
    smallest = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps           # (a step among the subnormal numbers)
    limit = half(dtype) * want.abs() * (1 + 2 * half(dtype)) + 2 * chain * STEP * size + smallest
    bad = ~((got - want).abs() <= limit) & ~(got == want) & ~(torch.isnan(got) & torch.isnan(want))
    assert not bad.any(), '%s: %d of %d off, worst %.3g at a limit of %.3g' % (
        name, int(bad.sum()), bad.numel(), float((got - want).abs()[bad].max()), float((limit * torch.ones_like(want))[bad].min()))


def rand(gen, *shape, scale=1.0, dtype=torch.float32):
    """Values that the type holds exactly, so that the reference sees the same inputs."""
    return (torch.randn(shape, generator=gen) * scale).to(dtype)


def on_gpu(*tensors, grad=False):
    out = []
    for t in tensors:
        if t is not None:
            t = t.cuda()
            if grad and t.is_floating_point():
                t.requires_grad_(True)
        out.append(t)
    return out


def wide(t):
    return None if t is None else t.double().requires_grad_(t.is_floating_point())


# ---- the definitions -----------------------------------------------------------------------------------------------------------------

def conv_definition(x, weight, bias, silu, starts, initial):
    b, t, d = x.shape
    k = weight.shape[1]
    window = torch.zeros((b, k - 1, d), dtype=torch.float64) if initial is None else initial
    ys = []
    for i in range(t):
        if starts is not None:
            window = torch.where(starts[:, i, None, None], torch.zeros_like(window), window)
        rows = torch.cat([window, x[:, i:i + 1]], 1)
        s = (rows * weight.t()).sum(1) + (0 if bias is None else bias)
        ys.append(s * torch.sigmoid(s) if silu else s)
        window = rows[:, 1:]
    y = torch.stack(ys, 1) if ys else torch.zeros_like(x)
    return y, window


def scan_definition(x, dt, A, B, C, D, z, dt_bias, soft, starts, initial):
    b, t, d = x.shape
    of = d // B.shape[2]
    h = torch.zeros((b, d, A.shape[1]), dtype=torch.float64) if initial is None else initial
    ys = []
    for i in range(t):
        delta = dt[:, i] + (0 if dt_bias is None else dt_bias)
        if soft:
            delta = torch.nn.functional.softplus(delta, threshold=1000)
        if starts is not None:
            h = torch.where(starts[:, i, None, None], torch.zeros_like(h), h)
        bb, cc = (v[:, i].repeat_interleave(of, 1) for v in (B, C))
        h = torch.exp(delta[..., None] * A) * h + (delta * x[:, i])[..., None] * bb
        y = (h * cc).sum(-1) + (0 if D is None else D * x[:, i])
        ys.append(y * z[:, i] * torch.sigmoid(z[:, i]) if z is not None else y)
    return (torch.stack(ys, 1) if ys else torch.zeros_like(x)), h


def loss_definition(hidden, weight, target, allowed, ignore=-100):
    logits = hidden @ weight.t()
    if allowed is not None:
        logits = logits.masked_fill(~allowed, -float('inf'))
    v = weight.shape[0]
    none = torch.zeros(len(target), dtype=torch.bool) if allowed is None else ~allowed.any(1)
    out = []
    for i in range(len(target)):
        t = int(target[i])
        if t == ignore or none[i]:
            out.append(torch.zeros((), dtype=torch.float64))
        elif not 0 <= t < v:
            out.append(logits[i][torch.isfinite(logits[i])].sum() * float('nan'))
        else:
            out.append(torch.logsumexp(logits[i], 0) - logits[i, t].detach().clone().fill_(-float('inf')) if torch.isinf(logits[i, t])
                       else torch.logsumexp(logits[i], 0) - logits[i, t])
    return torch.stack(out) if out else torch.zeros((0,), dtype=torch.float64)


# ---- what is refused (no GPU needed: nothing is launched) -----------------------------------------------------------------------------

def test_structs_match_the_header():
    from pypownet_amd import _lib
    prog = '#include <stdio.h>\n#include <stddef.h>\n#include "ppn.h"\nint main(void) {\n'
    for name, fields in _lib.POLICY_STRUCTS.items():
        prog += 'printf("%%zu", sizeof(%s));\n' % name
        for f in fields:
            prog += 'printf(" %%zu", offsetof(%s, %s));\n' % (name, f)
        prog += 'printf("\\n");\n'
    with tempfile.TemporaryDirectory() as d:
        open(os.path.join(d, 't.c'), 'w').write(prog + 'return 0;\n}\n')
        subprocess.check_call(['gcc', '-I', os.path.join(ROOT, 'include'), os.path.join(d, 't.c'), '-o', os.path.join(d, 't')])
        lines = subprocess.check_output([os.path.join(d, 't')]).decode().splitlines()
    for line, (name, fields) in zip(lines, _lib.POLICY_STRUCTS.items()):
        assert [int(v) for v in line.split()] == [8 * len(fields)] + [8 * i for i in range(len(fields))], name


def test_entry_points_refuse_a_bad_struct():
    import __graft_entry__ as g
    import struct
    from pypownet_amd import _lib
    g.build_hip()
    lib = _lib.load_library()
    calls = {'ppn_conv_args': ['ppn_conv_forward', 'ppn_conv_backward'], 'ppn_conv_step_args': ['ppn_conv_step'],
             'ppn_scan_args': ['ppn_scan_forward', 'ppn_scan_backward'], 'ppn_scan_step_args': ['ppn_scan_step'],
             'ppn_loss_args': ['ppn_loss_forward', 'ppn_loss_backward']}

    def packed(name, **values):
        fields = _lib.POLICY_STRUCTS[name]
        values.setdefault('struct_bytes', 8 * len(fields))
        assert set(values) <= set(fields)
        return struct.pack('%dq' % len(fields), *[values.get(f, 0) for f in fields])
    for name, functions in calls.items():
        for f in functions:
            assert getattr(lib, f)(packed(name, struct_bytes=8), None) == -1, f
            assert b'struct_bytes' in lib.ppn_policy_error()
            assert getattr(lib, f)(None, None) == -1, f
    conv = dict(batch=1, time=1, channels=4, taps=4)
    for bad in (dict(conv, taps=1), dict(conv, taps=9), dict(conv, type=3), dict(conv, batch=-1), dict(conv, channels=0), conv):
        assert lib.ppn_conv_forward(packed('ppn_conv_args', **bad), None) == -1, bad
    step = dict(rows=2, environments=1, channels=4, taps=4)
    for bad in (step, dict(step, environments=2), dict(step, rows=-1)):
        assert lib.ppn_conv_step(packed('ppn_conv_step_args', **bad), None) == -1, bad
    scan = dict(batch=1, time=1, channels=4, groups=1, states=4)
    for bad in (dict(scan, states=65), dict(scan, states=0), dict(scan, groups=3), dict(scan, groups=0), dict(scan, type=-1), scan):
        assert lib.ppn_scan_forward(packed('ppn_scan_args', **bad), None) == -1, bad
        assert lib.ppn_scan_backward(packed('ppn_scan_args', **bad), None) == -1, bad
    assert lib.ppn_scan_step(packed('ppn_scan_step_args', rows=2, environments=1, channels=4, groups=1, states=4), None) == -1
    loss = dict(rows=2, actions=40, features=4)
    for bad in (loss, dict(loss, actions=0), dict(loss, type=9), dict(loss, hidden=16, weight=16, target=16, loss=16, lse=16, allowed=16, allowed_row=1)):
        assert lib.ppn_loss_forward(packed('ppn_loss_args', **bad), None) == -1, bad
    # a workspace that is too small is refused, not overrun
    ready = dict(loss, hidden=16, weight=16, target=16, loss=16, lse=16, dloss=16, workspace=256, workspace_bytes=255, hidden_row=4, weight_row=4)
    assert lib.ppn_loss_forward(packed('ppn_loss_args', **ready), None) == -1 and b'workspace' in lib.ppn_policy_error()
    assert lib.ppn_loss_backward(packed('ppn_loss_args', **ready), None) == -1 and b'workspace' in lib.ppn_policy_error()


def packed_args(name, **values):
    from pypownet_amd import _lib
    fields = _lib.POLICY_STRUCTS[name]
    values.setdefault('struct_bytes', 8 * len(fields))
    assert set(values) <= set(fields)
    return struct.pack('%dq' % len(fields), *[values.get(f, 0) for f in fields])


def test_entry_points_refuse_what_is_too_large():
    """... before anything is launched: the pointers here are none."""
    from pypownet_amd import _lib
    lib = _lib.load_library()
    conv = dict(rows=1, environments=1 << 19, channels=4, taps=4, x=16, weight=16, y=16, state=16)
    scan = dict(rows=1, environments=1 << 19, channels=4, groups=1, states=4, x=16, dt=16, A=16, B=16, C=16, y=16, state=16)
    for name, function, values in (('ppn_conv_step_args', lib.ppn_conv_step, conv), ('ppn_scan_step_args', lib.ppn_scan_step, scan)):
        assert function(packed_args(name, **dict(values, rows=(1 << 18) + 1, env_ids=16)), None) == -1 and b'env_ids' in lib.ppn_policy_error()
        assert function(packed_args(name, **dict(values, rows=(1 << 19) + 1)), None) == -1 and b'more rows than environments' in lib.ppn_policy_error()
        assert function(packed_args(name, **dict(values, channels=(1 << 24) + 4)), None) == -1
    loss = dict(rows=1, actions=1, features=1)
    for field, most in (('rows', 22), ('actions', 23), ('features', 20)):
        args = packed_args('ppn_loss_args', **dict(loss, **{field: (1 << most) + 1}))
        assert lib.ppn_loss_forward(args, None) == -1 and ('2^%d %s' % (most, field)).encode() in lib.ppn_policy_error()
        assert lib.ppn_loss_forward_workspace(args) == -1 and lib.ppn_loss_backward_workspace(args) == -1
    window = dict(batch=1, time=1, channels=1, groups=1, states=1)
    for values in (dict(window, channels=(1 << 22) + 1), dict(window, x_time=(1 << 27) + 1), dict(window, states=65), dict(window, groups=2)):
        args = packed_args('ppn_scan_args', **values)
        assert lib.ppn_scan_forward(args, None) == -1 and lib.ppn_scan_backward_workspace(args) == -1 and lib.ppn_scan_checkpoint_bytes(args) == -1
    args = packed_args('ppn_conv_args', batch=(1 << 31) - 300, time=1, channels=1, taps=2, x=16, weight=16, y=16)
    assert lib.ppn_conv_forward(args, None) == -1 and b'environments' in lib.ppn_policy_error()


@pytest.mark.parametrize('shape', [(1, 1, 1, 1, 1), (3, 17, 200, 2, 12), (5, 8, 64, 1, 64), (2, 0, 7, 1, 3)])
def test_checkpoints_are_as_large_as_the_library_says(shape):
    from pypownet_amd import _lib, policy_ops as ops
    b, t, d, g, n = shape
    lib = _lib.load_library()
    args = packed_args('ppn_scan_args', batch=b, time=t, channels=d, groups=g, states=n)
    assert lib.ppn_scan_checkpoint_bytes(args) == 4 * b * -(-t // ops._CHECKPOINT_ROWS) * n * d


def test_policy_kernels_mir_has_no_vector_code_in_front_of_an_exec_restore():
    """The machine-IR lint of the engine's kernels over the policy operators' three units: the same compiler, the same hazard."""
    import sys
    if not os.path.exists(os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')):
        pytest.skip('no hipcc')
    r = subprocess.run([sys.executable, os.path.join(ROOT, 'tools', 'dev', 'mir_lint_exec_restore.py'), '--policy'], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.count(' 0 vector instruction(s) in front of one') == 3, r.stdout


def missing_waits(assembly):
    """Lines of one unit's assembly where a wait state is missing that the compiler does not add for inline assembly: a transfer into LDS needs one
    between a scalar write of M0 and itself, a memory operation in inline assembly five between a vector instruction's write of a scalar register and
    itself.  Instructions count as one, s_nop n as n + 1; what was written lately is followed along the branches."""
    import re

    def scalars(text):
        return [r for a, b, c in re.findall(r'\bs(?:\[(\d+):(\d+)\]|(\d+)\b)', text) for r in (range(int(a), int(b) + 1) if a else [int(c)])]
    lines, inline = [], False
    for line in assembly.splitlines():
        inline = '#ASMSTART' in line or inline and '#ASMEND' not in line
        text = line.split(';')[0].strip()
        if text.endswith(':') or text and not text.startswith('.'):
            op, _, rest = text.partition(' ')
            lines.append((text, op, [t.strip() for t in rest.split(',')], rest, inline))
    arriving, found, again = {}, set(), True      # label -> register (or 'm0') -> wait states since it was written, of the branches to it
    while again:
        again, since = False, {}
        for text, op, operands, rest, inline in lines:
            if op.endswith(':'):
                since = {r: min(since.get(r, 9), arriving.get(op[:-1], {}).get(r, 9)) for r in {*since, *arriving.get(op[:-1], {})}}
                continue
            if '_load_lds_' in op and 'm0' in since and since['m0'] < 1:
                found.add('M0: ' + text)
            if inline and op.startswith(('global_', 'buffer_', 'flat_', 'scratch_')) and any(r in since for r in scalars(rest)):
                found.add('vector write: ' + text)
            passed = int(operands[0], 0) + 1 if op == 's_nop' else 1
            since = {r: n + passed for r, n in since.items() if n + passed < 5}
            if op.startswith('v_'):
                since.update({r: 0 for r in scalars(operands[0]) + (scalars(operands[1]) if '_co_' in op else [])})
            elif op.startswith(('s_branch', 's_cbranch')):
                before = arriving.setdefault(operands[0], {})
                for r, n in since.items():
                    if n < before.get(r, 9):
                        before[r], again = n, True
                if op == 's_branch':
                    since = {}
            elif op == 's_endpgm':
                since = {}
            elif op.startswith('s_'):
                for r in scalars(operands[0]):
                    since.pop(r, None)
                if operands[0] == 'm0':
                    since['m0'] = 0
    return sorted(found)


def test_missing_waits_are_found():
    def asm(*lines):
        return '\n'.join([';;#ASMSTART', *lines, ';;#ASMEND'])
    move, load = 's_mov_b32 m0, s20', 'global_load_lds_dwordx4 v1, s[4:5]'
    assert len(missing_waits(asm(move, load))) == 1 and not missing_waits(asm(move, 's_nop 0', load)) and not missing_waits(asm(move, 'v_mov_b32 v2, 0', load))
    first = 'v_readfirstlane_b32 s5, v3\n'
    assert len(missing_waits(first + asm('s_nop 3', load))) == 1 and not missing_waits(first + asm('s_nop 4', load))
    assert not missing_waits(first + 's_add_u32 s5, s5, 4\n' + asm(load)) and not missing_waits('v_readfirstlane_b32 s6, v3\n' + asm(load))
    over = first + 's_branch .L1\n.L0:\n' + asm(load) + '\ns_endpgm\n.L1:\n'
    assert not missing_waits(over) and len(missing_waits(over + 's_cbranch_scc1 .L0\n')) == 1 and not missing_waits(over + 's_nop 3\ns_branch .L0\n')


def test_loss_kernels_assembly_has_its_wait_states(tmp_path):
    import __graft_entry__ as g
    hipcc = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')
    if not os.path.exists(hipcc):
        pytest.skip('no hipcc')
    csrc, out = os.path.join(ROOT, 'pypownet_amd', 'csrc'), str(tmp_path / 'unit.s')
    subprocess.run([hipcc, '--offload-arch=gfx950', '-O3', '-std=c++17', '-fPIC', *g.POLICY_FLAGS, '--cuda-device-only', '-S', os.path.join(csrc, 'ppn_loss.hip'),
                    '-o', out], check=True, stderr=subprocess.DEVNULL, timeout=300)
    assembly = open(out).read()
    assert assembly.count('global_load_lds_dwordx4') > 0 and missing_waits(assembly) == []
    for unit in g.POLICY_UNITS:      # (the only unit whose inline assembly reads or writes memory)
        text = open(os.path.join(csrc, unit + '.hip')).read()
        assert unit == 'ppn_loss' or not any(w in text for w in ('global_load', 'global_store', 'buffer_load', 'buffer_store')), unit


def test_cpu_tensors_are_refused():
    from pypownet_amd import policy_ops as ops
    x = torch.zeros((2, 3, 4))
    with pytest.raises(ValueError, match='GPU'):
        ops.short_conv(x, torch.zeros((4, 4)))
    with pytest.raises(ValueError, match='GPU'):
        ops.selective_scan(x, x, torch.zeros((4, 4)), torch.zeros((2, 3, 1, 4)), torch.zeros((2, 3, 1, 4)))
    with pytest.raises(ValueError, match='GPU'):
        ops.action_cross_entropy(torch.zeros((2, 4)), torch.zeros((5, 4)), torch.zeros((2,), dtype=torch.int64))
    with pytest.raises(TypeError):
        ops.short_conv([1.0], torch.zeros((4, 4)))
    with pytest.raises(TypeError, match='float32, bfloat16 or float16'):
        ops.short_conv(x.double(), torch.zeros((4, 4)))


def test_pack_allowed():
    from pypownet_amd import policy_ops as ops
    gen = torch.Generator().manual_seed(3)
    for n, v in ((0, 5), (3, 1), (4, 31), (5, 32), (2, 33), (3, 177), (2, 347)):
        mask = torch.rand((n, v), generator=gen) < 0.5
        bits = ops.pack_allowed(mask)
        assert bits.dtype == torch.int32 and bits.shape == (n, (v + 31) // 32)
        for i in range(n):
            for a in range(v):
                assert bool((int(bits[i, a >> 5]) >> (a & 31)) & 1) == bool(mask[i, a])
            if v % 32:
                assert (int(bits[i, -1]) & 0xffffffff) >> (v % 32) == 0


@pytest.mark.gpu
def test_gpu_arguments_are_refused():
    from pypownet_amd import policy_ops as ops
    f = lambda *s, **k: torch.zeros(s, device='cuda', **k)      # noqa: E731
    x, w = f(2, 3, 4), f(4, 4)
    bad = [
        (ValueError, lambda: ops.short_conv(f(3, 4), w)), (ValueError, lambda: ops.short_conv(x, f(4, 1))), (ValueError, lambda: ops.short_conv(x, f(4, 9))),
        (ValueError, lambda: ops.short_conv(x, f(5, 4))), (TypeError, lambda: ops.short_conv(x, w.half())), (ValueError, lambda: ops.short_conv(x, w, f(5))),
        (ValueError, lambda: ops.short_conv(x, w, activation='relu')), (ValueError, lambda: ops.short_conv(x, w.cpu())),
        (TypeError, lambda: ops.short_conv(x, w, starts=f(2, 3))), (ValueError, lambda: ops.short_conv(x, w, starts=f(3, 2, dtype=torch.bool))),
        (ValueError, lambda: ops.short_conv(x, w, initial_state=f(2, 4, 4))), (TypeError, lambda: ops.short_conv(x, w, initial_state=f(2, 3, 4).half())),
        (ValueError, lambda: ops.short_conv_step(f(5, 4), f(4, 3, 4), w)), (TypeError, lambda: ops.short_conv_step(f(5, 4), f(5, 3, 4).half(), w)),
        (ValueError, lambda: ops.short_conv_step(f(2, 4), f(3, 5, 4).transpose(0, 1)[:, :3], w)),
        (TypeError, lambda: ops.short_conv_step(f(2, 4), f(4, 3, 4), w, env_ids=f(2))),
        (ValueError, lambda: ops.short_conv_step(f(2, 4), f(4, 3, 4), w, env_ids=f(3, dtype=torch.int32))),
        (ValueError, lambda: ops.short_conv_step(f(2, 4).requires_grad_(), f(4, 3, 4), w)),
        (ValueError, lambda: ops.selective_scan(x, x, f(4, 65), f(2, 3, 1, 65), f(2, 3, 1, 65))),
        (ValueError, lambda: ops.selective_scan(x, x, w, f(2, 3, 3, 4), f(2, 3, 3, 4))), (ValueError, lambda: ops.selective_scan(x, x, w, f(2, 3, 4), f(2, 3, 4))),
        (ValueError, lambda: ops.selective_scan(x, f(2, 4, 4), w, f(2, 3, 1, 4), f(2, 3, 1, 4))),
        (TypeError, lambda: ops.selective_scan(x, x, w, f(2, 3, 1, 4).half(), f(2, 3, 1, 4))),
        (TypeError, lambda: ops.selective_scan(x, x, w.bfloat16(), f(2, 3, 1, 4), f(2, 3, 1, 4))),
        (ValueError, lambda: ops.selective_scan(x, x, w, f(2, 3, 1, 4), f(2, 3, 1, 4), initial_state=f(2, 4, 5))),
        (ValueError, lambda: ops.selective_scan_step(f(2, 4), f(2, 4), w, f(2, 1, 4), f(2, 1, 4), f(1, 4, 4))),
        (TypeError, lambda: ops.selective_scan_step(f(2, 4), f(2, 4), w, f(2, 1, 4), f(2, 1, 4), f(2, 4, 4).half())),
        (ValueError, lambda: ops.selective_scan_step(f(2, 4), f(2, 4), w.requires_grad_(), f(2, 1, 4), f(2, 1, 4), f(2, 4, 4))),
        (ValueError, lambda: ops.action_cross_entropy(f(2, 4), f(5, 3), f(2, dtype=torch.int64))),
        (TypeError, lambda: ops.action_cross_entropy(f(2, 4), f(5, 4), f(2, dtype=torch.int32))),
        (TypeError, lambda: ops.action_cross_entropy(f(2, 4), f(5, 4).half(), f(2, dtype=torch.int64))),
        (ValueError, lambda: ops.action_cross_entropy(f(2, 4), f(40, 4), f(2, dtype=torch.int64), allowed=f(2, 1, dtype=torch.int32))),
        (ValueError, lambda: ops.action_cross_entropy(f(2, 4), f(0, 4), f(2, dtype=torch.int64))),
    ]
    for i, (error, call) in enumerate(bad):
        with pytest.raises(error):
            call()
            pytest.fail('call %d was not refused' % i)


# ---- short causal convolution -----------------------------------------------------------------------------------------------------------

CONV = [  # batch, time, channels, taps, silu, bias, starts, initial, time_major
    (1, 1, 1, 2, False, False, False, False, False), (2, 5, 8, 4, True, True, True, True, False), (3, 67, 20, 3, True, True, True, True, True),
    (4, 33, 136, 4, True, False, True, False, True), (2, 3, 64, 8, False, True, True, True, False), (5, 130, 16, 5, True, True, False, True, False),
    (1, 300, 72, 6, True, True, True, True, False), (3, 16, 1032, 7, True, True, True, True, True), (2, 17, 520, 4, True, True, True, True, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('case', CONV, ids=str)
def test_gpu_short_conv(case, dtype):
    from pypownet_amd import policy_ops as ops
    b, t, d, k, silu, has_bias, has_starts, has_initial, time_major = case
    gen = torch.Generator().manual_seed(1)
    x = rand(gen, t, b, d, dtype=dtype).transpose(0, 1) if time_major else rand(gen, b, t, d, dtype=dtype)
    weight, bias = rand(gen, d, k, scale=0.5), rand(gen, d, scale=0.5) if has_bias else None
    initial = rand(gen, b, k - 1, d, dtype=dtype) if has_initial else None
    starts = torch.rand((b, t), generator=gen) < 0.15 if has_starts else None
    dy, dfinal = rand(gen, b, t, d, dtype=dtype), rand(gen, b, k - 1, d, dtype=dtype)
    ref = [wide(v) for v in (x, weight, bias, initial)]
    y64, last64 = conv_definition(ref[0], ref[1], ref[2], silu, starts, ref[3])
    leaves64 = [v for v in ref if v is not None]
    grads64 = torch.autograd.grad([y64, last64], leaves64, [dy.double(), dfinal.double()], allow_unused=True)
    gx = x.cuda() if not time_major else x.transpose(0, 1).cuda().transpose(0, 1)
    gx.requires_grad_(True)
    own = [gx] + on_gpu(weight, bias, initial, grad=True)
    kw = dict(activation='silu' if silu else None, starts=None if starts is None else starts.cuda(), initial_state=own[3], return_final_state=True)
    y, last = ops.short_conv(own[0], own[1], own[2], **kw)
    assert y.stride() == (gx.stride() if time_major and b > 1 and t > 1 else y.contiguous().stride())
    with torch.no_grad():
        again, _ = ops.short_conv(own[0], own[1], own[2], **kw)
    assert torch.equal(again, y)
    grads = torch.autograd.grad([y, last], [v for v in own if v is not None], [dy.cuda(), dfinal.cuda()])
    size = (float(x.abs().max()) * float(weight.abs().sum(1).max()) + 2) * (float(initial.abs().max()) + 1 if has_initial else 1)
    close('y', y, y64, dtype, 16 + k, size)
    assert torch.equal(last.cpu().double(), last64.detach()), 'final state'
    # a gradient of x sums k terms of |dy| |weight| (times silu', at most 1.1); one of a parameter sums b t terms
    up = 1.1 * float(dy.abs().max()) * float(weight.abs().sum(1).max()) * (1 + size) + float(dfinal.abs().max())
    names = ['dx', 'dweight'] + (['dbias'] if has_bias else []) + (['dinitial'] if has_initial else [])
    for name, got, want in zip(names, grads, grads64):
        want = torch.zeros(got.shape, dtype=torch.float64) if want is None else want
        if name in ('dx', 'dinitial'):
            close(name, got, want, dtype, 16 + 2 * k, up)
        else:
            close(name, got, want, torch.float32, 32 + 2 * k, b * t * 1.1 * (1 + size) * float(dy.abs().max()) * (1 + float(x.abs().max())))
    assert all(torch.equal(p, q) for p, q in zip(grads, torch.autograd.grad(
        ops.short_conv(own[0], own[1], own[2], **kw), [v for v in own if v is not None], [dy.cuda(), dfinal.cuda()])))


@pytest.mark.gpu
def test_gpu_short_conv_sizes_of_zero():
    from pypownet_amd import policy_ops as ops
    w = torch.randn((8, 4), device='cuda', requires_grad=True)
    init = torch.randn((2, 3, 8), device='cuda', requires_grad=True)
    for b, t in ((0, 5), (2, 0)):
        x = torch.zeros((b, t, 8), device='cuda', requires_grad=True)
        i = init[:b].detach().clone().requires_grad_(True)
        y, last = ops.short_conv(x, w, initial_state=i, return_final_state=True)
        assert y.shape == (b, t, 8)
        up = torch.randn_like(last)
        dx, dw, di = torch.autograd.grad([y, last], [x, w, i], [torch.zeros_like(y), up])
        assert dx.shape == x.shape and not dw.any()
        if t == 0:
            assert torch.equal(last, i) and torch.equal(di, up)
    state = torch.randn((4, 3, 8), device='cuda')
    kept = state.clone()
    assert ops.short_conv_step(torch.zeros((0, 8), device='cuda'), state, w.detach()).shape == (0, 8) and torch.equal(state, kept)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('d,k', [(1, 2), (24, 4), (250, 3), (1032, 8), (256, 4)])
def test_gpu_short_conv_step_follows_the_window(d, k, dtype):
    """Rows one by one through the step form leave what the window form leaves, bit for bit."""
    from pypownet_amd import policy_ops as ops
    gen = torch.Generator().manual_seed(2)
    b, t = 5, 9
    x, weight, bias = rand(gen, b, t, d, dtype=dtype).cuda(), rand(gen, d, k).cuda(), rand(gen, d).cuda()
    starts = (torch.rand((b, t), generator=gen) < 0.2).cuda()
    initial = rand(gen, b, k - 1, d, dtype=dtype).cuda()
    y, last = ops.short_conv(x, weight, bias, activation='silu', starts=starts, initial_state=initial, return_final_state=True)
    places = torch.tensor([6, 0, 3, 7, 2], device='cuda')
    state = torch.full((8, k - 1, d), 7.0, dtype=dtype, device='cuda')
    state[places] = initial
    for i in range(t):
        order = torch.randperm(b, generator=gen).cuda()
        row = ops.short_conv_step(x[order, i], state, weight, bias, activation='silu', env_ids=places[order], starts=starts[order, i])
        close('row %d' % i, row, y[order, i].double().cpu(), dtype, 16 + k, 40.0)
    assert torch.equal(state[places], last) and (state[[1, 4, 5]] == 7).all()


# ---- selective scan ---------------------------------------------------------------------------------------------------------------------

SCAN = [  # batch, time, channels, groups, states, D, z, dt_bias, softplus, starts, initial, time_major
    (1, 1, 1, 1, 1, False, False, False, False, False, False, False), (2, 7, 64, 1, 16, True, True, True, True, True, True, False),
    (3, 33, 70, 1, 12, True, True, True, True, True, True, True), (2, 50, 96, 3, 16, True, False, True, True, True, False, False),
    (2, 19, 40, 2, 32, False, True, False, True, True, True, True), (1, 24, 24, 1, 64, True, True, True, True, False, True, False),
    (1, 130, 130, 1, 8, True, True, True, True, True, True, False), (2, 65, 20, 1, 23, True, True, True, False, True, True, False),
    (1, 400, 32, 1, 16, True, True, True, True, True, True, False), (2, 9, 33, 1, 45, True, True, True, True, True, True, True),
    (1, 300, 20, 2, 40, True, True, True, True, True, True, False),
]


def scan_inputs(case, dtype, seed=5):
    b, t, d, g, n, has_D, has_z, has_bias, soft, has_starts, has_initial, time_major = case
    gen = torch.Generator().manual_seed(seed)

    def rows(*tail, scale=1.0):
        return rand(gen, t, b, *tail, scale=scale, dtype=dtype).transpose(0, 1) if time_major else rand(gen, b, t, *tail, scale=scale, dtype=dtype)
    v = dict(x=rows(d), dt=rows(d, scale=0.5) if soft else (rows(d, scale=0.2).abs()), A=-(torch.rand((d, n), generator=gen) * 4 + 0.05), B=rows(g, n), C=rows(g, n))
    v['D'] = rand(gen, d) if has_D else None
    v['z'] = rows(d) if has_z else None
    v['dt_bias'] = (rand(gen, d) - 2 if soft else rand(gen, d).abs() * 0.1) if has_bias else None
    v['initial'] = rand(gen, b, d, n) if has_initial else None
    starts = torch.rand((b, t), generator=gen) < 0.08 if has_starts else None
    return v, starts, rand(gen, b, t, d, dtype=dtype), rand(gen, b, d, n)


ORDER = ('x', 'dt', 'A', 'B', 'C', 'D', 'z', 'dt_bias', 'initial')


def own_scan(own, soft, starts):
    from pypownet_amd import policy_ops as ops
    return ops.selective_scan(own['x'], own['dt'], own['A'], own['B'], own['C'], D=own['D'], z=own['z'], dt_bias=own['dt_bias'], dt_softplus=soft,
                              starts=starts, initial_state=own['initial'], return_final_state=True)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('case', SCAN, ids=str)
def test_gpu_selective_scan(case, dtype):
    soft = case[8]
    v, starts, dy, dfinal = scan_inputs(case, dtype)
    ref = {k: wide(v[k]) for k in ORDER}
    y64, last64 = scan_definition(*[ref[k] for k in ORDER[:8]], soft, starts, ref['initial'])
    names = [k for k in ORDER if v[k] is not None]
    grads64 = torch.autograd.grad([y64, last64], [ref[k] for k in names], [dy.double(), dfinal.double()], allow_unused=True)
    # the same formulas over absolute values bound every partial sum
    big = {k: None if v[k] is None else (v[k].double().abs() if k not in ('A', 'dt', 'dt_bias', 'z') else v[k].double()).requires_grad_(True) for k in ORDER}
    if v['z'] is not None:
        big['z'] = v['z'].double().abs().requires_grad_(True)
    ybig, lastbig = scan_definition(*[big[k] for k in ORDER[:8]], soft, starts, big['initial'])
    gbig = torch.autograd.grad([ybig, lastbig], [big[k] for k in names], [dy.double().abs(), dfinal.double().abs()], allow_unused=True)
    own = {k: None if v[k] is None else v[k].transpose(0, 1).cuda().transpose(0, 1) if case[11] and v[k].dim() > 2 and k != 'initial' else v[k].cuda() for k in ORDER}
    for k in names:
        own[k].requires_grad_(True)
    gstarts = None if starts is None else starts.cuda()
    y, last = own_scan(own, soft, gstarts)
    with torch.no_grad():
        again, last_again = own_scan(own, soft, gstarts)
    assert torch.equal(again, y) and torch.equal(last_again, last), 'the form that keeps checkpoints differs'
    grads = torch.autograd.grad([y, last], [own[k] for k in names], [dy.cuda(), dfinal.cuda()])
    t, n = case[1], case[4]
    # a state's chain: per row one exponential (argument below 8: 8 steps, and its own) and two operations, but errors fade as the state does; 16 rows'
    # worth is what an average decay of exp(-0.3) leaves, and t rows bounds it
    chain = min(t, 64) * 12 + n + 32
    close('y', y, y64, dtype, chain, float(ybig.detach().abs().max()))
    close('final', last, last64, torch.float32, chain, float(lastbig.detach().abs().max()))
    for k, got, want, bound in zip(names, grads, grads64, gbig):
        want = torch.zeros(got.shape, dtype=torch.float64) if want is None else want
        size = max(float(want.abs().max()), 0.0 if bound is None else float(bound.abs().max()))
        close('d' + k, got, want, dtype if k in ('x', 'dt', 'B', 'C', 'z') else torch.float32, 2 * chain + 32, 3 * size)
    y2, last2 = own_scan(own, soft, gstarts)
    assert all(torch.equal(p, q) for p, q in zip(grads, torch.autograd.grad([y2, last2], [own[k] for k in names], [dy.cuda(), dfinal.cuda()])))


@pytest.mark.gpu
def test_gpu_selective_scan_against_differences():
    """A directional derivative of the kernel's own forward pass, in 32 bits: (f(+h) - f(-h)) / 2h over every input at once."""
    case = (2, 23, 12, 1, 6, True, True, True, True, True, True, False)
    v, starts, dy, dfinal = scan_inputs(case, torch.float32, seed=8)
    own = {k: v[k].cuda().requires_grad_(True) for k in ORDER}
    y, last = own_scan(own, True, starts.cuda())
    grads = torch.autograd.grad([y, last], [own[k] for k in ORDER], [dy.cuda(), dfinal.cuda()])
    gen = torch.Generator().manual_seed(9)
    move = {k: torch.randn(v[k].shape, generator=gen).cuda() for k in ORDER}
    slope = sum(float((g.double() * move[k].double()).sum()) for k, g in zip(ORDER, grads))
    step = 2.0 ** -8

    def value(s):
        with torch.no_grad():
            yy, ll = own_scan({k: own[k] + s * move[k] for k in ORDER}, True, starts.cuda())
        return float((yy.double() * dy.cuda().double()).sum() + (ll.double() * dfinal.cuda().double()).sum())
    # the difference's own error: third derivative times step^2 / 6 (of the order of the slope times 1e-4 here), and 32-bit rounding of f over 2 step
    assert abs((value(step) - value(-step)) / (2 * step) - slope) <= 4e-3 * sum(float((g.double().abs() * move[k].double().abs()).sum()) for k, g in zip(ORDER, grads))


@pytest.mark.gpu
def test_gpu_selective_scan_sizes_of_zero():
    from pypownet_amd import policy_ops as ops
    A = -torch.rand((8, 4), device='cuda') - 0.1
    A.requires_grad_(True)
    for b, t in ((0, 5), (2, 0)):
        x = torch.zeros((b, t, 8), device='cuda', requires_grad=True)
        bc = torch.zeros((b, t, 1, 4), device='cuda')
        init = torch.randn((b, 8, 4), device='cuda', requires_grad=True)
        y, last = ops.selective_scan(x, x, A, bc, bc, initial_state=init, return_final_state=True)
        assert y.shape == (b, t, 8) and torch.equal(last, init)
        up = torch.randn_like(last)
        dA, di = torch.autograd.grad([y, last], [A, init], [torch.zeros_like(y), up])
        assert not dA.any() and torch.equal(di, up)
    state = torch.randn((3, 8, 4), device='cuda')
    kept = state.clone()
    e = torch.zeros((0, 8), device='cuda')
    assert ops.selective_scan_step(e, e, A.detach(), torch.zeros((0, 1, 4), device='cuda'), torch.zeros((0, 1, 4), device='cuda'), state).shape == (0, 8)
    assert torch.equal(state, kept)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('d,g,n', [(1, 1, 1), (64, 1, 16), (70, 2, 12), (36, 1, 11), (20, 1, 64), (48, 1, 32), (513, 1, 4)])
def test_gpu_selective_scan_step_follows_the_window(d, g, n, dtype):
    from pypownet_amd import policy_ops as ops
    b, t = 5, 9
    v, starts, _, _ = scan_inputs((b, t, d, g, n, True, True, True, True, True, True, False), dtype, seed=11)
    own = {k: v[k].cuda() for k in ORDER}
    y, last = own_scan(own, True, starts.cuda())
    y64, last64 = scan_definition(*[None if v[k] is None else v[k].double() for k in ORDER[:8]], True, starts, v['initial'].double())
    places = torch.tensor([6, 0, 3, 7, 2], device='cuda', dtype=torch.int32)
    state = torch.full((8, d, n), 7.0, device='cuda')
    state[places.long()] = own['initial']
    gen = torch.Generator().manual_seed(12)
    size = float(y64.abs().max()) * (n + 4)
    for i in range(t):
        order = torch.randperm(b, generator=gen).cuda()
        row = ops.selective_scan_step(own['x'][order, i], own['dt'][order, i], own['A'], own['B'][order, i], own['C'][order, i], state, D=own['D'], z=own['z'][order, i],
                                      dt_bias=own['dt_bias'], dt_softplus=True, env_ids=places[order], starts=starts.cuda()[order, i])
        close('row %d' % i, row, y64[order.cpu(), i], dtype, 12 * t + n + 32, size)
    close('state', state[places.long()], last64, torch.float32, 12 * t + 32, float(last64.abs().max()) * 4)
    close('window', last, last64, torch.float32, 12 * t + 32, float(last64.abs().max()) * 4)
    assert (state[[1, 4, 5]] == 7).all()


@pytest.mark.gpu
def test_gpu_step_ids_padding_repeats_and_ranges():
    from pypownet_amd import policy_ops as ops
    n, d = 300, 24
    gen = torch.Generator().manual_seed(13)
    ids = torch.arange(n, dtype=torch.int32)
    ids[5], ids[17], ids[250], ids[260], ids[261] = -1, 400, 3, 100000, 250      # padding, out of range, a repeat, out of range; 250 itself is free
    x, w = rand(gen, n, d).cuda(), rand(gen, d, 4).cuda()
    conv = rand(gen, 300, 3, d).cuda()
    before = conv.clone()
    want = ops.short_conv_step(x, conv.clone(), w)
    y = ops.short_conv_step(x, conv, w, env_ids=ids.cuda())
    refused, padding = [17, 250, 260], [5]
    live = torch.ones(n, dtype=torch.bool)
    live[refused + padding] = False
    live[261] = False                                         # environment 250 seen through row 261: compared below
    assert torch.isnan(y[refused]).all() and not y[padding].any()
    assert torch.equal(y[live], want[live])
    assert torch.equal(conv[3, -1], x[3]) and torch.equal(conv[250, -1], x[261])
    for e in (5, 17, 260, 261):
        assert torch.equal(conv[e], before[e])
    A = -torch.rand((d, 8), generator=gen).cuda()
    bc = [rand(gen, n, 1, 8).cuda() for _ in range(2)]
    dt = rand(gen, n, d).cuda()
    state = rand(gen, 300, d, 8).cuda()
    before = state.clone()
    clean = state.clone()
    want = ops.selective_scan_step(x, dt, A, *bc, clean, dt_softplus=True)
    y = ops.selective_scan_step(x, dt, A, *bc, state, dt_softplus=True, env_ids=ids.long().cuda())
    assert torch.isnan(y[refused]).all() and not y[padding].any() and torch.equal(y[live], want[live]) and torch.equal(state[3], clean[3])
    for e in (5, 17, 260, 261):
        assert torch.equal(state[e], before[e])
    far = torch.tensor([2 ** 32 + 1, -2 ** 40], device='cuda')   # ids that 32 bits cannot hold
    y = ops.selective_scan_step(x[:2], dt[:2], A, bc[0][:2], bc[1][:2], state, env_ids=far)
    assert torch.isnan(y[0]).all() and not y[1].any()


@pytest.mark.gpu
def test_gpu_an_episode_does_not_see_the_one_before():
    """Infinities and NaN in front of a start reach nothing behind it, forward or backward; those behind it reach no gradient in front."""
    from pypownet_amd import policy_ops as ops
    b, t, d, n, at = 2, 40, 16, 16, 21
    v, _, dy, _ = scan_inputs((b, t, d, 1, n, True, True, True, True, False, True, False), torch.float32, seed=15)
    own = {k: v[k].cuda() for k in ORDER}
    starts = torch.zeros((b, t), dtype=torch.bool, device='cuda')
    starts[:, at] = True
    clean, _ = own_scan(own, True, starts)
    bad = dict(own, x=own['x'].clone(), initial=own['initial'] * float('inf'))
    bad['x'][:, at - 2] = float('nan')
    for k in ORDER:
        bad[k].requires_grad_(True)
    y, last = own_scan(bad, True, starts)
    assert torch.equal(y[:, at:], clean[:, at:]) and torch.isnan(y[:, at - 2]).all()
    only = torch.zeros_like(y)
    only[:, at:] = dy.cuda()[:, at:]
    dx, = torch.autograd.grad(y, [bad['x']], only, retain_graph=True)
    good = {k: own[k].detach().clone().requires_grad_(True) for k in ORDER}
    dx2, = torch.autograd.grad(own_scan(good, True, starts)[0], [good['x']], only)
    assert torch.equal(dx[:, at:], dx2[:, at:])
    w = torch.randn((d, 4), device='cuda')
    assert torch.equal(ops.short_conv(bad['x'].detach(), w, starts=starts)[:, at:], ops.short_conv(own['x'].detach(), w, starts=starts)[:, at:])


# ---- cross entropy ------------------------------------------------------------------------------------------------------------------------

LOSS = [  # rows, actions, features, masked
    (1, 1, 1, False), (3, 33, 17, True), (70, 177, 64, True), (64, 347, 96, False), (130, 500, 40, True), (257, 129, 128, True), (5, 3000, 32, True),
    (300, 2100, 200, True), (1100, 12099, 64, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('case', LOSS, ids=str)
def test_gpu_action_cross_entropy(case, dtype):
    from pypownet_amd import policy_ops as ops
    n, v, f, masked = case
    gen = torch.Generator().manual_seed(21)
    hidden, weight = rand(gen, n, f, dtype=dtype), rand(gen, v, f, scale=2 / f ** 0.5, dtype=dtype)
    target = torch.randint(0, v, (n,), generator=gen)
    allowed = None
    if masked:
        allowed = torch.rand((n, v), generator=gen) < 0.7
        allowed[torch.arange(n), target] = True
        allowed[n // 2] = False                       # nothing allowed
    if n > 3:
        target[n // 3] = -100
    dloss = rand(gen, n)
    ref = [wide(hidden), wide(weight)]
    loss64 = loss_definition(ref[0], ref[1], target, allowed)
    g64 = torch.autograd.grad(loss64, ref, dloss.double()) if loss64.requires_grad else [torch.zeros_like(r) for r in ref]
    own = on_gpu(hidden, weight, grad=True)
    bits = None if allowed is None else ops.pack_allowed(allowed.cuda())
    loss = ops.action_cross_entropy(own[0], own[1], target.cuda(), allowed=bits)
    with torch.no_grad():
        assert torch.equal(ops.action_cross_entropy(own[0], own[1], target.cuda(), allowed=bits), loss)
    size = (hidden.double().abs() @ weight.double().abs().t()).max()
    close('loss', loss, loss64, torch.float32, f + 64, float(size) + 16)
    grads = torch.autograd.grad(loss, own, dloss.cuda())
    with torch.no_grad():
        logits = hidden.double() @ weight.double().t()
        if allowed is not None:
            logits[~allowed] = -float('inf')
        p = torch.softmax(logits, 1).nan_to_num(0)
        counted = (target != -100) & (torch.ones(n, dtype=torch.bool) if allowed is None else allowed.any(1))
        one = torch.zeros_like(p)
        one[torch.arange(n), target.clamp(min=0)] = 1
        dl = (p - one).abs() * (dloss.double().abs() * counted)[:, None]
        # entries of dl: rounded to the type (below its normal range: by a step of the smallest, which the scale puts 2^28 below the largest |dloss|),
        # and off by the exponential's 32-bit error: a probability's by (f + 32) 2^-23 (size)
        each = half(dtype) * dl + (2 * (f + 32) * STEP * (float(size) + 16)) * p * (dloss.double().abs() * counted)[:, None]
        if dtype == torch.float16:
            each = each + float(dloss.abs().max()) * 2.0 ** -38 * counted[:, None]
        for name, got, want, slack, total in (('dhidden', grads[0], g64[0], each @ weight.double().abs(), dl @ weight.double().abs()),
                                              ('dweight', grads[1], g64[1], each.t() @ hidden.double().abs(), dl.t() @ hidden.double().abs())):
            limit = slack + half(dtype) * want.abs() * 1.01 + 2 * (max(n, v) + 8) * STEP * total + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
            off = (got.double().cpu() - want).abs()
            assert (off <= limit).all(), '%s: worst %.3g of its limit' % (name, float((off / limit).max()))
    if n > 3:
        assert not grads[0][n // 3].any()
    if masked:
        assert not grads[0][n // 2].any() and loss[n // 2] == 0
    again = torch.autograd.grad(ops.action_cross_entropy(own[0], own[1], target.cuda(), allowed=bits), own, dloss.cuda())
    assert all(torch.equal(a, b) for a, b in zip(again, grads))
    only, = torch.autograd.grad(ops.action_cross_entropy(own[0], own[1].detach(), target.cuda(), allowed=bits), own[:1], dloss.cuda())
    assert torch.equal(only, grads[0])
    only, = torch.autograd.grad(ops.action_cross_entropy(own[0].detach(), own[1], target.cuda(), allowed=bits), own[1:], dloss.cuda())
    assert torch.equal(only, grads[1])


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_gpu_action_cross_entropy_in_pieces(dtype):
    """So many logits that the backward pass takes the catalogue in several pieces, the last one shorter."""
    from pypownet_amd import policy_ops as ops
    gen = torch.Generator().manual_seed(25)
    n, v, f = 16400, 9001, 24
    hidden, weight = rand(gen, n, f, dtype=dtype), rand(gen, v, f, scale=0.3, dtype=dtype)
    target = torch.randint(0, v, (n,), generator=gen)
    dloss = rand(gen, n)
    own = on_gpu(hidden, weight, grad=True)
    loss = ops.action_cross_entropy(own[0], own[1], target.cuda())
    grads = torch.autograd.grad(loss, own, dloss.cuda())
    h, w, g = hidden.cuda().double(), weight.cuda().double(), dloss.cuda().double()[:, None]
    logits = h @ w.t()
    size = float((h.abs() @ w.abs().t()).max())
    p = torch.softmax(logits, 1)
    at = torch.arange(n, device='cuda')
    close('loss', loss, (torch.logsumexp(logits, 1) - logits[at, target.cuda()]).cpu(), torch.float32, f + 64, size + 16)
    p[at, target.cuda()] -= 1
    dl = p * g
    # as in test_gpu_action_cross_entropy, |p - one| being a probability's size or more
    each = (half(dtype) + 2 * (f + 32) * STEP * (size + 16)) * dl.abs() + (2 * (f + 32) * STEP * (size + 16)) * g.abs() * (p < 0)
    if dtype == torch.float16:
        each = each + float(dloss.abs().max()) * 2.0 ** -38
    for name, got, want, slack, total in (('dhidden', grads[0], dl @ w, each @ w.abs(), dl.abs() @ w.abs()),
                                          ('dweight', grads[1], dl.t().contiguous() @ h, each.t().contiguous() @ h.abs(), dl.abs().t().contiguous() @ h.abs())):
        limit = slack + half(dtype) * want.abs() * 1.01 + 2 * (n + 8) * STEP * total + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        off = (got.double() - want).abs()
        assert (off <= limit).all(), '%s: worst %.3g of its limit' % (name, float((off / limit).max()))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_gpu_action_cross_entropy_of_bad_targets_and_values(dtype):
    from pypownet_amd import policy_ops as ops
    gen = torch.Generator().manual_seed(22)
    n, v, f = 8, 100, 32
    hidden, weight = rand(gen, n, f, dtype=dtype).cuda(), rand(gen, v, f, scale=0.3, dtype=dtype).cuda()
    mask = torch.ones((n, v), dtype=torch.bool, device='cuda')
    mask[2, 7] = False
    target = torch.tensor([0, v, 7, -1, 99, -100, 5, 6], device='cuda')
    hidden[6] = float('nan')
    hidden.requires_grad_(True)
    loss = ops.action_cross_entropy(hidden, weight, target, allowed=ops.pack_allowed(mask))
    assert torch.isfinite(loss[[0, 4, 7]]).all() and torch.isnan(loss[[1, 3, 6]]).all() and loss[2] == float('inf') and loss[5] == 0
    dh, = torch.autograd.grad(loss, hidden, torch.ones_like(loss))
    assert torch.isfinite(dh[[0, 2, 4, 5, 7]]).all() and torch.isnan(dh[[1, 3, 6]]).all() and not dh[5].any()
    # logits far from zero: the maximum is taken out before the exponential
    far = torch.full((2, f), 30.0, dtype=dtype, device='cuda')
    loss = ops.action_cross_entropy(far, weight, torch.tensor([1, 2], device='cuda'))
    want = loss_definition(far.double().cpu(), weight.double().cpu(), torch.tensor([1, 2]), None)
    close('far', loss, want, torch.float32, f + 64, float((far.double().cpu().abs() @ weight.double().cpu().abs().t()).max()))
    ninf = weight.clone()
    ninf[3] = -float('inf')
    loss = ops.action_cross_entropy(far, ninf, torch.tensor([1, 2], device='cuda'))
    keep = [i for i in range(v) if i != 3]
    want = loss_definition(far.double().cpu(), weight.double().cpu()[keep], torch.tensor([1, 2]), None)
    close('a logit of -inf', loss, want, torch.float32, f + 64, float((far.double().cpu().abs() @ weight.double().cpu().abs().t()).max()))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_gpu_action_cross_entropy_strides_and_small_upstream(dtype):
    from pypownet_amd import policy_ops as ops
    gen = torch.Generator().manual_seed(23)
    n, v, f = 65, 177, 64
    h, w = rand(gen, n, f, dtype=dtype).cuda(), rand(gen, v, f, scale=0.3, dtype=dtype).cuda()
    target = torch.randint(0, v, (n,), generator=gen).cuda()
    base = ops.action_cross_entropy(h, w, target)
    wide_h = torch.full((n, f + 3), 9.0, dtype=dtype, device='cuda')
    wide_h[:, 2:2 + f] = h
    assert torch.equal(ops.action_cross_entropy(wide_h[:, 2:2 + f], w, target), base)
    assert torch.equal(ops.action_cross_entropy(h, w.t().contiguous().t(), target), base)
    assert torch.equal(ops.action_cross_entropy(h[:1].expand(n, f), w, target)[:1], base[:1])
    # upstream gradients of any size: the scale of dl follows them
    hs = h.clone().requires_grad_(True)
    ones, = torch.autograd.grad(ops.action_cross_entropy(hs, w, target), hs, torch.ones(n, device='cuda'))
    tiny, = torch.autograd.grad(ops.action_cross_entropy(hs, w, target), hs, torch.full((n,), 2.0 ** -10, device='cuda'))
    big = torch.finfo(dtype).smallest_normal
    keep = tiny.float().abs() > big
    assert keep.float().mean() > 0.5 and torch.equal((tiny.float() * 2 ** 10)[keep], ones.float()[keep])
    assert not torch.autograd.grad(ops.action_cross_entropy(hs, w, target), hs, torch.zeros(n, device='cuda'))[0].any()


# ---- streams, graphs, threads ---------------------------------------------------------------------------------------------------------------

def _block(leaves, starts, target, bits):
    """The three operators as a policy runs them: convolution, scan, loss."""
    from pypownet_amd import policy_ops as ops
    x, w, dt, A, B, C, head = leaves
    y = ops.short_conv(x, w, activation='silu', starts=starts)
    h = ops.selective_scan(y, dt, A, B, C, dt_softplus=True, starts=starts)
    return ops.action_cross_entropy(h.reshape(-1, h.shape[-1]), head, target, allowed=bits)


def _block_inputs(dtype=torch.float32, seed=31):
    from pypownet_amd import policy_ops as ops
    gen = torch.Generator().manual_seed(seed)
    b, t, d, n, v = 3, 40, 64, 16, 177
    leaves = [rand(gen, b, t, d, dtype=dtype), rand(gen, d, 4, scale=0.5), rand(gen, b, t, d, scale=0.5, dtype=dtype), -torch.rand((d, n), generator=gen) - 0.1,
              rand(gen, b, t, 1, n, dtype=dtype), rand(gen, b, t, 1, n, dtype=dtype), rand(gen, v, d, scale=0.2, dtype=dtype)]
    leaves = [v_.cuda().requires_grad_(True) for v_ in leaves]
    starts = (torch.rand((b, t), generator=gen) < 0.1).cuda()
    target = torch.randint(0, v, (b * t,), generator=gen)
    mask = torch.rand((b * t, v), generator=gen) < 0.8
    mask[torch.arange(b * t), target] = True
    return leaves, starts, target.cuda(), ops.pack_allowed(mask.cuda())


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_gpu_operators_together(dtype):
    leaves, starts, target, bits = _block_inputs(dtype)
    loss = _block(leaves, starts, target, bits)
    grads = torch.autograd.grad(loss.mean(), leaves)
    ref = [v.detach().cpu().double().requires_grad_(True) for v in leaves]
    y = conv_definition(ref[0], ref[1], None, True, starts.cpu(), None)[0]
    h = scan_definition(y, ref[2], ref[3], ref[4], ref[5], None, None, None, True, starts.cpu(), None)[0]
    place = torch.arange(32)
    mask = ((bits.cpu()[..., None] >> place) & 1).bool().view(len(target), -1)[:, :ref[6].shape[0]]
    want = loss_definition(h.reshape(-1, h.shape[-1]), ref[6], target.cpu(), mask)
    g64 = torch.autograd.grad(want.mean(), ref)
    # two roundings to the type between the operators (y, h) reach the logits through |head|, the gradients through their own formulas: the
    # relative error of a whole tensor stays within a few half steps
    assert ((loss.detach().cpu().double() - want).norm() / want.norm()) < 8 * half(dtype) + 1e-5
    for got, ref_g in zip(grads, g64):
        assert ((got.cpu().double() - ref_g).norm() / ref_g.norm()) < 16 * half(dtype) + 1e-5


@pytest.mark.gpu
def test_gpu_operators_on_another_stream_and_from_two_threads():
    import threading
    leaves, starts, target, bits = _block_inputs()
    want = torch.autograd.grad(_block(leaves, starts, target, bits).sum(), leaves)
    torch.cuda.synchronize()
    results, errors = {}, []

    def run(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(5):
                    mine = [v.detach().clone().requires_grad_(True) for v in leaves]
                    results[i] = torch.autograd.grad(_block(mine, starts, target, bits).sum(), mine)
            stream.synchronize()
        except Exception as e:                                   # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors, errors
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(results[i], want))


@pytest.mark.gpu
def test_gpu_operators_in_a_graph():
    """Captured forward and backward, replayed between eager calls of the same operators, and two graphs whose workspaces must not meet."""
    leaves, starts, target, bits = _block_inputs()
    inputs = [[v.detach().clone().requires_grad_(True) for v in leaves] for _ in range(2)]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(2):
            torch.autograd.grad(_block(inputs[i], starts, target, bits).sum(), inputs[i])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            loss = _block(inputs[i], starts, target, bits)
            outs.append((loss.detach(), torch.autograd.grad(loss, inputs[i], torch.ones_like(loss))))
        graphs.append(g)
    gen = torch.Generator().manual_seed(33)
    for turn in range(4):
        fresh = [[(torch.randn(v.shape, generator=gen) * 0.3).cuda() if j not in (1, 3) else v.detach().clone() for j, v in enumerate(leaves)] for _ in range(2)]
        for i in range(2):
            with torch.no_grad():
                for dst, src in zip(inputs[i], fresh[i]):
                    dst.copy_(src)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            mine = [v.detach().clone().requires_grad_(True) for v in fresh[i]]
            loss = _block(mine, starts, target, bits)
            want = torch.autograd.grad(loss, mine, torch.ones_like(loss))
            assert torch.equal(outs[i][0], loss.detach()), (turn, i)
            assert all(torch.equal(a, b) for a, b in zip(outs[i][1], want)), (turn, i)


@pytest.mark.gpu
def test_gpu_step_in_a_graph():
    from pypownet_amd import policy_ops as ops
    gen = torch.Generator().manual_seed(35)
    n, d, m = 37, 64, 16
    x, w, dt = (rand(gen, *s).cuda() for s in ((n, d), (d, 4), (n, d)))
    A, bc = -torch.rand((d, m), generator=gen).cuda(), rand(gen, n, 1, m).cuda()
    ids = torch.randperm(64, generator=gen)[:n].to(torch.int32).cuda()
    conv, state = rand(gen, 64, 3, d).cuda(), rand(gen, 64, d, m).cuda()

    def step(c, s):
        return ops.selective_scan_step(ops.short_conv_step(x, c, w, env_ids=ids), dt, A, bc, bc, s, dt_softplus=True, env_ids=ids)
    eager_c, eager_s = conv.clone(), state.clone()
    step(conv.clone(), state.clone())
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = step(conv, state)
    for _ in range(4):
        x.copy_(rand(gen, n, d).cuda())
        g.replay()
        want = step(eager_c, eager_s)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(conv, eager_c) and torch.equal(state, eager_s)


@pytest.mark.gpu
def test_gpu_gradients_of_gradients_are_refused():
    """A graph of the backward pass may be asked for (the gradients are the same); differentiating through it is an error, not a wrong number."""
    from pypownet_amd import policy_ops as ops
    leaves, starts, target, bits = _block_inputs()
    want = torch.autograd.grad(_block(leaves, starts, target, bits).sum(), leaves)
    got = torch.autograd.grad(_block(leaves, starts, target, bits).sum(), leaves, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(got[0].sum(), leaves[0])
    gen = torch.Generator().manual_seed(41)
    h, w = rand(gen, 5, 8).cuda().requires_grad_(True), rand(gen, 9, 8).cuda().requires_grad_(True)
    dh, = torch.autograd.grad(ops.action_cross_entropy(h, w, torch.arange(5, device='cuda')).sum(), h, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dh.sum(), h)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_gpu_a_state_stepped_between_a_window_and_its_backward_pass(dtype):
    """The convolution's backward pass reads its initial rows again: moving them on in between is an error, as with torch's own operations in place.  The
    scan's does not: its gradients are those of the state the window began with."""
    from pypownet_amd import policy_ops as ops
    gen = torch.Generator().manual_seed(41)
    b, t, d, n = 3, 11, 24, 8
    x, w = rand(gen, b, t, d, dtype=dtype).cuda().requires_grad_(True), rand(gen, d, 4).cuda().requires_grad_(True)
    window = rand(gen, b, 3, d, dtype=dtype).cuda()
    y = ops.short_conv(x, w, activation='silu', initial_state=window)
    ops.short_conv_step(x.detach()[:, 0], window, w.detach(), activation='silu')
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.float().sum().backward()
    A, bc = -torch.rand((d, n), generator=gen).cuda().requires_grad_(True) - 0.1, [rand(gen, b, t, 1, n, dtype=dtype).cuda() for _ in range(2)]
    first = rand(gen, b, d, n).cuda()
    for stepped in (False, True):
        state = first.clone().requires_grad_(True)
        y = ops.selective_scan(x, x, A, *bc, dt_softplus=True, initial_state=state)
        before = state._version
        if stepped:
            with torch.no_grad():
                ops.selective_scan_step(x.detach()[:, 0], x.detach()[:, 0], A.detach(), bc[0][:, 0], bc[1][:, 0], state, dt_softplus=True)
            assert state._version > before
        grads = torch.autograd.grad(y, [x, state], torch.ones_like(y))
        if stepped:
            assert all(torch.equal(p, q) for p, q in zip(grads, kept))
        kept = grads
    with torch.inference_mode():      # (a tensor without a version counter)
        ops.short_conv_step(x.detach()[:, 0], torch.zeros((b, 3, d), dtype=dtype, device='cuda'), w.detach())


@pytest.mark.gpu
def test_gpu_forward_mode_derivatives_and_tracing_are_refused():
    """... not answered without the tangent, or with a recording that holds no kernel."""
    import torch.autograd.forward_ad as forward
    from pypownet_amd import policy_ops as ops
    r = lambda *s: torch.randn(s, device='cuda')      # noqa: E731
    x, row, w, A, bc, bc_row = r(2, 5, 8), r(2, 8), r(8, 4), -torch.rand((8, 4), device='cuda'), r(2, 5, 1, 4), r(2, 1, 4)
    target = torch.zeros((2,), dtype=torch.int64, device='cuda')
    calls = {
        'conv': (lambda v: ops.short_conv(v, w), x), 'conv weight': (lambda v: ops.short_conv(x, v), w), 'conv step': (lambda v: ops.short_conv_step(v, r(2, 3, 8), w), row),
        'scan': (lambda v: ops.selective_scan(v, x, A, bc, bc), x), 'scan D': (lambda v: ops.selective_scan(x, x, A, bc, bc, D=v), r(8)),
        'scan step': (lambda v: ops.selective_scan_step(v, row, A, bc_row, bc_row, r(2, 8, 4)), row),
        'scan state': (lambda v: ops.selective_scan_step(row, row, A, bc_row, bc_row, v), r(2, 8, 4)),
        'loss': (lambda v: ops.action_cross_entropy(v, r(6, 8), target), row),
    }
    for name, (call, v) in calls.items():
        plain = call(v.clone())
        for mode in (torch.no_grad(), torch.enable_grad()):
            with mode, forward.dual_level():
                with pytest.raises(ValueError, match='forward-mode'):
                    call(forward.make_dual(v.clone(), torch.ones_like(v)))
                    pytest.fail(name)
                assert call(v.clone()).shape == plain.shape      # (a level without a tangent of ours is no reason to refuse)
        with pytest.raises(Exception):
            torch.func.jvp(call, (v.clone(),), (torch.ones_like(v),))
            pytest.fail(name)
        with pytest.raises(ValueError, match='traced'), torch.no_grad():
            torch.jit.trace(call, (v.clone(),), check_trace=False)
            pytest.fail(name)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_gpu_action_cross_entropy_with_one_mask_for_all_rows(dtype):
    """A row of bits expanded over the rows, or rows of bits that overlap, are as good as copies of them."""
    from pypownet_amd import policy_ops as ops
    gen = torch.Generator().manual_seed(42)
    n, v, f = 70, 177, 40
    h, w = rand(gen, n, f, dtype=dtype).cuda().requires_grad_(True), rand(gen, v, f, scale=0.3, dtype=dtype).cuda().requires_grad_(True)
    mask = torch.rand((1, v), generator=gen) < 0.6
    mask[0, 5] = True
    target, up = torch.full((n,), 5, device='cuda'), rand(gen, n).cuda()
    one = ops.pack_allowed(mask.cuda())
    words = torch.randint(-2 ** 31, 2 ** 31, (n + 5,), generator=gen).to(torch.int32).cuda() | 32
    for bits in (one.expand(n, -1), words.as_strided((n, 6), (1, 1)), one.expand(n, -1)[:1]):
        rows = bits.shape[0]
        loss = ops.action_cross_entropy(h[:rows], w, target[:rows], allowed=bits)
        want = ops.action_cross_entropy(h[:rows], w, target[:rows], allowed=bits.contiguous().clone())
        assert torch.equal(loss, want) and torch.isfinite(loss).all()
        assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(loss, [h, w], up[:rows]), torch.autograd.grad(want, [h, w], up[:rows])))


@pytest.mark.gpu
@pytest.mark.parametrize('v', [3, 200, 20000])
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_gpu_action_cross_entropy_where_every_allowed_logit_is_minus_infinity(dtype, v):
    """... is not a row that allows nothing: its loss is not defined, and says so."""
    from pypownet_amd import policy_ops as ops
    gen = torch.Generator().manual_seed(43)
    n, f = 260, 24
    h, w = rand(gen, n, f, dtype=dtype).abs() + 0.125, rand(gen, v, f, scale=0.3, dtype=dtype)
    w[1:] = -float('inf')                                     # action 0 alone has a finite logit
    mask = torch.rand((n, v), generator=gen) < 0.5
    mask[:, 1] = True
    mask[:, 0] = torch.arange(n) % 3 != 0
    mask[7] = False
    mask[8] = torch.arange(v) == 1
    target = torch.zeros((n,), dtype=torch.int64)
    target[4] = 1
    target[mask[:, 0].logical_not()] = 1
    target[7], target[10] = 1, -100
    want = loss_definition(h.double(), w.double(), target, mask)
    lost = torch.isnan(want)
    assert lost[3] and lost[8] and want[7] == 0 and want[10] == 0 and want[4] == float('inf') and want[5] == 0
    hg = h.cuda().requires_grad_(True)
    loss = ops.action_cross_entropy(hg, w.cuda(), target.cuda(), allowed=ops.pack_allowed(mask.cuda()))
    got = loss.detach().double().cpu()
    assert torch.equal(torch.isnan(got), lost)
    # (the logarithm of one exponential: zero but for the rounding of logits below 16 in size, summed over 24 features)
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and (got[torch.isfinite(want)].abs() <= 2 * (f + 16) * STEP * 16).all()


@pytest.mark.gpu
@pytest.mark.parametrize('t,n', [(1, 16), (5, 12), (13, 16), (16, 16), (61, 16), (61, 40)])
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_gpu_selective_scan_rows_past_the_last_one_do_not_count(dtype, t, n):
    """Lengths that are no multiple of a block: a last row that is infinite, and channels that forget at once (A = -infinity), keep their values."""
    case = (2, t, 70, 1, n, True, True, True, True, False, True, False)
    v, _, dy, dfinal = scan_inputs(case, dtype, seed=44)
    v['B'], v['C'], v['D'], v['z'] = v['B'].abs(), v['C'].abs(), v['D'].abs(), v['z'].abs() + 0.5
    v['A'][3] = -float('inf')
    if n == 16:      # (elsewhere an infinity times the zeros that fill the last lane's states is NaN)
        v['x'][1, -1, 5] = float('inf')
    y64, last64 = scan_definition(*[v[k].double() for k in ORDER[:8]], True, None, v['initial'].double())
    assert torch.isinf(y64[1, -1, 5]) == (n == 16) and torch.isfinite(y64[:, :, 3]).all()
    own = {k: v[k].cuda().requires_grad_(True) for k in ORDER}
    chain = min(t, 64) * 12 + n + 32
    for keep in (False, True):
        with torch.set_grad_enabled(keep):
            y, last = own_scan(own, True, None)
        close('y', y, y64, dtype, chain, 4 * float(y64[torch.isfinite(y64)].abs().max()))
        close('final', last, last64, torch.float32, chain, 4 * float(last64[torch.isfinite(last64)].abs().max()))
    # behind the infinity nothing is finite, but for the channel that forgets in the other environment
    ref = {k: v[k].double() for k in ORDER}
    ref['x'].requires_grad_(True)
    y64, last64 = scan_definition(*[ref[k] for k in ORDER[:8]], True, None, ref['initial'])
    want, = torch.autograd.grad([y64, last64], ref['x'], [dy.double(), dfinal.double()])
    got, = torch.autograd.grad([y, last], own['x'], [dy.cuda(), dfinal.cuda()])
    assert torch.isfinite(want[0, :, 3]).all()
    close('dx', got[0, :, 3], want[0, :, 3], dtype, 2 * chain + 32, 8 * float(want[0].abs().max()))


@pytest.mark.gpu
@pytest.mark.parametrize('t', [48, 300, 1000])
def test_gpu_selective_scan_chunks_that_grow(t):
    """A state that grows by e^6 a row: what a chunk of rows does to a state outgrows 32 bits, but the states and gradients do not, since they are zero for so long
    (in front of the last eight rows, and behind the first eight)."""
    b, d, n = 1, 40, 8
    gen = torch.Generator().manual_seed(45)
    v = dict(x=rand(gen, b, t, d), dt=torch.ones((b, t, d)), A=5.9 + 0.1 * torch.rand((d, n), generator=gen), B=rand(gen, b, t, 1, n), C=rand(gen, b, t, 1, n))
    v.update({k: None for k in ORDER if k not in v})
    v['x'][:, :-8] = 0
    dy = rand(gen, b, t, d)
    y64, last64 = scan_definition(*[None if v[k] is None else v[k].double() for k in ORDER[:8]], False, None, None)
    own = {k: None if v[k] is None else v[k].cuda().requires_grad_(True) for k in ORDER}
    y, last = own_scan(own, False, None)
    assert not y[:, :-8].any()
    # eight rows of an exponential (argument 6) and two operations; sums of 8
    big = float(y64.abs().max())
    close('y', y, y64, torch.float32, 8 * 12 + n + 32, 4 * big)
    close('final', last, last64, torch.float32, 8 * 12 + 32, 4 * float(last64.abs().max()))
    with torch.no_grad():
        assert torch.equal(own_scan(own, False, None)[0], y)
    # gradients: those of the first eight rows' outputs (behind them there is none, in front of them no state)
    up = dy.clone()
    up[:, 8:] = 0
    names = ['x', 'dt', 'A', 'B', 'C']
    ref = {k: v[k].double().requires_grad_(True) for k in names}
    yr, _ = scan_definition(*[ref.get(k) for k in ORDER[:8]], False, None, None)
    want = torch.autograd.grad(yr, [ref[k] for k in names], up.double())
    got = torch.autograd.grad(y, [own[k] for k in names], up.cuda())
    for k, p, q in zip(names, got, want):
        close('d' + k, p, q, torch.float32, 2 * (8 * 12 + n + 32), 8 * float(want[0].abs().max()) + float(q.abs().max()))


def test_entry_points_refuse_what_no_launch_can_hold():
    """2^32 lanes along an axis, before anything is launched: the pointers here are none."""
    from pypownet_amd import _lib
    lib = _lib.load_library()
    step = dict(rows=1 << 24, environments=1 << 24, channels=4, x=16, y=16, state=16)
    assert lib.ppn_conv_step(packed_args('ppn_conv_step_args', taps=4, weight=16, **step), None) == -1 and b'rows' in lib.ppn_policy_error()
    assert lib.ppn_scan_step(packed_args('ppn_scan_step_args', groups=1, states=4, dt=16, A=16, B=16, C=16, **step), None) == -1 and b'rows' in lib.ppn_policy_error()
    conv = dict(batch=1 << 26, time=1, channels=1, taps=2, x=16, weight=16, y=16)
    assert lib.ppn_conv_forward(packed_args('ppn_conv_args', **conv), None) == -1 and b'environments' in lib.ppn_policy_error()
    scan = dict(channels=1, groups=1, states=1, x=16, dt=16, A=16, B=16, C=16, y=16, dy=16, dx=16, ddt=16, dB=16, dC=16, checkpoints=16, workspace=256, workspace_bytes=1 << 62)
    for sizes in (dict(batch=1 << 26, time=1), dict(batch=1 << 15, time=1 << 15)):
        if sizes['time'] == 1:
            assert lib.ppn_scan_forward(packed_args('ppn_scan_args', **scan, **sizes), None) == -1 and b'environments' in lib.ppn_policy_error()
        assert lib.ppn_scan_backward(packed_args('ppn_scan_args', **scan, **sizes), None) == -1 and b'rows' in lib.ppn_policy_error()
    loss = dict(hidden=16, weight=16, target=16, loss=16, lse=16, dloss=16, dhidden=16, dweight=16, workspace=256, workspace_bytes=1 << 62)
    for rows, actions, features, backward in ((1 << 22, 1 << 18, 8, False), (1, 1 << 23, 1023, True), (1 << 22, 1 << 10, 1 << 14, True)):
        args = packed_args('ppn_loss_args', rows=rows, actions=actions, features=features, hidden_row=features, weight_row=features, **loss)
        calls = [lib.ppn_loss_backward] if backward else []
        if actions != 1 << 10:
            calls.append(lib.ppn_loss_forward)
        for call in calls:
            assert call(args, None) == -1 and b'too many rows' in lib.ppn_policy_error(), (rows, actions, features)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('d,k,silu', [(1, 2, True), (24, 4, True), (250, 3, False), (1032, 8, True), (256, 4, True), (512, 5, False)])
def test_gpu_short_conv_step_is_the_window_bit_for_bit(d, k, silu, dtype):
    from pypownet_amd import policy_ops as ops
    gen = torch.Generator().manual_seed(46)
    b, t = 3, 9
    x, weight, bias = rand(gen, b, t, d, dtype=dtype).cuda(), rand(gen, d, k).cuda(), rand(gen, d).cuda()
    starts, state = (torch.rand((b, t), generator=gen) < 0.2).cuda(), rand(gen, b, k - 1, d, dtype=dtype).cuda()
    activation = 'silu' if silu else None
    y = ops.short_conv(x, weight, bias, activation=activation, starts=starts, initial_state=state)
    for i in range(t):
        assert torch.equal(ops.short_conv_step(x[:, i], state, weight, bias, activation=activation, starts=starts[:, i]), y[:, i]), i


@pytest.mark.parametrize('kind,size', [(0, 4), (1, 2), (2, 2)])
def test_the_loss_workspace_stays_within_what_is_said(kind, size):
    """Backward: copies of both operands (twice where their rows are not whole 16 bytes), dl and its transpose, 32-bit sums."""
    from pypownet_amd import _lib
    lib = _lib.load_library()
    for rows in (1, 63, 256, 4096, 16384, 20480, 61440, 131072, 245760, 1 << 22):
        for actions in (1, 347, 12099, 24129, 1 << 20):
            for features in (24, 64, 250, 512, 4096):
                args = packed_args('ppn_loss_args', type=kind, rows=rows, actions=actions, features=features, hidden=16, weight=16, hidden_row=features,
                                   weight_row=features)
                up = lambda v, to: -(-v // to) * to      # noqa: E731
                operands = (up(rows, 64) + up(actions, 64)) * up(features, 8) * size * 2
                # (a piece is a multiple of 128 actions, so up to 127 more rows of the transpose)
                dl = 2 * max((256 << 20) + 128 * up(rows, 64) * size, 1024 * up(rows, 64) * size)
                piece = min(up(actions, 64), max(1024, up((256 << 20) // (up(rows, 64) * size), 128)))
                sums = max(128 << 20, 4 * (rows + piece) * features)
                assert 0 < lib.ppn_loss_backward_workspace(args) <= operands + dl + sums + 4096, (rows, actions, features)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_gpu_action_cross_entropy_of_many_rows(dtype):
    """A window of thousands of environments: pieces of the catalogue at their smallest, the inner dimension of dweight's product at its longest."""
    from pypownet_amd import policy_ops as ops
    gen = torch.Generator().manual_seed(47)
    n, v, f = 140003, 1100, 24
    hidden, weight = rand(gen, n, f, dtype=dtype).cuda(), rand(gen, v, f, scale=0.3, dtype=dtype).cuda()
    target, dloss = torch.randint(0, v, (n,), generator=gen).cuda(), rand(gen, n).cuda()
    own = [hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)]
    loss = ops.action_cross_entropy(own[0], own[1], target)
    grads = torch.autograd.grad(loss, own, dloss)
    h, w, g = hidden.double(), weight.double(), dloss.double()[:, None]
    size = max(float((h[i:i + 20000].abs() @ w.abs().t()).max()) for i in range(0, n, 20000))
    slack_w, total_w, want_w = (torch.zeros((v, f), dtype=torch.float64, device='cuda') for _ in range(3))
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    probability = 2 * (f + 32) * STEP * (size + 16)      # (limits as in test_gpu_action_cross_entropy_in_pieces)
    for i in range(0, n, 20000):
        rows = slice(i, min(n, i + 20000))
        logits = h[rows] @ w.t()
        p, at = torch.softmax(logits, 1), torch.arange(logits.shape[0], device='cuda')
        close('loss', loss[rows], (torch.logsumexp(logits, 1) - logits[at, target[rows]]).cpu(), torch.float32, f + 64, size + 16)
        p[at, target[rows]] -= 1
        dl = p * g[rows]
        each = (half(dtype) + probability) * dl.abs() + probability * g[rows].abs() * (p < 0)
        if dtype == torch.float16:
            each = each + float(dloss.abs().max()) * 2.0 ** -38
        want = dl @ w
        limit = each @ w.abs() + half(dtype) * want.abs() * 1.01 + 2 * (v + 8) * STEP * (dl.abs() @ w.abs()) + tiny
        assert ((grads[0][rows].double() - want).abs() <= limit).all()
        slack_w += each.t().contiguous() @ h[rows].abs()
        total_w += dl.abs().t().contiguous() @ h[rows].abs()
        want_w += dl.t().contiguous() @ h[rows]
    limit = slack_w + half(dtype) * want_w.abs() * 1.01 + 2 * (n + 8) * STEP * total_w + tiny
    assert ((grads[1].double() - want_w).abs() <= limit).all()


def _one_free_block():
    """Small tensors in every free place of torch's small memory but one segment: what is allocated and freed there next is what is allocated behind it."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    kept, reserved = [], torch.cuda.memory_reserved()
    while torch.cuda.memory_reserved() == reserved:
        kept.append(torch.empty((512,), dtype=torch.uint8, device='cuda'))
    kept.pop()
    return kept


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('n,v,f', [(7, 40, 25), (300, 177, 65), (2000, 347, 64)])
def test_gpu_upstream_gradients_that_are_no_memory_of_their_own(n, v, f, dtype):
    """sum() and mean() hand back one number expanded over the rows, a slice of a larger gradient has strides: the copy that is made of it lives as long as
    the kernels that read it are queued."""
    from pypownet_amd import policy_ops as ops
    gen = torch.Generator().manual_seed(49)
    h, w = rand(gen, n, f, dtype=dtype).cuda().requires_grad_(True), rand(gen, v, f, scale=0.3, dtype=dtype).cuda().requires_grad_(True)
    target, wide_up = torch.randint(0, v, (n,), generator=gen).cuda(), rand(gen, n, 3).cuda()
    x, weight = rand(gen, 3, n, 24, dtype=dtype).cuda().requires_grad_(True), rand(gen, 24, 4).cuda().requires_grad_(True)
    state, A = rand(gen, 3, 24, 8).cuda().requires_grad_(True), (-torch.rand((24, 8), generator=gen) - 0.1).cuda().requires_grad_(True)
    bc = rand(gen, 3, n, 1, 8, dtype=dtype).cuda().requires_grad_(True)

    def conv():
        return ops.short_conv(x, weight, activation='silu', initial_state=x[:, :3], return_final_state=True)

    def scan():
        return ops.selective_scan(x, x, A, bc, bc, dt_softplus=True, initial_state=state, return_final_state=True)
    loss = lambda: (ops.action_cross_entropy(h, w, target),)      # noqa: E731
    one = torch.ones((), device='cuda')
    for call, leaves in ((loss, [h, w]), (conv, [x, weight]), (scan, [x, A, bc, state])):
        for k in range(3):
            outs = call()
            ups = [one.to(o.dtype).expand_as(o) if k < 2 else wide_up[:, 1] if o.dim() == 1 else rand(gen, *o.shape[::-1], dtype=o.dtype).cuda().permute(2, 1, 0) for o in outs]
            kept = [u.contiguous().clone() for u in ups]
            want = torch.autograd.grad(outs, leaves, kept)
            del outs
            outs = call()
            full = _one_free_block() if k == 1 else None
            got = torch.autograd.grad(outs, leaves, ups)
            del full, outs
            assert all(torch.equal(p, q) for p, q in zip(got, want)), (call, k)
    for reduce, up in ((lambda y: y.sum(), torch.ones((n,), device='cuda')), (lambda y: y.mean(), torch.full((n,), 1.0, device='cuda') / n)):
        want = torch.autograd.grad(loss()[0], [h, w], up)
        reduced = reduce(loss()[0])
        full = _one_free_block()
        got = torch.autograd.grad(reduced, [h, w])
        del full
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def _far(t, stride):
    """The same values with what lies along the first axis `stride` elements apart."""
    far = torch.empty(((t.shape[0] - 1) * stride + t[0].numel(),), dtype=t.dtype, device='cuda').as_strided(t.shape, (stride, *t[0].contiguous().stride()))
    return far.copy_(t)


@pytest.mark.gpu
def test_gpu_offsets_past_32_bits():
    """Environments, rows and states more than 2^32 bytes apart in memory are the same as close together."""
    from pypownet_amd import policy_ops as ops
    gen = torch.Generator().manual_seed(48)
    dtype, apart = torch.bfloat16, (1 << 31) + 64
    b, t, d, n = 3, 13, 256, 16
    v = dict(x=rand(gen, b, t, d, dtype=dtype), dt=rand(gen, b, t, d, dtype=dtype), B=rand(gen, b, t, 1, n, dtype=dtype), C=rand(gen, b, t, 1, n, dtype=dtype))
    w, A, up, starts = rand(gen, d, 4).cuda(), -torch.rand((d, n), generator=gen).cuda() - 0.1, rand(gen, b, t, d, dtype=dtype), torch.rand((b, t), generator=gen) < 0.1
    close_by, far = [{k: put(q.cuda()) for k, q in v.items()} for put in (lambda q: q.clone(), lambda q: _far(q, apart))]
    up, starts = [up.cuda(), _far(up.cuda(), apart)], [starts.cuda(), _far(starts.cuda(), 1 << 32)]
    results = []
    for u, s, up_, starts_ in ((close_by, 0, *(q[0] for q in (up, starts))), (far, 1, *(q[1] for q in (up, starts)))):
        for q in u.values():
            q.requires_grad_(True)
        y = ops.short_conv(u['x'], w, activation='silu', starts=starts_)
        h = ops.selective_scan(u['x'], u['dt'], A, u['B'], u['C'], dt_softplus=True, starts=starts_)
        results.append([y, h, *torch.autograd.grad(y, u['x'], up_), *torch.autograd.grad(h, list(u.values()), up_)])
    assert all(torch.equal(p, q) for p, q in zip(*results))
    del far, up, starts, results, u, up_, starts_, y, h
    # one row of environments far into a state
    environments = (1 << 32) // (d * n * 4) + 3
    state, window = torch.zeros((environments, d, n), device='cuda'), torch.zeros(((1 << 32) // (3 * d * 2) + 3, 3, d), dtype=dtype, device='cuda')
    rows = [v[k][:2, 0].cuda() for k in ('x', 'dt', 'B', 'C')]
    for big, call in ((state, lambda s, ids: ops.selective_scan_step(*rows[:2], A, *rows[2:], s, dt_softplus=True, env_ids=ids)),
                      (window, lambda s, ids: ops.short_conv_step(rows[0], s, w, env_ids=ids))):
        last = big.shape[0] - 1
        big[last] = rand(gen, *big.shape[1:], dtype=big.dtype).cuda()
        small = big[[0, last]].contiguous()
        assert torch.equal(call(big, torch.tensor([0, last], device='cuda')), call(small, None)) and torch.equal(big[[0, last]], small)
        assert not big[1:last].any()
    del state, window, big
    rows, actions, f = 300, 177, 64
    h, weight, target = rand(gen, rows, f, dtype=dtype).cuda(), rand(gen, actions, f, dtype=dtype).cuda(), torch.randint(0, actions, (rows,), generator=gen).cuda()
    bits = ops.pack_allowed(torch.ones((rows, actions), dtype=torch.bool, device='cuda'))
    results = []
    for hh, ww, bb in ((h.clone(), weight.clone(), bits), (_far(h, 1 << 23), _far(weight, 1 << 23), _far(bits, 1 << 23)), (_far(h, (1 << 23) + 8), _far(weight, (1 << 23) + 8), bits)):
        hh.requires_grad_(True), ww.requires_grad_(True)
        loss = ops.action_cross_entropy(hh, ww, target, allowed=bb)
        results.append([loss, *torch.autograd.grad(loss.sum(), [hh, ww])])
        del hh, ww, bb
    assert all(torch.equal(p, q) for p, q in zip(results[0], results[1])) and all(torch.equal(p, q) for p, q in zip(results[0], results[2]))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_gpu_results_do_not_depend_on_what_memory_held(dtype):
    """Outputs, workspaces and checkpoints out of memory full of zeros, of NaN and of large numbers: the same bits."""
    from pypownet_amd import policy_ops as ops
    gen = torch.Generator().manual_seed(50)

    def fill(byte):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        kept = [torch.full((1 << k,), byte, dtype=torch.uint8, device='cuda') for k in (9, 12, 14, 16, 17, 18, 19, 20, 21, 22, 23, 24, 26) for _ in range(8)]
        del kept
    calls = []
    for b, t, d, k in ((3, 67, 20, 3), (2, 17, 520, 4), (5, 40, 136, 5)):
        x, w, up = (q.cuda().requires_grad_(True) for q in (rand(gen, b, t, d, dtype=dtype), rand(gen, d, k), rand(gen, b, t, d, dtype=dtype)))
        starts = (torch.rand((b, t), generator=gen) < 0.1).cuda()
        calls.append((lambda x, w, s=starts: ops.short_conv(x, w, activation='silu', starts=s), [x, w], up))
    for case in (SCAN[2], SCAN[3], SCAN[8], SCAN[10]):
        v, starts, dy, _ = scan_inputs(case, dtype)
        names = [k for k in ORDER if v[k] is not None]
        leaves = [v[k].cuda().requires_grad_(True) for k in names]

        def scan(*leaves, names=names, soft=case[8], starts=None if starts is None else starts.cuda()):
            return own_scan({**dict.fromkeys(ORDER), **dict(zip(names, leaves))}, soft, starts)[0]
        calls.append((scan, leaves, dy.cuda()))
    for n, actions, f in ((65, 40, 25), (300, 177, 64), (700, 1100, 72)):
        h, w, up = (q.cuda().requires_grad_(True) for q in (rand(gen, n, f, dtype=dtype), rand(gen, actions, f, scale=0.3, dtype=dtype), rand(gen, n)))
        target = torch.randint(0, actions, (n,), generator=gen)
        mask = torch.rand((n, actions), generator=gen) < 0.7
        mask[torch.arange(n), target] = True
        calls.append((lambda h, w, t=target.cuda(), m=ops.pack_allowed(mask.cuda()): ops.action_cross_entropy(h, w, t, allowed=m), [h, w], up))
    for call, leaves, up in calls:
        results = []
        for byte in (0, 0xff, 0x41):
            fill(byte)
            y = call(*leaves)
            fill(byte)
            results.append([y.detach(), *torch.autograd.grad(y, leaves, up.detach())])
        assert torch.isfinite(results[0][0]).all()
        assert all(torch.equal(p, q) for other in results[1:] for p, q in zip(results[0], other))
