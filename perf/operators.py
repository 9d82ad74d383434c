"""The operators of learned switching policies, as cases to be measured.

A policy that acts on a batch of grids remembers what it has seen (a short causal convolution and a selective state
space scan over the rows an environment has shown) and chooses from a catalogue of switching actions (one line, or one
substation's node configuration: 12099 entries on the 118-bus grid with node configurations counted up to relabelling of
the two nodes, 24129 with every switch pattern).  Its training reads recorded rollouts: `batch` environments, `time` rows
each, an episode's first row marked in `starts`; its acting form takes one row of every environment that is due.

    conv        y[t] = silu(bias + sum_k w[k] x[t - K + 1 + k])      taps in front of the episode's first row are zero
    scan        h[t] = exp(d[t] A) h[t - 1] + d[t] B[t] x[t],  d = softplus(dt + dt_bias),  h = 0 in front of a start
                y[t] = (sum_n C[t, n] h[t, n] + D x[t]) silu(z[t])
    loss        l[i] = log sum_v exp(hidden[i] . weight[v]) - hidden[i] . weight[target[i]]   over the allowed actions

`own` chooses between plain torch operations in 32 bits and the calls of the package.
"""
import math

import torch

own = False

TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
WIDTH = {'f32': 4, 'bf16': 2, 'f16': 2}
IGNORED = -100


def listed():
    return [
        # acting: the environments one receive returned, their convolution windows kept by environment
        dict(name='conv_step_64', op='conv_step', type='f32', rows=64, environments=256, channels=256, taps=4),
        # the rows a few environments played so far, read again in one go (727 rows: a chronic of the 14-bus grid)
        dict(name='conv_prompt_odd', op='conv', type='f16', batch=3, time=727, channels=250, taps=3, train=False, time_major=False),
        # training on windows of 60 steps of 1024 environments, recorded step by step (time first in memory)
        dict(name='conv_train', op='conv', type='bf16', batch=1024, time=60, channels=1024, taps=4, train=True, time_major=True),
        # acting: a handful of environments, an odd model
        dict(name='scan_step_37', op='scan_step', type='f32', rows=37, environments=64, channels=200, states=12, groups=1),
        # acting: the whole batch of 4096 environments
        dict(name='scan_step_4096', op='scan_step', type='bf16', rows=4096, environments=4096, channels=512, states=16, groups=1),
        # two environments' twelve chronics of 727 rows back to back: few rows, a long axis
        dict(name='scan_prompt_long', op='scan', type='f16', batch=2, time=8724, channels=768, states=16, groups=1, train=False, time_major=False),
        # training on the windows of conv_train
        dict(name='scan_train', op='scan', type='bf16', batch=1024, time=60, channels=512, states=16, groups=1, train=True, time_major=True),
        # training in 32 bits on whole chronics of the 118-bus grid (167 rows), odd sizes, two heads of B and C
        dict(name='scan_train_odd', op='scan', type='f32', batch=75, time=167, channels=200, states=12, groups=2, train=True, time_major=False),
        # log-probabilities of the chosen actions of one step of 4096 environments
        dict(name='loss_value', op='loss', type='bf16', rows=4096, actions=24129, features=512, masked=True, train=False),
        # a small policy on the 14-bus grid's catalogue, in 32 bits
        dict(name='loss_train_small', op='loss', type='f32', rows=256, actions=347, features=128, masked=False, train=True),
        # imitation of a search's best actions, odd sizes
        dict(name='loss_train_odd', op='loss', type='f16', rows=999, actions=12099, features=392, masked=True, train=True),
        # the largest: a batch of 16384 rows on the whole catalogue
        dict(name='loss_train', op='loss', type='bf16', rows=16384, actions=24129, features=512, masked=True, train=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(['conv_step', 'conv', 'scan_step', 'scan', 'loss'])
    case = dict(op=op, type=rng.choice(['f32', 'bf16', 'f16']))
    if op in ('conv_step', 'scan_step'):
        rows = _log(rng, 1, 4096)
        case.update(rows=rows, environments=rows + rng.choice([0, 0, _log(rng, 1, 512)]))
        if op == 'conv_step':
            case.update(channels=_log(rng, 64, 1024), taps=rng.randint(2, 6))
        else:
            groups = rng.choice([1, 1, 2, 4])
            case.update(channels=groups * _log(rng, 32, 512 // groups), states=rng.choice([8, 11, 12, 16, 16, 24, 32]), groups=groups)
    elif op == 'conv':
        channels, taps = _log(rng, 64, 1024), rng.randint(2, 6)
        time = _log(rng, 1, 4096)
        batch = _log(rng, 1, max(1, 60 * 1024 * 1024 // (time * channels * 2)))
        case.update(batch=batch, time=time, channels=channels, taps=taps, train=rng.random() < 0.5, time_major=rng.random() < 0.5)
    elif op == 'scan':
        groups = rng.choice([1, 1, 2, 4])
        channels, states = groups * _log(rng, 32, 512 // groups), rng.choice([8, 11, 12, 16, 16, 24, 32])
        train = rng.random() < 0.5
        time = _log(rng, 1, 700 if train else 8000)
        batch = _log(rng, 1, max(1, 20 * 1024 * 512 * 16 // (time * channels * states)))
        case.update(batch=batch, time=time, channels=channels, states=states, groups=groups, train=train, time_major=rng.random() < 0.5)
    else:
        actions, features = _log(rng, 100, 24129), _log(rng, 64, 512)
        case.update(rows=_log(rng, 1, 8192), actions=actions, features=features, masked=rng.random() < 0.5, train=rng.random() < 0.6)
        if case['type'] == 'f32':
            case['rows'] = max(1, case['rows'] // 4)
    return case


# ---- inputs ------------------------------------------------------------------------------------------------------------------------

def _starts(case, gen, shape):
    """First rows of episodes: one in fifty (a game over restarts the environment behind the step that ended it)."""
    return torch.rand(shape, generator=gen, device='cuda') < 0.02


def _rows(case, gen, *tail, scale=1.0):
    b, t = case['batch'], case['time']
    first, second = (t, b) if case['time_major'] else (b, t)
    x = (torch.randn((first, second) + tail, generator=gen, device='cuda') * scale).to(TYPES[case['type']])
    return x.transpose(0, 1) if case['time_major'] else x


def _scan_parameters(case, gen):
    d, n = case['channels'], case['states']
    a = -torch.arange(1, n + 1, device='cuda', dtype=torch.float32).repeat(d, 1)
    a = a * (1 + 0.05 * torch.randn((d, n), generator=gen, device='cuda'))
    skip = 1 + 0.1 * torch.randn((d,), generator=gen, device='cuda')
    step = torch.exp(torch.rand((d,), generator=gen, device='cuda') * math.log(100.0) + math.log(1e-3))
    return a, skip, torch.log(torch.expm1(step))      # softplus(dt_bias) spread over 0.001 .. 0.1


def _allowed(case, gen):
    """Bit-packed legality of every action in every row: the actions of a substation on cooldown are out (one in thirty)."""
    n, v = case['rows'], case['actions']
    words = (v + 31) // 32
    blocks = min(118, v)
    group = (torch.arange(words * 32, device='cuda') * blocks) // (words * 32)
    place = torch.arange(32, device='cuda', dtype=torch.int64)
    bits = torch.empty((n, words), dtype=torch.int32, device='cuda')
    for i in range(0, n, 1024):
        free = torch.rand((min(1024, n - i), blocks), generator=gen, device='cuda') > 1 / 30
        ok = free[:, group]
        ok[:, 0] = True                                # doing nothing is always allowed
        ok[:, v:] = False
        word = (ok.view(-1, words, 32).to(torch.int64) << place).sum(-1)
        bits[i:i + 1024] = torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32)
    return bits


def _unpack(bits, v):
    place = torch.arange(32, device=bits.device, dtype=torch.int32)
    return (((bits[..., None] >> place) & 1) != 0).view(bits.shape[0], -1)[:, :v]


def prepare(case, seed):
    gen = torch.Generator(device='cuda')
    gen.manual_seed(seed)
    op, dtype = case['op'], TYPES[case['type']]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device='cuda')

    s = dict(case=case)
    if op in ('conv_step', 'scan_step'):
        n, e, d = case['rows'], case['environments'], case['channels']
        s['env_ids'] = torch.randperm(e, generator=gen, device='cuda')[:n].to(torch.int32)
        s['starts'] = _starts(case, gen, (n,))
        s['x'] = normal(n, d).to(dtype)
        if op == 'conv_step':
            k = case['taps']
            s.update(state=normal(e, k - 1, d).to(dtype), weight=normal(d, k) / math.sqrt(k), bias=0.1 * normal(d))
        else:
            g, m = case['groups'], case['states']
            s['A'], s['D'], s['dt_bias'] = _scan_parameters(case, gen)
            s.update(dt=(0.5 * normal(n, d)).to(dtype), B=normal(n, g, m).to(dtype), C=normal(n, g, m).to(dtype), z=normal(n, d).to(dtype),
                     state=normal(e, d, m))
    elif op == 'conv':
        b, d, k = case['batch'], case['channels'], case['taps']
        s.update(x=_rows(case, gen, d), weight=normal(d, k) / math.sqrt(k), bias=0.1 * normal(d), initial_state=normal(b, k - 1, d).to(dtype),
                 starts=_starts(case, gen, (b, case['time'])))
        if case['train']:
            s['grad'] = _rows(case, gen, d)
    elif op == 'scan':
        b, d, g, m = case['batch'], case['channels'], case['groups'], case['states']
        s['A'], s['D'], s['dt_bias'] = _scan_parameters(case, gen)
        s.update(x=_rows(case, gen, d), dt=_rows(case, gen, d, scale=0.5), B=_rows(case, gen, g, m), C=_rows(case, gen, g, m), z=_rows(case, gen, d),
                 initial_state=normal(b, d, m), starts=_starts(case, gen, (b, case['time'])))
        if case['train']:
            s['grad'] = _rows(case, gen, d)
    else:
        n, v, f = case['rows'], case['actions'], case['features']
        s.update(hidden=normal(n, f).to(dtype), weight=(2 * normal(v, f) / math.sqrt(f)).to(dtype))
        s['allowed'] = _allowed(case, gen) if case['masked'] else None
        target = torch.randint(0, v, (n,), generator=gen, device='cuda')
        if case['masked']:                             # what is taught is allowed: elsewhere the row teaches doing nothing
            word = s['allowed'].gather(1, (target >> 5)[:, None])[:, 0]
            target = torch.where(((word >> (target & 31).to(torch.int32)) & 1) != 0, target, torch.zeros_like(target))
        quiet = torch.rand((n,), generator=gen, device='cuda')
        target = torch.where(quiet < 0.3, torch.zeros_like(target), target)
        s['target'] = torch.where(quiet > 0.99, torch.full_like(target, IGNORED), target)   # rows behind an episode's end
        if case['train']:
            s['grad'] = normal(n) / n                  # advantages over the number of rows
    if case.get('train'):
        for name in _LEAVES[op]:
            s[name].requires_grad_(True)
    return s


_LEAVES = {'conv': ('x', 'weight', 'bias', 'initial_state'),
           'scan': ('x', 'dt', 'A', 'B', 'C', 'D', 'z', 'dt_bias', 'initial_state'),
           'loss': ('hidden', 'weight')}


# ---- the package's calls -----------------------------------------------------------------------------------------------------------

def _run_own(s):
    from pypownet_amd import policy_ops as ops
    op = s['case']['op']
    if op == 'conv_step':
        y = ops.short_conv_step(s['x'], s['state'], s['weight'], s['bias'], activation='silu', env_ids=s['env_ids'], starts=s['starts'])
        return y, s['state']
    if op == 'scan_step':
        y = ops.selective_scan_step(s['x'], s['dt'], s['A'], s['B'], s['C'], s['state'], D=s['D'], z=s['z'], dt_bias=s['dt_bias'], dt_softplus=True,
                                    env_ids=s['env_ids'], starts=s['starts'])
        return y, s['state']
    train = s['case']['train']
    if op == 'conv':
        y, last = ops.short_conv(s['x'], s['weight'], s['bias'], activation='silu', starts=s['starts'], initial_state=s['initial_state'],
                                 return_final_state=True)
    elif op == 'scan':
        y, last = ops.selective_scan(s['x'], s['dt'], s['A'], s['B'], s['C'], D=s['D'], z=s['z'], dt_bias=s['dt_bias'], dt_softplus=True,
                                     starts=s['starts'], initial_state=s['initial_state'], return_final_state=True)
    else:
        y = ops.action_cross_entropy(s['hidden'], s['weight'], s['target'], allowed=s['allowed'], ignore_index=IGNORED)
        last = None
    out = (y.detach(),) if last is None else (y.detach(), last.detach())
    if not train:
        return out
    return out + torch.autograd.grad(y, [s[name] for name in _LEAVES[op]], s['grad'])


# ---- plain forms -------------------------------------------------------------------------------------------------------------------

def _silu(x):
    return x / (1 + torch.exp(-x))


def _softplus(x):
    return torch.where(x > 20, x, torch.log(1 + torch.exp(torch.clamp(x, max=20))))


def _plain_conv(x, weight, bias, initial, starts):
    """The K - 1 rows in front of the window, then x; a tap counts if no episode has begun between it and the row."""
    b, t, d = x.shape
    k = weight.shape[1]
    rows = torch.cat([initial.float(), x.float()], dim=1)
    begun = torch.cat([torch.zeros((b, k - 1), device=x.device, dtype=torch.int32), starts.to(torch.int32)], dim=1).cumsum(1)
    total = bias[None, None, :]
    for j in range(k):
        same = (begun[:, k - 1:] == begun[:, j:j + t]).to(torch.float32)
        total = total + weight[:, j] * rows[:, j:j + t] * same[..., None]
    y = _silu(total).to(x.dtype)
    kept = (begun[:, t:] == begun[:, -1:])[..., None]
    last = torch.where(kept, rows[:, t:], torch.zeros_like(rows[:, t:])).to(initial.dtype)
    return y, last


def _plain_scan_cell(h, x, dt, A, B, C, D, z, dt_bias, starts):
    """One row: h [rows, channels, states]; x, dt, z [rows, channels]; B, C [rows, groups, states]."""
    d = A.shape[0]
    of = d // B.shape[1]
    delta = _softplus(dt.float() + dt_bias)
    b, c = (v.float().repeat_interleave(of, dim=1) for v in (B, C))
    h = torch.where(starts[:, None, None], torch.zeros_like(h), h)
    h = torch.exp(delta[..., None] * A) * h + (delta * x.float())[..., None] * b
    y = ((h * c).sum(-1) + D * x.float()) * _silu(z.float())
    return h, y.to(x.dtype)


def _run_plain(s):
    op = s['case']['op']
    if op == 'conv_step':
        ids = s['env_ids'].long()
        state = torch.where(s['starts'][:, None, None], torch.zeros_like(s['state'][ids]), s['state'][ids])
        rows = torch.cat([state, s['x'][:, None, :]], dim=1)
        y = _silu((rows.float() * s['weight'].t()).sum(1) + s['bias'])
        s['state'][ids] = rows[:, 1:]
        return y.to(s['x'].dtype), s['state']
    if op == 'scan_step':
        ids = s['env_ids'].long()
        h, y = _plain_scan_cell(s['state'][ids], s['x'], s['dt'], s['A'], s['B'], s['C'], s['D'], s['z'], s['dt_bias'], s['starts'])
        s['state'][ids] = h
        return y, s['state']
    if op == 'loss':
        return _plain_loss(s)
    train = s['case']['train']
    with torch.set_grad_enabled(train):
        if op == 'conv':
            y, last = _plain_conv(s['x'], s['weight'], s['bias'], s['initial_state'], s['starts'])
        else:
            h, ys = s['initial_state'], []
            for t in range(s['case']['time']):
                h, row = _plain_scan_cell(h, s['x'][:, t], s['dt'][:, t], s['A'], s['B'][:, t], s['C'][:, t], s['D'], s['z'][:, t], s['dt_bias'],
                                          s['starts'][:, t])
                ys.append(row)
            y, last = torch.stack(ys, dim=1), h
        out = (y.detach(), last.detach())
        if not train:
            return out
        return out + torch.autograd.grad(y, [s[name] for name in _LEAVES[op]], s['grad'])


def _plain_loss(s):
    with torch.no_grad():
        h, w = s['hidden'].float(), s['weight'].float()
        target, counted = s['target'], s['target'] != IGNORED
        at = torch.where(counted, target, torch.zeros_like(target))[:, None]
        logits = h @ w.t()
        if s['allowed'] is not None:
            logits = logits.masked_fill(~_unpack(s['allowed'], w.shape[0]), -math.inf)
        top = logits.max(dim=1, keepdim=True).values
        wanted = logits.gather(1, at)
        e = torch.exp(logits - top)
        total = e.sum(dim=1, keepdim=True)
        loss = torch.where(counted, (torch.log(total) + top - wanted)[:, 0], torch.zeros_like(top[:, 0]))
        if not s['case']['train']:
            return (loss,)
        grad = torch.where(counted, s['grad'], torch.zeros_like(s['grad']))[:, None]
        d = e * (grad / total)
        d.scatter_add_(1, at, -grad)
        return loss, (d @ w).to(s['hidden'].dtype), (d.t() @ h).to(s['weight'].dtype)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the work that cannot be done without --------------------------------------------------------------------------------------------

def work(case):
    op, size = case['op'], WIDTH[case['type']]
    if op == 'conv_step':
        n, d, k = case['rows'], case['channels'], case['taps']
        return dict(bytes=n * d * size * (2 + 2 * (k - 1)) + d * (k + 1) * 4 + 5 * n, flops=n * d * (2 * k + 5))
    if op == 'scan_step':
        n, d, m, g = case['rows'], case['channels'], case['states'], case['groups']
        return dict(bytes=n * d * (4 * size + 8 * m) + n * g * m * 2 * size + d * (m + 2) * 4 + 5 * n, flops=n * d * (6 * m + 12))
    if op == 'conv':
        e, d, k, b = case['batch'] * case['time'] * case['channels'], case['channels'], case['taps'], case['batch']
        moved = 2 * e * size + 2 * b * (k - 1) * d * size + d * (k + 1) * 4 + b * case['time']
        flops = e * (2 * k + 5)
        if case['train']:        # x and the gradient of y in, the gradient of x out, the parameters' gradients
            moved += 3 * e * size + b * (k - 1) * d * size + 2 * d * (k + 1) * 4
            flops += e * (6 * k + 12)
        return dict(bytes=moved, flops=flops)
    if op == 'scan':
        b, t, d, m, g = case['batch'], case['time'], case['channels'], case['states'], case['groups']
        e, bc = b * t * d, 2 * b * t * g * m
        moved = e * 4 * size + bc * size + 8 * b * d * m + d * (m + 2) * 4 + b * t
        flops = e * (6 * m + 12)
        if case['train']:        # x, dt, z, B, C and the gradient of y in; the gradients of the first five out
            moved += e * 7 * size + 2 * bc * size + 8 * b * d * m + 2 * d * (m + 2) * 4
            flops += e * (16 * m + 30)
        return dict(bytes=moved, flops=flops)
    n, v, f = case['rows'], case['actions'], case['features']
    moved = (n + v) * f * size + 12 * n + (n * ((v + 31) // 32) * 4 if case['masked'] else 0)
    flops = 2 * n * v * f + 3 * n * v
    if case['train']:
        moved += 2 * (n + v) * f * size + 4 * n
        flops = 3 * 2 * n * v * f + 6 * n * v
    return dict(bytes=moved, flops=flops)


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    v = {k: (t.detach().double() if torch.is_tensor(t) and t.is_floating_point() else t) for k, t in s.items()}
    with torch.no_grad():
        return {'conv_step': _exact_conv_step, 'scan_step': _exact_scan_step, 'conv': _exact_conv, 'scan': _exact_scan, 'loss': _exact_loss}[case['op']](case, v)


def _exact_conv_step(case, v):
    k = case['taps']
    state = v['state'].clone()
    window = state[v['env_ids'].long()] * (~v['starts'])[:, None, None]
    pre = v['bias'] + v['x'] * v['weight'][:, k - 1]
    for j in range(k - 1):
        pre = pre + window[:, j] * v['weight'][:, j]
    state[v['env_ids'].long()] = torch.cat([window, v['x'][:, None]], 1)[:, 1:]
    return pre * torch.sigmoid(pre), state


def _exact_cell(v, h, t=None):
    """d, exp(d A), and the new state of one row (rows t of the sequences, or the row itself)."""
    at = (lambda a: a) if t is None else (lambda a: a[:, t])
    of = v['A'].shape[0] // at(v['B']).shape[1]
    pre = at(v['dt']) + v['dt_bias']
    d = torch.clamp(pre, min=0) + torch.log1p(torch.exp(-pre.abs()))
    b, c = (at(a).repeat_interleave(of, 1) for a in (v['B'], v['C']))
    decay = torch.exp(torch.einsum('rd,dn->rdn', d, v['A'])) * (~at(v['starts']))[:, None, None]
    return pre, d, decay, b, c, decay * h + (d * at(v['x']))[..., None] * b, of


def _exact_scan_step(case, v):
    state = v['state'].clone()
    ids = v['env_ids'].long()
    _, _, _, _, c, h, _ = _exact_cell(v, state[ids])
    state[ids] = h
    return ((h * c).sum(-1) + v['D'] * v['x']) * v['z'] * torch.sigmoid(v['z']), state


def _exact_conv(case, v):
    b, t, d, k = case['batch'], case['time'], case['channels'], case['taps']
    x, w = v['x'], v['weight']
    padded = torch.cat([v['initial_state'], x], 1)
    episode = torch.cat([torch.zeros((b, k - 1), dtype=torch.int64, device=x.device), v['starts'].long()], 1).cumsum(1)
    live = [(episode[:, j:j + t] == episode[:, k - 1:])[..., None].double() for j in range(k)]
    pre = v['bias'] + sum(live[j] * padded[:, j:j + t] * w[:, j] for j in range(k))
    sig = torch.sigmoid(pre)
    last = padded[:, t:] * (episode[:, t:] == episode[:, -1:])[..., None]
    if not case['train']:
        return pre * sig, last
    dpre = v['grad'] * sig * (1 + pre * (1 - sig))
    dpadded = torch.zeros_like(padded)
    dw = torch.zeros_like(w)
    for j in range(k):
        dpadded[:, j:j + t] += dpre * live[j] * w[:, j]
        dw[:, j] = (dpre * live[j] * padded[:, j:j + t]).sum((0, 1))
    return pre * sig, last, dpadded[:, k - 1:], dw, dpre.sum((0, 1)), dpadded[:, :k - 1]


def _exact_scan(case, v):
    b, t, d, g, m = case['batch'], case['time'], case['channels'], case['groups'], case['states']
    h, states, y = v['initial_state'], [], torch.empty((b, t, d), dtype=torch.float64, device='cuda')
    gate = v['z'] * torch.sigmoid(v['z'])
    for i in range(t):
        if case['train']:
            states.append(h)
        _, _, _, _, c, h, _ = _exact_cell(v, h, i)
        y[:, i] = (h * c).sum(-1) + v['D'] * v['x'][:, i]
    if not case['train']:
        return y * gate, h
    dy = v['grad'] * gate
    sig = torch.sigmoid(v['z'])
    dz = v['grad'] * y * sig * (1 + v['z'] * (1 - sig))
    dx, ddt = torch.empty_like(y), torch.empty_like(y)
    dB, dC = (torch.empty((b, t, g, m), dtype=torch.float64, device='cuda') for _ in range(2))
    dA, dh = torch.zeros_like(v['A']), torch.zeros_like(h)
    for i in range(t - 1, -1, -1):
        pre, delta, decay, bb, c, now, of = _exact_cell(v, states[i], i)
        dC[:, i] = (dy[:, i, :, None] * now).view(b, g, of, m).sum(2)
        dh = dh + dy[:, i, :, None] * c
        dB[:, i] = (dh * (delta * v['x'][:, i])[..., None]).view(b, g, of, m).sum(2)
        through = (dh * bb).sum(-1)
        dx[:, i] = through * delta + dy[:, i] * v['D']
        dlog = dh * decay * states[i]
        dA += torch.einsum('rdn,rd->dn', dlog, delta)
        ddt[:, i] = ((dlog * v['A']).sum(-1) + through * v['x'][:, i]) * torch.sigmoid(pre)
        dh = dh * decay
        states[i] = None
    return y * gate, h, dx, ddt, dA, dB, dC, (dy * v['x']).sum((0, 1)), dz, ddt.sum((0, 1)), dh


def _exact_loss(case, v):
    h, w, target = v['hidden'], v['weight'], v['target']
    n = h.shape[0]
    loss = torch.zeros((n,), dtype=torch.float64, device='cuda')
    dh, dw = torch.zeros_like(h), torch.zeros_like(w)
    for i in range(0, n, 2048):
        rows = slice(i, min(n, i + 2048))
        logits = h[rows] @ w.t()
        if v['allowed'] is not None:
            logits[~_unpack(v['allowed'][rows], w.shape[0])] = -math.inf
        logp = logits - torch.logsumexp(logits, 1, keepdim=True)
        counted = target[rows] != IGNORED
        at = target[rows].clamp(min=0)[:, None]
        loss[rows] = -logp.gather(1, at)[:, 0] * counted
        if case['train']:
            p = torch.exp(logp)
            p.scatter_add_(1, at, -torch.ones_like(p[:, :1]))
            p *= (v['grad'][rows] * counted)[:, None]
            dh[rows] = p @ w
            dw += p.t() @ h[rows]
    return (loss, dh, dw) if case['train'] else (loss,)
