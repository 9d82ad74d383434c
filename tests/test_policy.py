"""The action catalogue and the recurrent policy (pypownet_amd.policy) on batched environments.

Tolerance of a network in 32 bits against the same network in 64, in the Euclidean norm over all entries: a layer is a chain of nine stages (norm, two
products, convolution, three products, scan, gate), each with sums of at most 256 terms, off by at most 2 (256 + 8) 2^-24 of their size; sums of random
signs are smaller than their sizes by up to 16 (the root of 256).  Two layers and the two ends are 20 stages forward and as many backward:
40 x 16 x 264 x 2^-23 = 0.02 at worst, where every error has the same direction; a wrong term changes a result by far more."""
import os
import types

import numpy as np
import pytest
import torch

from helpers import ENVS, load_env
from pypownet_amd.policy import ActionCatalogue, PolicyMemory, RecurrentPolicy, imitate
from test_policy_ops import conv_definition, loss_definition, scan_definition

NETWORK = 0.02


# ---- CPU ------------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize('name,count', [('default14', 177), ('default30', 347), ('default118', 12099)])
def test_catalogue(name, count):
    case = load_env(name)[0]
    c = ActionCatalogue(case)
    assert len(c) == count and c.vectors.shape == (count, case.action_length) and set(np.unique(c.vectors)) <= {0, 1}
    assert not c.vectors[0].any() and c.asset[0] == 0
    lines = c.vectors[:, case.n_topo:]
    assert np.array_equal(lines[1:1 + case.nl], np.eye(case.nl, dtype=np.uint8)) and not lines[1 + case.nl:].any()
    topo = c.vectors[1 + case.nl:, :case.n_topo]
    for row, asset in zip(topo, c.asset[1 + case.nl:]):
        assert set(case.elem_sub[np.flatnonzero(row)]) == {asset - 1 - case.nl}
    assert not c.vectors[:1 + case.nl, :case.n_topo].any()
    # no two of a substation's actions are equal or each other's complement
    for sub in range(case.nS):
        mine = topo[c.asset[1 + case.nl:] == 1 + case.nl + sub][:, case.mapping_array[sub]]
        assert len(mine) == 2 ** (len(case.mapping_array[sub]) - 1) - 1
        assert len({tuple(r) for r in mine} | {tuple(1 - r) for r in mine}) == 2 * len(mine)


@pytest.mark.parametrize('most', [1, 2, 3])
def test_catalogue_of_small_sets(most):
    from pypownet_amd.policy import _sets_up_to
    case = load_env('default14')[0]
    whole, some = ActionCatalogue(case), ActionCatalogue(case, max_swapped=most)
    keep = []
    for i, row in enumerate(whole.vectors):
        k = len(case.mapping_array[whole.asset[i] - 1 - case.nl]) if whole.asset[i] > case.nl else 0
        on = int(row[:case.n_topo].sum())
        keep.append(min(on, k - on) <= most if k else True)
    assert np.array_equal(some.vectors, whole.vectors[keep]) and np.array_equal(some.asset, whole.asset[keep])
    # substations with too many elements to list every set of take another way to the same sets
    for k in range(2, 9):
        every = (np.arange(1, 1 << (k - 1))[:, None] >> np.arange(k - 1)) & 1
        size = every.sum(axis=1)
        assert {tuple(r) for r in _sets_up_to(k, most)} == {tuple(r) for r in every[np.minimum(size, k - size) <= most]}


def test_catalogue_of_a_large_substation():
    case = types.SimpleNamespace(mapping_array=[list(range(24)), [24], []], nl=0, nS=3, n_topo=25, action_length=25)
    with pytest.raises(ValueError, match='max_swapped'):
        ActionCatalogue(case)
    c = ActionCatalogue(case, max_swapped=1)
    assert len(c) == 1 + 24 and (c.asset[1:] == 1).all()
    with pytest.raises(ValueError):
        ActionCatalogue(case, max_swapped=0)


def test_allowed_actions():
    case = load_env('default14')[0]
    c = ActionCatalogue(case)
    lines, subs = torch.ones((2, case.nl), dtype=torch.bool), torch.ones((2, case.nS), dtype=torch.bool)
    lines[1, 3] = False
    subs[1] = False
    mask = c.allowed(lines, subs)
    assert mask[0].all() and mask.dtype == torch.bool
    assert mask[1].nonzero()[:, 0].tolist() == [i for i in range(1 + case.nl) if i != 4]


def test_policy_arguments_are_refused():
    c = ActionCatalogue(load_env('default14')[0])
    with pytest.raises(TypeError):
        RecurrentPolicy(c, 538, dtype=torch.float64)
    for bad in (dict(taps=9), dict(taps=1), dict(states=65), dict(states=0), dict(layers=0), dict(features=0)):
        with pytest.raises(ValueError):
            RecurrentPolicy(c, 538, **bad)
    policy = RecurrentPolicy(c, 538, features=8, layers=2)
    with pytest.raises(ValueError, match='538'):
        policy.window(torch.zeros(2, 3, 537))
    with pytest.raises(ValueError, match='layers'):
        policy.window(torch.zeros(2, 3, 538), memory=RecurrentPolicy(c, 538, features=8, layers=1).memory(2))
    with pytest.raises(ValueError, match='environments'):
        policy.window(torch.zeros(2, 3, 538), memory=policy.memory(3))
    with pytest.raises(ValueError, match='GPU'):
        policy.window(torch.zeros(2, 3, 538))
    with pytest.raises(ValueError, match='GPU'):
        policy.act(torch.zeros(2, 538), policy.memory(2))
    with pytest.raises(ValueError, match='candidates'):
        imitate(None, policy, None, policy.memory(2), steps=1, candidates=1)


# ---- GPU ------------------------------------------------------------------------------------------------------------------------------

def near(name, got, want, limit=NETWORK):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    off = float((got - want).norm()) / float(want.norm())
    assert off <= limit, '%s: off by %.3g of its norm' % (name, off)


def rows_of(env_name, batch, steps, length):
    """Smooth made-up observation rows in the range of the real ones."""
    gen = torch.Generator().manual_seed(len(env_name))
    return torch.randn((batch, steps, length), generator=gen).cumsum(1) * torch.logspace(-1, 2, length)


@pytest.mark.gpu
def test_gpu_policy_gradients(monkeypatch):
    """The loss of a window and every parameter's gradient against the same network on the operators' definitions in 64 bits."""
    import pypownet_amd.policy as module
    c = ActionCatalogue(load_env('default14')[0])
    torch.manual_seed(3)
    policy = RecurrentPolicy(c, 538, features=32, layers=2, states=16, taps=4, dtype=torch.float32)
    gen = torch.Generator().manual_seed(4)
    b, t = 5, 23
    obs = rows_of('default14', b, t, 538)
    starts = torch.rand((b, t), generator=gen) < 0.1
    allowed = torch.rand((b, t, len(c)), generator=gen) < 0.6
    target = torch.randint(0, len(c), (b, t), generator=gen)
    allowed.scatter_(2, target[..., None], True)
    target[1, 3] = -100
    bits = module.ops.pack_allowed(allowed.view(b * t, -1)).view(b, t, -1)
    policy.cuda()
    begun = policy.window(obs[:, :4].cuda())[1]
    loss, after = policy.loss(obs.cuda(), target.cuda(), bits.cuda(), starts.cuda(), begun)
    grads = torch.autograd.grad(loss.mean(), list(policy.parameters()))
    again, _ = policy.loss(obs.cuda(), target.cuda(), bits.cuda(), starts.cuda(), begun)
    assert torch.equal(again, loss)
    policy.cpu().double()
    policy.dtype = torch.float64

    def conv(x, weight, bias, activation, starts, initial, final):
        return conv_definition(x, weight, bias, True, starts, initial)

    def scan(x, dt, A, B, C, D, z, dt_bias, soft, starts, initial, final):
        return scan_definition(x, dt, A, B, C, D, z, dt_bias, soft, starts, initial)

    def cross(hidden, weight, target, allowed_bits):
        return loss_definition(hidden, weight, target, allowed.view(b * t, -1))
    monkeypatch.setattr(module, 'ops', types.SimpleNamespace(short_conv=conv, selective_scan=scan, action_cross_entropy=cross))
    memory = PolicyMemory([w.cpu().double() for w in begun.windows], [s.cpu().double() for s in begun.states])
    want, after64 = policy.loss(obs, target, bits, starts, memory)
    wanted = torch.autograd.grad(want.mean(), list(policy.parameters()))
    near('loss', loss, want)
    assert loss[1, 3] == 0
    for (name, _), got, g in zip(policy.named_parameters(), grads, wanted):
        near(name, got, g)
    for got, m in zip(after.windows + after.states, after64.windows + after64.states):
        near('memory', got, m)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_gpu_acting_row_by_row_remembers_what_the_window_does(dtype):
    """Environments advance at their own pace: their memories are those of their own rows in one window."""
    c = ActionCatalogue(load_env('default14')[0])
    torch.manual_seed(5)
    policy = RecurrentPolicy(c, 538, features=32, layers=1, dtype=dtype).cuda()
    b, t = 7, 12
    obs = rows_of('x', b, t, 538).cuda()
    starts = torch.zeros((b, t), dtype=torch.uint8)
    starts[2, 5] = starts[4, 0] = starts[6, 11] = 1
    starts = starts.cuda()
    memory = policy.memory(b)
    gen = torch.Generator().manual_seed(6)
    at = [0] * b
    while min(at) < t:
        ids = [i for i in torch.randperm(b, generator=gen).tolist() if at[i] < t][:1 + int(torch.randint(0, 4, (), generator=gen))]
        index, when = torch.tensor(ids, device='cuda'), torch.tensor([at[i] for i in ids], device='cuda')
        policy.act(obs[index, when], memory, env_ids=index, starts=starts[index, when])
        for i in ids:
            at[i] += 1
    _, after = policy.window(obs, starts)
    # the products' rounding to the type, once per row of a state; each at most half a step of what it rounds, the five in front of a state alike
    limit = NETWORK if dtype == torch.float32 else 16 * torch.finfo(dtype).eps
    for got, want in zip(memory.windows + memory.states, after.windows + after.states):
        near('memory', got, want, limit)


def environments(batch, name='default14', **kw):
    from pypownet_amd.batched import BatchedRunEnv
    env = BatchedRunEnv(os.path.join(ENVS, name), 'level0', batch, device=0, config_overrides={'solver': 'newton'}, **kw)
    env.reset()
    env.engine.process_game_over()
    return env


@pytest.mark.gpu
@pytest.mark.parametrize('sample', [False, True])
def test_gpu_policy_acts_on_environments(sample):
    env = environments(96)
    c = ActionCatalogue(env.case)
    torch.manual_seed(7)
    policy = RecurrentPolicy(c, env.engine.observation_length('minimalist'), features=32).cuda()
    memory = policy.memory(96)
    acted = ended = 0
    for _ in range(25):
        rows, starts, allowed = env.policy_rows(policy, layout='minimalist')
        assert np.array_equal(starts.cpu().numpy() != 0, env.engine.read('DONE') != 0)
        assert allowed[:, 0].all()
        actions = env.policy_actions(policy, memory=memory, layout='minimalist', sample=sample)
        assert actions.dtype == torch.uint8 and tuple(actions.shape) == (96, env.action_length)
        acted += int(actions.any(dim=1).sum())
        _, done, _, illegal = env.step(actions, auto_reset=True, want_obs=False)
        assert not illegal.any()
        ended += int(done.sum())
    assert acted > 0 and all(torch.isfinite(m).all() for m in memory.windows + memory.states)
    memory.clear()
    assert not any(m.any() for m in memory.windows + memory.states)
    with pytest.raises(ValueError, match='memory'):
        env.policy_actions(policy)
    with pytest.raises(ValueError, match='environments'):
        env.policy_actions(policy, memory=policy.memory(95))
    with pytest.raises(ValueError, match='length'):
        env.policy_actions(RecurrentPolicy(ActionCatalogue(load_env('default30')[0]), 538, features=8).cuda(), memory=policy.memory(96))


@pytest.mark.gpu
@pytest.mark.parametrize('candidates', [2, 5])
def test_gpu_policy_learns_from_the_search(candidates):
    """Acting, searching, recording and one update, as a user runs them; the memory behind the window is that of the rows that were played."""
    env = environments(48, 'default30')
    c = ActionCatalogue(env.case)
    torch.manual_seed(8)
    policy = RecurrentPolicy(c, env.engine.observation_length(), features=32).cuda()
    before = [p.detach().clone() for p in policy.parameters()]
    memory = policy.memory(48)
    optimizer = torch.optim.SGD(policy.parameters(), lr=1e-3)
    for _ in range(2):
        loss, reward = imitate(env, policy, optimizer, memory, steps=9, candidates=candidates)
        assert torch.isfinite(loss) and float(loss) > 0 and np.isfinite(reward)
        assert all(torch.isfinite(m).all() for m in memory.windows + memory.states)
    for (name, p), old in zip(policy.named_parameters(), before):
        assert torch.isfinite(p).all() and not torch.equal(p, old), name
    # ... and acting goes on from it
    env.step(env.policy_actions(policy, memory=memory), want_obs=False)


@pytest.mark.gpu
def test_gpu_policy_with_environments_at_their_own_pace():
    """send / recv: whichever environments are ready are decided for, their memories looked up by id."""
    env = environments(64)
    c = ActionCatalogue(env.case)
    torch.manual_seed(9)
    policy = RecurrentPolicy(c, env.engine.observation_length(), features=32, layers=1).cuda()
    memory = policy.memory(64)
    for rows in (16, 64):      # (libraries load their code here, not beside the resident step server)
        policy.act(torch.zeros((rows, policy.observation_length), device='cuda'), memory, env_ids=torch.arange(rows, dtype=torch.int32, device='cuda'))
    memory.clear()
    torch.cuda.synchronize()
    env.async_start(obs_dtype='float32', idle_timeout_ms=2000)
    stream = env.async_stream()
    steps = np.zeros(64, dtype=np.int64)
    try:
        with torch.cuda.stream(stream):
            env.send(np.arange(64), torch.zeros((64, env.action_length), dtype=torch.uint8, device='cuda'))
            while steps.min() < 6:
                ids, obs, report = env.recv(min_ready=16, timeout_ms=20000)
                assert len(ids)
                choice = policy.act(obs, memory, env_ids=ids, starts=report[:, 0] != 0)
                ids = ids.cpu().numpy()
                steps[ids] += 1
                on = steps[ids] < 6
                if on.any():
                    env.send(ids[on], policy.vectors[choice[torch.from_numpy(on).cuda()]])
        stream.synchronize()
    finally:
        env.async_stop()
    assert (steps == 6).all()
    assert all(torch.isfinite(m).all() for m in memory.windows + memory.states)
    assert (memory.states[0].abs().amax(dim=(1, 2)) > 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=str)
def test_gpu_acting_between_a_loss_and_its_backward_pass(dtype):
    """Acting moves a memory on in place; a window that began with it cannot be learned from any more, and says so.  From a copy of it, it can."""
    c = ActionCatalogue(load_env('default14')[0])
    torch.manual_seed(10)
    policy = RecurrentPolicy(c, 538, features=16, layers=2, dtype=dtype).cuda()
    b, t = 4, 9
    obs, target = rows_of('x', b, t, 538).cuda(), torch.zeros((b, t), dtype=torch.int64, device='cuda')
    memory = policy.memory(b)
    policy.act(obs[:, 0], memory)
    copy = PolicyMemory([w.clone() for w in memory.windows], [s.clone() for s in memory.states])
    want = torch.autograd.grad(policy.loss(obs, target, memory=copy)[0].mean(), list(policy.parameters()))
    again, _ = policy.loss(obs, target, memory=copy)
    shared, _ = policy.loss(obs, target, memory=memory)
    policy.act(obs[:, 1], memory)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(again.mean(), list(policy.parameters())), want))
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        shared.mean().backward()


@pytest.mark.gpu
@pytest.mark.parametrize('b,t', [(0, 5), (3, 0)])
def test_gpu_policy_loss_of_no_rows(b, t):
    c = ActionCatalogue(load_env('default14')[0])
    policy = RecurrentPolicy(c, 538, features=16, layers=1).cuda()
    words = (len(c) + 31) // 32
    memory = policy.memory(b)
    if b:
        policy.act(torch.randn((b, 538), device='cuda'), memory)
    kept = [m.clone() for m in memory.windows + memory.states]
    loss, after = policy.loss(torch.zeros((b, t, 538), device='cuda'), torch.zeros((b, t), dtype=torch.int64, device='cuda'),
                              torch.zeros((b, t, words), dtype=torch.int32, device='cuda'), torch.zeros((b, t), dtype=torch.bool, device='cuda'), memory)
    assert loss.shape == (b, t) and all(torch.equal(m, k) for m, k in zip(after.windows + after.states, kept))
    loss.sum().backward()
    assert all(p.grad is not None and not p.grad.any() for p in policy.parameters())


@pytest.mark.gpu
def test_gpu_the_memory_behind_imitate_is_that_of_the_rows_played(monkeypatch):
    import copy
    env = environments(20, 'default30')
    c = ActionCatalogue(env.case)
    torch.manual_seed(11)
    policy = RecurrentPolicy(c, env.engine.observation_length(), features=32).cuda()
    memory = policy.memory(20)
    optimizer = torch.optim.SGD(policy.parameters(), lr=1e-2)
    seen, rows = [], env.policy_rows

    def recording(*args, **kw):
        seen.append(rows(*args, **kw))
        return seen[-1]
    monkeypatch.setattr(env, 'policy_rows', recording)
    for _ in range(2):
        seen.clear()
        before, old = copy.deepcopy(policy), PolicyMemory([w.clone() for w in memory.windows], [s.clone() for s in memory.states])
        imitate(env, policy, optimizer, memory, steps=7, candidates=3)
        assert len(seen) == 7
        _, after = before.window(torch.stack([o for o, _, _ in seen], dim=1), torch.stack([s for _, s, _ in seen], dim=1), old)
        for mine, want, had in zip(memory.windows + memory.states, after.windows + after.states, old.windows + old.states):
            assert torch.equal(mine, want) and not torch.equal(mine, had)
