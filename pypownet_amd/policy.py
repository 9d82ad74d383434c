"""A policy with a memory for ``BatchedRunEnv``: a numbered catalogue of switching actions, and a recurrent network over the observation rows that
chooses from it.  Its memory is ``policy_ops``'s short convolution and selective scan: stepped row by row while it acts (state per environment, so
environments may advance at their own pace), run over whole recorded windows while it learns; its loss is ``policy_ops.action_cross_entropy``.

    catalogue = ActionCatalogue(env.case)
    policy = RecurrentPolicy(catalogue, env.engine.observation_length()).cuda()
    memory = policy.memory(env.batch)
    env.step(env.policy_actions(policy, memory=memory), want_obs=False)         # acting
    imitate(env, policy, optimizer, memory, steps=32)                           # learning from BatchedRunEnv.search

The reference's agents are one greedy search per step (pypownet/agent.py:161-325) and learn nothing; the teacher here is that search.
"""
import math

import numpy as np
import torch
import torch.nn.functional as F

from . import policy_ops as ops


class ActionCatalogue(object):
    """The single-asset actions of a case, numbered: 0 does nothing, 1 .. n_lines switch one line each, the others swap the nodes of some of one
    substation's elements.  Swapping a set of elements and swapping all the others leave the same grid up to the names of the two nodes, so a
    substation of k elements has 2^(k-1) - 1 of them, the ones that leave its last element where it is; ``max_swapped`` keeps those where the set, or
    the others, are at most that many.  ``vectors`` [actions x action_length] are the action vectors ``BatchedRunEnv.step`` takes."""

    def __init__(self, case, max_swapped=None):
        if max_swapped is not None and max_swapped < 1:
            raise ValueError('max_swapped must be at least 1')
        sets = []
        for sub, elements in enumerate(case.mapping_array):
            k = len(elements)
            if max_swapped is None and k > 21:
                raise ValueError('substation %d has %d elements, 2^%d sets of them: say max_swapped' % (sub, k, k - 1))
            if k < 2:
                continue
            if max_swapped is None or k <= 21:
                chosen = np.unpackbits(np.arange(1, 1 << (k - 1), dtype='<u4').view(np.uint8).reshape(-1, 4), axis=1, bitorder='little')[:, :k - 1]
                if max_swapped is not None:
                    size = chosen.sum(axis=1)
                    chosen = chosen[np.minimum(size, k - size) <= max_swapped]
            else:
                chosen = _sets_up_to(k, max_swapped)
            sets.append((sub, elements, chosen))
        count = 1 + case.nl + sum(len(c) for _, _, c in sets)
        self.n_lines, self.n_substations, self.action_length = case.nl, case.nS, case.action_length
        self.vectors = np.zeros((count, case.action_length), dtype=np.uint8)
        # what an action touches: 0 nothing, 1 + line, 1 + n_lines + substation
        self.asset = np.zeros((count,), dtype=np.int64)
        lines = np.arange(case.nl)
        self.vectors[1 + lines, case.n_topo + lines] = 1
        self.asset[1:1 + case.nl] = 1 + lines
        at = 1 + case.nl
        for sub, elements, chosen in sets:
            self.vectors[at:at + len(chosen), elements[:chosen.shape[1]]] = chosen
            self.asset[at:at + len(chosen)] = 1 + case.nl + sub
            at += len(chosen)

    def __len__(self):
        return len(self.vectors)

    def allowed(self, lines_free, substations_free, asset=None):
        """[rows x actions] bool: the actions whose line / substation may be switched now (``lines_free`` [rows x lines], ``substations_free``
        [rows x substations], bool tensors).  Doing nothing always may.  ``asset``: this catalogue's, as a tensor that is on the device already."""
        asset = torch.from_numpy(self.asset).to(lines_free.device) if asset is None else asset
        free = torch.cat([torch.ones_like(lines_free[:, :1]), lines_free, substations_free], dim=1)
        return free.index_select(1, asset)


def _sets_up_to(k, most):
    """Sets without element k - 1 (as rows of k - 1 zeros and ones, the empty one left out) that have, or leave out, at most `most` elements of k."""
    from itertools import combinations
    rows = set()
    for size in range(1, min(most, k // 2) + 1):
        for some in combinations(range(k), size):
            row = np.zeros((k,), dtype=np.uint8)
            row[list(some)] = 1
            rows.add(tuple((row ^ row[-1])[:k - 1]))
    return np.array(sorted(rows), dtype=np.uint8)


class PolicyMemory(object):
    """What a ``RecurrentPolicy`` remembers of each environment: per layer the convolution's last rows and the scan's state; zeros at first."""

    def __init__(self, windows, states):
        self.windows, self.states = windows, states

    def clear(self):
        for t in self.windows + self.states:
            t.zero_()


class _Layer(torch.nn.Module):
    def __init__(self, features, channels, states, taps):
        super().__init__()
        rank = max(1, features // 16)
        self.sizes = [rank, states, states]
        self.norm = torch.nn.Parameter(torch.ones(features))
        self.wide = torch.nn.Parameter(torch.randn(2 * channels, features) / math.sqrt(features))
        self.taps = torch.nn.Parameter(torch.randn(channels, taps) / math.sqrt(taps))
        self.taps_bias = torch.nn.Parameter(torch.zeros(channels))
        self.select = torch.nn.Parameter(torch.randn(sum(self.sizes), channels) / math.sqrt(channels))
        self.rate = torch.nn.Parameter(torch.randn(channels, rank) / math.sqrt(rank))
        # steps of 0.001 to 0.1 at first (softplus of the bias), decays of 1 .. states
        steps = torch.exp(torch.empty(channels).uniform_(math.log(1e-3), math.log(1e-1)))
        self.rate_bias = torch.nn.Parameter(torch.log(torch.expm1(steps)))
        self.log_decay = torch.nn.Parameter(torch.log(torch.arange(1, states + 1, dtype=torch.float32)).repeat(channels, 1))
        self.through = torch.nn.Parameter(torch.ones(channels))
        self.narrow = torch.nn.Parameter(torch.randn(features, channels) / math.sqrt(channels))

    def selected(self, x):
        """dt, B, C of the convolved rows, by channel and state, one group."""
        low, b, c = F.linear(x, self.select.to(x.dtype)).split(self.sizes, dim=-1)
        return F.linear(low, self.rate.to(x.dtype)), b.unsqueeze(-2), c.unsqueeze(-2)

    def inward(self, rows):
        return F.linear(F.rms_norm(rows, rows.shape[-1:], self.norm.to(rows.dtype)), self.wide.to(rows.dtype)).chunk(2, dim=-1)

    def window(self, rows, starts, initial):
        x, z = self.inward(rows)
        x, last_rows = ops.short_conv(x, self.taps, self.taps_bias, 'silu', starts, initial[0], True)
        dt, b, c = self.selected(x)
        y, state = ops.selective_scan(x, dt, -self.log_decay.exp(), b, c, self.through, z, self.rate_bias, True, starts, initial[1], True)
        return rows + F.linear(y, self.narrow.to(y.dtype)), last_rows, state

    def step(self, rows, last_rows, state, env_ids, starts):
        x, z = self.inward(rows)
        x = ops.short_conv_step(x, last_rows, self.taps, self.taps_bias, 'silu', env_ids, starts)
        dt, b, c = self.selected(x)
        y = ops.selective_scan_step(x, dt, -self.log_decay.exp(), b, c, state, self.through, z, self.rate_bias, True, env_ids, starts)
        return rows + F.linear(y, self.narrow.to(y.dtype))


class RecurrentPolicy(torch.nn.Module):
    """Chooses actions of ``catalogue`` from observation rows.  Parameters are float32; products and activations run in ``dtype``, the scan's states and
    the loss in float32.  Lives on the GPU: the operators have no CPU form."""

    def __init__(self, catalogue, observation_length, features=64, layers=2, states=16, taps=4, dtype=torch.bfloat16):
        super().__init__()
        if dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise TypeError('dtype must be float32, bfloat16 or float16, got %s' % dtype)
        if not (2 <= taps <= 8 and 1 <= states <= 64 and features >= 1 and layers >= 1 and observation_length >= 1):
            raise ValueError('2 to 8 taps, 1 to 64 states, and at least one feature, layer and observation entry are needed')
        self.catalogue, self.observation_length, self.features, self.dtype = catalogue, int(observation_length), int(features), dtype
        self.channels, self.n_states, self.n_taps = 2 * int(features), int(states), int(taps)
        self.inlet = torch.nn.Parameter(torch.randn(features, observation_length) / math.sqrt(observation_length))
        self.layers = torch.nn.ModuleList([_Layer(features, self.channels, states, taps) for _ in range(layers)])
        self.norm = torch.nn.Parameter(torch.ones(features))
        self.head = torch.nn.Parameter(torch.randn(len(catalogue), features) / math.sqrt(features))
        self.register_buffer('vectors', torch.from_numpy(catalogue.vectors), persistent=False)
        self.register_buffer('asset', torch.from_numpy(catalogue.asset), persistent=False)

    def memory(self, environments):
        """An empty ``PolicyMemory`` for that many environments."""
        dev = self.inlet.device
        return PolicyMemory([torch.zeros((environments, self.n_taps - 1, self.channels), dtype=self.dtype, device=dev) for _ in self.layers],
                            [torch.zeros((environments, self.channels, self.n_states), dtype=torch.float32, device=dev) for _ in self.layers])

    def _inlet(self, observations):
        if observations.shape[-1] != self.observation_length:
            raise ValueError('observations must have %d entries a row, got %d' % (self.observation_length, observations.shape[-1]))
        # entries range from per-unit voltages over flows in MW to counters: compressed alike; what a grid in outage leaves undefined counts as zero
        rows = torch.asinh(torch.nan_to_num(observations.float(), 0.0, 0.0, 0.0))
        return F.linear(rows.to(self.dtype), self.inlet.to(self.dtype))

    def _outlet(self, rows):
        return F.rms_norm(rows, rows.shape[-1:], self.norm.to(rows.dtype))

    def _check_memory(self, memory, environments=None):
        if len(memory.states) != len(self.layers):
            raise ValueError('this memory is of a policy with %d layers' % len(memory.states))
        if environments is not None and memory.states[0].shape[0] != environments:
            raise ValueError('this memory is of %d environments, not %d' % (memory.states[0].shape[0], environments))

    def window(self, observations, starts=None, memory=None):
        """``observations [batch, time, observation_length]`` -> (features [batch, time, features], the memory behind the last row).  ``starts`` marks
        first rows of episodes; ``memory`` (untouched) is what was remembered in front of the first row, nothing when None.  Differentiable: the
        backward pass reads that memory again, so acting must not move it on in between (autograd raises); act on a copy, as ``imitate`` does."""
        if memory is not None:
            self._check_memory(memory, observations.shape[0])
        rows = self._inlet(observations)
        windows, states = [], []
        for i, layer in enumerate(self.layers):
            rows, w, s = layer.window(rows, starts, (None, None) if memory is None else (memory.windows[i], memory.states[i]))
            windows.append(w.detach())
            states.append(s.detach())
        return self._outlet(rows), PolicyMemory(windows, states)

    def loss(self, observations, actions, allowed=None, starts=None, memory=None):
        """Cross entropy [batch, time] of the recorded ``actions`` (int64 numbers of the catalogue, -100: not counted) under the policy; ``allowed``
        [batch, time, words] as ``policy_ops.pack_allowed`` makes them.  Returns (loss, memory behind the window)."""
        b, t = observations.shape[:2]
        hidden, after = self.window(observations, starts, memory)
        bits = None if allowed is None else allowed.reshape(b * t, allowed.shape[-1])
        return ops.action_cross_entropy(hidden.reshape(b * t, self.features), self.head.to(self.dtype), actions.reshape(b * t), bits).view(b, t), after

    @torch.no_grad()
    def act(self, observations, memory, env_ids=None, starts=None, allowed=None, sample=False):
        """One row of each listed environment (``env_ids`` as in ``policy_ops.short_conv_step``; row i is environment i when None): its memory moves on,
        and the number of the likeliest allowed action -- with ``sample`` one drawn from the distribution -- comes back, int64 [rows].
        ``allowed [rows, actions]`` is a bool mask (``ActionCatalogue.allowed``)."""
        self._check_memory(memory)
        rows = self._inlet(observations)
        for layer, last_rows, state in zip(self.layers, memory.windows, memory.states):
            rows = layer.step(rows, last_rows, state, env_ids, starts)
        logits = F.linear(self._outlet(rows), self.head.to(self.dtype)).float()
        if allowed is not None:
            logits = logits.masked_fill(~allowed, -math.inf)
        if sample:      # the largest of the logits plus independent Gumbel noise is distributed as the softmax
            logits = logits - torch.log(torch.empty_like(logits).exponential_())
        return logits.argmax(dim=1)


def imitate(env, policy, optimizer, memory, steps, candidates=8, layout='full'):
    """Plays ``steps`` steps of every environment of ``env`` and teaches ``policy`` to choose what a search would: at each step doing nothing, the
    policy's own choice and random legal actions, ``candidates`` in all, are simulated (``BatchedRunEnv.search``), the best rewarded one is played and
    recorded, and one optimizer step is made on the window's mean cross entropy.  ``memory`` is moved behind the window.  Returns the mean loss
    (a 0-dim tensor) and the mean reward of the played actions."""
    if candidates < 2 or steps < 1:
        raise ValueError('at least one step and two candidates are needed')
    policy._check_memory(memory, env.batch)
    acting = PolicyMemory([t.clone() for t in memory.windows], [t.clone() for t in memory.states])
    observations, starts, bits, targets, gained = [], [], [], [], 0.0
    every = torch.arange(env.batch, device=policy.inlet.device)
    for _ in range(steps):
        obs, first, allowed = env.policy_rows(policy, layout=layout)
        choice = policy.act(obs, acting, starts=first, allowed=allowed)
        tried = torch.stack([torch.zeros_like(choice), choice], dim=1)
        if candidates > 2:
            tried = torch.cat([tried, torch.multinomial(allowed.float(), candidates - 2, replacement=True)], dim=1)
        rewards, done, _, _ = env.search(policy.vectors[tried])
        rewards = torch.where(done, torch.full_like(rewards, -math.inf), rewards)      # (an action that ends the episode is the last to take)
        best = rewards.argmax(dim=1)
        target = tried[every, best]
        observations.append(obs), starts.append(first), bits.append(ops.pack_allowed(allowed)), targets.append(target)
        env.step(policy.vectors[target], auto_reset=True, want_obs=False)
        gained += float(env.rewards().mean())
    losses, after = policy.loss(torch.stack(observations, dim=1), torch.stack(targets, dim=1), torch.stack(bits, dim=1), torch.stack(starts, dim=1), memory)
    loss = losses.mean()
    optimizer.zero_grad(set_to_none=True)
    loss.backward()
    optimizer.step()
    for mine, new in zip(memory.windows + memory.states, after.windows + after.states):
        mine.copy_(new)
    return loss.detach(), gained / steps
