#!/usr/bin/env python
"""Closed-loop stepping without the batch barrier (GPU box): env-steps/s of ppn_rollout_policy (device-side policy, every environment
on its own clock) next to the synchronous forms on the bench workload.
    python tools/policy_rate.py [batch] [steps]
    python tools/policy_rate.py --recurrent [batch] [steps]      a RecurrentPolicy (pypownet_amd/policy.py) in the loop instead: acting, and learning
                                                                 from the search"""
import json
import os
import sys
import time

import numpy as np

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), '..'))
sys.path.insert(0, ROOT)


def recurrent(B, K):
    import torch
    import bench
    from pypownet_amd.batched import BatchedRunEnv
    from pypownet_amd.policy import ActionCatalogue, RecurrentPolicy, imitate
    case, _, _ = bench.load_workload()
    env = BatchedRunEnv(os.path.join(ROOT, 'tests', 'golden', 'envs', bench.ENV_NAME), 'level0', B, device=0, config_overrides={'solver': 'newton'},
                        thermal_limits=bench.bench_limits(case), max_active_buses=case.nS)
    env.reset()
    catalogue = ActionCatalogue(env.case)
    policy = RecurrentPolicy(catalogue, env.engine.observation_length('minimalist'), features=256).cuda()
    memory = policy.memory(B)

    def timed(f, n):
        f()
        torch.cuda.synchronize()
        t = time.perf_counter()
        for _ in range(n):
            f()
        torch.cuda.synchronize()
        return (time.perf_counter() - t) / n
    out = {'batch': B, 'steps': K, 'actions': len(catalogue), 'features': policy.features}
    obs, starts, allowed = env.policy_rows(policy, layout='minimalist')
    out['policy_rows_ms'] = 1e3 * timed(lambda: env.policy_rows(policy, layout='minimalist'), K)
    out['act_ms'] = 1e3 * timed(lambda: policy.act(obs, memory, starts=starts, allowed=allowed), K)
    step = timed(lambda: env.step(env.policy_actions(policy, memory=memory, layout='minimalist'), want_obs=False), K)
    out['closed_loop_env_steps_per_s'] = B / step
    window = [v[:, None].expand(v.shape[0], 32, *v.shape[1:]) for v in (obs, starts)]
    target = torch.zeros((B, 32), dtype=torch.int64, device='cuda')

    def learn():
        policy.loss(window[0], target, starts=window[1], memory=memory)[0].mean().backward()
    out['learn_32_rows_ms'] = 1e3 * timed(learn, 3)
    optimizer = torch.optim.SGD(policy.parameters(), lr=1e-3)
    out['imitate_4_steps_of_8_candidates_ms'] = 1e3 * timed(lambda: imitate(env, policy, optimizer, memory, steps=4, layout='minimalist'), 1)
    print(json.dumps(out))


def main():
    if '--recurrent' in sys.argv[1:]:
        given = [int(a) for a in sys.argv[1:] if a != '--recurrent']
        return recurrent(given[0] if given else 1024, given[1] if len(given) > 1 else 20)
    import torch
    import bench
    from pypownet_amd.engine import Engine
    B = int(sys.argv[1]) if len(sys.argv) > 1 else 4096
    K = int(sys.argv[2]) if len(sys.argv) > 2 else 60
    case, conf, chronics = bench.load_workload()
    out = {'batch': B, 'steps': K}
    for policy, params in (('do_nothing', []), ('line_relief', [1.0])):
        eng = Engine(case, conf, B, chronics=chronics, thermal_limits=bench.bench_limits(case), max_active_buses=case.nS)
        slots, t0 = bench.env_assignment(0, B, chronics)
        eng.reset(chronic_slot=slots, t0=t0)
        buf = torch.zeros((B, case.action_length), dtype=torch.uint8, device='cuda')
        torch.cuda.synchronize()
        for _ in range(5):
            eng.policy_actions(policy, params, buf.data_ptr())
            eng.step_device(buf.data_ptr(), auto_reset=1)
        eng.sync()
        # synchronous closed loop: policy kernel + step kernel per step
        n0 = int(eng.read('N_STEPS').astype(np.int64).sum())
        t = time.perf_counter()
        for _ in range(K):
            eng.policy_actions(policy, params, buf.data_ptr())
            eng.step_device(buf.data_ptr(), auto_reset=1)
        eng.sync()
        el = time.perf_counter() - t
        n1 = int(eng.read('N_STEPS').astype(np.int64).sum())
        out[policy + '_stepped_env_steps_per_s'] = (n1 - n0) / el
        # the same closed loop in one launch
        eng.rollout_policy(policy, params, 4)
        eng.sync()
        n0 = int(eng.read('N_STEPS').astype(np.int64).sum())
        t = time.perf_counter()
        eng.rollout_policy(policy, params, K)
        eng.sync()
        el = time.perf_counter() - t
        n1 = int(eng.read('N_STEPS').astype(np.int64).sum())
        out[policy + '_rollout_policy_env_steps_per_s'] = (n1 - n0) / el
        out[policy + '_envs_done_last_step'] = int(eng.read('DONE').sum())
        if policy == 'do_nothing':      # the open-loop rollout of round 3 for comparison (same agent)
            n0 = n1
            t = time.perf_counter()
            eng.rollout_device(buf.zero_().data_ptr(), K, per_step_actions=False, auto_reset=1)
            eng.sync()
            el = time.perf_counter() - t
            out['do_nothing_open_loop_rollout_env_steps_per_s'] = (int(eng.read('N_STEPS').astype(np.int64).sum()) - n0) / el
        eng.close()
    print(json.dumps(out))


if __name__ == '__main__':
    main()
