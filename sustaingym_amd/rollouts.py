"""Whole-episode evaluation of arithmetic-free policies for a BATCH of seeds in one engine call.

What the reference does with a Python loop — ``BaseAlgorithm.run(seeds)`` resets the environment
with every seed in turn and steps a ``GreedyAlgorithm`` / ``RandomAlgorithm`` until the episode ends
(sustaingym/algorithms/base.py:38-99, algorithms/evcharging/baselines.py:22-51) — is done here the
other way round: every seed becomes one environment of a batch, the policy lives on the GPU
(``EVC_ACTION_GREEDY`` / ``EVC_ACTION_RANDOM``) and ``evc_rollout`` plays all 288 periods of all
episodes in ONE kernel launch (csrc/evc_rollout.h: the environments' state stays in registers, no
per-period action read or observation write).  The result has the columns of the reference's DataFrame
(``seed``, ``return``, ``max_profit``, ``reward_breakdown``).

MPC / OfflineOptimal (baselines.py:54-223) are cvxpy programs that merely call ``step()``; they stay
out of scope.  Policies that need Python (a trained network, a user's controller) go
through :func:`run_policy`, which drives any environment of this package — ``EVChargingEnv``, a wrapped
one, the multi-agent one — through its own ``reset`` / ``step``.

A network that lives on the GPU plays the whole batch: :func:`collect` steps an ``EVChargingVectorEnv(output='torch',
discrete_bins=K)`` on the levels that it chooses (:func:`learner.choose_levels`) and returns the trajectory with advantages
(:func:`learner.advantages`); :func:`score` asks a policy again about the levels that were played, with gradients
(:func:`learner.level_logprobs`).
"""
from __future__ import annotations

from typing import Any, Iterable, NamedTuple, Sequence

import numpy as np

from . import _lib
from .hostio import to_host
from .engine import StepEngine
from .event_generation import AbstractTraceGenerator
from .network import site_str_to_site

POLICIES = ('greedy', 'random')
EPISODE_STEPS = _lib.EPISODE_STEPS


def _episode_bank(generator: AbstractTraceGenerator, seeds: Sequence[int], stride: int):
    """One episode per seed, exactly as ``env.reset(seed=seed)`` would create it (env.py:314-323:
    ``set_seed``, event table, then the MOER matrix of the already-advanced day)."""
    ns = np.zeros(len(seeds), np.int32)
    sessions = np.zeros((len(seeds), stride), dtype=_lib.SESSION_DTYPE)
    requested = np.zeros((len(seeds), stride), np.float64)
    moer = np.zeros((len(seeds), _lib.MOER_ROWS, _lib.MOER_COLS), np.float64)
    max_profit = np.zeros(len(seeds), np.float64)
    for i, seed in enumerate(seeds):
        generator.set_seed(int(seed))
        table = generator.get_event_table()
        if len(table) > stride:
            raise ValueError(f'seed {seed}: {len(table)} sessions exceed the engine capacity {stride}')
        ns[i] = len(table)
        sessions[i, :ns[i]] = table.sessions
        requested[i, :ns[i]] = table.requested
        max_profit[i] = table.max_profit()
        moer[i] = generator.get_moer()
    return ns, sessions, requested, moer, max_profit


class PolicyRollout:
    """Plays one episode per seed under a device-resident policy.

    Args:
        data_generator: a trace generator of this package (``RealTraceGenerator``,
            ``GMMsTraceGenerator``): seed ``s`` yields the episode ``EVChargingEnv.reset(seed=s)`` plays.
        policy: ``'greedy'`` — full rate wherever the observed demand is non-zero (baselines.py:32-35) —
            or ``'random'`` — uniform actions (baselines.py:45-51) from the engine's counter-based
            stream (``evc_set_policy_seed``; numpy's sequential ``default_rng`` cannot be drawn by
            thousands of wavefronts, so action values differ from the reference's stream by design).
        discrete_bins: ``> 0`` = the policy acts through ``DiscreteActionWrapper(bins)``
            (wrappers.py:13-45); greedy is unaffected (its maximum action maps to 1.0 either way).
    """

    def __init__(self, data_generator: AbstractTraceGenerator, policy: str = 'greedy',
                 moer_forecast_steps: int = 36, project_action_in_env: bool = True,
                 discrete_bins: int = -1, policy_seed: int = 0, device: int = 0,
                 max_sessions: int = _lib.MAX_SESSIONS, charge_calculation: str = 'continuous'):
        if policy not in POLICIES:
            raise ValueError(f'policy must be one of {POLICIES}')
        self.data_generator = data_generator
        self.policy = policy
        self.cn = site_str_to_site(data_generator.site)
        self.k = int(moer_forecast_steps)
        self.project = bool(project_action_in_env)
        self.bins = int(discrete_bins) if discrete_bins and discrete_bins > 0 else 0
        self.policy_seed = int(policy_seed)
        self.device = int(device)
        self.max_sessions = int(max_sessions)
        self.charge_calculation = charge_calculation

    def run(self, seeds: Iterable[int] | int, env_id_base: int = 0) -> dict[str, np.ndarray | list]:
        """All episodes at once.  Returns ``{'seed', 'return', 'max_profit', 'reward_breakdown',
        'status'}``; ``reward_breakdown`` is a list of dicts like the reference's ``info`` column."""
        import torch
        seeds = list(range(seeds)) if isinstance(seeds, int) else [int(s) for s in seeds]
        if not seeds:
            return {'seed': [], 'return': np.zeros(0), 'max_profit': np.zeros(0), 'reward_breakdown': [],
                    'status': np.zeros(0, np.int32)}
        B = len(seeds)
        ns, sessions, requested, moer, max_profit = _episode_bank(self.data_generator, seeds, self.max_sessions)
        eng = StepEngine(self.cn, B, moer_forecast_steps=self.k, project_action=self.project, autoreset=False,
                         device=self.device, bank_slots=B, max_sessions=self.max_sessions, moer_days=B,
                         charge_calculation=self.charge_calculation)
        try:
            eng.upload_moer(moer)
            eng.upload_episodes(ns, sessions, requested, np.arange(B, dtype=np.int32))
            eng.set_policy_seed(self.policy_seed, env_id_base)
            eng.reset()
            out = eng.rollout(policy=self.policy, steps=EPISODE_STEPS, bins=self.bins)
            torch.cuda.synchronize(self.device)
            assert bool(out['terminated'].all()), 'episodes must end after 288 periods'
            returns = to_host(out['returns']).copy()
            breakdown = to_host(out['breakdown']).copy()
            status = eng.env_scalars()['status']
        finally:
            eng.close()
        return {
            'seed': seeds, 'return': returns, 'max_profit': max_profit,
            'reward_breakdown': [{'profit': float(b[0]), 'carbon_cost': float(b[1]), 'excess_charge': float(b[2])}
                                 for b in breakdown],
            'status': status,
        }

    def run_frame(self, seeds: Iterable[int] | int):
        """``run`` as a pandas DataFrame (the reference's return type)."""
        import pandas as pd
        res = self.run(seeds)
        return pd.DataFrame({k: (list(v) if isinstance(v, np.ndarray) else v) for k, v in res.items()})


def evaluate(data_generator: AbstractTraceGenerator, policy: str, seeds: Iterable[int] | int, **kwargs):
    """Shorthand: ``PolicyRollout(data_generator, policy, **kwargs).run(seeds)``."""
    return PolicyRollout(data_generator, policy, **kwargs).run(seeds)


def run_policy(env, policy, seeds: Iterable[int] | int) -> dict[str, list]:
    """Evaluation of a host-side policy on ANY single environment of this package through its public API: one
    episode per seed, ``policy(observation) -> action`` asked once per period.  For callers of the reference's
    ``BaseAlgorithm.run`` whose controller is Python code (what the device-resident :class:`PolicyRollout` cannot
    take).  Multi-agent environments (dict-of-agents observations) work too: rewards are summed over agents and an
    episode ends when every agent is done.  Returns the columns of :meth:`PolicyRollout.run`."""
    seeds = list(range(seeds)) if isinstance(seeds, int) else [int(s) for s in seeds]
    out: dict[str, list] = {'seed': [], 'return': [], 'max_profit': [], 'reward_breakdown': []}
    for seed in seeds:
        obs, info = env.reset(seed=seed)
        total, finished = 0.0, False
        while not finished:
            obs, reward, terminated, truncated, info = env.step(policy(obs))
            if isinstance(reward, dict):                                  # PettingZoo-parallel style
                total += float(sum(reward.values()))
                finished = all(terminated.values()) or all(truncated.values()) or not terminated
                info = next(iter(info.values())) if info else {}
            else:
                total += float(reward)
                finished = bool(terminated) or bool(truncated)
        out['seed'].append(seed)
        out['return'].append(total)
        out['max_profit'].append(info.get('max_profit'))
        out['reward_breakdown'].append(info.get('reward_breakdown'))
    return out


class Trajectory(NamedTuple):
    """``T`` steps of ``N`` environments with ``n`` stations (device tensors; ``obs``: a dict of ``[T, N, ...]``)."""
    obs: dict
    levels: Any          # int64 [T, N, n], what was played
    logprobs: Any        # float32 [T, N, n], under the policy that played
    entropy: Any         # float32 [T, N, n]
    mask: Any            # bool [T, N, n, 1 or K] or None: what the policy allowed
    rewards: Any         # float64 [T, N]
    values: Any          # float32 [T, N], the policy's estimates
    ends: Any            # bool [T, N]: the episode ended with this step
    last_values: Any     # float32 [N]: of the observation behind the last step
    advantages: Any      # float32 [T, N]
    targets: Any         # float32 [T, N]: advantages + values


def _ask(policy, obs):
    answer = policy(obs)
    return answer if len(answer) == 3 else (*answer, None)


def collect(venv, policy, steps: int, obs=None, gamma: float = 0.99, lam: float = 0.95, greedy: bool = False, generator=None):
    """``steps`` steps of a batch under a policy on the GPU; returns ``(Trajectory, obs)``, the observation to go on from.

    venv: ``EVChargingVectorEnv(..., output='torch', discrete_bins=K)``; episodes begin anew by themselves.
    policy: ``policy(obs) -> (logits [N, n, K], values [N])`` or ``(logits, values, mask)``; mask: bool, broadcastable to the
        logits, True = allowed (a station that it leaves nothing gets level 0), given at every step or at none.  K is the
        environments' ``discrete_bins``; answers of other shapes raise ``ValueError`` before a step is taken on them.
    obs: the observation to begin with; None resets the environments.
    greedy: the most probable level instead of a sampled one (``generator``: the torch generator of the samples).

    The steps are enqueued on the current stream and no gradient is recorded.  The host waits for the GPU where the environments do:
    ``reset`` and a step that ends the episodes fetch the ``max_profit`` of episodes that were generated on the GPU."""
    import torch
    from . import learner
    if getattr(venv, 'output', None) != 'torch' or not venv.discrete_bins > 0:
        raise ValueError("collect needs an EVChargingVectorEnv with output='torch' and discrete_bins > 0")
    if steps < 1:
        raise ValueError(f'steps: at least 1, got {steps}')
    rows: dict[str, list] = {key: [] for key in ('levels', 'logprobs', 'entropy', 'mask', 'rewards', 'values', 'ends')}
    seen: list[dict] = []
    allowed = None
    rows_of = (venv.num_envs, venv.num_stations, venv.discrete_bins)

    def kept(values):                                # (a policy may answer in the same tensor every time)
        return values.to(torch.float32, copy=True)

    with torch.no_grad():
        if obs is None:
            obs, _ = venv.reset()
        for _ in range(steps):
            seen.append({key: val.clone() for key, val in obs.items()})      # (the environments overwrite theirs)
            logits, values, mask = _ask(policy, seen[-1])
            if tuple(logits.shape) != rows_of:
                raise ValueError(f'logits: {tuple(logits.shape)}, the environments take {rows_of} (environments, stations, discrete_bins)')
            if tuple(values.shape) != rows_of[:1]:
                raise ValueError(f'values: {tuple(values.shape)} instead of {rows_of[:1]}')
            kind = None if mask is None else mask.shape[-1] if mask.dim() else 1
            if len(seen) > 1 and kind != allowed:
                raise ValueError('mask: given at every step, with the same last dimension, or at none')
            allowed = kind
            noise = None if greedy else torch.empty(logits.shape, dtype=torch.float32, device=logits.device).exponential_(
                generator=generator).clamp_(min=1e-30).log_().neg_()         # Gumbel
            choice = learner.choose_levels(logits, noise, mask)
            obs, rewards, ends, _, _ = venv.step(choice.levels)
            for key, val in (*zip(('levels', 'logprobs', 'entropy'), choice), ('values', kept(values)), ('rewards', rewards.clone()),
                             ('ends', ends.clone())):
                rows[key].append(val)
            if mask is not None:
                rows['mask'].append(mask.expand((*rows_of[:2], kind)).clone())
        last_values = kept(_ask(policy, obs)[1])
        if tuple(last_values.shape) != rows_of[:1]:
            raise ValueError(f'values: {tuple(last_values.shape)} instead of {rows_of[:1]}')
        out = {key: torch.stack(val) if val else None for key, val in rows.items()}
        adv = learner.advantages(out['rewards'], out['values'], out['ends'], last_values, gamma, lam)
        return Trajectory(obs={key: torch.stack([o[key] for o in seen]) for key in seen[0]}, last_values=last_values,
                          advantages=adv.advantages, targets=adv.targets, **out), {key: val.clone() for key, val in obs.items()}


def score(trajectory: Trajectory, policy, top: int = 0):
    """The levels of a trajectory under ``policy`` as it is now: ``(learner.LevelScores, values [T, N])`` with gradients to its
    parameters.  The policy is asked once, about ``T * N`` observations; what was allowed is what the trajectory says."""
    from . import learner
    T, N = trajectory.rewards.shape
    logits, values, _ = _ask(policy, {key: val.flatten(0, 1) for key, val in trajectory.obs.items()})
    logits = logits.unflatten(0, (T, N))
    return learner.level_logprobs(logits, trajectory.levels, trajectory.mask, top), values.unflatten(0, (T, N))
