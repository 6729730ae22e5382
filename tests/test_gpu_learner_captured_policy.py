"""rollouts.collect with a policy that is captured into a graph: it answers in the graph's own tensors every time."""
import pytest
import torch

from tests.test_gpu_learner_rollout import K, Policy, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('masked', [True, False])
def test_a_captured_policy_gives_the_eager_ones_trajectory(masked):
    from sustaingym_amd import rollouts
    eager_env, env = make(), make()
    N, n, T = env.num_envs, env.num_stations, 40
    policy = Policy(n, masked=masked)
    demands = torch.zeros((N, n), device='cuda')
    with torch.no_grad():
        policy({'demands': demands})
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            answer = policy({'demands': demands})
    assert answer[0].shape == (N, n, K) and answer[1].dtype == torch.float32

    def captured(obs):
        demands.copy_(obs['demands'])
        graph.replay()
        return answer

    def play(venv, p):
        g = torch.Generator(device='cuda')
        g.manual_seed(4)
        first, _ = venv.reset(seed=1)
        first = {key: val.clone() for key, val in first.items()}
        for _ in range(100):                                            # (into the morning, where stations have demands)
            first, _, _, _, _ = venv.step(policy='greedy')
        return rollouts.collect(venv, p, T, obs={key: val.clone() for key, val in first.items()}, generator=g)[0]

    want, got = play(eager_env, policy), play(env, captured)
    assert float(want.values.std(0).max()) > 0
    for name in ('levels', 'logprobs', 'entropy', 'rewards', 'values', 'ends', 'last_values', 'advantages', 'targets', *(('mask',) if masked else ())):
        assert torch.equal(getattr(want, name), getattr(got, name)), name
    eager_env.close()
    env.close()
