"""rollouts.collect on the CPU, with a stand-in for the environments and the learner's operators in plain torch: what it keeps of a
policy's answers, and which answers it refuses."""
import pytest
import torch

from sustaingym_amd import learner, rollouts
from tests import learner_reference as ref

N, STATIONS, K = 4, 3, 5


class Environments:
    """Every observation is the number of steps so far."""
    output, discrete_bins, num_envs, num_stations = 'torch', K, N, STATIONS

    def __init__(self):
        self.obs, self.steps, self.played = {'demands': torch.zeros(N, STATIONS)}, 0, []

    def reset(self):
        self.obs['demands'].zero_()
        return self.obs, {}

    def step(self, levels):
        self.played.append(levels.clone())
        self.steps += 1
        self.obs['demands'] += 1.0
        return self.obs, torch.full((N,), float(self.steps), dtype=torch.float64), torch.zeros(N, dtype=torch.bool), None, {}


@pytest.fixture
def plain(monkeypatch):
    def choose_levels(logits, noise=None, mask=None):
        level, r = ref.choose(logits, noise, mask)
        return learner.LevelChoice(level, r.of_levels(level)[0].float(), r.entropy.float())

    def advantages(rewards, values, ends, last_values, gamma=0.99, lam=0.95):
        a = ref.advantages(rewards, values, ends, last_values, gamma, lam)[0].float()
        return learner.Advantages(a, a + values)
    monkeypatch.setattr(learner, 'choose_levels', choose_levels)
    monkeypatch.setattr(learner, 'advantages', advantages)


def test_a_policy_may_answer_in_the_same_tensors_every_time(plain):
    logits, values, mask = torch.zeros(N, STATIONS, K), torch.zeros(N), torch.ones((N, STATIONS, 1), dtype=torch.bool)

    def policy(obs):
        t = float(obs['demands'][0, 0])
        values.fill_(t)
        logits.zero_()
        logits[..., int(t) % K] = 9.0
        mask.fill_(True)
        mask[0] = int(t) % 2 == 0
        return logits, values, mask
    traj, obs = rollouts.collect(Environments(), policy, 4, greedy=True)
    assert traj.values[:, 0].tolist() == [0.0, 1.0, 2.0, 3.0] and traj.last_values.tolist() == [4.0] * N
    assert traj.levels[:, 1, 0].tolist() == [0, 1, 2, 3] and traj.mask[:, 0, 0, 0].tolist() == [True, False, True, False]
    want, _ = ref.advantages(traj.rewards, torch.arange(4.0)[:, None].expand(4, N), traj.ends, torch.full((N,), 4.0), 0.99, 0.95)
    assert torch.allclose(traj.advantages.double(), want, rtol=1e-6)
    values.fill_(77.0)                                        # what the policy does later changes nothing that was returned
    assert traj.last_values.tolist() == [4.0] * N and float(obs['demands'][0, 0]) == 4.0


@pytest.mark.parametrize('logits,values,match', [((N, STATIONS, K + 1), (N,), 'logits'), ((N, STATIONS, K - 1), (N,), 'logits'), ((N, STATIONS + 1, K), (N,), 'logits'),
                                                 ((N * STATIONS, K), (N,), 'logits'), ((N, STATIONS, K), (N, 1), 'values'), ((N, STATIONS, K), (), 'values')])
def test_answers_of_other_shapes_are_refused_before_a_step(plain, logits, values, match):
    venv = Environments()
    with pytest.raises(ValueError, match=match):
        rollouts.collect(venv, lambda obs: (torch.zeros(logits), torch.zeros(values)), 3)
    assert venv.steps == 0


@pytest.mark.parametrize('masks', [(None, 1), (1, None), (1, K), (K, 1)])
def test_masks_that_come_and_go_are_refused(plain, masks):
    """Stacked, they would be those of other steps."""
    def policy(obs):
        last = masks[int(obs['demands'][0, 0]) % 2]
        answer = torch.zeros(N, STATIONS, K), torch.zeros(N)
        return answer if last is None else (*answer, torch.ones((N, STATIONS, last), dtype=torch.bool))
    venv = Environments()
    with pytest.raises(ValueError, match='mask'):
        rollouts.collect(venv, policy, 4)
    assert venv.steps == 1


@pytest.mark.parametrize('shape', [(), (1,), (K,), (STATIONS, 1), (N, STATIONS, K)])
def test_masks_of_any_shape_that_broadcasts_are_kept(plain, shape):
    traj, _ = rollouts.collect(Environments(), lambda obs: (torch.zeros(N, STATIONS, K), torch.zeros(N), torch.ones(shape, dtype=torch.bool)), 2)
    assert traj.mask.shape == (2, N, STATIONS, shape[-1] if shape else 1) and bool(traj.mask.all())
