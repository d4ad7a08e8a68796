"""The Decision Transformer over recorded episodes: the seeds of its counter dropout, actions outside the environment's."""
import numpy as np
import pytest

from ray_memory_management_amd.rllib.algorithms import get_algorithm_class
from ray_memory_management_amd.rllib.offline import JsonWriter
from ray_memory_management_amd.rllib.sample_batch import SampleBatch


def _record(path, actions):
    """One episode of CartPole's shapes with the given actions."""
    n, w = len(actions), JsonWriter(str(path))
    w.write(SampleBatch({"obs": np.zeros((n, 4), np.float32), "actions": np.asarray(actions),
                         "rewards": np.ones(n, np.float32), "dones": np.eye(n, dtype=np.float32)[-1],
                         "eps_id": np.zeros(n, int)}))


def _config(path, seed=None):
    return (get_algorithm_class("DT").get_default_config().environment("CartPole-v1").offline_data(input_=str(path))
            .training(train_batch_size=4, target_return=5.0, embed_dim=8, max_seq_len=3, num_layers=1, counter_dropout=True)
            .debugging(seed=seed))


def test_counter_dropout_takes_a_seed_of_its_own(ray_shared, tmp_path):
    _record(tmp_path, [0, 1, 1, 0])
    seeds = []
    for seed in (None, None, 0, 5, 5):
        a = _config(tmp_path, seed).build()
        seeds.append(a.model.drop.seed)
        a.stop()
    assert seeds[2:] == [0, 5, 5] and len(set(seeds[:2])) == 2 and 0 not in seeds[:2]


@pytest.mark.parametrize("actions", [[0, 1, 3], [0, -1, 1]])
def test_recorded_actions_outside_the_environment_are_refused(ray_shared, tmp_path, actions):
    _record(tmp_path, actions)
    with pytest.raises(ValueError, match="recorded actions"):
        _config(tmp_path).build()
