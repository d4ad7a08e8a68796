"""Algorithm base: a Tune Trainable driving rollout workers + a learner.
Parity: reference rllib/algorithms/algorithm.py (setup: WorkerSet + policy; step ->
training_step + metrics; evaluate; compute_single_action; save/restore checkpoints; get_policy;
stop) and rllib/evaluation/metrics.py (episode_reward_mean/min/max, episode_len_mean, ...).
"""
from __future__ import annotations

import collections
import time
from typing import Any, Dict, Optional

import numpy as np

from ray_memory_management_amd.rllib.algorithms.algorithm_config import AlgorithmConfig
from ray_memory_management_amd.rllib.env import make_env
from ray_memory_management_amd.rllib.evaluation.rollout_worker import RolloutWorker
from ray_memory_management_amd.rllib.evaluation.worker_set import WorkerSet
from ray_memory_management_amd.tune.trainable import Trainable


class Algorithm(Trainable):
    _config_class = AlgorithmConfig
    # model["use_lstm"] / model["use_gated_scan"] / model["use_attention"]: only algorithms whose learners train sequence
    # models accept them (PPO, IMPALA / APPO; R2D2 brings its own recurrent Q-model); everywhere
    # else they raise instead of being silently ignored
    _supports_sequence_models = False

    @classmethod
    def get_default_config(cls) -> AlgorithmConfig:
        return cls._config_class(algo_class=cls)

    def __init__(self, config=None, env=None, logger_creator=None, **kw):
        if isinstance(config, dict) or config is None:
            cfg = self.get_default_config().update_from_dict(dict(config or {}))
        else:
            cfg = config.copy()
        if env is not None:
            cfg.env = env
        self.algo_config = cfg
        super().__init__(cfg.to_dict())

    def setup(self, config: Dict):
        import ray_memory_management_amd as ray

        if not ray.is_initialized():
            ray.init()
        c = self.algo_config
        self.validate_config(c)
        from ray_memory_management_amd.rllib.recurrent_net import wants_sequence_model

        if wants_sequence_model(c.model) and not self._supports_sequence_models:
            raise ValueError(f"{type(self).__name__} does not train recurrent / attention models: model config "
                             f"use_lstm / use_gated_scan / use_attention is supported by PPO, IMPALA and APPO (R2D2 for recurrent "
                             f"Q-learning)")
        env_creator = c.env if callable(c.env) and not isinstance(c.env, str) else None
        cfg = c.to_dict()
        self._placement_group = None
        strategy = self._rollout_worker_strategy(c)
        self.workers = WorkerSet(env_creator, cfg, num_workers=c.num_workers, worker_strategy=strategy)
        self._episode_history = collections.deque(maxlen=c.metrics_num_episodes_for_smoothing)
        self._episodes_total = 0
        self._timesteps_total = 0
        self._counters = collections.Counter()
        self._env_creator = env_creator
        self.callbacks = c.callbacks_class() if c.callbacks_class else None
        if self.callbacks is not None and hasattr(self.callbacks, "on_algorithm_init"):
            self._init_cb_pending = True
        self._multi_agent = c.is_multi_agent()
        if self._multi_agent:
            if not hasattr(self, "_ma_learner"):
                raise ValueError(f"{type(self).__name__} does not support multi-agent configs "
                                 "(multi-agent PG / A2C / PPO are supported)")
            self._setup_multi_agent()
        else:
            self._setup_learner()
        if getattr(self, "_init_cb_pending", False):
            self.callbacks.on_algorithm_init(algorithm=self)

    def _rollout_worker_strategy(self, c):
        """GPU rollout workers next to GPU learner actors: one placement-group bundle per learner
        GPU {GPU: 1}; learner k and its rollout workers share bundle k (fractional GPUs), so a
        fragment never leaves the GPU that trains on it."""
        gpu_workers = getattr(c, "gpu_rollouts", False) or (c.num_gpus_per_worker or 0) > 0
        if not (gpu_workers and getattr(c, "num_learner_workers", 0)):
            return None
        import ray_memory_management_amd as ray
        from ray_memory_management_amd.util.placement_group import placement_group
        from ray_memory_management_amd.util.scheduling_strategies import PlacementGroupSchedulingStrategy

        n = int(c.num_learner_workers)
        per = max(1, c.num_workers // n)
        cpus = c.num_cpus_per_learner_worker + per * c.num_cpus_per_worker
        gpus = min(1.0, float(c.num_gpus_per_learner_worker) + per * float(c.num_gpus_per_worker or 0))
        pg = placement_group([{"GPU": gpus, "CPU": float(cpus)} for _ in range(n)], strategy="PACK")
        ray.get(pg.ready())
        self._placement_group = pg
        # worker i feeds learner i % n (split_for_learners is round-robin): same bundle, same GPU
        return lambda i: PlacementGroupSchedulingStrategy(pg, placement_group_bundle_index=i % n)

    def learner_strategy(self):
        if getattr(self, "_placement_group", None) is None:
            return None
        from ray_memory_management_amd.util.scheduling_strategies import PlacementGroupSchedulingStrategy

        pg = self._placement_group
        return lambda r: PlacementGroupSchedulingStrategy(pg, placement_group_bundle_index=r)

    def validate_config(self, config: AlgorithmConfig):
        if config.env is None:
            raise ValueError("No env specified: use config.environment(env=...)")

    def _setup_learner(self):
        pass

    # ------------------------------------------------------------------ Trainable
    def step(self) -> Dict:
        t0 = time.time()
        c = self.algo_config
        results: Dict[str, Any] = {}
        ts0 = self._counters["num_env_steps_sampled"]
        while True:
            results = self.training_step()
            time_ok = not c.min_time_s_per_iteration or time.time() - t0 >= c.min_time_s_per_iteration
            steps_ok = self._counters["num_env_steps_sampled"] - ts0 >= (c.min_sample_timesteps_per_iteration or 0)
            if time_ok and steps_ok:
                break
        episodes = self.workers.collect_metrics()
        custom = self.workers.collect_custom_metrics() if hasattr(self.workers, "collect_custom_metrics") else {}
        for r, ln in episodes:
            self._episode_history.append((r, ln))
        self._episodes_total += len(episodes)
        hist = list(self._episode_history)
        out = {
            "episode_reward_mean": float(np.mean([h[0] for h in hist])) if hist else float("nan"),
            "episode_reward_min": float(np.min([h[0] for h in hist])) if hist else float("nan"),
            "episode_reward_max": float(np.max([h[0] for h in hist])) if hist else float("nan"),
            "episode_len_mean": float(np.mean([h[1] for h in hist])) if hist else float("nan"),
            "episodes_this_iter": len(episodes),
            "episodes_total": self._episodes_total,
            "timesteps_total": self._timesteps_total,
            "num_env_steps_sampled": self._counters["num_env_steps_sampled"],
            "num_env_steps_trained": self._counters["num_env_steps_trained"],
            "custom_metrics": __import__("ray_memory_management_amd.rllib.algorithms.callbacks",
                                         fromlist=["x"]).summarize_custom_metrics(custom),
            "info": {"learner": ({pid: {"learner_stats": st} for pid, st in results.items()}
                                 if getattr(self, "_multi_agent", False) else
                                 {"default_policy": {"learner_stats": results}}), **dict(self._counters)},
        }
        if c.evaluation_interval and (self.iteration + 1) % c.evaluation_interval == 0:
            out.update(self.evaluate())
        if self.callbacks is not None and hasattr(self.callbacks, "on_train_result"):
            self.callbacks.on_train_result(algorithm=self, result=out)
        return out

    def training_step(self) -> Dict:
        raise NotImplementedError

    # ------------------------------------------------------------------ multi-agent
    def _setup_multi_agent(self):
        """One learner per trainable policy (reference: policy_map + policies_to_train)."""
        local = self.workers.local_worker()
        self.ma_learners = {pid: self._ma_learner(pid, local.policy_map[pid]) for pid in local.policies_to_train}
        self._ma_sync()

    def _ma_sync(self):
        w = {pid: ln.get_weights() for pid, ln in self.ma_learners.items()}
        self.workers.local_worker().set_weights(w)
        self.workers.sync_weights(w)

    def _ma_training_step(self) -> Dict:
        import ray_memory_management_amd as ray
        from ray_memory_management_amd.rllib.sample_batch import concat_samples

        c = self.algo_config
        parts, steps = {}, 0
        while steps < c.train_batch_size:
            if self.workers.remote_workers():
                new = ray.get([w.sample.remote() for w in self.workers.remote_workers()])
            else:
                new = [self.workers.local_worker().sample()]
            for mb in new:
                steps += mb.count
                for pid, b in mb.policy_batches.items():
                    parts.setdefault(pid, []).append(b)
        self._counters["num_env_steps_sampled"] += steps
        self._timesteps_total += steps
        stats = {}
        for pid, ln in self.ma_learners.items():
            if pid in parts:
                b = concat_samples(parts[pid])
                stats[pid] = self._ma_update(ln, b)
                self._counters["num_agent_steps_trained"] += b.count
        self._counters["num_env_steps_trained"] += steps
        self._ma_sync()
        return stats

    def _ma_update(self, learner, batch) -> Dict:
        return learner.update(batch)

    def evaluate(self) -> Dict:
        c = self.algo_config
        rewards, lens = RolloutWorker.evaluate_episodes(self.get_policy(), self._env_creator, c.env, c.env_config,
                                                        int(c.evaluation_duration), seed=c.seed)
        # reference rllib/algorithms/algorithm.py evaluate(): metrics under the "evaluation" key
        return {"evaluation": {"episode_reward_mean": float(np.mean(rewards)),
                               "episode_reward_max": float(np.max(rewards)),
                               "episode_reward_min": float(np.min(rewards)), "episode_len_mean": float(np.mean(lens)),
                               "episodes_this_iter": len(rewards)}}

    def get_policy(self, policy_id: str = "default_policy"):
        if getattr(self, "_multi_agent", False):
            return self.workers.local_worker().get_policy(policy_id)
        return self.workers.local_worker().policy

    def compute_single_action(self, observation, *, explore: Optional[bool] = None, policy_id="default_policy"):
        return self.get_policy(policy_id).compute_single_action(observation, explore=bool(explore))

    def get_weights(self):
        return self.get_policy().get_weights()

    def set_weights(self, weights):
        self.get_policy().set_weights(weights)
        self.workers.sync_weights(weights)

    def save_checkpoint(self, checkpoint_dir: str):
        return {"weights": self.get_weights(), "counters": dict(self._counters),
                "timesteps_total": self._timesteps_total, "episodes_total": self._episodes_total,
                "extra": self._extra_state()}

    def load_checkpoint(self, ck):
        self.set_weights(ck["weights"])
        self._counters = collections.Counter(ck.get("counters", {}))
        self._timesteps_total = ck.get("timesteps_total", 0)
        self._episodes_total = ck.get("episodes_total", 0)
        self._load_extra_state(ck.get("extra") or {})

    def _extra_state(self):
        return {}

    def _load_extra_state(self, s):
        pass

    def cleanup(self):
        self.workers.stop()
        if getattr(self, "_placement_group", None) is not None:
            from ray_memory_management_amd.util.placement_group import remove_placement_group

            try:
                remove_placement_group(self._placement_group)
            except Exception:
                pass
            self._placement_group = None

    @classmethod
    def default_resource_request(cls, config):
        from ray_memory_management_amd.tune.trainable import PlacementGroupFactory

        cfg = config if isinstance(config, dict) else config.to_dict()
        head = {"CPU": cfg.get("num_cpus_for_local_worker", 1), "GPU": cfg.get("num_gpus", 0)}
        workers = [{"CPU": cfg.get("num_cpus_per_worker", 1), "GPU": cfg.get("num_gpus_per_worker", 0)}
                   for _ in range(cfg.get("num_workers", 0))]
        return PlacementGroupFactory([{k: v for k, v in head.items() if v}] +
                                     [{k: v for k, v in w.items() if v} for w in workers])
