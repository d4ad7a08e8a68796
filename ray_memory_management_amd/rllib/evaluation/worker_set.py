"""WorkerSet: one local RolloutWorker + N remote RolloutWorker actors.
Parity: reference rllib/evaluation/worker_set.py (local_worker, remote_workers, sync_weights,
foreach_worker, add_workers, recreate failed workers) and
rllib/execution/rollout_ops.py:synchronous_parallel_sample.
Weights are broadcast with ONE ray.put per sync (every worker reads the same shm object)."""
from __future__ import annotations

import os
from typing import Callable, List, Optional

import ray_memory_management_amd as ray
from ray_memory_management_amd.rllib.evaluation.rollout_worker import RolloutWorker
from ray_memory_management_amd.rllib.recurrent_net import wants_sequence_model
from ray_memory_management_amd.rllib.sample_batch import SampleBatch, concat_samples


class WorkerSet:
    def __init__(self, env_creator=None, config: Optional[dict] = None, num_workers: int = 0,
                 local_worker: bool = True, worker_strategy: Optional[Callable[[int], object]] = None):
        """`worker_strategy(i)` (optional) gives remote worker i's scheduling strategy, e.g. the
        placement-group bundle it shares with its learner GPU."""
        self._config = dict(config or {})
        self._env_creator = env_creator
        cls = RolloutWorker
        if (self._config.get("multiagent") or {}).get("policies"):
            from ray_memory_management_amd.rllib.evaluation.multi_agent_worker import MultiAgentRolloutWorker

            cls = MultiAgentRolloutWorker
        self._local = cls(env_creator, self._config, 0, num_workers) if local_worker else None
        if cls is not RolloutWorker:
            pass
        elif self._config.get("gpu_rollouts"):
            from ray_memory_management_amd.rllib.evaluation.gpu_rollout_worker import GPURolloutWorker

            cls = GPURolloutWorker
        elif self._config.get("num_gpus_per_worker", 0) and env_creator is None and not wants_sequence_model(
                self._config.get("model")):
            from ray_memory_management_amd.rllib.env import _VECTOR_REGISTRY

            env = self._config.get("env")
            if isinstance(env, str) and env in _VECTOR_REGISTRY:
                # CPU vector env + policy on the worker's GPU (RLlib num_gpus_per_worker > 0)
                from ray_memory_management_amd.rllib.evaluation.gpu_rollout_worker import HybridRolloutWorker

                cls = HybridRolloutWorker
        opts = dict(num_cpus=self._config.get("num_cpus_per_worker", 1),
                    num_gpus=self._config.get("num_gpus_per_worker", 0))
        if cls.__name__ in ("HybridRolloutWorker", "GPURolloutWorker"):
            # rollout workers drive one stream: one hardware queue each keeps many co-located worker
            # processes from oversubscribing the GPU's queue slots (the learner keeps the default)
            q = self._config.get("rollout_worker_hw_queues", int(os.environ.get("RMM_ROLLOUT_HW_QUEUES", "1")))
            if q:
                opts["runtime_env"] = {"env_vars": {"GPU_MAX_HW_QUEUES": str(int(q))}}
        self.remote_worker_class = cls  # which rollout-worker class the remote actors run
        self._remote_cls = ray.remote(cls).options(**opts)
        self._strategy = worker_strategy
        self._remote: List = []
        self.add_workers(num_workers)

    def add_workers(self, n: int):
        start = len(self._remote)
        for i in range(n):
            cls = self._remote_cls
            if self._strategy is not None:
                cls = cls.options(scheduling_strategy=self._strategy(start + i))
            self._remote.append(cls.remote(self._env_creator, self._config, start + i + 1, start + n))

    def local_worker(self) -> RolloutWorker:
        return self._local

    def remote_workers(self) -> List:
        return list(self._remote)

    def num_remote_workers(self) -> int:
        return len(self._remote)

    def sync_weights(self, weights=None, from_worker=None, ref=None):
        """Broadcast weights to the remote workers through ONE store object (`ref` if the caller
        already has one, e.g. the learner actor's returned weights)."""
        if ref is not None:
            if self._remote:
                ray.get([w.set_weights.remote(ref) for w in self._remote])
            return
        if weights is None:
            weights = (from_worker or self._local).get_weights()
        if self._remote:
            ref = ray.put(weights)
            ray.get([w.set_weights.remote(ref) for w in self._remote])
        if self._local is not None and from_worker is not None and from_worker is not self._local:
            self._local.set_weights(weights)

    def foreach_worker(self, fn: Callable, local_worker: bool = True):
        out = [fn(self._local)] if local_worker and self._local is not None else []
        if self._remote:
            out += ray.get([w.apply.remote(fn) for w in self._remote])
        return out

    def synchronous_parallel_sample(self, max_env_steps: int, concat: bool = True):
        """Sample until >= max_env_steps were collected (reference rollout_ops.py). concat=False
        returns the list of per-worker batches (fragments keep their layout for learner ingest)."""
        batches, steps = [], 0
        while steps < max_env_steps:
            if self._remote:
                new = ray.get([w.sample.remote() for w in self._remote])
            else:
                new = [self._local.sample()]
            for b in new:
                steps += b.count
            batches += new
        return concat_samples(batches) if concat else batches

    def collect_metrics(self) -> List[tuple]:
        out = list(self._local.get_metrics()) if self._local is not None else []
        if self._remote:
            for m in ray.get([w.get_metrics.remote() for w in self._remote]):
                out += m
        return out

    def collect_custom_metrics(self):
        """Per-metric value lists recorded by episode callbacks since the last call."""
        out = {}
        parts = []
        if self._local is not None and hasattr(self._local, "get_custom_metrics"):
            parts.append(self._local.get_custom_metrics())
        if self._remote and self._config.get("callbacks") is not None:
            parts += ray.get([w.get_custom_metrics.remote() for w in self._remote])
        for p in parts:
            for k, v in (p or {}).items():
                out.setdefault(k, []).extend(v)
        return out

    def recreate_failed_workers(self):
        alive = []
        for i, w in enumerate(self._remote):
            try:
                ray.get(w.get_metrics.remote(), timeout=30)
                alive.append(w)
            except Exception:
                alive.append(self._remote_cls.remote(self._env_creator, self._config, i + 1, len(self._remote)))
        self._remote = alive

    def stop(self):
        for w in self._remote:
            try:
                ray.kill(w)
            except Exception:
                pass
        self._remote = []
