"""Operators of token and sequence models: embedding with a sorted gradient, counter-based dropout and the gated
linear recurrence (kernels K22-K24 in ``csrc/hip/{embedding,dropout,scan}_kernels.hip``, their torch operators with
autograd in ``csrc/hip/seq_torch.cc``).

CUDA(ROCm) tensors run the HIP kernels on the current stream of their device; CPU tensors the same formulas in torch.
fp32, bf16 and fp16 are taken on the GPU; sums and states are held in fp32. Everything here can be captured into a
graph: nothing synchronises, and what a call keeps for its backward pass belongs to that call. (A capture refuses leaves
that a graph made outside it still holds: torch's engine would have the captured backward pass wait on their stream.)
Second and forward-mode derivatives are refused on the GPU.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from ray_memory_management_amd._native import require_seq

__all__ = ["embedding", "Embedding", "dropout", "Dropout", "repeatable", "gated_scan", "gated_scan_step"]

_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # the type codes of the kernels


def _code(who: str, t: torch.dtype) -> int:
    c = _CODE.get(t)
    if c is None:
        raise ValueError(f"{who}: fp32, bf16 or fp16 tensors on the GPU, not {t}")
    return c


def _same_device(who: str, ref: torch.Tensor, **tensors) -> None:
    dev = ref.device
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{who}: {name} is on {t.device}, not on {dev}")


# ------------------------------------------------------------------------------------------ embedding
def _embedding_cpu(ids, weight, scale, padding_idx, dtype):
    w = weight if weight.dtype in (torch.float32, torch.float64) else weight.float()
    pad = padding_idx if padding_idx >= 0 else None
    if weight.shape[0] == 0:
        out = w.sum() + w.new_zeros((*ids.shape, w.shape[1]))
    else:
        try:
            out = nn.functional.embedding(ids, w, pad)
        except (IndexError, RuntimeError):  # torch looks at each id on the CPU, and most calls have none outside
            ok = (ids >= 0) & (ids < weight.shape[0])
            out = nn.functional.embedding(torch.where(ok, ids, torch.zeros_like(ids)), w, pad)
            out = torch.where(ok.unsqueeze(-1), out, torch.zeros((), dtype=out.dtype))
    return (out if scale == 1.0 else out * scale).to(dtype)


def embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, padding_idx: Optional[int] = None,
              dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``out[...] = scale * weight[ids[...]]``, rounded once to ``dtype`` (weight's type by default).

    ids: int32 / int64 of any shape; an id outside ``[0, len(weight))`` gives a row of zeros and no gradient, so -1
    can mark padded places. weight: [V, D]. Its gradient is dense, ``scale * sum of dy over the places of an id``,
    summed in fp32 in a grouping that the sizes and types alone choose (the same bits every time) and rounded once; the row ``padding_idx``
    (negative counts from the end) is read as any other and gets no gradient."""
    if ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"embedding: int32 or int64 ids, not {ids.dtype}")
    if weight.dim() != 2:
        raise ValueError(f"embedding: weight must be [V, D], not {tuple(weight.shape)}")
    _same_device("embedding", weight, ids=ids)
    V, pad, dtype = weight.shape[0], -1, dtype or weight.dtype
    if padding_idx is not None:
        if not -V <= padding_idx < V:
            raise ValueError(f"embedding: padding_idx {padding_idx} outside the {V} rows")
        pad = int(padding_idx) % V
    if not dtype.is_floating_point or not weight.dtype.is_floating_point:
        raise ValueError("embedding: floating-point weight and output types")
    if not weight.is_cuda:
        return _embedding_cpu(ids, weight, float(scale), pad, dtype)
    _code("embedding", weight.dtype), _code("embedding", dtype)
    if max(ids.numel(), V) >= 2 ** 31 - 1:
        raise ValueError("embedding: fewer than 2^31 - 1 ids and rows")
    return require_seq().embedding(ids, weight, scale, pad, _CODE[dtype])


class Embedding(nn.Embedding):
    """``nn.Embedding`` through :func:`embedding`: the same parameters and state dict, with a ``scale`` on the output.
    ``max_norm``, ``scale_grad_by_freq`` and ``sparse`` are not supported."""

    def __init__(self, num_embeddings: int, embedding_dim: int, padding_idx: Optional[int] = None, *,
                 scale: float = 1.0, **kw):
        for k in ("max_norm", "scale_grad_by_freq", "sparse"):
            if kw.get(k):
                raise ValueError(f"Embedding: {k} is not supported")
        super().__init__(num_embeddings, embedding_dim, padding_idx=padding_idx, **kw)
        self.scale = float(scale)

    def forward(self, ids):
        return embedding(ids, self.weight, self.scale, self.padding_idx)


# ------------------------------------------------------------------------------------------ dropout
_M32 = 0xFFFFFFFF


def _mulhilo(m: int, x: torch.Tensor):
    """High and low word of m * x for 32-bit words held in int64 (the product itself could pass 63 bits)."""
    low, high = (m & 0xFFFF) * x, (m >> 16) * x
    mid = (low >> 16) + high
    return mid >> 16, ((mid & 0xFFFF) << 16) | (low & 0xFFFF)


def _philox_words(index: torch.Tensor, offset: int, seed: int) -> torch.Tensor:
    """The four 32-bit words (int64, [n, 4]) of Philox4x32-10 (Salmon et al. 2011) at counter (index, offset)."""
    a, b = index & _M32, (index >> 32) & _M32
    c, d = torch.full_like(index, offset & _M32), torch.full_like(index, (offset >> 32) & _M32)
    k0, k1 = seed & _M32, (seed >> 32) & _M32
    for _ in range(10):
        h0, l0 = _mulhilo(0xD2511F53, a)
        h1, l1 = _mulhilo(0xCD9E8D57, c)
        a, b, c, d = h1 ^ b ^ k0, l1, h0 ^ d ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    return torch.stack([a, b, c, d], dim=-1)


def _threshold(p: float) -> int:
    return int(round(p * 65536))


def _dropout_cpu(x, p, seed, offset, residual):
    n, t = x.numel(), _threshold(p)
    w = _philox_words(torch.arange((n + 7) // 8), int(offset), seed)
    keep = torch.stack([w & 0xFFFF, w >> 16], dim=-1).reshape(-1)[:n].reshape(x.shape) >= t
    acc = x if x.dtype == torch.float64 else x.float()
    # the dropped places go out before the product, so that what they hold reaches neither result nor gradient
    y = torch.where(keep, acc, torch.zeros((), dtype=acc.dtype)) * (65536.0 / (65536 - t) if t < 65536 else 0.0)
    return (y if residual is None else y + residual.to(y.dtype)).to(x.dtype)


def dropout(x: torch.Tensor, p: float, seed: int, offset: Union[int, torch.Tensor] = 0,
            residual: Optional[torch.Tensor] = None, training: bool = True) -> torch.Tensor:
    """``residual + dropout(x)`` whose mask is a function of (seed, offset, element index) and never stored.

    An element is dropped (zero, whatever it held) where its 16 random bits are below ``t = round(65536 p)``, else
    scaled by ``65536 / (65536 - t)``; the bits are those of Philox4x32-10 with key ``seed`` and counter
    (index // 8, offset), so the CPU and the GPU draw the same mask. Elements are numbered in row-major order. (p above
    1 - 2^-17 drops everything; the GPU takes fewer than 2^35 elements.)

    offset: the call's own number under the seed: an int, or an int64 tensor on x's device whose first element is read
    when the kernel runs (a graph replay then draws a new mask after each advance); the backward pass uses the value
    that its forward pass read. A call that activation checkpointing repeats reads the tensor again: there, give it one
    that stays as it is until the backward pass. residual: same shape and type as x."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout: p must be in [0, 1], not {p}")
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError(f"dropout: residual must match x: {tuple(residual.shape)} {residual.dtype} against "
                             f"{tuple(x.shape)} {x.dtype}")
        _same_device("dropout", x, residual=residual)
    ctr = None
    if isinstance(offset, torch.Tensor):
        if offset.dtype != torch.int64 or offset.numel() < 1:
            raise ValueError("dropout: an offset tensor holds int64")
        _same_device("dropout", x, offset=offset)
        ctr, offset = offset, 0
    if not x.dtype.is_floating_point:
        raise ValueError(f"dropout: a floating-point tensor, not {x.dtype}")
    if not training:
        return x if residual is None else x + residual
    p, seed, offset = float(p), int(seed) & 0xFFFFFFFFFFFFFFFF, int(offset) & 0xFFFFFFFFFFFFFFFF
    if not x.is_cuda:
        return _dropout_cpu(x, p, seed, offset if ctr is None else int(ctr.reshape(-1)[0]), residual)
    _code("dropout", x.dtype)
    return require_seq().dropout(x, residual, p, seed, offset, ctr)


def _in_backward() -> bool:
    """Whether this thread runs a backward pass, which calls layers only to recompute what they gave."""
    return torch._C._current_graph_task_id() != -1


class Dropout(nn.Module):
    """Dropout layer over :func:`dropout`. Its call counter is a buffer on the layer's device that every training call
    advances there, so a captured graph draws a new mask on each replay and a restored state dict goes on where it was
    saved. Masks follow from the seed and the counter alone: layers of one model take different seeds, and so do the
    ranks of a data-parallel group.

    Activation checkpointing calls the layer again in the backward pass, when the counter has moved on. Checkpoint
    ``ops.repeatable(block)`` in place of ``block``; without it the second call raises."""

    _repeats = 0  # above 0 while :class:`repeatable` has set the counter back

    def __init__(self, p: float = 0.5, seed: int = 0):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"Dropout: p must be in [0, 1], not {p}")
        self.p, self.seed = float(p), int(seed)
        self.register_buffer("counter", torch.zeros(1, dtype=torch.int64))

    def forward(self, x, residual=None):
        if not self.training or self.p == 0.0:
            return dropout(x, self.p, self.seed, residual=residual, training=False)
        if not self._repeats and _in_backward():
            raise RuntimeError("Dropout: called again in a backward pass, where its counter has moved on and would draw "
                               "another mask: checkpoint ops.repeatable(block) in place of the block")
        y = dropout(x, self.p, self.seed, self.counter, residual)
        self.counter.add_(1)
        return y

    def extra_repr(self):
        return f"p={self.p}, seed={self.seed}"


class repeatable:
    """``fn`` for one checkpointed call, ``checkpoint(ops.repeatable(block), x)``, with either ``use_reentrant``.

    The first call notes the counters of the :class:`Dropout` layers in ``fn``; the later ones, of the recomputation,
    start from these and leave the layers as they were, so they draw the masks of the first. modules: where the layers
    are if ``fn`` is no module itself. Each checkpointed call takes a wrapper of its own."""

    def __init__(self, fn, *modules: nn.Module):
        roots = [m for m in (fn, *modules) if isinstance(m, nn.Module)]
        if not roots:
            raise ValueError("repeatable: fn is no module: name the modules whose Dropout layers it calls")
        self.fn, self.start = fn, None
        self.layers = list({id(m): m for r in roots for m in r.modules() if isinstance(m, Dropout)}.values())

    def __call__(self, *args, **kw):
        again = _in_backward()
        if self.start is None:
            if again and not all(m._repeats for m in self.layers):
                raise RuntimeError("repeatable: first called in a backward pass: the region around it has to be "
                                   "repeatable too")
            self.start = [m.counter.clone() for m in self.layers]
            return self.fn(*args, **kw)
        if not again:
            raise RuntimeError("repeatable: each checkpointed call takes a wrapper of its own")
        now = [m.counter.clone() for m in self.layers]
        for m, start in zip(self.layers, self.start):
            m.counter.copy_(start)
            m._repeats += 1
        try:
            return self.fn(*args, **kw)
        finally:
            for m, c in zip(self.layers, now):
                m.counter.copy_(c)
                m._repeats -= 1


# ------------------------------------------------------------------------------------------ gated scan
def _held(v):
    """A sigmoid, a little more than zero also where the type has none for it: for a finite gate it is not zero, and zero
    times an infinite state or input would be NaN."""
    return v.clamp(min=torch.finfo(v.dtype).smallest_normal * torch.finfo(v.dtype).eps)


class _Gate(torch.autograd.Function):
    """z = sigmoid(g) and the state's factor 1 - z with their relative precision on both sides, in the gradient too (that of
    torch.sigmoid takes 1 - z by a subtraction, which has none left near z = 1)."""

    @staticmethod
    def forward(ctx, g):
        z, a = torch.sigmoid(g), torch.sigmoid(-g)
        ctx.save_for_backward(z, a)
        return z, _held(a)

    @staticmethod
    @once_differentiable
    def backward(ctx, dz, da):
        z, a = ctx.saved_tensors
        return (dz - da) * z * a


def _scan_cpu(x, gate, h0, resets, lengths):
    B, L, D = x.shape
    ct = torch.promote_types(x.dtype, torch.float32)
    st = torch.promote_types(ct, h0.dtype)
    x, gate, h, zero = x.to(ct), gate.to(ct), h0.to(st), torch.zeros((), dtype=ct)
    live = None
    if lengths is not None:
        live = (torch.arange(L) < lengths.unsqueeze(1)).unsqueeze(-1)
        x, gate = torch.where(live, x, zero), torch.where(live, gate, zero)
    z, a = _Gate.apply(gate)
    u = torch.where(z != 0, z * x, (_held(z) * x).detach())
    ys = []
    for t in range(L):
        prev = h if resets is None else torch.where((resets != 0)[:, t, None], torch.zeros((), dtype=st), h)
        new = a[:, t] * prev + u[:, t]
        h = new if live is None else torch.where(live[:, t], new, h)
        ys.append(new if live is None else torch.where(live[:, t], new, torch.zeros((), dtype=new.dtype)))
    return (torch.stack(ys, dim=1), h) if L else (u.to(st), h + u.sum(dim=1))


def _scan_parts(who, x, gate):
    """Checks x and gate; the channel count."""
    if x.dim() != (3 if who == "gated_scan" else 2):
        raise ValueError(f"{who}: x must be {'[B, L, D]' if who == 'gated_scan' else '[B, D]'}, not {tuple(x.shape)}")
    if not x.dtype.is_floating_point:
        raise ValueError(f"{who}: a floating-point tensor, not {x.dtype}")
    if gate is None:
        if x.shape[-1] % 2:
            raise ValueError(f"{who}: without a gate, x holds the inputs and the gates in halves of one size; "
                             f"{x.shape[-1]} channels")
        return x.shape[-1] // 2
    if gate.shape != x.shape or gate.dtype != x.dtype:
        raise ValueError(f"{who}: gate must match x: {tuple(gate.shape)} {gate.dtype} against {tuple(x.shape)} {x.dtype}")
    return x.shape[-1]


def gated_scan(x: torch.Tensor, gate: Optional[torch.Tensor] = None, h0: Optional[torch.Tensor] = None,
               resets: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None
               ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Gated linear recurrence over [B, L, D]: ``h_t = (1 - z_t) h_{t-1} + z_t x_t`` with ``z = sigmoid(gate)``.

    Returns (y, h_last): y [B, L, D] the states in x's type, h_last [B, D] the fp32 state behind the last step.
    Differentiable in x, gate and h0.

    x, gate: same shape and type; any strides with consecutive channels are read in place. Without ``gate``, x is
    [B, L, 2D], inputs and gates in its halves as one projection gives them, and so is its gradient.
    h0: [B, D] state before the first step (zeros by default). resets: [B, L], non-zero where the state is dropped
    before the step (an episode or document begins), whatever it held. Without one, an infinite state stays infinite under
    any gate (an infinite gate counts as a very large one).
    lengths: [B] integers, steps of each sequence (clamped to [0, L]): later places take no part whatever they hold, their
    y and gradients are 0."""
    D = _scan_parts("gated_scan", x, gate)
    B, L = x.shape[:2]
    _same_device("gated_scan", x, gate=gate, h0=h0, resets=resets, lengths=lengths)
    if h0 is not None and tuple(h0.shape) != (B, D):
        raise ValueError(f"gated_scan: h0 must be {(B, D)}, not {tuple(h0.shape)}")
    if lengths is not None and (tuple(lengths.shape) != (B,) or lengths.dtype.is_floating_point
                                or lengths.dtype.is_complex or lengths.dtype == torch.bool):
        raise ValueError(f"gated_scan: lengths must be {B} integers, not {tuple(lengths.shape)} {lengths.dtype}")
    if resets is not None and tuple(resets.shape) != (B, L):
        raise ValueError(f"gated_scan: resets must be {(B, L)}, not {tuple(resets.shape)}")
    if not x.is_cuda:
        if gate is None:
            x, gate = x[..., :D], x[..., D:]
        h0 = x.new_zeros((B, D), dtype=torch.promote_types(x.dtype, torch.float32)) if h0 is None else h0
        y, h = _scan_cpu(x, gate, h0, resets, lengths)
        return y.to(x.dtype), h.to(torch.promote_types(x.dtype, torch.float32))
    _code("gated_scan", x.dtype)
    return require_seq().gated_scan(x, gate, h0, resets, lengths)


def gated_scan_step(x: torch.Tensor, gate: Optional[torch.Tensor], state: torch.Tensor,
                    resets: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None
                    ) -> Tuple[torch.Tensor, torch.Tensor]:
    """One step of :func:`gated_scan` for B running sequences: returns (y [B, D] in x's type, new state [B, D] fp32).

    x, gate: [B, D] (or x [B, 2D] and gate None). state: [B, D] fp32, consecutive. resets: [B]. out: where the new state
    goes; ``out=state`` updates it in place. Not differentiable: with gradients, call :func:`gated_scan` with L = 1."""
    D = _scan_parts("gated_scan_step", x, gate)
    B = x.shape[0]
    _same_device("gated_scan_step", x, gate=gate, state=state, resets=resets, out=out)
    for name, t in (("state", state), ("out", out)):
        if t is not None and (tuple(t.shape) != (B, D) or t.dtype != torch.float32 or not t.is_contiguous()):
            raise ValueError(f"gated_scan_step: {name} must be {(B, D)}, fp32 and contiguous")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, gate, state, out)):
        raise ValueError("gated_scan_step is not differentiable: call gated_scan with L = 1, or under torch.no_grad()")
    if out is not None:
        delta = abs(out.data_ptr() - state.data_ptr())
        if 0 < delta < state.numel() * 4:
            raise ValueError("gated_scan_step: out overlaps state without being it")
    if resets is not None and tuple(resets.shape) != (B,):
        raise ValueError(f"gated_scan_step: resets must be {(B,)}, not {tuple(resets.shape)}")
    if not x.is_cuda:
        if gate is None:
            x, gate = x[..., :D], x[..., D:]
        prev = state if resets is None else torch.where((resets != 0).unsqueeze(-1), torch.zeros(()), state)
        h = _held(torch.sigmoid(-gate.float())) * prev + _held(torch.sigmoid(gate.float())) * x.float()
        out = h if out is None else out.copy_(h)
        return out.to(x.dtype, copy=True), out
    _code("gated_scan_step", x.dtype)
    return require_seq().gated_scan_step(x, gate, state, resets, out)
