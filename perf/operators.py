"""Timed cases of the sequence operators: embedding, counter-based dropout and the gated scan.

Each case is one call as a training step or a serving loop makes it. ``own`` chooses between the
framework's kernels (``ray_memory_management_amd.ops``) and the same formulas in elementary torch
operations; ``exact`` gives the formulas' values in 64 bits.

  embedding   out[i] = scale * W[id_i]; ids outside [0, V) give a row of zeros. The gradient is
              dW[v] = scale * sum of dy[i] over the i with id_i = v, zero for the padding row.
  dropout     out = residual + (u >= t ? x * 65536 / (65536 - t) : 0) with t = round(65536 p) and u the
              element's 16 random bits: Philox4x32-10 (Salmon et al. 2011) keyed by the seed, counter =
              (element index / 8, offset), 8 elements to a counter, low half of each word first.
  gated scan  h_t = (1 - z_t) h_{t-1} + z_t x_t with z = sigmoid(gate), h_{t-1} taken as 0 where a reset
              is set; steps behind a sequence's length leave the state and give y = 0.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_M32 = 0xFFFFFFFF


def listed():
    return [
        # ---- embedding
        # an offline sequence policy's timestep table: 128 segments of 5 steps, embedding width 128
        dict(name="embed train segments", op="embed", n=640, v=501, d=128, w="f32", out="f32", scale=1.0, pad=False,
             train=True),
        # next-token lookup of a decode batch
        dict(name="embed decode", op="embed", n=64, v=100003, d=4096, w="bf16", out="bf16", scale=1.0, pad=False,
             train=False),
        # a training batch of 8 sequences of 1024 tokens, padded at the end, scaled by sqrt(width)
        dict(name="embed train batch", op="embed", n=8192, v=32768, d=1024, w="bf16", out="bf16", scale=32.0, pad=True,
             train=True),
        # a long-context step with fp32 weights under bf16 activations; an odd token count
        dict(name="embed train long", op="embed", n=131071, v=100003, d=1536, w="f32", out="bf16", scale=1.0, pad=False,
             train=True),
        # ---- dropout
        # the same policy's token block [128, 15, 128]
        dict(name="dropout train segments", op="dropout", shape="128,15,128", t="f32", p=0.1, residual=False, train=True),
        # a residual branch of a training batch
        dict(name="dropout train residual", op="dropout", shape="8192,1024", t="bf16", p=0.1, residual=True, train=True),
        # a wide hidden layer, rows of odd width
        dict(name="dropout train wide", op="dropout", shape="32768,4097", t="f16", p=0.5, residual=False, train=True),
        # ---- gated scan
        # one token for each of 64 running sequences
        dict(name="scan step", op="scan", b=64, l=1, d=1024, t="bf16", train=False, resets=False, ragged=False,
             packed=True, step=True),
        # a recurrent policy's minibatch: 256 sequences of 20 steps with episode ends inside
        dict(name="scan train sequences", op="scan", b=256, l=20, d=256, t="f32", train=True, resets=True, ragged=False,
             packed=True, step=False),
        # an ordinary training batch of packed documents
        dict(name="scan train batch", op="scan", b=8, l=2048, d=1024, t="bf16", train=True, resets=True, ragged=False,
             packed=True, step=False),
        # prefill of prompts of different lengths, separate projections
        dict(name="scan prefill ragged", op="scan", b=16, l=3001, d=2048, t="bf16", train=False, resets=False,
             ragged=True, packed=False, step=False),
        # one very long sequence, trained with its carried state
        dict(name="scan train long", op="scan", b=1, l=65537, d=1024, t="bf16", train=True, resets=False, ragged=False,
             packed=False, step=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embed", "dropout", "scan"])
    if op == "embed":
        train = rng.random() < 0.75
        n = _log_int(rng, 1, 131072)
        v = _log_int(rng, 2, 131072)
        most = min(4096, (1 << 27) // max(n, v))  # rows and table within the largest listed case
        d = _log_int(rng, 16, max(most, 17))
        w, out = rng.choice([("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16")])
        return dict(op="embed", n=n, v=v, d=d, w=w, out=out, scale=rng.choice([1.0, math.sqrt(d), 0.125]),
                    pad=rng.random() < 0.4, train=train)
    if op == "dropout":
        total = _log_int(rng, 64, 1 << 26)
        cols = _log_int(rng, 1, 8192)
        return dict(op="dropout", shape="%d,%d" % (max(1, total // cols), cols), t=rng.choice(["f32", "bf16", "f16"]),
                    p=rng.choice([0.1, 0.5, round(rng.uniform(0.01, 0.99), 3)]), residual=rng.random() < 0.5,
                    train=rng.random() < 0.75)
    t = rng.choice(["f32", "bf16", "f16"])
    if rng.random() < 0.2:
        return dict(op="scan", b=_log_int(rng, 1, 512), l=1, d=_log_int(rng, 32, 8192), t=t, train=False,
                    resets=rng.random() < 0.5, ragged=False, packed=rng.random() < 0.5, step=True)
    l = _log_int(rng, 1, 65536)
    d = _log_int(rng, 16, 4096)
    b = _log_int(rng, 1, max(2, min(512, (1 << 25) // (l * d))))
    while b * l * d > 1 << 25 and l > 1:
        l = l // 2 + 1 if l > 2 else 1
    return dict(op="scan", b=b, l=l, d=d, t=t, train=rng.random() < 0.6, resets=rng.random() < 0.5,
                ragged=rng.random() < 0.4, packed=rng.random() < 0.5, step=False)


# ------------------------------------------------------------------------------------------ inputs
def _randn(shape, g, t, scale=1.0, shift=0.0):
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    return x.mul_(scale).add_(shift).to(t)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    s = {"case": case}
    if case["op"] == "embed":
        n, v, d = case["n"], case["v"], case["d"]
        u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
        s["ids"] = (torch.pow(float(v), u).long() - 1).clamp_(0, v - 1)  # log-uniform: frequent tokens first
        if case["pad"]:
            tail = torch.rand(n, generator=g, device="cuda") < 0.1
            s["ids"][tail] = 0
        s["w"] = _randn((v, d), g, _TYPES[case["w"]], 0.02).requires_grad_(case["train"])
        if case["train"]:
            s["dy"] = _randn((n, d), g, _TYPES[case["out"]])
    elif case["op"] == "dropout":
        shape, t = [int(k) for k in case["shape"].split(",")], _TYPES[case["t"]]
        s["x"] = _randn(shape, g, t).requires_grad_(case["train"])
        s["res"] = _randn(shape, g, t).requires_grad_(case["train"]) if case["residual"] else None
        s["seed"], s["offset"] = 1234567 + 31 * int(seed), 5 + int(seed)
        if case["train"]:
            s["dy"] = _randn(shape, g, t)
    else:
        b, l, d, t = case["b"], case["l"], case["d"], _TYPES[case["t"]]
        if case["packed"]:
            xg = _randn((b, l, 2 * d), g, torch.float32)
            xg[..., d:].mul_(1.5).sub_(2.0)
            s["x"], s["gate"] = xg.to(t).requires_grad_(case["train"]), None
        else:
            s["x"] = _randn((b, l, d), g, t).requires_grad_(case["train"])
            s["gate"] = _randn((b, l, d), g, t, 1.5, -2.0).requires_grad_(case["train"])  # slow forgetting
        s["h0"] = _randn((b, d), g, torch.float32).requires_grad_(case["train"])
        s["resets"] = s["lengths"] = None
        if case["resets"]:
            s["resets"] = torch.rand((b, l), generator=g, device="cuda") < (0.02 if not case["step"] else 0.1)
        if case["ragged"]:
            s["lengths"] = torch.randint(0 if b > 1 else 1, l + 1, (b,), generator=g, device="cuda")
            s["lengths"][0] = l
        if case["train"]:
            s["dy"] = _randn((b, l, d), g, t)
            s["dh"] = _randn((b, d), g, torch.float32)
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(state):
    c = state["case"]
    if own:
        return {"embed": _own_embed, "dropout": _own_dropout, "scan": _own_scan}[c["op"]](state, c)
    with torch.no_grad():
        return {"embed": _embed, "dropout": _dropout, "scan": _scan}[c["op"]](state, c)


def _own_embed(s, c):
    from ray_memory_management_amd import ops

    out = ops.embedding(s["ids"], s["w"], scale=c["scale"], padding_idx=0 if c["pad"] else None, dtype=_TYPES[c["out"]])
    if not c["train"]:
        return out
    return out, torch.autograd.grad(out, s["w"], s["dy"])[0]


def _own_dropout(s, c):
    from ray_memory_management_amd import ops

    y = ops.dropout(s["x"], c["p"], s["seed"], offset=s["offset"], residual=s["res"])
    if not c["train"]:
        return y
    leaves = (s["x"], s["res"]) if c["residual"] else (s["x"],)
    return (y,) + torch.autograd.grad(y, leaves, s["dy"])


def _own_scan(s, c):
    from ray_memory_management_amd import ops

    if c["step"]:
        gate = None if c["packed"] else s["gate"][:, 0]
        return ops.gated_scan_step(s["x"][:, 0], gate, s["h0"],
                                   resets=None if s["resets"] is None else s["resets"][:, 0])
    y, h = ops.gated_scan(s["x"], s["gate"], h0=s["h0"], resets=s["resets"], lengths=s["lengths"])
    if not c["train"]:
        return y, h
    leaves = (s["x"], s["h0"]) if c["packed"] else (s["x"], s["gate"], s["h0"])
    return (y, h) + torch.autograd.grad((y, h), leaves, (s["dy"], s["dh"]))


# ------------------------------------------------------------------------------------------ plain forms
def _embed(s, c):
    ids, w = s["ids"], s["w"]
    ok = (ids >= 0) & (ids < c["v"])
    rows = w[ids.clamp(0, c["v"] - 1)].float() * c["scale"]
    out = torch.where(ok[:, None], rows, torch.zeros_like(rows)).to(_TYPES[c["out"]])
    if not c["train"]:
        return out
    if c["pad"]:
        ok = ok & (ids != 0)
    dy = torch.where(ok[:, None], s["dy"].float(), torch.zeros((), device=ids.device))
    dw = torch.zeros((c["v"], c["d"]), dtype=torch.float32, device=ids.device)
    dw.index_add_(0, ids.clamp(0, c["v"] - 1), dy)
    return out, (dw * c["scale"]).to(w.dtype)


def _mulhilo(m, x):
    """Halves of the 64-bit product of a 32-bit constant and 32-bit words held in int64."""
    low = (m & 0xFFFF) * x
    high = (m >> 16) * x
    mid = (low >> 16) + high
    return mid >> 16, ((mid & 0xFFFF) << 16) | (low & 0xFFFF)


def _bits16(n, seed, offset, device):
    q = torch.arange((n + 7) // 8, dtype=torch.int64, device=device)
    a, b = q & _M32, q >> 32
    c, d = torch.full_like(q, offset & _M32), torch.full_like(q, (offset >> 32) & _M32)
    k0, k1 = seed & _M32, (seed >> 32) & _M32
    for _ in range(10):
        h0, l0 = _mulhilo(0xD2511F53, a)
        h1, l1 = _mulhilo(0xCD9E8D57, c)
        a, b, c, d = h1 ^ b ^ k0, l1, h0 ^ d ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    w = torch.stack([a, b, c, d], dim=1)
    return torch.stack([w & 0xFFFF, w >> 16], dim=2).reshape(-1)[:n]


def _dropout(s, c):
    x, t = s["x"], int(round(c["p"] * 65536))
    keep = (_bits16(x.numel(), s["seed"], s["offset"], x.device) >= t).view(x.shape)
    k, zero = 65536.0 / (65536 - t), torch.zeros((), device=x.device)
    y = torch.where(keep, x.float() * k, zero)
    if c["residual"]:
        y = y + s["res"].float()
    y = y.to(x.dtype)
    if not c["train"]:
        return y
    dx = torch.where(keep, s["dy"].float() * k, zero).to(x.dtype)
    return (y, dx, s["dy"].clone()) if c["residual"] else (y, dx)


def _doubling(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1 from h = 0, by combining spans of doubling length."""
    k = 1
    while k < a.shape[1]:
        b = torch.cat([b[:, :k], b[:, k:] + a[:, k:] * b[:, :-k]], dim=1)
        a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], dim=1)
        k *= 2
    return b


def _halves(s, c):
    return s["x"].chunk(2, dim=-1) if c["packed"] else (s["x"], s["gate"])


def _scan(s, c):
    x, gate = _halves(s, c)
    b, l, d, t = c["b"], c["l"], c["d"], _TYPES[c["t"]]
    x, z, a = x.float(), torch.sigmoid(gate.float()), torch.sigmoid(-gate.float())
    carry = torch.ones((b, l, 1), dtype=torch.bool, device=x.device)  # the state before step t reaches it
    live = torch.ones_like(carry)
    if s["resets"] is not None:
        carry = ~s["resets"][:, :, None]
    if s["lengths"] is not None:
        live = (torch.arange(l, device=x.device)[None] < s["lengths"][:, None])[:, :, None]
    keep = torch.where(live, a * carry, torch.ones_like(a))
    u = torch.where(live, z * x, torch.zeros_like(x))
    u[:, 0] += keep[:, 0] * s["h0"]
    h = _doubling(keep, u)
    y = torch.where(live, h, torch.zeros_like(h)).to(t)
    last = h[:, -1].clone()
    if c["step"]:
        return y[:, 0], last
    if not c["train"]:
        return y, last
    dy = torch.where(live, s["dy"].float(), torch.zeros_like(h))
    dy[:, -1] += s["dh"]
    nxt = torch.cat([keep[:, 1:], torch.zeros_like(keep[:, :1])], dim=1)
    dh = _doubling(nxt.flip(1), dy.flip(1)).flip(1)
    prev = torch.cat([s["h0"][:, None], h[:, :-1]], dim=1) * carry
    dx = torch.where(live, dh * z, torch.zeros_like(h)).to(t)
    dg = torch.where(live, dh * (x - prev) * z * a, torch.zeros_like(h)).to(t)
    dh0 = keep[:, 0] * dh[:, 0]
    if c["packed"]:
        return y, last, torch.cat([dx, dg], dim=-1), dh0
    return y, last, dx, dg, dh0


# ------------------------------------------------------------------------------------------ exact values
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"embed": _exact_embed, "dropout": _exact_dropout, "scan": _exact_scan}[case["op"]](s, case)


def _exact_embed(s, c):
    w = s["w"].double() * c["scale"]
    out = torch.index_select(torch.cat([w, w.new_zeros(1, c["d"])]), 0,
                             torch.where((s["ids"] < 0) | (s["ids"] >= c["v"]), c["v"], s["ids"]))
    if not c["train"]:
        return out
    order = torch.argsort(s["ids"], stable=True)
    ids, rows = s["ids"][order], order
    dw = torch.zeros((c["v"], c["d"]), dtype=torch.float64, device=w.device)
    for at in range(0, c["n"], 16384):  # sums of whole blocks: 64-bit rows of the full batch are large
        dw.index_add_(0, ids[at:at + 16384], s["dy"][rows[at:at + 16384]].double())
    if c["pad"]:
        dw[0] = 0
    return out, dw * c["scale"]


def _exact_dropout(s, c):
    # the generator with numpy's unsigned 64-bit products, on the host
    import numpy as np

    n, t = s["x"].numel(), int(round(c["p"] * 65536))
    q = np.arange((n + 7) // 8, dtype=np.uint64)
    m = np.uint64(_M32)
    w = [q & m, q >> np.uint64(32), np.full_like(q, s["offset"] & _M32), np.full_like(q, s["offset"] >> 32)]
    key = [s["seed"] & _M32, s["seed"] >> 32]
    for _ in range(10):
        p0, p1 = w[0] * np.uint64(0xD2511F53), w[2] * np.uint64(0xCD9E8D57)
        w = [(p1 >> np.uint64(32)) ^ w[1] ^ np.uint64(key[0]), p1 & m,
             (p0 >> np.uint64(32)) ^ w[3] ^ np.uint64(key[1]), p0 & m]
        key = [(key[0] + 0x9E3779B9) & _M32, (key[1] + 0xBB67AE85) & _M32]
    u = np.stack(w, axis=1).astype("<u4").view("<u2").reshape(-1)[:n]
    keep = torch.from_numpy((u >= t)).to(s["x"].device).view(s["x"].shape).double()
    y = s["x"].double() * keep * 65536.0 / (65536 - t)
    if c["residual"]:
        y += s["res"].double()
    if not c["train"]:
        return y
    dx = s["dy"].double() * keep * 65536.0 / (65536 - t)
    return (y, dx, s["dy"].double()) if c["residual"] else (y, dx)


def _exact_scan(s, c):
    x, gate = _halves(s, c)
    x, gate = x.double().transpose(0, 1).contiguous(), gate.double().transpose(0, 1).contiguous()
    l, b = c["l"], c["b"]
    end = s["lengths"] if s["lengths"] is not None else torch.full((b,), l, device=x.device)
    live = (torch.arange(l, device=x.device)[:, None] < end[None])[:, :, None]
    f = torch.sigmoid(-gate)  # the share of the old state that stays
    if s["resets"] is not None:
        f = f.masked_fill(s["resets"].t()[:, :, None], 0.0)
    f = torch.where(live, f, torch.ones_like(f))
    u = torch.where(live, torch.sigmoid(gate) * x, torch.zeros_like(x))
    h, cur = torch.empty_like(x), s["h0"].double()
    for t in range(l):
        cur = torch.addcmul(u[t], f[t], cur)
        h[t] = cur
    y = torch.where(live, h, torch.zeros_like(h)).transpose(0, 1)
    if c["step"]:
        return y[:, 0], cur
    if not c["train"]:
        return y, cur
    dy = torch.where(live, s["dy"].double().transpose(0, 1), torch.zeros_like(h))
    dh, back = torch.empty_like(x), s["dh"].double()
    for t in range(l - 1, -1, -1):
        back = dy[t] + back
        dh[t] = back
        back = back * f[t]
    prev = torch.cat([s["h0"].double()[None], h[:-1]])
    if s["resets"] is not None:
        prev = prev.masked_fill(s["resets"].t()[:, :, None], 0.0)
    z = torch.sigmoid(gate)
    dx = torch.where(live, dh * z, torch.zeros_like(h)).transpose(0, 1)
    dg = torch.where(live, dh * (x - prev) * z * torch.sigmoid(-gate), torch.zeros_like(h)).transpose(0, 1)
    return (y, cur, torch.cat([dx, dg], dim=-1), back) if c["packed"] else (y, cur, dx, dg, back)


# ------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    c = case
    if c["op"] == "embed":
        n, v, d, w, o = c["n"], c["v"], c["d"], size[c["w"]], size[c["out"]]
        rows = v * (1.0 - math.exp(-min(n, 4 * v) / (v * max(1.0, math.log(v) / 2))))  # distinct rows read, about
        total = 8 * n + min(n, rows) * d * w + n * d * o
        if c["train"]:
            total += 8 * n + n * d * o + v * d * w
        return {"bytes": int(total), "flops": n * d * (2 if c["train"] else 1)}
    if c["op"] == "dropout":
        n = 1
        for k in c["shape"].split(","):
            n *= int(k)
        e = size[c["t"]]
        units = 2 + (1 if c["residual"] else 0) + (2 if c["train"] else 0)
        return {"bytes": n * e * units, "flops": n * (2 + (1 if c["residual"] else 0) + (2 if c["train"] else 0))}
    n, e, bd = c["b"] * c["l"] * c["d"], size[c["t"]], c["b"] * c["d"]
    total = 3 * n * e + 8 * bd
    flops = 10 * n
    if c["train"]:
        total += 5 * n * e + 8 * bd  # x, gate and dy again, both gradients; the state's two
        flops += 20 * n
    if c["resets"]:
        total += c["b"] * c["l"] * (2 if c["train"] else 1)
    return {"bytes": int(total), "flops": flops}
