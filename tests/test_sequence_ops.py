"""ops.embedding / dropout / gated_scan against plain implementations in 64 bits.

Every tolerance is a bound computed beside the reference: u = 2^-24 for each fp32 rounding (counted per term), and
half a step of the output type for the one rounding at the end. The CPU runs the torch forms, the GPU the kernels."""
import math

import pytest
import torch

from ray_memory_management_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(params=DEVICES)
def dev(request):
    if request.param == "cuda":
        if not torch.cuda.is_available():
            pytest.skip("no GPU")
        from ray_memory_management_amd._native import require_hip

        require_hip()
    return torch.device(request.param)


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """Half the spacing of the subnormals: what a result near zero may be off by."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def check(got, want, bound, t):
    """|got - want| within the bound on the fp32 value before rounding plus the rounding to t."""
    assert got.dtype == t and got.shape == want.shape
    got = got.detach().cpu().double()
    tol = bound + (want.abs() + bound) * half_step(t) + tiny(t) + tiny(torch.float32)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / tol).max()):.3g} "
                           f"times the bound, first at {bad.nonzero()[0].tolist()}")


def rand(*shape, seed, t=torch.float32, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * scale + shift).to(t)


# ------------------------------------------------------------------------------------------ embedding
def embed_reference(ids, w, scale, pad, dy):
    V = w.shape[0]
    flat = ids.reshape(-1).long()
    ok = (flat >= 0) & (flat < V)
    w64, dy64 = w.double(), dy.double().reshape(flat.numel(), -1)
    out = torch.zeros(flat.numel(), w.shape[1], dtype=torch.float64)
    dw, mag, cnt = torch.zeros_like(w64), torch.zeros_like(w64), torch.zeros(V, 1, dtype=torch.float64)
    out[ok] = w64[flat[ok]] * scale
    use = ok if pad is None else ok & (flat != pad)
    dw.index_add_(0, flat[use], dy64[use])
    mag.index_add_(0, flat[use], dy64[use].abs())
    cnt.index_add_(0, flat[use], torch.ones(int(use.sum()), 1, dtype=torch.float64))
    # forward: the scale to fp32 and one product; gradient: cnt additions of the magnitudes, then the same two
    return (out.reshape(*ids.shape, -1), 2 * U * out.reshape(*ids.shape, -1).abs(), dw * scale,
            (cnt + 2) * U * mag * abs(scale))


def embed_case(dev, ids, V, D, wt, ot, scale=1.0, pad=None, seed=0, w=None):
    w = rand(V, D, seed=seed, t=wt) if w is None else w
    dy = rand(*ids.shape, D, seed=seed + 1, t=ot)
    out, ob, dw, db = embed_reference(ids, w, scale, pad, dy)
    wd = w.to(dev).requires_grad_()
    got = ops.embedding(ids.to(dev), wd, scale, pad, ot)
    check(got, out, ob, ot)
    got.backward(dy.to(dev))
    check(wd.grad, dw, db, wt)


def some_ids(n, V, seed, kind="log"):
    g = torch.Generator().manual_seed(seed)
    u = torch.rand(n, generator=g, dtype=torch.float64)
    if kind == "log":
        return (torch.pow(float(V), u).long() - 1).clamp_(0, V - 1)
    return (u * V).long().clamp_(0, V - 1)


@pytest.mark.parametrize("wt,ot", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (1, 5000, 8), (63, 7, 130), (640, 501, 128), (2049, 3, 33),
                                   (5000, 70001, 16), (4097, 300, 264)])
def test_embedding(dev, n, V, D, wt, ot):
    embed_case(dev, some_ids(n, V, n), V, D, TYPES[wt], TYPES[ot], scale=math.sqrt(D))


@pytest.mark.parametrize("kind", ["log", "uniform"])
@pytest.mark.parametrize("n,V", [(40000, 1000), (30011, 65536), (33000, 2), (20000, 511), (20000, 512)])
def test_embedding_many_tokens(dev, n, V, kind):
    embed_case(dev, some_ids(n, V, n, kind), V, 40, torch.float32, torch.bfloat16, scale=0.5)


@pytest.mark.parametrize("n", [1, 64, 257, 1025, 4096, 4097, 9000])
def test_embedding_one_token_everywhere(dev, n):
    embed_case(dev, torch.full((n,), 6), 9, 24, torch.float32, torch.float32)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_embedding_padding_and_ids_outside(dev, dtype):
    ids = some_ids(600, 50, 3).reshape(20, 30)
    ids[:, 25:] = 7
    ids[3] = -1
    ids[4, :5] = 50
    if dtype == torch.int64:
        ids[5, :5] = 1 << 40
        ids[6, :5] = -(1 << 40)
        ids[7, :2] = (1 << 32) + 3
    embed_case(dev, ids.to(dtype), 50, 24, torch.float32, torch.float32, scale=2.0, pad=7)
    w = rand(50, 24, seed=1).to(dev).requires_grad_()
    out = ops.embedding(ids.to(dtype).to(dev), w, padding_idx=-43)   # from the end: row 7
    assert (out[3] == 0).all() and torch.equal(out[0, 29], w[7])
    out.sum().backward()                                             # a broadcast gradient
    assert (w.grad[7] == 0).all() and float(w.grad.sum()) > 0


def test_embedding_rows_none_use_and_no_ids(dev):
    w = rand(300, 16, seed=0).to(dev).requires_grad_()
    ids = torch.empty(0, 4, dtype=torch.long, device=dev)
    out = ops.embedding(ids, w)
    assert out.shape == (0, 4, 16)
    out.sum().backward()
    assert (w.grad == 0).all()
    w.grad = None
    ops.embedding(torch.full((5,), -1, device=dev), w).sum().backward()
    assert (w.grad == 0).all()


def test_embedding_weight_strides(dev):
    big = rand(40, 50, seed=4)
    ids = some_ids(100, 40, 0)
    for w in (big[:, 3:27], big[:, :24], big.t()[:24].t(), big[::2][:, :24], big[:1, :24].expand(40, 24)):
        out, ob, _, _ = embed_reference(ids.clamp_max(len(w) - 1), w, 1.0, None, torch.zeros(100, 24))
        wd = torch.empty_strided(big.size(), big.stride()).copy_(big).to(dev)
        wd = wd.as_strided(w.size(), w.stride(), w.storage_offset())
        check(ops.embedding(ids.clamp_max(len(w) - 1).to(dev), wd), out, ob, torch.float32)


def test_embedding_gradient_strides(dev):
    """dy rows apart from each other, and dy whose channels are not consecutive."""
    ids = some_ids(50, 30, 0)
    for cut in (lambda b: b[:, 8:24], lambda b: b[:, 1:17], lambda b: b[:, ::2][:, :16]):
        dy = cut(rand(50, 40, seed=9))
        _, _, dw, db = embed_reference(ids, torch.zeros(30, 16), 1.0, None, dy)
        w = torch.zeros(30, 16, device=dev, requires_grad=True)
        ops.embedding(ids.to(dev), w).backward(cut(rand(50, 40, seed=9).to(dev)))
        check(w.grad, dw, db, torch.float32)


def test_embedding_gradient_is_the_difference_quotient(dev):
    """The loss is linear in the weight, so a difference of any size gives the gradient: (f(W + e) - f(W - e)) / 2."""
    ids, v = some_ids(200, 17, 0), rand(200, 8, seed=5, t=torch.float32)
    w, e = rand(17, 8, seed=6), rand(17, 8, seed=7)
    f = lambda wt: (ops.embedding(ids.to(dev), wt.to(dev), 3.0).cpu().double() * v.double()).sum()  # noqa: E731
    wd = w.to(dev).requires_grad_()
    (g,) = torch.autograd.grad(ops.embedding(ids.to(dev), wd, 3.0), wd, v.to(dev))
    quotient = (f(w + e) - f(w - e)) / 2
    mag = float((v.abs().double().sum() * 3 * (w.abs() + e.abs()).max()).detach())
    assert abs(float((g.cpu().double() * e.double()).sum()) - float(quotient)) <= 220 * U * mag


def test_embedding_same_bits_every_time(dev):
    ids, w = some_ids(20000, 90, 1).to(dev), rand(90, 64, seed=0).to(dev).requires_grad_()
    dy = rand(20000, 64, seed=1, t=torch.float32).to(dev)
    a, b = (torch.autograd.grad(ops.embedding(ids, w), w, dy)[0] for _ in range(2))
    assert torch.equal(a, b)


def test_embedding_module_matches_torch(dev):
    m = ops.Embedding(30, 12, padding_idx=2).to(dev)
    r = torch.nn.Embedding(30, 12, padding_idx=2).to(dev)
    r.load_state_dict(m.state_dict())
    ids = some_ids(50, 30, 0).to(dev)
    assert torch.equal(m(ids), r(ids))
    m(ids).sum().backward()
    r(ids).sum().backward()
    assert torch.equal(m.weight.grad, r.weight.grad)  # sums of ones: exact in any order
    assert torch.equal(ops.Embedding.from_pretrained(r.weight.detach()).to(dev)(ids), r(ids))
    for bad in ({"sparse": True}, {"max_norm": 1.0}, {"scale_grad_by_freq": True}):
        with pytest.raises(ValueError, match="not supported"):
            ops.Embedding(3, 4, **bad)


def test_embedding_refusals(dev):
    w, ids = torch.zeros(4, 3, device=dev), torch.zeros(2, dtype=torch.long, device=dev)
    for a, kw in (((ids.float(), w), {}), ((ids, w[0]), {}), ((ids, w), {"padding_idx": 4}),
                  ((ids, w), {"padding_idx": -5}), ((ids, w.long()), {}), ((ids, w), {"dtype": torch.int32}),
                  ((ids.bool(), w), {})):
        with pytest.raises(ValueError, match="embedding"):
            ops.embedding(*a, **kw)


# ------------------------------------------------------------------------------------------ dropout
def philox_reference(n, seed, offset):
    """16 bits an element, with Python's integers."""
    bits = []
    for q in range((n + 7) // 8):
        c = [q & 0xFFFFFFFF, q >> 32, offset & 0xFFFFFFFF, offset >> 32]
        k = [seed & 0xFFFFFFFF, seed >> 32]
        for _ in range(10):
            p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & 0xFFFFFFFF, (p0 >> 32) ^ c[3] ^ k[1], p0 & 0xFFFFFFFF]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        for w in c:
            bits += [w & 0xFFFF, w >> 16]
    return torch.tensor(bits[:n])


def test_generator_known_answers():
    """The published test vectors of Philox4x32-10."""
    from ray_memory_management_amd.ops.sequence import _philox_words

    for index, offset, seed, want in (
            (0, 0, 0, [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]),
            (-1, 2 ** 64 - 1, 2 ** 64 - 1, [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]),
            (0x85a308d3243f6a88 - 2 ** 64, 0x0370734413198a2e, 0x299f31d0a4093822,
             [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1])):
        assert _philox_words(torch.tensor([index]), offset, seed)[0].tolist() == want


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("shape,p", [((1,), 0.5), ((7,), 0.1), ((8,), 0.9), ((2, 0, 3), 0.5), ((33, 65), 0.25),
                                     ((5, 2051), 0.999), ((64, 64), 0.0), ((100,), 1.0), ((40, 50), 1e-6)])
def test_dropout(dev, shape, p, residual, t):
    T, seed, offset = TYPES[t], (77 << 33) + 5, (3 << 32) + 9
    n = math.prod(shape)
    x, r, dy = (rand(*shape, seed=s, t=T) for s in (1, 2, 3))
    thr = round(p * 65536)
    keep = (philox_reference(n, seed, offset) >= thr).reshape(shape) if n else torch.zeros(shape, dtype=torch.bool)
    k = 65536 / (65536 - thr) if thr < 65536 else 0.0
    want = torch.where(keep, x.double() * k, 0.0)
    full = want + r.double() if residual else want
    xd, rd = x.to(dev).requires_grad_(), r.to(dev).requires_grad_()
    y = ops.dropout(xd, p, seed, offset, rd if residual else None)
    # the scale to fp32, the product, and with a residual the sum
    check(y, full, 2 * U * want.abs() + (U * full.abs() * (1 + 3 * U) + 3 * U * U if residual else 0), T)
    y.backward(dy.to(dev))
    dwant = torch.where(keep, dy.double() * k, 0.0)
    check(xd.grad, dwant, 2 * U * dwant.abs(), T)
    if residual:
        assert torch.equal(rd.grad.cpu(), dy)
    assert ((y.detach().cpu() == 0) | keep).all() or residual


def test_dropout_rate_and_expectation(dev):
    """2^18 elements: the count of dropped ones within 6 standard deviations of p n."""
    n, p = 1 << 18, 0.3
    y = ops.dropout(torch.ones(n, device=dev), p, 11, 4)
    assert abs(int((y == 0).sum()) - p * n) < 6 * math.sqrt(n * p * (1 - p))
    a, b, c = (ops.dropout(torch.ones(n, device=dev), p, s, o) for s, o in ((11, 5), (12, 4), (11, 4)))
    assert not torch.equal(a, y) and not torch.equal(b, y) and torch.equal(c, y)


def test_dropout_ignores_what_it_drops(dev):
    x = torch.full((4096,), float("nan"), device=dev)
    x[::2] = float("inf")
    y = ops.dropout(x.requires_grad_(), 1.0, 1)
    assert (y == 0).all()
    y.sum().backward()
    assert (x.grad == 0).all()
    dy = torch.full((4096,), float("inf"), device=dev)
    x = torch.ones(4096, device=dev, requires_grad=True)
    y = ops.dropout(x, 0.5, 3)
    y.backward(dy)
    assert torch.equal(torch.isinf(x.grad), y.detach() != 0) and not torch.isnan(x.grad).any()


def test_dropout_strides_and_alignment(dev):
    base = rand(40, 70, seed=0, t=torch.bfloat16).to(dev)
    flat = base.reshape(-1)
    for x in (base.t(), base[:, 3:61], base[::2], flat[1:1000], flat[3:3 + 2048], base[:1].expand(9, 70)):
        want = ops.dropout(x.contiguous().clone(), 0.4, 5, 6, residual=torch.ones_like(x.contiguous()))
        assert torch.equal(ops.dropout(x, 0.4, 5, 6, residual=torch.ones(x.shape, dtype=x.dtype, device=dev)), want)
        leaf = x.detach().clone().requires_grad_()
        gy = x.detach().clone()
        g = torch.autograd.grad(ops.dropout(leaf, 0.4, 5, 6), leaf, gy)[0]
        assert torch.equal(g, ops.dropout(gy.contiguous(), 0.4, 5, 6))


def test_dropout_offset_tensor_read_once(dev):
    """The backward pass uses the counter value its forward pass read, also after the counter went on."""
    x = rand(1000, seed=0).to(dev).requires_grad_()
    ctr = torch.tensor([41, 7], device=dev)
    y = ops.dropout(x, 0.5, 9, ctr)
    ctr.add_(100)
    assert torch.equal(y, ops.dropout(x, 0.5, 9, 41))
    y.sum().backward()
    assert torch.equal(x.grad, ops.dropout(torch.ones(1000, device=dev), 0.5, 9, 41))


def test_dropout_module(dev):
    m = ops.Dropout(0.5, seed=3).to(dev)
    x = torch.ones(512, device=dev)
    a, b = m(x), m(x)
    assert not torch.equal(a, b) and torch.equal(a, ops.dropout(x, 0.5, 3, 0)) and int(m.counter) == 2
    r = ops.Dropout(0.5, seed=3).to(dev)
    r.load_state_dict(m.state_dict())
    assert torch.equal(r(x), ops.dropout(x, 0.5, 3, 2))
    m.eval()
    assert torch.equal(m(x), x) and torch.equal(m(x, residual=x), x + x) and int(m.counter) == 2


def test_dropout_refusals(dev):
    x = torch.ones(4, device=dev)
    for a, kw in (((x, -0.1, 0), {}), ((x, 1.5, 0), {}), ((x, float("nan"), 0), {}), ((x.long(), 0.5, 0), {}),
                  ((x, 0.5, 0), {"residual": torch.ones(5, device=dev)}),
                  ((x, 0.5, 0), {"residual": x.to(torch.bfloat16)}),
                  ((x, 0.5, 0, torch.zeros(1, device=dev)), {}),
                  ((x, 0.5, 0, torch.zeros(0, dtype=torch.long, device=dev)), {})):
        with pytest.raises(ValueError, match="dropout"):
            ops.dropout(*a, **kw)


# ------------------------------------------------------------------------------------------ gated scan
def scan_reference(x, g, h0, resets, lengths, dy, dh):
    """Values in 64 bits by the definition, and error bounds: E_t = a E_{t-1} + k u H_t, where H is the same recurrence
    over magnitudes (nothing cancels in it, so it also covers a sum taken in another order) and k counts the roundings
    of a step: an exponential and reciprocal good to (|g| + 8) u on each of two factors of a span, and the sums."""
    B, L, D = x.shape
    x, g, dy, dh = x.double(), g.double(), dy.double(), dh.double()
    h = torch.zeros(B, D, dtype=torch.float64) if h0 is None else h0.double()
    end = torch.full((B,), L) if lengths is None else lengths.clamp(0, L)
    z, a = torch.sigmoid(g), torch.sigmoid(-g)
    H, E = h.abs(), torch.zeros_like(h)
    k = 2 * (torch.nan_to_num(g).abs() + 8) + 4
    out = {n: torch.zeros(B, L, D, dtype=torch.float64) for n in ("y", "ey", "dx", "ex", "dg", "eg")}
    hp, Ep, Hp = (torch.zeros(B, L, D, dtype=torch.float64) for _ in range(3))
    for b in range(B):
        for t in range(int(end[b])):
            if resets is not None and bool(resets[b, t]):
                h[b], H[b], E[b] = 0, 0, 0
            hp[b, t], Ep[b, t], Hp[b, t] = h[b], E[b], H[b]
            h[b] = a[b, t] * h[b] + z[b, t] * x[b, t]
            H[b] = a[b, t] * H[b] + z[b, t] * x[b, t].abs()
            E[b] = a[b, t] * E[b] + k[b, t] * U * H[b]
            out["y"][b, t], out["ey"][b, t] = h[b], E[b]
    out["h"], out["eh"] = h.clone(), E.clone()
    back, Bm, Be = dh.clone(), dh.abs(), torch.zeros_like(dh)
    for b in range(B):
        for t in range(int(end[b]) - 1, -1, -1):
            zz, aa = z[b, t], a[b, t]
            back[b], Bm[b] = back[b] + dy[b, t], Bm[b] + dy[b, t].abs()
            Be[b] = Be[b] + k[b, t] * U * Bm[b]
            out["dx"][b, t], out["ex"][b, t] = back[b] * zz, zz * (Be[b] + k[b, t] * U * Bm[b])
            diff = (x[b, t].abs() + Hp[b, t])
            out["dg"][b, t] = back[b] * (x[b, t] - hp[b, t]) * zz * aa
            out["eg"][b, t] = zz * aa * (Be[b] * diff + Bm[b] * Ep[b, t] + 2 * k[b, t] * U * Bm[b] * diff)
            if resets is not None and bool(resets[b, t]):
                back[b], Bm[b], Be[b] = 0, 0, 0
            else:
                back[b], Bm[b], Be[b] = back[b] * aa, Bm[b] * aa, Be[b] * aa + k[b, t] * U * Bm[b] * aa
    out["dh0"], out["eh0"] = back, Be
    return out


def scan_case(dev, B, L, D, t, resets=None, lengths=None, h0=True, packed=False, seed=0, x=None, g=None, layout=None):
    T = TYPES[t]
    x = rand(B, L, D, seed=seed, t=T) if x is None else x
    g = rand(B, L, D, seed=seed + 1, t=T, scale=1.5, shift=-1.0) if g is None else g
    h0 = rand(B, D, seed=seed + 2) if h0 else None
    dy, dh = rand(B, L, D, seed=seed + 3, t=T), rand(B, D, seed=seed + 4)
    ref = scan_reference(x, g, h0, resets, lengths, dy, dh)
    mv = lambda v: None if v is None else v.to(dev)  # noqa: E731
    h0d = None if h0 is None else mv(h0).requires_grad_()
    if packed:
        xg = mv(torch.cat([x, g], dim=-1)).requires_grad_()
        y, h = ops.gated_scan(xg, h0=h0d, resets=mv(resets), lengths=mv(lengths))
        leaves = [xg]
    else:
        leaves = [mv(x).requires_grad_(), mv(g).requires_grad_()]
        xi, gi = leaves
        if layout == "time-major":
            xi, gi = (v.transpose(0, 1).contiguous().transpose(0, 1) for v in leaves)
        elif layout == "cut":  # rows of a wider projection, at an odd element
            xi, gi = (torch.nn.functional.pad(v, (3, 2))[..., 3:3 + D] for v in leaves)
        elif layout == "channels first":
            xi, gi = (v.transpose(1, 2).contiguous().transpose(1, 2) for v in leaves)
        y, h = ops.gated_scan(xi, gi, h0d, mv(resets), mv(lengths))
    check(y, ref["y"], ref["ey"], T)
    check(h, ref["h"], ref["eh"], torch.float32)
    ins = leaves + ([h0d] if h0 is not None else [])
    dyd = mv(dy) if layout != "channels first" else mv(dy).transpose(1, 2).contiguous().transpose(1, 2)
    gr = torch.autograd.grad((y, h), ins, (dyd, mv(dh)))
    dx, dg = (gr[0][..., :D], gr[0][..., D:]) if packed else gr[:2]
    check(dx, ref["dx"], ref["ex"], T)
    check(dg, ref["dg"], ref["eg"], T)
    if h0 is not None:
        check(gr[-1], ref["dh0"], ref["eh0"], torch.float32)


def some_resets(B, L, seed, rate=0.1):
    return torch.rand(B, L, generator=torch.Generator().manual_seed(seed)) < rate


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,L,D", [(1, 1, 1), (2, 3, 5), (3, 17, 64), (2, 33, 130), (1, 130, 72), (5, 20, 256)])
@pytest.mark.parametrize("packed", [False, True])
def test_gated_scan(dev, B, L, D, packed, t):
    scan_case(dev, B, L, D, t, packed=packed)


@pytest.mark.parametrize("B,L,D", [(2, 700, 8), (1, 1100, 64), (1, 2500, 4), (3, 257, 96)])
@pytest.mark.parametrize("packed", [False, True])
def test_gated_scan_long(dev, B, L, D, packed):
    scan_case(dev, B, L, D, "f32", resets=some_resets(B, L, L, 0.004), packed=packed)
    scan_case(dev, B, L, D, "bf16", h0=False, packed=packed)


@pytest.mark.parametrize("rate", [0.05, 0.6, 1.0])
def test_gated_scan_resets(dev, rate):
    for L in (1, 20, 150):
        scan_case(dev, 4, L, 40, "f32", resets=some_resets(4, L, L, rate), packed=L == 20)
        scan_case(dev, 4, L, 40, "bf16", resets=some_resets(4, L, L, rate).to(torch.float32), h0=False)


@pytest.mark.parametrize("L", [1, 16, 70, 300])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_gated_scan_lengths(dev, L, t):
    lengths = torch.tensor([L, 0, 1, max(L - 1, 0), L // 2, L + 9, -3])
    scan_case(dev, 7, L, 24, t, lengths=lengths, resets=some_resets(7, L, 1), packed=True)
    scan_case(dev, 7, L, 24, t, lengths=lengths.to(torch.int32))


@pytest.mark.parametrize("layout", ["time-major", "cut", "channels first"])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_gated_scan_strides(dev, layout, t):
    scan_case(dev, 3, 50, 48, t, layout=layout, resets=some_resets(3, 50, 2))
    scan_case(dev, 3, 50, 37, t, layout=layout)


def test_gated_scan_gates_at_the_ends(dev):
    """Gates that let all or nothing through: z and 1 - z keep their relative precision on both sides."""
    g = torch.tensor([-200.0, -87.0, -30.0, -8.0, 0.0, 8.0, 30.0, 87.0, 200.0]).repeat(20)
    g = g[torch.randperm(180, generator=torch.Generator().manual_seed(1))].reshape(1, 180, 1).repeat(1, 1, 3)
    scan_case(dev, 1, 180, 3, "f32", g=g)
    scan_case(dev, 1, 180, 3, "bf16", g=g.to(torch.bfloat16))
    inf = torch.full((1, 40, 2), float("inf"))
    x = rand(1, 40, 2, seed=0)
    y, h = ops.gated_scan(x.to(dev), inf.to(dev))
    assert torch.equal(y.cpu(), x)
    y, h = ops.gated_scan(x.to(dev), -inf.to(dev), h0=torch.ones(1, 2, device=dev))
    assert (y == 1).all() and (h == 1).all()


@pytest.mark.parametrize("junk", [float("nan"), float("inf")])
def test_gated_scan_masked_places_take_no_part(dev, junk):
    """Whatever stands behind a sequence's end, in its dy too, and before a reset, reaches nothing else."""
    B, L, D = 3, 150, 16
    lengths = torch.tensor([100, 150, 0])
    x, g, dy = (rand(B, L, D, seed=s) for s in (1, 2, 3))
    clean = [v.clone() for v in (x, g, dy)]
    pad = torch.arange(L)[None, :, None] >= lengths[:, None, None]
    for v in (x, g, dy):
        v.masked_fill_(pad, junk)
    res = []
    for vs in (clean, (x, g, dy)):
        xi, gi = (v.to(dev).requires_grad_() for v in vs[:2])
        h0 = torch.ones(B, D, device=dev, requires_grad=True)
        y, h = ops.gated_scan(xi, gi, h0, lengths=lengths.to(dev))
        res.append([y, h, *torch.autograd.grad((y, h), (xi, gi, h0), (vs[2].to(dev), torch.ones_like(h)))])
    for a, b in zip(*res):
        assert torch.equal(a, b)
    assert (res[1][0].cpu()[pad.expand(B, L, D)] == 0).all() and (res[1][2].cpu()[pad.expand(B, L, D)] == 0).all()
    # a spoiled document before a reset, and a spoiled carried state
    x = rand(1, L, D, seed=5)
    x[:, :60] = junk
    resets = torch.zeros(1, L, dtype=torch.bool)
    resets[0, 60] = True
    y, h = ops.gated_scan(x.to(dev), torch.zeros(1, L, D, device=dev), torch.full((1, D), junk, device=dev),
                          resets=resets.to(dev))
    assert torch.isfinite(y[:, 60:]).all() and torch.isfinite(h).all() and not torch.isfinite(y[:, 59]).any()
    # the gradient of what follows a reset reaches nothing before it
    xi = rand(1, L, D, seed=6).to(dev).requires_grad_()
    y, h = ops.gated_scan(xi, torch.zeros(1, L, D, device=dev), resets=resets.to(dev))
    gy = torch.ones(1, L, D)
    gy[:, 60:] = junk
    (gx,) = torch.autograd.grad(y, xi, gy.to(dev))
    assert torch.isfinite(gx[:, :60]).all() and not torch.isfinite(gx[:, 60]).any()


def test_gated_scan_carries_infinities_forward(dev):
    """An infinite input stays in the state until a reset, over spans of any length."""
    x = torch.zeros(1, 400, 2)
    x[0, 3, 0] = float("inf")
    y, h = ops.gated_scan(x.to(dev), torch.zeros(1, 400, 2, device=dev))
    assert torch.isinf(y[0, 3:, 0]).all() and torch.isinf(h[0, 0]) and (y[0, :, 1] == 0).all()


def test_gated_scan_partial_gradients_and_empty(dev):
    x, g = (rand(2, 30, 8, seed=s).to(dev) for s in (0, 1))
    xr = x.clone().requires_grad_()
    y, h = ops.gated_scan(xr, g)
    a = torch.autograd.grad(h.sum(), xr, retain_graph=True)[0]           # no gradient of y
    b = torch.autograd.grad(y.sum(), xr)[0]                             # none of h_last
    y, h = ops.gated_scan(xr, g)
    c = torch.autograd.grad(y.sum() + h.sum(), xr)[0]
    torch.testing.assert_close(a + b, c, rtol=1e-5, atol=1e-6)           # a sum of two fp32 results
    h0 = torch.ones(2, 8, device=dev, requires_grad=True)
    y, h = ops.gated_scan(x[:, :0], g[:, :0], h0)
    assert y.shape == (2, 0, 8) and torch.equal(h, h0)
    h.sum().backward()
    assert (h0.grad == 1).all()
    y, h = ops.gated_scan(x[:0], g[:0])
    assert y.shape == (0, 30, 8) and h.shape == (0, 8)
    one = torch.ones(8, device=dev, requires_grad=True)                  # a learned initial state, shared
    y, h = ops.gated_scan(x, g, one.expand(2, 8))
    h.sum().backward()
    h2 = torch.ones(2, 8, device=dev, requires_grad=True)
    ops.gated_scan(x, g, h2)[1].sum().backward()
    torch.testing.assert_close(one.grad, h2.grad.sum(0))


def test_gated_scan_gradient_is_the_difference_quotient(dev):
    """Central differences of a 64-bit loss over the fp32 outputs, with a step that a third derivative bounds: the
    gate's logistic has derivatives below 1, so step 2^-5 leaves an error below 2^-10 of the magnitudes."""
    B, L, D = 2, 12, 6
    x, g, h0 = rand(B, L, D, seed=1), rand(B, L, D, seed=2), rand(B, D, seed=3)
    wy, wh = rand(B, L, D, seed=4).double(), rand(B, D, seed=5).double()

    def loss(x, g, h0):
        y, h = ops.gated_scan(x.to(dev), g.to(dev), h0.to(dev))
        return float((y.cpu().double() * wy).sum() + (h.cpu().double() * wh).sum())

    ins = [v.clone().to(dev).requires_grad_() for v in (x, g, h0)]
    y, h = ops.gated_scan(*ins)
    grads = torch.autograd.grad((y, h), ins, (wy.float().to(dev), wh.float().to(dev)))
    mag = float(wy.abs().sum() + wh.abs().sum()) * 4
    for k, v in enumerate((x, g, h0)):
        e = torch.sign(rand(*v.shape, seed=10 + k)) / v.numel() ** 0.5  # a unit direction
        s = 2.0 ** -5
        up, down = [[w + (s if i == k else 0) * d * e if i == k else w for i, w in enumerate((x, g, h0))]
                    for d in (1, -1)]
        quotient = (loss(*up) - loss(*down)) / (2 * s)
        assert abs(float((grads[k].cpu().double() * e.double()).sum()) - quotient) < mag * (s * s + 64 * U / s)


def test_gated_scan_step_matches_scan(dev):
    for t in TYPES.values():
        x, g = rand(5, 6, 70, seed=0, t=t).to(dev), rand(5, 6, 70, seed=1, t=t).to(dev)
        resets = some_resets(5, 6, 1, 0.3).to(dev)
        h0 = rand(5, 70, seed=2).to(dev)
        y, h = ops.gated_scan(x, g, h0, resets=resets)
        state = h0.clone()
        for s in range(6):
            if s % 2:
                ys, state = ops.gated_scan_step(torch.cat([x[:, s], g[:, s]], -1), None, state, resets[:, s])
            else:
                keep = state.clone()
                ys, new = ops.gated_scan_step(x[:, s], g[:, s], state, resets[:, s], out=state)
                assert new is state and not torch.equal(keep, state)
            # both round the same chain of a few products; k u H per step as above
            torch.testing.assert_close(ys.float(), y[:, s].float(), rtol=2 * half_step(t) * 2, atol=64 * U * 4)
        torch.testing.assert_close(state, h, rtol=0, atol=64 * U * 4)


def test_gated_scan_refusals(dev):
    x = torch.zeros(2, 3, 4, device=dev)
    for a, kw in (((x[0],), {}), ((x[..., :3],), {}), ((x, x[:, :2]), {}), ((x, x.to(torch.bfloat16)), {}),
                  ((x, x), {"h0": torch.zeros(2, 3, device=dev)}), ((x.long(), x.long()), {}),
                  ((x, x), {"resets": torch.zeros(2, 4, device=dev)}), ((x, x), {"lengths": torch.ones(2, device=dev)}),
                  ((x, x), {"lengths": torch.ones(3, dtype=torch.long, device=dev)}),
                  ((x, x), {"lengths": torch.ones(2, dtype=torch.bool, device=dev)})):
        with pytest.raises(ValueError, match="gated_scan"):
            ops.gated_scan(*a, **kw)
    s = torch.zeros(2, 4, device=dev)
    big = torch.zeros(3, 4, device=dev)
    v = x[:, 0].contiguous()
    for a, kw in (((x, x, s), {}), ((v, v, s.double()), {}), ((v, v, s[:, :3]), {}), ((v, v, s.t().reshape(4, 2)), {}),
                  ((v, v, torch.zeros(2, 8, device=dev)[:, :4]), {}), ((v, None, s), {}),
                  ((v, v, big[:2]), {"out": big[1:]}), ((v, v, s), {"resets": torch.zeros(3, device=dev)}),
                  ((v.clone().requires_grad_(), v, s), {})):
        with pytest.raises(ValueError, match="gated_scan_step"):
            ops.gated_scan_step(*a, **kw)


# ------------------------------------------------------------------------------------------ together
def test_a_token_model_trains_through_all_three(dev):
    """ids -> embedding * sqrt(D) -> dropout -> projection -> gated scan -> tied logits: loss and gradients against the
    same model in 64 bits with the same mask."""
    V, D, B, L, p = 61, 32, 3, 40, 0.2
    w, proj, h0 = rand(V, D, seed=0, scale=0.2), rand(2 * D, D, seed=1, scale=0.2), rand(1, D, seed=2)
    ids = some_ids(B * (L + 1), V, 3).reshape(B, L + 1)
    lengths = torch.tensor([L, 25, 7])
    resets = some_resets(B, L, 4, 0.05)
    tgt = ids[:, 1:].masked_fill(torch.arange(L)[None] >= lengths[:, None], -100)

    def run(w, proj, h0, mine):
        if mine:
            e = ops.embedding(ids[:, :L].to(dev), w, math.sqrt(D), padding_idx=0)
            e = ops.dropout(e, p, seed=5, offset=1)
            y, h = ops.gated_scan(e @ proj.t(), h0=h0.expand(B, D), resets=resets.to(dev), lengths=lengths.to(dev))
        else:
            e = torch.nn.functional.embedding(ids[:, :L], w, padding_idx=0) * math.sqrt(D)
            thr = round(p * 65536)
            keep = (philox_reference(e.numel(), 5, 1) >= thr).view(e.shape)
            xg = (e * keep * 65536 / (65536 - thr)) @ proj.t()
            x, z = xg[..., :D], torch.sigmoid(xg[..., D:])
            hs, h = [], h0.expand(B, D)
            for t in range(L):
                live = (t < lengths)[:, None]
                new = (1 - z[:, t]) * h * (~resets[:, t, None]) + z[:, t] * x[:, t]
                h = torch.where(live, new, h)
                hs.append(torch.where(live, new, torch.zeros_like(new)))
            y = torch.stack(hs, 1)
        loss = torch.nn.functional.cross_entropy((y @ w.t()).reshape(-1, V), tgt.reshape(-1).to(y.device),
                                                 ignore_index=-100)
        return loss, torch.autograd.grad(loss, (w, proj, h0))

    want = run(*(v.double().requires_grad_() for v in (w, proj, h0)), False)
    got = run(*(v.to(dev).requires_grad_() for v in (w, proj, h0)), True)
    # fp32 throughout: dot products of 32 to 120 terms of size ~1 and the scan's bound, well under 2^12 roundings
    got_loss, want_loss = float(got[0].detach()), float(want[0].detach())
    assert abs(got_loss - want_loss) < 4096 * U * want_loss
    for a, b in zip(got[1], want[1]):
        assert float((a.cpu().double() - b).abs().max()) < 4096 * U * float(b.abs().max())


def test_gated_scan_with_some_gradients_wanted(dev):
    """Any subset of the inputs may want gradients, and one tensor may be both input and gate."""
    x, g, h0 = (rand(*s, seed=k).to(dev) for k, s in enumerate(((2, 9, 6), (2, 9, 6), (2, 6))))
    full = [v.clone().requires_grad_() for v in (x, g, h0)]
    y, h = ops.gated_scan(*full)
    want = torch.autograd.grad(y.sum() + h.sum(), full)
    for k in range(3):
        ins = [v.clone().requires_grad_(i == k) for i, v in enumerate((x, g, h0))]
        y, h = ops.gated_scan(*ins)
        assert torch.equal(torch.autograd.grad(y.sum() + h.sum(), ins[k])[0], want[k])
    both = x.clone().requires_grad_()
    y, h = ops.gated_scan(both, both)
    (got,) = torch.autograd.grad(y.sum() + h.sum(), both)
    two = [x.clone().requires_grad_() for _ in range(2)]
    y, h = ops.gated_scan(*two)
    assert torch.equal(got, sum(torch.autograd.grad(y.sum() + h.sum(), two)))
