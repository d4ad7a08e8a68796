"""The sequence operators on the GPU where it can go wrong beside the arithmetic: captured graphs, several streams and
threads at once, second derivatives, sizes that pass 32 bits. Results are compared with the same call made plainly."""
import threading

import pytest
import torch

from ray_memory_management_amd import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _need_gpu(cuda):
    from ray_memory_management_amd._native import require_seq

    require_seq()


def scan_inputs(B, L, D, seed, t=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    xg = torch.randn(B, L, 2 * D, generator=g, device="cuda")
    xg[..., D:] -= 2
    return (xg.to(t), torch.randn(B, D, generator=g, device="cuda"),
            torch.rand(B, L, generator=g, device="cuda") < 0.02, torch.randint(0, L + 1, (B,), generator=g, device="cuda"))


def scan_all(xg, h0, resets, lengths, dy, dh):
    xg, h0 = xg.detach().requires_grad_(), h0.detach().requires_grad_()
    y, h = ops.gated_scan(xg, h0=h0, resets=resets, lengths=lengths)
    return (y, h, *torch.autograd.grad((y, h), (xg, h0), (dy, dh)))


def embed_all(ids, w, dy):
    w = w.detach().requires_grad_()
    out = ops.embedding(ids, w, 2.0, padding_idx=0)
    return out, torch.autograd.grad(out, w, dy)[0]


def capture(fn):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out


@pytest.mark.parametrize("B,L,D", [(1, 3000, 128), (4, 20, 64), (200, 130, 130)])
def test_gated_scan_in_a_graph(B, L, D):
    """Forward and backward replayed with new inputs, with eager calls and synchronisations between the replays."""
    bufs = list(scan_inputs(B, L, D, 0)) + [torch.randn(B, L, D, device="cuda").bfloat16(), torch.randn(B, D, device="cuda")]
    graph, out = capture(lambda: scan_all(*bufs))
    for seed in (1, 2, 3, 4):
        new = list(scan_inputs(B, L, D, seed)) + [torch.randn_like(bufs[4]), torch.randn_like(bufs[5])]
        for b, v in zip(bufs, new):
            b.copy_(v)
        graph.replay()
        want = scan_all(*new)
        torch.cuda.synchronize()
        for a, w in zip(out, want):
            assert torch.equal(a, w)


@pytest.mark.parametrize("n,V,D", [(700, 90, 24), (20000, 3000, 64)])
def test_embedding_in_a_graph(n, V, D):
    ids, w, dy = torch.randint(0, V, (n,), device="cuda"), torch.randn(V, D, device="cuda"), torch.randn(n, D, device="cuda")
    graph, out = capture(lambda: embed_all(ids, w, dy))
    for seed in range(4):
        torch.manual_seed(seed)
        ids.random_(0, V)
        w.normal_()
        dy.normal_()
        graph.replay()
        want = embed_all(ids, w, dy)
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_dropout_in_a_graph_draws_anew_with_its_counter():
    x, dy, ctr = torch.randn(3001, device="cuda"), torch.randn(3001, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")

    def step():
        leaf = x.detach().requires_grad_()
        y = ops.dropout(leaf, 0.3, 7, ctr)
        ctr.add_(1)
        return y, torch.autograd.grad(y, leaf, dy)[0]

    graph, (y, dx) = capture(step)
    masks = []
    for _ in range(4):
        k = int(ctr)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.dropout(x, 0.3, 7, k)) and torch.equal(dx, ops.dropout(dy, 0.3, 7, k))
        assert int(ctr) == k + 1
        masks.append(y == 0)
    assert not any(torch.equal(a, b) for i, a in enumerate(masks) for b in masks[:i])


def test_two_graphs_replayed_at_once():
    """Each graph has its own workspace: replays on two streams do not disturb each other."""
    sets = [list(scan_inputs(1, 4000, 128, s)) + [torch.randn(1, 4000, 128, device="cuda").bfloat16(),
                                                 torch.randn(1, 128, device="cuda")] for s in (0, 1)]
    e = [(torch.randint(0, 500, (9000,), device="cuda"), torch.randn(500, 32, device="cuda"),
          torch.randn(9000, 32, device="cuda")) for _ in (0, 1)]
    graphs = [capture(lambda i=i: (*scan_all(*sets[i]), *embed_all(*e[i]))) for i in (0, 1)]
    want = [(*scan_all(*sets[i]), *embed_all(*e[i])) for i in (0, 1)]
    streams = [torch.cuda.Stream() for _ in (0, 1)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (_, out), w in zip(graphs, want):
        for a, b in zip(out, w):
            assert torch.equal(a, b)


def test_streams_and_threads_at_once():
    """Calls from four threads, each on a stream of its own, against the same calls alone."""
    jobs = []
    for k in range(4):
        sc = list(scan_inputs(2, 2500, 96, k)) + [torch.randn(2, 2500, 96, device="cuda").bfloat16(),
                                                 torch.randn(2, 96, device="cuda")]
        jobs.append((sc, (torch.randint(0, 700, (12000,), device="cuda"), torch.randn(700, 40, device="cuda"),
                          torch.randn(12000, 40, device="cuda"))))
    want = [(*scan_all(*s), *embed_all(*e)) for s, e in jobs]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(k):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(5):
                    got[k] = (*scan_all(*jobs[k][0]), *embed_all(*jobs[k][1]))
            stream.synchronize()
        except Exception as e:  # pragma: no cover - shown by the assert below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors, errors
    for g, w in zip(got, want):
        for a, b in zip(g, w):
            assert torch.equal(a, b)


def test_a_capture_over_leaves_of_a_living_eager_graph_is_refused():
    x = torch.randn(2, 6, 4, device="cuda", requires_grad=True)
    w = torch.randn(5, 4, device="cuda", requires_grad=True)
    ids = torch.zeros(3, dtype=torch.long, device="cuda")
    calls = [lambda: ops.dropout(x, 0.5, 1), lambda: ops.gated_scan(x, x.detach())[0], lambda: ops.embedding(ids, w)]
    alive = [c() for c in calls]
    for c in calls:
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="outside the capture"):
            with torch.cuda.graph(graph):
                c()
    del alive
    for c in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = c()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, c())
        del out


def test_a_step_in_place_is_noticed_by_autograd(cuda):
    state = torch.randn(2, 4, device=cuda)
    y = torch.ones(2, 4, device=cuda, requires_grad=True) * state
    with torch.no_grad():
        ops.gated_scan_step(torch.zeros(2, 4, device=cuda), torch.zeros(2, 4, device=cuda), state, out=state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_second_derivatives_are_refused():
    x = torch.randn(2, 5, 8, device="cuda", requires_grad=True)
    w = torch.randn(6, 8, device="cuda", requires_grad=True)
    v = torch.randn(2, 5, 8, device="cuda", requires_grad=True)
    for y, leaf in ((ops.gated_scan(x, x * 1.0)[0], x), (ops.dropout(x, 0.5, 1), x),
                    (ops.embedding(torch.zeros(2, 5, dtype=torch.long, device="cuda"), w), w)):
        (g,) = torch.autograd.grad(y, leaf, v, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            g.sum().backward()  # as with torch's own once-differentiable functions, said when the pass gets there


def test_large_tables_and_batches_pass_32_bits():
    """A table of 2^32 + 2^13 elements and a batch of 2^32 + 2^14 (fp16 / bf16): rows at both ends."""
    V, D = (1 << 19) + 1, 1 << 13
    w = torch.zeros(V, D, dtype=torch.float16, device="cuda")
    w[0], w[V - 1], w[V // 2] = 1, 2, 3
    w.requires_grad_()
    ids = torch.tensor([V - 1, 0, V // 2, V - 1, V], device="cuda")
    out = ops.embedding(ids, w)
    assert out[:, 0].tolist() == [2, 1, 3, 2, 0] and out[:, -1].tolist() == [2, 1, 3, 2, 0]
    (dw,) = torch.autograd.grad(out, w, torch.ones_like(out))
    assert (dw[V - 1] == 2).all() and (dw[0] == 1).all() and (dw[V // 2] == 1).all()
    assert float(dw.sum(dtype=torch.float64)) == 4 * D
    del out, dw, w
    n = (1 << 32) + (1 << 14)
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = ops.dropout(x, 0.5, 5, 6)
    tail = ((1 << 32) // 8) * 8
    from ray_memory_management_amd.ops.sequence import _philox_words

    q = torch.arange(tail // 8, tail // 8 + 100)
    words = _philox_words(q, 6, 5)
    keep = torch.stack([words & 0xFFFF, words >> 16], dim=-1).reshape(-1) >= 32768
    assert torch.equal(y[tail:tail + 800].cpu() != 0, keep)
    assert not torch.equal(y[:800], y[tail:tail + 800])
    del x, y
    B, L, D = 3, (1 << 20) + 1, 1 << 11                       # sequences of 2^31 + 2^11 elements
    x = torch.zeros(1, L, D, dtype=torch.bfloat16, device="cuda").expand(B, L, D)
    gate = torch.full((1, 1, D), 0.0, dtype=torch.bfloat16, device="cuda").expand(B, L, D)
    h0 = torch.ones(B, D, device="cuda")
    resets = torch.zeros(B, L, dtype=torch.bool, device="cuda")
    y, h = ops.gated_scan(x[:, -40:], gate[:, -40:], h0)
    assert torch.equal(h, torch.full_like(h, 2.0 ** -40))
    lengths = torch.tensor([L, 3, L - 1], device="cuda")
    y, h = ops.gated_scan(x, gate, h0, resets=resets, lengths=lengths)
    assert (h[1] == 0.125).all() and (h[0] == 0).all() and y[1, 2, -1] == 0.125 and (y[2, :4, -1].float() == torch.tensor(
        [0.5, 0.25, 0.125, 0.0625], device="cuda")).all()
    assert (y[:, 64:200] < 1e-18).all() and (y[1, 3:] == 0).all()


def test_inputs_of_a_call_may_change_after_it(cuda):
    """What a backward pass needs is either kept by autograd, which notices a change, or belongs to the call."""
    lengths = torch.tensor([5, 3], device=cuda)
    x = torch.randn(2, 5, 8, device=cuda, requires_grad=True)
    y, h = ops.gated_scan(x, torch.zeros_like(x).requires_grad_(), lengths=lengths)
    lengths.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_a_batch_of_many_short_sequences(cuda):
    """More sequences than a grid dimension other than the first may have."""
    x = torch.randn(70000, 2, 3, device=cuda)
    y, h = ops.gated_scan(x, torch.zeros_like(x))
    want = x[:, 0] / 2
    assert torch.equal(y[:, 0], want) and torch.allclose(y[:, 1], want / 2 + x[:, 1] / 2) and torch.equal(h, y[:, 1])


def batch_reference(x, g, h0, resets, lengths, dy, dh):
    """test_sequence_ops.scan_reference (values and bounds) for all sequences at once."""
    u = 2.0 ** -24
    x, g, dy = x.double(), g.double(), dy.double()
    B, L, D = x.shape
    live = (torch.arange(L, device=x.device)[None] < lengths[:, None])[:, :, None]
    z, a = torch.sigmoid(g), torch.sigmoid(-g)
    k = (2 * (g.abs() + 8) + 4) * u
    cut = resets[:, :, None]
    h, H = h0.double(), h0.double().abs()
    E = torch.zeros_like(h)
    out = {n: torch.zeros(B, L, D, dtype=torch.float64, device=x.device) for n in ("y", "ey", "dx", "ex", "dg", "eg")}
    hp, Hp, Ep = (torch.zeros_like(out["y"]) for _ in range(3))
    for t in range(L):
        keep = (~cut[:, t]).double()
        hp[:, t], Hp[:, t], Ep[:, t] = h * keep, H * keep, E * keep
        nh = a[:, t] * hp[:, t] + z[:, t] * x[:, t]
        nH = a[:, t] * Hp[:, t] + z[:, t] * x[:, t].abs()
        nE = a[:, t] * Ep[:, t] + k[:, t] * nH
        h, H, E = (torch.where(live[:, t], n, o) for n, o in ((nh, h), (nH, H), (nE, E)))
        out["y"][:, t], out["ey"][:, t] = nh, nE
    out["h"], out["eh"] = h, E
    back, M = dh.double(), dh.double().abs()
    F = torch.zeros_like(back)
    for t in range(L - 1, -1, -1):
        b, m = back + dy[:, t], M + dy[:, t].abs()
        f = F + k[:, t] * m
        diff = x[:, t].abs() + Hp[:, t]
        out["dx"][:, t], out["ex"][:, t] = b * z[:, t], z[:, t] * (f + k[:, t] * m)
        out["dg"][:, t] = b * (x[:, t] - hp[:, t]) * z[:, t] * a[:, t]
        out["eg"][:, t] = z[:, t] * a[:, t] * (f * diff + m * Ep[:, t] + 2 * k[:, t] * m * diff)
        keep = (~cut[:, t]).double() * a[:, t]
        back, M, F = (torch.where(live[:, t], n, o) for n, o in (
            (b * keep, back), (m * keep, M), (f * keep + k[:, t] * m * keep, F)))
    out["dh0"], out["eh0"] = back, F
    for n in ("y", "ey", "dx", "ex", "dg", "eg"):
        out[n] = torch.where(live, out[n], 0.0)
    return out


@pytest.mark.parametrize("B,L,D,t", [
    (130, 2600, 6, torch.bfloat16), (140, 700, 130, torch.float32), (3, 9000, 20, torch.float16), (128, 400, 64, torch.bfloat16),
    (2, 5000, 34, torch.float32), (40, 600, 1, torch.bfloat16), (1, 12345, 7, torch.float32), (70, 900, 257, torch.float16)])
def test_gated_scan_over_many_tiles_and_segments(cuda, B, L, D, t):
    """Whole and cut chains, wide and narrow rows, odd widths, with resets and lengths."""
    from test_sequence_ops import check

    g = torch.Generator(device="cuda").manual_seed(B * L + D)
    x = torch.randn(B, L, D, generator=g, device=cuda).to(t)
    gate = (torch.randn(B, L, D, generator=g, device=cuda) * 1.5 - 2).to(t)
    resets = torch.rand(B, L, generator=g, device=cuda) < 0.005
    lengths = torch.randint(0, L + 1, (B,), generator=g, device=cuda)
    lengths[0] = L
    h0, dh = (torch.randn(B, D, generator=g, device=cuda) for _ in range(2))
    dy = torch.randn(B, L, D, generator=g, device=cuda).to(t)
    ref = {n: v.cpu() for n, v in batch_reference(x, gate, h0, resets, lengths, dy, dh).items()}
    leaves = [v.clone().requires_grad_() for v in (x, gate, h0)]
    y, h = ops.gated_scan(*leaves, resets=resets, lengths=lengths)
    check(y, ref["y"], ref["ey"], t)
    check(h, ref["h"], ref["eh"], torch.float32)
    gx, gg, gh = torch.autograd.grad((y, h), leaves, (dy, dh))
    check(gx, ref["dx"], ref["ex"], t)
    check(gg, ref["dg"], ref["eg"], t)
    check(gh, ref["dh0"], ref["eh0"], torch.float32)
