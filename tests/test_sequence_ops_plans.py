"""The sequence kernels' plans on the GPU: sizes that take each of the ways a call can be cut up, against 64 bits under the
bounds of test_sequence_ops.py."""
import pytest
import torch

from ray_memory_management_amd import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _need_gpu(cuda):
    from ray_memory_management_amd._native import require_seq

    require_seq()


# Chains cut into segments of several tiles: wide and narrow rows, each type. (100, 1100, 128): 2 segments of 5 tiles of 8
# chunks; (60, 9000, 20): 4 of 5; (50, 900, 128) fp32: 5 of 3; (1, 9000, 3000): 9 of 8; and single channels, whole.
@pytest.mark.parametrize("B,L,D,t", [(100, 1100, 128, torch.bfloat16), (60, 9000, 20, torch.float16),
                                     (50, 900, 128, torch.float32), (1, 9000, 3000, torch.bfloat16),
                                     (12, 5000, 1, torch.float16)])
@pytest.mark.parametrize("grads", ["both", "h_last", "y"])
def test_gated_scan_over_segments_of_several_tiles(cuda, B, L, D, t, grads):
    from test_sequence_ops import check
    from test_sequence_ops_gpu import batch_reference

    g = torch.Generator(device="cuda").manual_seed(B * L + D)
    x = torch.randn(B, L, D, generator=g, device=cuda).to(t)
    gate = (torch.randn(B, L, D, generator=g, device=cuda) * 1.5 - 2).to(t)
    resets = torch.rand(B, L, generator=g, device=cuda) < 0.001
    lengths = torch.randint(0, L + 1, (B,), generator=g, device=cuda)
    lengths[0] = L
    if B > 2:
        lengths[1:3] = torch.tensor([0, L - 1], device=cuda)
    h0, dh = (torch.randn(B, D, generator=g, device=cuda) for _ in range(2))
    dy = torch.randn(B, L, D, generator=g, device=cuda).to(t)
    if grads == "h_last":
        dy.zero_()
    if grads == "y":
        dh.zero_()
    ref = {n: v.cpu() for n, v in batch_reference(x, gate, h0, resets, lengths, dy, dh).items()}
    # What the bounds relative to the values leave out: a gradient of h_last alone fades through the denormals, where each
    # step's product rounds by up to 2^-150 of its own, a product of factors that underflows is held at 2^-149 (times what
    # it multiplies), and a factor at most 1 passes that on: L steps together.
    floor = L * 2.0 ** -149 * (1 + max(float(v.abs().max()) for v in (x, h0, dh, dy)))
    for n in ("ey", "eh", "ex", "eg", "eh0"):
        ref[n] += floor
    leaves = [v.clone().requires_grad_() for v in (x, gate, h0)]
    y, h = ops.gated_scan(*leaves, resets=resets, lengths=lengths)
    check(y, ref["y"], ref["ey"], t)
    check(h, ref["h"], ref["eh"], torch.float32)
    out, seeds = {"both": ((y, h), (dy, dh)), "h_last": ((h,), (dh,)), "y": ((y,), (dy,))}[grads]
    gx, gg, gh = torch.autograd.grad(out, leaves, seeds)
    check(gx, ref["dx"], ref["ex"], t)
    check(gg, ref["dg"], ref["eg"], t)
    check(gh, ref["dh0"], ref["eh0"], torch.float32)


# 300001 ids of 300000 rows: three passes of the tiled sort, two rounds of each wave in them; long pieces whose sums are
# joined: 70000 ids of 50 rows (64 positions a piece) and 200000 of 7 (256); 4099 ids x 2053 columns: two rounds of a lane's
# columns in the lookup, with a remainder; 9000 ids x 3 columns: rows shorter than a lane.
@pytest.mark.parametrize("n,V,D,wt,ot", [
    (300001, 300000, 16, torch.float32, torch.float32), (300001, 300000, 17, torch.float32, torch.bfloat16),
    (70000, 50, 520, torch.bfloat16, torch.bfloat16), (200000, 7, 1032, torch.float32, torch.bfloat16),
    (4099, 500, 2053, torch.float16, torch.float16), (9000, 40, 3, torch.bfloat16, torch.bfloat16)])
def test_embedding_over_its_plans(cuda, n, V, D, wt, ot):
    from test_sequence_ops import U, check

    g = torch.Generator(device="cuda").manual_seed(n + D)
    ids = (torch.rand(n, generator=g, device=cuda) ** 2 * V).long().clamp_(0, V - 1)
    ids[torch.rand(n, generator=g, device=cuda) < 0.02] = -1
    ids[torch.rand(n, generator=g, device=cuda) < 0.02] = V
    pad, scale = V // 2, 0.75  # a scale that takes no rounding
    ids[n // 3:n // 3 + n // 50] = pad
    w = torch.randn(V, D, generator=g, device=cuda).to(wt).requires_grad_()
    dy = torch.randn(n, D, generator=g, device=cuda).to(ot)
    out = ops.embedding(ids, w, scale, pad, ot)
    (dw,) = torch.autograd.grad(out, w, dy)
    with torch.no_grad():
        ok = (ids >= 0) & (ids < V)
        want = torch.where(ok[:, None], w[ids.clamp(0, V - 1)].double() * scale, 0.0)
        check(out, want.cpu(), (U * want.abs()).cpu(), ot)
        use = torch.where(ok & (ids != pad), ids, V)
        total, mag = (torch.zeros(V + 1, D, dtype=torch.float64, device=cuda) for _ in range(2))
        for at in range(0, n, 50000):
            rows = dy[at:at + 50000].double()
            total.index_add_(0, use[at:at + 50000], rows)
            mag.index_add_(0, use[at:at + 50000], rows.abs())
        count = torch.bincount(use, minlength=V + 1)[:V, None]
        # count additions of fp32 in any grouping, and the scale's product
        check(dw, (total[:V] * scale).cpu(), ((count + 1) * U * mag[:V] * scale).cpu(), wt)
        assert (dw[pad] == 0).all()
    again = torch.autograd.grad(ops.embedding(ids, w, scale, pad, ot), w, dy)[0]
    assert torch.equal(dw, again)
