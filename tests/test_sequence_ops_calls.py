"""Calls of the sequence operators beside the ordinary ones: recomputation, forward-mode derivatives, closed gates,
aliased outputs, sizes at the ends of the launches."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from ray_memory_management_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.fixture(params=DEVICES)
def dev(request):
    if request.param == "cuda":
        if not torch.cuda.is_available():
            pytest.skip("no GPU")
        from ray_memory_management_amd._native import require_seq

        require_seq()
    return torch.device(request.param)


# ------------------------------------------------------------------------------------------ recomputation
class Block(torch.nn.Module):
    """Two dropout layers, one of them called twice, around products elementwise (so that gradients have no sums)."""

    def __init__(self, dev):
        super().__init__()
        self.a, self.b = ops.Dropout(0.5, seed=3), ops.Dropout(0.25, seed=4)
        self.w = torch.nn.Parameter(torch.linspace(0.5, 1.5, 3000))
        self.to(dev)

    def forward(self, x):
        return self.a(torch.tanh(self.b(self.a(x) * self.w)), residual=x)


@pytest.mark.parametrize("use_reentrant", [False, True])
def test_a_recomputed_block_draws_the_same_masks(dev, use_reentrant):
    plain, block = Block(dev), Block(dev)
    for step in range(3):
        x = torch.linspace(1, 2, 3000, device=dev) + step
        xs = [x.clone().requires_grad_() for _ in (0, 1)]
        plain.w.grad = block.w.grad = None  # then a gradient is the sum of two terms, the same in either order
        mid = [plain(xs[0]), checkpoint(ops.repeatable(block), xs[1], use_reentrant=use_reentrant)]
        out = [plain(mid[0]), checkpoint(ops.repeatable(block), mid[1], use_reentrant=use_reentrant)]
        for o, v in zip(out, xs):
            o.backward(torch.linspace(-1, 1, 3000, device=dev))
        assert torch.equal(*out) and torch.equal(xs[0].grad, xs[1].grad) and torch.equal(plain.w.grad, block.w.grad)
        for m in (plain, block):  # each training call counts once, whether recomputed or not
            assert int(m.a.counter) == 4 * (step + 1) and int(m.b.counter) == 2 * (step + 1)
    assert block.a._repeats == 0


@pytest.mark.parametrize("use_reentrant", [False, True])
def test_a_recomputed_layer_drops_the_same_places(dev, use_reentrant):
    m = ops.Dropout(0.5, seed=3).to(dev)
    for _ in range(3):
        x = torch.ones(4096, device=dev, requires_grad=True)
        y = checkpoint(ops.repeatable(m), x, use_reentrant=use_reentrant)
        y.sum().backward()
        assert torch.equal(y == 0, x.grad == 0) and bool((y == 0).any())
    fn = lambda v: m(v) * 2.0  # noqa: E731
    x = torch.ones(4096, device=dev, requires_grad=True)
    y = checkpoint(ops.repeatable(fn, m), x, use_reentrant=use_reentrant)
    y.sum().backward()
    assert torch.equal(y == 0, x.grad == 0) and int(m.counter) == 4


def test_a_recomputation_in_a_recomputation(dev):
    block, plain = Block(dev), Block(dev)
    x, r = (torch.linspace(1, 2, 3000, device=dev).requires_grad_() for _ in (0, 1))
    inner = lambda v: checkpoint(ops.repeatable(block), v, use_reentrant=False) + block.b(v)  # noqa: E731
    y = checkpoint(ops.repeatable(inner, block), x, use_reentrant=False)
    want = plain(r) + plain.b(r)
    assert torch.equal(y, want)
    y.sum().backward()
    want.sum().backward()
    assert torch.equal(x.grad, r.grad) and torch.equal(block.w.grad, plain.w.grad)
    assert int(block.a.counter) == 2 and int(block.b.counter) == 2 and block.a._repeats == block.b._repeats == 0


@pytest.mark.parametrize("use_reentrant", [False, True])
def test_a_recomputation_with_another_mask_is_refused(dev, use_reentrant):
    m = ops.Dropout(0.5, seed=3).to(dev)
    x = torch.ones(64, device=dev, requires_grad=True)
    y = checkpoint(m, x, use_reentrant=use_reentrant)
    with pytest.raises(RuntimeError, match="repeatable"):
        y.sum().backward()
    wrapped = ops.repeatable(m)
    y = checkpoint(wrapped, x, use_reentrant=use_reentrant)
    with pytest.raises(RuntimeError, match="a wrapper of its own"):
        wrapped(x)
    y.sum().backward()
    # an ordinary region around a repeatable one whose result it needs again
    y = checkpoint(lambda v: checkpoint(ops.repeatable(m), v, use_reentrant=use_reentrant).exp(), x,
                   use_reentrant=use_reentrant)
    with pytest.raises(RuntimeError, match="around it"):
        y.sum().backward()
    with pytest.raises(ValueError, match="repeatable"):
        ops.repeatable(lambda v: m(v))
    m.eval()
    checkpoint(m, x, use_reentrant=use_reentrant).sum().backward()  # nothing is drawn


@pytest.mark.gpu
def test_a_recomputed_layer_in_a_graph(cuda):
    """Each replay draws a new mask, and its recomputation the same one."""
    m = ops.Dropout(0.5, seed=3).to(cuda)
    src = torch.ones(3000, device=cuda)

    def step():
        x = src.detach().requires_grad_()
        y = checkpoint(ops.repeatable(m), x, use_reentrant=False, preserve_rng_state=False)
        return y, torch.autograd.grad(y, x, torch.ones_like(y))[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, g = step()
    at = int(m.counter)
    for k in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.dropout(src, 0.5, 3, at + k)) and torch.equal(g, y)
    assert int(m.counter) == at + 4


# ------------------------------------------------------------------------------------------ derivatives
@pytest.mark.gpu
def test_forward_mode_derivatives_are_refused(cuda):
    """A dual tensor without requires_grad would come out without its tangent."""
    import torch.autograd.forward_ad as fw

    def both(*shape):
        v = torch.randn(*shape, device=cuda)
        return v, fw.make_dual(v.clone(), torch.ones_like(v))

    with fw.dual_level():
        (x, xd), (w, wd), (h, hd) = both(2, 5, 8), both(6, 8), both(2, 8)
        ids = torch.zeros(3, dtype=torch.long, device=cuda)
        calls = [lambda: ops.embedding(ids, wd), lambda: ops.dropout(xd, 0.5, 1), lambda: ops.dropout(x, 0.5, 1, residual=xd),
                 lambda: ops.gated_scan(xd, x), lambda: ops.gated_scan(x, xd), lambda: ops.gated_scan(xd),
                 lambda: ops.gated_scan(x, x, hd), lambda: ops.gated_scan(x, x, hd.requires_grad_()),
                 lambda: ops.gated_scan_step(xd[:, 0], x[:, 0], h), lambda: ops.gated_scan_step(x[:, 0], x[:, 0], hd)]
        for call in calls:
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call()
            with pytest.raises((NotImplementedError, ValueError), match="forward-mode|not differentiable"):
                call()
        dy = fw.make_dual(torch.ones(2, 5, 8, device=cuda), torch.ones(2, 5, 8, device=cuda))
        leaf, table = x.clone().requires_grad_(), w.clone().requires_grad_()
        for y in (ops.dropout(leaf, 0.5, 1), ops.gated_scan(leaf, x)[0], ops.embedding(ids.new_zeros(2, 5), table)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                y.backward(dy)
    ops.gated_scan(x, x, h)  # outside the level nothing is refused
