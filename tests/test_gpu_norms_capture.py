"""Captured backward passes of dropout and the norms beside eager graphs: refused where the pass would reach one on the default
stream, however far behind the operator, and only there."""
import gc

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 1e-6


def rows(n, d, seed, dtype=torch.float32):
    return torch.randn(n, d, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


# leaf -> what the norm takes as its weight
BETWEEN = {
    "cast": lambda w: w.to(torch.bfloat16),
    "view": lambda w: w.view(-1),
    "slice and product": lambda w: (w.view(2, 32) * 2.0).reshape(64),
}


@pytest.mark.parametrize("name", sorted(BETWEEN))
def test_a_leaf_behind_other_operations(name):
    from t5vqvae_amd import norms
    h, g = rows(50, 64, 601, torch.bfloat16), rows(50, 64, 602, torch.bfloat16)
    w = rows(1, 64, 603)[0].requires_grad_(True)

    def forward():
        return norms.norm(h, BETWEEN[name](w), eps=EPS)
    eager = forward()
    (want,) = torch.autograd.grad(eager, w, g, retain_graph=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = h * 2.0
        out = forward()
        with pytest.raises(RuntimeError, match="eager graph"):
            torch.autograd.grad(out, w, g)
        with pytest.raises(RuntimeError, match="eager graph"):
            forward().backward(g)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, h * 2.0) and w.grad is None
    del eager, out
    gc.collect()                                                  # what the refusals' tracebacks held
    again = torch.cuda.CUDAGraph()
    with torch.cuda.graph(again):
        (got,) = torch.autograd.grad(forward(), w, g)
    for _ in range(3):
        again.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_a_stream_of_layers_behind_the_last_one():
    """The last of a few add + norm and dropout layers sees the first one's leaf."""
    from t5vqvae_amd import norms
    h, g = rows(40, 64, 611), rows(40, 64, 612)
    ws = [rows(1, 64, 613 + k)[0].requires_grad_(True) for k in range(3)]
    t = torch.tensor([5, 16], device="cuda")

    def forward():
        x = h
        for w in ws:
            out, x = norms.add_norm(x, norms.dropout(x, 0.2, ticket=t), w, branch_p=0.1, ticket=t)
            x = norms.dropout(out, 0.3, x, ticket=t)
        return x
    want = torch.autograd.grad(forward(), ws, g)
    first = norms.norm(h, ws[0], eps=EPS)                        # keeps the first leaf's accumulator on the default stream
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = forward()
        with pytest.raises(RuntimeError, match="eager graph"):
            torch.autograd.grad(out, ws, g)
        # the other leaves alone do not run that accumulator
        got = torch.autograd.grad(out, ws[1:], g)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[1:]))
    del first


def test_an_eager_operation_in_front_of_the_captured_ones():
    """Not a leaf: the tensor itself was computed eagerly on the default stream, and its gradient is asked for."""
    from t5vqvae_amd import norms
    leaf, g, w = rows(50, 64, 621).requires_grad_(True), rows(50, 64, 622), rows(1, 64, 623)[0]
    x = leaf * 2.0
    t = torch.tensor([5, 16], device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = g * 2.0
        for call in (lambda: norms.norm(x, w, eps=EPS), lambda: norms.dropout(x, 0.5, ticket=t)):
            with pytest.raises(RuntimeError, match="eager graph"):
                torch.autograd.grad(call(), leaf, g)
        inside = x.detach().requires_grad_(True)
        (got,) = torch.autograd.grad(norms.norm(inside, w, eps=EPS), inside, g)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, g * 2.0)
    outside = x.detach().requires_grad_(True)
    assert torch.equal(got, torch.autograd.grad(norms.norm(outside, w, eps=EPS), outside, g)[0])


def test_an_eager_graph_on_the_capturing_stream_is_no_obstacle():
    """Accumulators that a warm-up on a side stream keeps: the pass reaches no default-stream node and is captured."""
    from t5vqvae_amd import norms
    h, g = rows(50, 64, 631), rows(50, 64, 632)
    w = rows(1, 64, 633)[0].requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        living = norms.norm(h, w, eps=EPS)
        (want,) = torch.autograd.grad(living, w, g, retain_graph=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        (got,) = torch.autograd.grad(norms.norm(h, w, eps=EPS), w, g)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    del living


def test_captured_autograd_steps_draw_from_the_generator():
    """No ticket: every replay draws anew, and its backward drops what its forward dropped."""
    from t5vqvae_amd import norms
    x, g = torch.ones(200, 768, device="cuda"), torch.ones(200, 768, device="cuda")
    zero, one = torch.zeros(768, device="cuda"), torch.ones(768, device="cuda")

    def step():
        leaf, branch = x.detach().requires_grad_(True), x.detach().requires_grad_(True)
        y = norms.dropout(leaf, 0.5)
        total = norms.add_norm(torch.zeros_like(x), branch, zero, one, branch_p=0.5, p=0.5)
        return (y.detach(), torch.autograd.grad(y, leaf, g)[0], total[1].detach(),
                torch.autograd.grad(total[1], branch, g)[0])
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    seen = []
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        y, gx, total, gb = res
        assert torch.equal(y, gx) and torch.equal(total, gb) and not torch.equal(y != 0, total != 0)
        assert 0.45 < float((y != 0).float().mean()) < 0.55
        assert not any(torch.equal(y, s) for s in seen)
        seen.append(y.clone())
        step()                                                    # the program's own eager draws in between


def test_graphed_callables():
    """torch captures a module's forward and backward into two graphs of its own: the same results as eager."""
    from t5vqvae_amd import norms
    class Layer(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.first, self.last = norms.Norm(96), norms.Norm(96, "rms")

        def forward(self, h, br):
            out, total = self.first(h, br)
            return self.last(out) * 2.0 + total
    h, br, g = rows(64, 96, 641), rows(64, 96, 642), rows(64, 96, 643)
    layer = Layer().cuda()
    with torch.no_grad():
        for k, p in enumerate(layer.parameters()):
            p.copy_(rows(1, 96, 644 + k)[0])

    def step(f):
        a, b = h.detach().requires_grad_(True), br.detach().requires_grad_(True)
        y = f(a, b)
        return (y.detach().clone(),) + tuple(t.clone() for t in torch.autograd.grad(y, [a, b, *layer.parameters()], g))
    want = step(layer)
    graphed = torch.cuda.make_graphed_callables(layer, (h.detach().requires_grad_(True), br.detach().requires_grad_(True)))
    for _ in range(3):
        for a, b in zip(step(graphed), want):
            assert torch.equal(a, b)
        torch.cuda.synchronize()
