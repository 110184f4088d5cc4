"""Gradients of dropout and the norms under create_graph: their values, and that a second derivative through them is refused
wherever it is asked for -- none is left out without a word."""
import pytest
import torch

pytestmark = pytest.mark.gpu

AGAIN = "cannot be differentiated again"


def tensors(n=37, d=96):
    g = torch.Generator(device="cuda").manual_seed(511)
    h, br, go, gs = (torch.randn(n, d, generator=g, device="cuda") for _ in range(4))
    return h, br, torch.randn(d, generator=g, device="cuda"), torch.randn(d, generator=g, device="cuda"), go, gs


def ticket():
    return torch.tensor([3, 8], device="cuda")


def test_gradients_that_record_a_graph_are_the_plain_ones():
    from t5vqvae_amd import norms
    h, br, w, b, go, gs = tensors()
    leaves = [t.requires_grad_(True) for t in (h, br, w, b)]
    for create in (False, True):
        out, total = norms.add_norm(*leaves, ticket=ticket(), branch_p=0.2, p=0.1)
        grads = torch.autograd.grad((out, total), leaves, (go, gs), create_graph=create)
        if not create:
            want = grads
    for got, plain in zip(grads, want):
        assert got.requires_grad and not plain.requires_grad and torch.equal(got, plain)
        for leaf in leaves[:3]:
            with pytest.raises(RuntimeError, match=AGAIN):
                torch.autograd.grad(got.sum(), leaf, retain_graph=True)
    with pytest.raises(RuntimeError, match=AGAIN):
        sum(g.sum() for g in grads).backward()


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("branch", [False, True])
def test_a_penalty_on_the_gradient_is_refused_beside_a_first_derivative(branch, strided):
    """The loss reaches the leaf by itself as well: the second derivative must not go missing from the sum."""
    from t5vqvae_amd import norms
    h, br, w, b, go, _ = tensors()
    leaf = (h.t().contiguous() if strided else h).requires_grad_(True)
    x = leaf.t() if strided else leaf
    w = w.requires_grad_(True)
    out = norms.add_norm(x, br, w, b)[0] if branch else norms.norm(x, w, b)
    gx, gw = torch.autograd.grad(out, (leaf, w), go, create_graph=True)
    for grad in (gx, gw):
        loss = (out * go).sum() + grad.square().sum()
        for wanted in (leaf, w):
            with pytest.raises(RuntimeError, match=AGAIN):
                torch.autograd.grad(loss, wanted, retain_graph=True)
        with pytest.raises(RuntimeError, match=AGAIN):
            torch.autograd.grad(loss, [leaf], retain_graph=True, allow_unused=True)


def test_second_derivatives_by_the_incoming_gradient():
    """Both operators' gradients are linear in the incoming one; that derivative does not exist here either.  What passes
    through unchanged (a residual's gradient, the sum's) is differentiated as such."""
    from t5vqvae_amd import norms
    h, br, w, b, go, gs = tensors()
    h.requires_grad_(True), br.requires_grad_(True), go.requires_grad_(True), gs.requires_grad_(True)
    y = norms.dropout(br, 0.4, h, ticket=ticket())
    gh, gbr = torch.autograd.grad(y, (h, br), go, create_graph=True)
    with pytest.raises(RuntimeError, match=AGAIN):
        torch.autograd.grad(gbr.sum(), go, retain_graph=True)
    assert torch.equal(gh, go) and torch.equal(torch.autograd.grad((3 * gh).sum(), go)[0], torch.full_like(go, 3))
    out, total = norms.add_norm(h, br, w, b, branch_p=0.4, ticket=ticket())
    gh, gbr = torch.autograd.grad(total, (h, br), gs, create_graph=True)
    with pytest.raises(RuntimeError, match=AGAIN):
        torch.autograd.grad(gbr.sum(), gs, retain_graph=True)
    assert torch.equal(gh, gs) and torch.equal(torch.autograd.grad((3 * gh).sum(), gs)[0], torch.full_like(gs, 3))
    for out in (norms.norm(h, w, b), norms.add_norm(h, br, w, b)[0]):
        (gh,) = torch.autograd.grad(out, h, go, create_graph=True)
        with pytest.raises(RuntimeError, match=AGAIN):
            torch.autograd.grad(gh.sum(), go)


def test_a_dropout_whose_incoming_gradient_is_a_constant_has_no_second_derivative_to_leave_out():
    from t5vqvae_amd import norms
    h, _, _, _, go, _ = tensors()
    h.requires_grad_(True)
    y = norms.dropout(h, 0.4, ticket=ticket())
    (gh,) = torch.autograd.grad(y, h, go, create_graph=True)
    assert not gh.requires_grad                                   # mask * go: no function of h
    (first,) = torch.autograd.grad((y * go).sum() + gh.square().sum(), h)
    assert torch.equal(first, gh)
