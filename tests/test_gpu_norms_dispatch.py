"""Dropout and the norms under torch's dispatch modes on the device: what the modes see, that results do not depend on them,
and that a refused call leaves the generator where it was."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode, UnsupportedOperatorException
from torch.utils._python_dispatch import TorchDispatchMode

pytestmark = pytest.mark.gpu


class Log(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func.namespace == "t5vq":
            self.names.append(func._opname)
        return func(*args, **(kwargs or {}))


def tensors(n=37, d=96):
    g = torch.Generator(device="cuda").manual_seed(501)
    h, br, go, gs = (torch.randn(n, d, generator=g, device="cuda") for _ in range(4))
    w, b = torch.randn(d, generator=g, device="cuda"), torch.randn(d, generator=g, device="cuda")
    return h, br, w, b, go, gs


def step(h, br, w, b, go, gs):
    from t5vqvae_amd import norms
    leaves = [t.detach().requires_grad_(True) for t in (h, br, w, b)]
    out, total = norms.add_norm(*leaves, branch_p=0.2, p=0.1)
    y = norms.dropout(out, 0.3, total)
    return (y.detach(), total.detach()) + torch.autograd.grad((y, total), leaves, (go, gs))


def test_a_mode_sees_the_operators_and_changes_nothing():
    from t5vqvae_amd import norms
    x = tensors()
    torch.manual_seed(7)
    plain = step(*x)
    torch.manual_seed(7)
    with Log() as log:
        seen = step(*x)
    assert log.names == ["norm_forward", "dropout_add", "dropout_backward", "norm_backward"]
    assert all(torch.equal(a, b) for a, b in zip(plain, seen))
    with torch.no_grad(), Log() as log:
        norms.norm(x[0], x[2])
        norms.dropout(x[0], 0.5)
    assert log.names == ["norm_forward", "dropout_add"]


def test_fake_tensors_leave_the_generator_alone():
    from t5vqvae_amd import norms
    torch.manual_seed(3)
    state = torch.cuda.get_rng_state()
    for grad in (False, True):
        with FakeTensorMode():
            x = torch.empty(4, 8, device="cuda", requires_grad=grad)
            w = torch.empty(8, device="cuda", requires_grad=grad)
            for call in (lambda: norms.dropout(x, 0.5), lambda: norms.norm(x, w, p=0.5),
                         lambda: norms.add_norm(x, x, w, branch_p=0.5)):
                with pytest.raises(UnsupportedOperatorException):
                    call()
    assert torch.equal(torch.cuda.get_rng_state(), state)


def test_tensors_that_stand_for_their_negative():
    """A view whose negation torch has put off (the imaginary part of a conjugate) is negated before a kernel reads it: rows,
    parameters and incoming gradients."""
    from t5vqvae_amd import norms
    h, br, w, b, go, gs = tensors()
    t = torch.tensor([3, 8], device="cuda")

    def run(view):
        leaves = [v.detach().requires_grad_(True) for v in (h, br, w, b)]
        x = [view(v) for v in leaves]
        out, total = norms.add_norm(*x, branch_p=0.2, p=0.1, ticket=t)
        y = norms.dropout(x[0], 0.3, out, ticket=t)
        plain = norms.norm(x[1], x[2], x[3])
        with torch.no_grad():
            quiet = norms.norm(x[0], x[2], x[3], p=0.1, ticket=t)
        grads = torch.autograd.grad((y, total, plain), leaves, (view(go), view(gs), view(go)))
        return (y.detach(), total.detach(), plain.detach(), quiet) + grads
    lazy, done = run(torch._neg_view), run(torch.neg)
    assert torch._neg_view(h).is_neg()
    for a, c in zip(lazy, done):
        assert torch.equal(a, c)


def test_inference_mode_and_saved_tensors_kept_elsewhere():
    from t5vqvae_amd import norms
    h, br, w, b, go, gs = tensors()
    t = torch.tensor([3, 8], device="cuda")

    def run():
        return norms.add_norm(h, br, w, b, branch_p=0.2, p=0.1, ticket=t) + (norms.dropout(h, 0.3, br, ticket=t),)
    plain = run()
    with torch.inference_mode():
        quiet = run()
    assert all(torch.equal(a, c) for a, c in zip(plain, quiet))
    grads = []
    for away in (False, True):
        leaves = [v.detach().requires_grad_(True) for v in (h, br, w, b)]
        with torch.autograd.graph.save_on_cpu() if away else torch.autograd.graph.saved_tensors_hooks(lambda v: v, lambda v: v):
            out, total = norms.add_norm(*leaves, branch_p=0.2, p=0.1, ticket=t)
            y = norms.dropout(out, 0.3, total, ticket=t)
        grads.append(torch.autograd.grad((y, total), leaves, (go, gs)))
    assert all(torch.equal(a, c) for a, c in zip(*grads))
