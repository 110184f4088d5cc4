"""Dropout and the norms under torch's dispatch modes, without a GPU: what a tracer or a logging mode sees of them."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode, UnsupportedOperatorException

CALLS = {
    "dropout": (lambda n, x, w: n.dropout(x, 0.5), "t5vq.dropout_add"),
    "dropout + residual": (lambda n, x, w: n.dropout(x, 0.5, x), "t5vq.dropout_add"),
    "norm": (lambda n, x, w: n.norm(x, w), "t5vq.norm_forward"),
    "norm with dropout": (lambda n, x, w: n.norm(x, w, p=0.5), "t5vq.norm_forward"),
    "add_norm": (lambda n, x, w: n.add_norm(x, x, w, w, branch_p=0.5, p=0.5)[0], "t5vq.norm_forward"),
}


@pytest.mark.parametrize("name", sorted(CALLS))
@pytest.mark.parametrize("grad", [False, True])
def test_fake_tensors_are_refused_like_those_of_the_other_operators(name, grad):
    """A fake device tensor has no memory and its mode no rule for these operators: the mode's own refusal, which a
    compiler breaks its graph on, comes before any stream, generator or pointer is asked for."""
    from t5vqvae_amd import _lib, norms
    ops = _lib.load_torch_ops()
    call, op = CALLS[name]
    with FakeTensorMode():
        x = torch.empty(4, 8, device="cuda", requires_grad=grad)
        w = torch.empty(8, device="cuda", requires_grad=grad)
        with pytest.raises(UnsupportedOperatorException):
            ops.code_sqnorms(w.detach().view(1, 8))
        with pytest.raises(UnsupportedOperatorException, match=op):
            call(norms, x, w)
