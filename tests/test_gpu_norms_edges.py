"""Backward of norms whose rows are far from zero and do not fill their lanes: what stands behind a row's end stays out of it."""
import pytest
import torch

from oracle import norm_oracle as no

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


# (rows, columns, the rows' constant, eps): |constant| / sqrt(eps) passes fp32's largest number, columns * |constant| does not,
# and columns * fl(1 / columns) rounds to 1, so that the kernel's mean is the constant exactly and the deviation sqrt(eps)
@pytest.mark.parametrize("n,d,power,eps", [(3, 5, 119, 1e-6), (3, 100, 116, 1e-8), (3, 300, 116, 1e-8), (3, 1030, 117, 1e-8),
                                           (3, 4100, 115, 1e-8), (3, 10000, 112, 1e-10), (2, 20001, 112, 1e-10),
                                           (900, 513, 116, 1e-8), (3, 2, 122, 1e-6)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_constant_rows_far_from_zero(n, d, power, eps, dtype):
    """n = 0 in every column, so grad_hidden = r (a - mean a) and grad_weight = 0."""
    from t5vqvae_amd import ops
    inv = torch.tensor(1.0) / d
    assert float(torch.tensor(float(d)) * inv) == 1.0 and d * 2.0 ** power < 2.0 ** 128 < 2.0 ** power / eps ** 0.5
    g = torch.Generator().manual_seed(701)
    h = torch.full((n, d), 2.0 ** power, dtype=dtype)
    go, w = torch.randn(n, d, generator=g).to(dtype), torch.randn(d, generator=g)
    out, _, stats, _, _ = ops.norm_forward(h.cuda(), w.cuda(), None, kind="layer", eps=eps)
    r = float(torch.tensor(eps, dtype=torch.float32).double() ** -0.5)
    assert bool((out == 0).all()) and bool((stats[:, 0] == 2.0 ** power).all())
    assert bool(((stats[:, 1].double() / r - 1.0).abs() <= 4 * U).all())
    for branch_dtype in (None, dtype):
        gh, gb, gw, gbias = ops.norm_backward(go.cuda(), None, h.cuda(), w.cuda(), stats, kind="layer",
                                              branch_dtype=branch_dtype)
        a = go.double() * w.double()
        want = (a - a.mean(1, keepdim=True)) * r
        # products, the mean's chain of ceil(d / 64) + 16, the subtraction, the product with r (r off by 4 u), the rounding
        size = a.abs() + a.abs().mean(1, keepdim=True)
        bound = r * (-(-d // 64) + 16 + 10) * U * size
        bound = bound + torch.finfo(dtype).eps / 2 * (want.abs() + bound)
        assert bool(((gh.cpu().double() - want).abs() <= bound).all())
        assert bool((gw == 0).all()) and bool(torch.isfinite(gbias).all())
        assert (gb is None) == (branch_dtype is None) and (gb is None or torch.equal(gb, gh))


def test_waves_without_a_row_add_nothing():
    """Calls past the caches keep a workgroup's waves together, also those that have run out of rows: behind a last row of that
    kind they still add nothing to the parameters' gradients."""
    from t5vqvae_amd import ops
    n, d, power, eps = 65541, 1024, 117, 1e-8
    h = torch.full((n, d), 2.0 ** power, device="cuda")
    g = torch.randn(n, d, generator=torch.Generator(device="cuda").manual_seed(702), device="cuda")
    w = torch.ones(d, device="cuda")
    _, _, stats, _, _ = ops.norm_forward(h, w, None, kind="layer", eps=eps)
    assert bool((stats[:, 0] == 2.0 ** power).all())
    for branch_dtype in (None, torch.float32):
        gh, _, gw, gbias = ops.norm_backward(g, None, h, w, stats, kind="layer", branch_dtype=branch_dtype)
        assert bool((gw == 0).all()) and bool(torch.isfinite(gh).all())
        total, size = g.double().sum(0), g.double().abs().sum(0)
        assert bool(((gbias.double() - total).abs() <= (n / 2048 + 68) * U * size).all())
