"""Dropout and the norms at the sizes where a wave walks several rows, where calls go past the caches, and at every width where
lanes and chunks change: the forms that small calls do not reach.  First, middle and last rows against the 64-bit oracle (its
masks counted from those rows), the parameters' gradients against float64 sums over all rows.

Those sums run, a column each, over the rows that one wave walks (n / (256 ROWS) at most, ROWS rows a workgroup, 256 workgroups
at least), the workgroup's rows (48 at most), and the slices (8, then a tree of 6): chains of n / (256 ROWS) + 64 at most."""
import pytest
import torch

from oracle import norm_oracle as no
from test_gpu_norms import BF16, EPS, F16, F32, TICKET, U, check, check_backward, check_forward, half_step, ticket, tiny

pytestmark = pytest.mark.gpu


def rows_at_once(d):
    """A lower bound of the rows that the workgroups of a backward call hold at once."""
    return 256 * (32 if d <= 256 else 8 if d <= 1024 else 4 if d <= 2048 else 2 if d <= 4096 else 1)


def mask(n, d, p, site):
    """All of a site's mask, as the dropout kernel draws it: site 1 of an offset is site 0 of the offset 4 further on."""
    from t5vqvae_amd import ops
    if no.keep_count(p) == 65536:
        return None
    ones = torch.ones(n, d, dtype=F16, device="cuda")
    return ops.dropout_add(ones, p, None, ticket(TICKET[0], TICKET[1] + 4 * site))[0] != 0


def parts(n):
    return [(0, min(n, 37)), (n // 2, min(n - n // 2, 41)), (max(0, n - 29), min(n, 29))]


def check_call(n, d, hidden, branch, out, wdtype, kind, bp, p, seed, with_sum=True):
    """One forward and one backward call; branch None: the plain norm."""
    from t5vqvae_amd import ops
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(dtype, *shape):
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)
    h, w, b = normal(hidden, n, d), normal(wdtype, d), normal(wdtype, d)
    br = None if branch is None else normal(branch, n, d)
    g, gs = normal(out, n, d), normal(hidden, n, d) if branch is not None and with_sum else None
    y, total, stats, _, _ = ops.norm_forward(h, w, b, kind=kind, eps=EPS, branch=br, branch_p=bp, p=p, ticket=ticket(),
                                             out_dtype=out)
    rows = h if branch is None else total
    got = ops.norm_backward(g, gs, rows, w, stats, kind=kind, branch_p=bp, p=p, ticket=ticket(), branch_dtype=branch)
    if branch is not None:
        assert torch.equal(total, ops.dropout_add(br, bp, h, ticket())[0])
    for first, count in parts(n):
        part = slice(first, first + count)
        keep0 = no.keep_mask(count, d, bp, TICKET, 0, first_row=first)
        keep1 = no.keep_mask(count, d, p, TICKET, 1, first_row=first)
        if branch is not None:
            want = h[part].double().cpu() + no.drop(br[part].double().cpu(), keep0, bp)
            off = 3 * U * (h[part].double().cpu().abs() + want.abs())
            check(total[part], want, half_step(hidden) * (want.abs() + off) + off + tiny(hidden), "sum")
        check_forward(y[part], rows[part], w, b, kind, keep1, p, out)
        check_backward((got[0][part], None if got[1] is None else got[1][part], None, None), g[part], rows[part], w, kind,
                       keep1, p, None if gs is None else gs[part], keep0, bp)
    m = mask(n, d, p, 1)
    gy = g.double() if m is None else torch.where(m, g.double() * no.scale_of(p), 0.0)
    unit = (rows.double() - stats[:, :1].double()) * stats[:, 1:].double()
    chain = -(-n // rows_at_once(d)) + 64
    # n is off by 2 u (a subtraction and a product); the scale is rounded, and applied at the end
    for name, grad, terms in (("weight", got[2], gy * unit), ("bias", got[3], gy)):
        want, bound = terms.sum(0), (chain + 6) * U * terms.abs().sum(0)
        check(grad, want.cpu(), (half_step(wdtype) * (want.abs() + bound) + bound + tiny(wdtype)).cpu(), name)


# ---- every width where lanes and chunks change, whole and one column beside it ------------------------------------------------
@pytest.mark.parametrize("d", [4, 63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 257, 511, 512, 513, 767, 768, 769, 1023, 1024,
                               1025, 2047, 2048, 2049, 4095, 4096, 4097, 6143, 6144, 6145, 8191, 8192, 8193])
@pytest.mark.parametrize("hidden,branch,out,wdtype,kind", [
    (F32, None, F32, F32, "layer"), (BF16, None, BF16, F32, "rms"), (F16, None, F32, F16, "layer"),
    (F32, F32, F32, F32, "layer"), (F32, BF16, F32, F32, "rms"), (BF16, BF16, BF16, BF16, "layer"), (F16, F16, F32, F32, "rms")])
def test_widths(d, hidden, branch, out, wdtype, kind):
    check_call(45, d, hidden, branch, out, wdtype, kind, 0.2 if branch else 0.0, 0.1, 801 + d)


# ---- several rows a wave, one site dropping: the last chunk's bits come with the row before -----------------------------------
# (calls of less than 192 MB, then of more)
TURNS = [(70001, 64, F32), (70001, 64, BF16), (40009, 192, BF16), (40009, 191, F16), (20011, 768, BF16), (12007, 768, F32),
         (12007, 765, BF16), (2003, 6144, BF16), (2003, 6141, F16)]
STREAMED = [(800005, 64, F32), (200003, 192, BF16), (131083, 768, BF16), (65541, 768, F32), (131083, 768, F16), (10003, 6144, F32)]


@pytest.mark.parametrize("n,d,dtype", TURNS + STREAMED)
def test_plain_norm_over_many_rows(n, d, dtype):
    check_call(n, d, dtype, None, dtype, F32, "layer", 0.0, 0.1, 851)


@pytest.mark.parametrize("n,d,dtype", TURNS + STREAMED)
@pytest.mark.parametrize("bp,p", [(0.2, 0.0), (0.0, 0.1)])
def test_add_norm_over_many_rows_with_one_site(n, d, dtype, bp, p):
    check_call(n, d, dtype, dtype, dtype, F32, "rms", bp, p, 852)


# ---- whole rows past the caches: every width ----------------------------------------------------------------------------------
@pytest.mark.parametrize("d", [64, 128, 192, 256, 512, 768, 1024, 2048, 4096, 6144, 8192])
@pytest.mark.parametrize("hidden,branch,out,with_sum", [(F32, None, F32, True), (BF16, None, BF16, True), (BF16, None, F32, True),
                                                        (F16, F16, F32, True), (F32, BF16, F32, True), (F32, F16, F32, False)])
def test_past_the_caches(d, hidden, branch, out, with_sum):
    """Rows of one type with an output of another, and a stream with a branch of another, at 192 MB and more in forward as in
    backward."""
    size = {F32: 4, BF16: 2, F16: 2}
    forward = size[hidden] + size[out] + (size[branch] + size[hidden] if branch else 0)
    n = (192 << 20) // (forward * d) + 37
    check_call(n, d, hidden, branch, out, F32, "layer", 0.2 if branch else 0.0, 0.1, 861 + d, with_sum)


# ---- dropout ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,d", [(30011, 768), (65541, 768), (30011, 771), (200003, 3)])
@pytest.mark.parametrize("x_type,y_type", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F32), (F32, BF16)])
def test_dropout_over_many_rows(n, d, x_type, y_type):
    """With and without a residual of y's type, all elements; the gradient on the way back."""
    from t5vqvae_amd import ops
    p = 0.1
    gen = torch.Generator(device="cuda").manual_seed(871)
    x = torch.randn(n, d, generator=gen, device="cuda").to(x_type)
    res, g = (torch.randn(n, d, generator=gen, device="cuda").to(y_type) for _ in range(2))
    keep = mask(n, d, p, 0)
    for first, count in parts(n):
        assert torch.equal(keep[first:first + count].cpu(), no.keep_mask(count, d, p, TICKET, 0, first_row=first))

    def close(got, want, off):
        bound = half_step(got.dtype) * (want.abs() + off) + off + tiny(got.dtype)
        assert bool(((got.double() - want).abs() <= bound).all())
    want = torch.where(keep, x.double() * no.scale_of(p), 0.0)
    y = ops.dropout_add(x, p, res, ticket())[0]
    assert y.dtype == y_type
    total = want + res.double()
    close(y, total, 2 * U * want.abs() + U * total.abs())
    if x_type == y_type:
        close(ops.dropout_add(x, p, None, ticket())[0], want, 2 * U * want.abs())
    back = torch.where(keep, g.double() * no.scale_of(p), 0.0)
    gx = ops.dropout_backward(g, p, ticket(), x_type)
    assert gx.dtype == x_type and bool((gx[~keep] == 0).all())
    close(gx, back, 2 * U * back.abs())
