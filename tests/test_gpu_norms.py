"""Dropout from a counter, layer / RMS norm and add + norm (t5vqvae_amd.norms, ops, EncoderTailVQ's counter form) against
the 64-bit oracle.  Masks are compared exactly, values element by element with bounds that count the roundings:

u_T = half a step of the output's type, u = 2^-24.  A sum of n fp32 terms in chains of at most c terms is off by at most
(c - 1) u sum|terms|; a row's sums run in chains of ceil(D / 64) + 16 at most (a lane's groups, the four values of a group,
the tree over lanes), a column's in N / 8 + 160 (a wave's rows -- at least min(N, 8) slices --, four waves, the slices' tree)
for the sizes below.  With C the row's chain: the mean is off by (C + 1) u mean|h|, h - mean by that plus u |h - mean|, 1 / deviation relatively
by (C + 8) u / 2 + 2 u (the sum of squares, division, eps, root, reciprocal; the mean's own error enters squared), so
n = (h - mean) r by   dn = (C + 1) u mean|h| r + (C / 2 + 8) u |n|   (the same for the n a backward makes from the statistics)."""
import copy

import numpy as np
import pytest
import torch

from oracle import norm_oracle as no

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
EPS = 1e-6
TICKET = (0x0123456789ABCDEF, (5 << 33) + 16)


def ticket(seed=TICKET[0], offset=TICKET[1]):
    return torch.tensor([seed, offset], dtype=torch.int64, device="cuda")


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):      # below the smallest normal number a rounding is off by half a subnormal step at most
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps


def rows(n, d, seed, dtype=F32, scale=1.0, offset=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, d, generator=g) * scale + offset).to(dtype)


def check(got, want, bound, name):
    got, want, bound = got.detach().cpu().double(), want.double(), bound.double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    off = (got - want).abs() - bound
    assert bool(torch.isfinite(got).all()), name
    worst = int(off.argmax())
    assert float(off.max()) <= 0, (name, worst, float(got.reshape(-1)[worst]), float(want.reshape(-1)[worst]),
                                   float(bound.reshape(-1)[worst]))


def chain(d):
    return -(-d // 64) + 16


def check_forward(out, h, weight, bias, kind, keep, p, dtype, name="out"):
    """out against the norm of the rows h (as the kernel read them)."""
    h, w = h.double().cpu(), weight.double().cpu()
    b = None if bias is None else bias.double().cpu()
    want = no.norm(h, w, b, kind, EPS, keep, p)
    mean, r = no.stats(h, kind, EPS)
    n, c = (h - mean) * r, chain(h.shape[1])
    dn = (c + 1) * U * h.abs().mean(1, keepdim=True) * r + (c / 2 + 8) * U * n.abs()
    y = (n * w).abs() + (0 if b is None else b.abs())
    bound = (dn * w.abs() + 4 * U * y) * (no.scale_of(p) if p else 1.0)
    check(out, want, half_step(dtype) * (want.abs() + bound) + bound + tiny(dtype), name)
    if p:
        assert bool((out.cpu()[~keep] == 0).all())


def check_backward(got, g, h, weight, kind, keep, p, g_sum=None, branch_keep=None, branch_p=0.0, n_slices=8):
    gh, gb, gw, gbias = got
    g, h, w = g.double().cpu(), h.double().cpu(), weight.double().cpu()
    gs = None if g_sum is None else g_sum.double().cpu()
    want = no.norm_backward(g, h, w, kind, EPS, keep, p, gs, branch_keep, branch_p)
    mean, r = no.stats(h, kind, EPS)
    n, c = (h - mean) * r, chain(h.shape[1])
    dn = (c + 1) * U * h.abs().mean(1, keepdim=True) * r + (c / 2 + 8) * U * n.abs()
    gy = g if keep is None else no.drop(g, keep, p)
    a = (gy * w).abs()
    m1 = a.mean(1, keepdim=True) if kind == "layer" else torch.zeros(1, 1, dtype=torch.float64)
    m2 = (a * n.abs()).mean(1, keepdim=True)
    # every term of the formula with its own roundings, the two means with their chains, n and r with their errors
    bound = r * ((c + 8) * U * (a + m1 + n.abs() * m2) + dn * m2 + n.abs() * (a * dn).mean(1, keepdim=True)
                 + (c / 2 + 8) * U * (a + m1 + n.abs() * m2))
    if gs is not None:
        bound = bound + 2 * U * (gs.abs() + want[0].abs())
    check(gh, want[0], half_step(gh.dtype) * (want[0].abs() + bound) + bound + tiny(gh.dtype), "grad_hidden")
    if gb is not None:
        bb = (bound + 2 * U * want[0].abs()) * (no.scale_of(branch_p) if branch_p else 1.0)
        check(gb, want[1], half_step(gb.dtype) * (want[1].abs() + bb) + bb + tiny(gb.dtype), "grad_branch")
        if branch_p:
            assert bool((gb.cpu()[~branch_keep] == 0).all())
    rows_chain = h.shape[0] / n_slices + 160
    if gw is not None:
        bound = (gy.abs() * dn).sum(0) + (rows_chain + 3) * U * (gy * n).abs().sum(0)
        check(gw, want[2], half_step(gw.dtype) * (want[2].abs() + bound) + bound + tiny(gw.dtype), "grad_weight")
    if gbias is not None:
        bound = (rows_chain + 3) * U * gy.abs().sum(0)
        check(gbias, want[3], half_step(gbias.dtype) * (want[3].abs() + bound) + bound + tiny(gbias.dtype), "grad_bias")


# ---- dropout ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,d", [(1, 1), (1, 768), (3, 5), (45, 771), (257, 64), (100, 2049), (2, 100003), (1030, 8),
                                 (70000, 3)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_dropout_forward_and_backward(n, d, dtype):
    from t5vqvae_amd import ops
    p = 0.1
    x, res, g = rows(n, d, 1, dtype), rows(n, d, 2, dtype), rows(n, d, 3, dtype)
    keep = no.keep_mask(n, d, p, TICKET, 0)
    for r in (None, res):
        y, drawn = ops.dropout_add(x.cuda(), p, None if r is None else r.cuda(), ticket())
        assert drawn is None and y.dtype == dtype
        want = no.drop(x.double(), keep, p)
        off = 2 * U * want.abs()
        if r is not None:
            off = off + U * (want + r.double()).abs()
            want = want + r.double()
        check(y, want, half_step(dtype) * (want.abs() + off) + off + tiny(dtype), "y")
        assert bool((y.cpu()[~keep] == (0 if r is None else r[~keep])).all())
    gx = ops.dropout_backward(g.cuda(), p, ticket())
    want = no.drop(g.double(), keep, p)
    check(gx, want, (half_step(dtype) + 2 * U) * want.abs() + tiny(dtype), "gx")
    assert bool((gx.cpu()[~keep] == 0).all())


@pytest.mark.parametrize("half", [BF16, F16])
def test_dropout_of_a_half_branch_beside_an_fp32_stream(half):
    from t5vqvae_amd import norms
    n, d, p = 33, 100, 0.25
    x, res, g = rows(n, d, 1, half), rows(n, d, 2), rows(n, d, 3)
    xg, rg = x.cuda().requires_grad_(True), res.cuda().requires_grad_(True)
    y = norms.dropout(xg, p, rg, ticket=ticket())
    assert y.dtype == F32
    keep = no.keep_mask(n, d, p, TICKET, 0)
    want = no.drop(x.double(), keep, p)
    check(y, want + res.double(), 3 * U * (want.abs() + res.double().abs()), "y")
    y.backward(g.cuda())
    assert xg.grad.dtype == half and torch.equal(rg.grad.cpu(), g)
    want = no.drop(g.double(), keep, p)
    check(xg.grad, want, (half_step(half) + 2 * U) * want.abs() + tiny(half), "gx")


def test_dropout_probabilities_at_their_ends_and_values_that_are_not_numbers():
    from t5vqvae_amd import norms, ops
    x = rows(50, 77, 5).cuda()
    assert torch.equal(ops.dropout_add(x, 0.0)[0], x) and ops.dropout_add(x, 0.0)[1] is None
    assert torch.equal(ops.dropout_add(x, 2.0 ** -18)[0], x)                # rounds to no dropout at all
    assert bool((ops.dropout_add(x, 1.0)[0] == 0).all())
    assert torch.equal(ops.dropout_add(x, 1.0, x)[0], x)
    assert bool((ops.dropout_backward(x, 1.0, ticket()) == 0).all())
    one = 1.0 - 1.0 / 65536                                                   # one draw in 65536 keeps: scale 65536
    y = ops.dropout_add(x, one, None, ticket())[0].cpu()
    keep = no.keep_mask(50, 77, one, TICKET, 0)
    assert torch.equal(y, torch.where(keep, x.cpu() * 65536, torch.zeros(())))
    bad = torch.full((40, 40), float("nan"), device="cuda")
    bad[::2] = float("inf")
    y = ops.dropout_add(bad, 0.5, None, ticket())[0].cpu()
    keep = no.keep_mask(40, 40, 0.5, TICKET, 0)
    assert bool((y[~keep] == 0).all()) and not bool(torch.isfinite(y[keep]).any())
    assert norms.dropout(x, 0.3, training=False) is x
    assert torch.equal(norms.dropout(x, 0.3, x, training=False), x + x)


def test_dropout_behind_four_gigabytes():
    """Element offsets past 2^32 (fp16: 8.6 GB in, 8.6 GB out): the last rows against the oracle, rows behind none."""
    from t5vqvae_amd import ops
    n, d, p = (1 << 16) + 40, 1 << 16, 0.1
    x = torch.zeros(n, d, dtype=F16, device="cuda")
    x[-3:] = 1.0
    x[0] = 2.0
    y, _ = ops.dropout_add(x, p, None, ticket())
    for first, count in ((n - 3, 3), (0, 1)):
        keep = no.keep_mask(count, d, p, TICKET, 0, first_row=first)
        want = torch.where(keep, (x[first:first + count].float().cpu() * np.float32(no.scale_of(p))), torch.zeros(())).half()
        assert torch.equal(y[first:first + count].cpu(), want)
    assert float(y[1:-3].abs().max()) == 0.0


# ---- norms, forward ---------------------------------------------------------------------------------------------------
SHAPES = [(1, 1), (1, 768), (5, 3), (37, 64), (30, 130), (45, 771), (64, 1024), (9, 2048), (7, 2051), (3, 4096), (2, 8200),
          (1, 20001), (2880, 768), (33, 190), (50, 256), (10, 300), (21, 513)]


@pytest.mark.parametrize("n,d", SHAPES)
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("dtype,out,wdtype", [(F32, F32, F32), (BF16, BF16, F32), (BF16, F32, BF16), (F16, F16, F16),
                                              (F16, F32, F32)])
def test_norm_forward(n, d, kind, dtype, out, wdtype):
    from t5vqvae_amd import ops
    h = rows(n, d, 11, dtype, 3.0, 0.7)
    w, b = rows(1, d, 12, wdtype)[0], (rows(1, d, 13, wdtype)[0] if kind == "layer" else None)
    for p in (0.0, 0.1):
        got, total, stats, xx, drawn = ops.norm_forward(h.cuda(), w.cuda(), None if b is None else b.cuda(), kind=kind, eps=EPS,
                                                        p=p, ticket=ticket(), out_dtype=out)
        assert got.dtype == out and total is None and xx is None and drawn is None
        keep = no.keep_mask(n, d, p, TICKET, 1)
        check_forward(got, h, w, b, kind, keep, p, out)
        mean, r = no.stats(h.double(), kind, EPS)
        c = chain(d)
        check(stats[:, :1], mean, (c + 1) * U * h.double().abs().mean(1, keepdim=True), "mean")
        # with a single column (h - mean) is rounding alone, far below eps
        check(stats[:, 1:], r, (c / 2 + 8) * U * r, "r")


@pytest.mark.parametrize("n,d", SHAPES)
@pytest.mark.parametrize("hidden,branch,out,wdtype,kind", [
    (F32, F32, F32, F32, "rms"), (F32, BF16, F32, F32, "layer"), (F32, F16, F32, F32, "rms"), (BF16, BF16, BF16, BF16, "layer"),
    (BF16, BF16, F32, F32, "rms"), (F16, F16, F16, F32, "layer"), (F16, F16, F32, F16, "rms")])
def test_add_norm_forward_and_its_parts(n, d, hidden, branch, out, wdtype, kind):
    """sum and out against the oracle, and bit for bit what the two operators in turn give from the same ticket."""
    from t5vqvae_amd import ops
    h, br = rows(n, d, 21, hidden, 3.0, 0.7), rows(n, d, 22, branch)
    w, b = rows(1, d, 23, wdtype)[0], rows(1, d, 24, wdtype)[0]
    p0, p1 = 0.2, 0.1
    got, total, stats, _, _ = ops.norm_forward(h.cuda(), w.cuda(), b.cuda(), kind=kind, eps=EPS, branch=br.cuda(), branch_p=p0,
                                               p=p1, ticket=ticket(), out_dtype=out)
    keep0, keep1 = no.keep_mask(n, d, p0, TICKET, 0), no.keep_mask(n, d, p1, TICKET, 1)
    dropped = no.drop(br.double(), keep0, p0)
    want = h.double() + dropped
    off = 3 * U * (h.double().abs() + dropped.abs())
    check(total, want, half_step(hidden) * (want.abs() + off) + off + tiny(hidden), "sum")
    check_forward(got, total, w, b, kind, keep1, p1, out)
    alone, _ = ops.dropout_add(br.cuda(), p0, h.cuda(), ticket())
    assert torch.equal(alone, total)
    again, _, stats2, _, _ = ops.norm_forward(alone, w.cuda(), b.cuda(), kind=kind, eps=EPS, p=p1, ticket=ticket(), out_dtype=out)
    assert torch.equal(again, got) and torch.equal(stats2, stats)
    plain, total0, _, _, _ = ops.norm_forward(h.cuda(), w.cuda(), b.cuda(), kind=kind, eps=EPS, branch=br.cuda(), out_dtype=out)
    assert torch.equal(total0, ops.dropout_add(br.cuda(), 0.0, h.cuda())[0])
    check_forward(plain, total0, w, b, kind, None, 0.0, out)


def test_norm_of_hard_rows():
    """Constant rows, rows far from zero, rows of one huge element, rows with NaN or infinity beside good ones."""
    from t5vqvae_amd import ops
    d = 768
    h = rows(8, d, 31)
    h[0] = 5.0                                             # variance 0: eps alone
    h[1] = h[1] + 1000.0                                   # mean large against the deviation
    h[2] = 0.0
    h[3, 7] = 1e15
    h[4] = h[4] * 1e-18                                    # squares below the smallest normal number
    w, b = rows(1, d, 32)[0], rows(1, d, 33)[0]
    for kind in ("layer", "rms"):
        got = ops.norm_forward(h.cuda(), w.cuda(), b.cuda(), kind=kind, eps=EPS)[0]
        check_forward(got, h, w, b, kind, None, 0.0, F32)
    for bad in (float("nan"), float("inf")):
        k = h.clone()
        k[5, 100] = bad
        for kind in ("layer", "rms"):
            got = ops.norm_forward(k.cuda(), w.cuda(), b.cuda(), kind=kind, eps=EPS)[0].cpu()
            assert bool(torch.isnan(got[5]).any())
            good = [0, 1, 2, 3, 4, 6, 7]
            check_forward(got[good], h[good], w, b, kind, None, 0.0, F32)


def test_norm_behind_four_gigabytes():
    from t5vqvae_amd import ops
    n, d = (1 << 21) + 5, 2048                            # fp16: 8.6 GB of rows
    h = torch.zeros(n, d, dtype=F16, device="cuda")
    tail = rows(3, d, 41, F16)
    h[-3:] = tail.cuda()
    w = rows(1, d, 42)[0]
    out, _, stats, _, _ = ops.norm_forward(h, w.cuda(), None, kind="rms", eps=EPS, p=0.1, ticket=ticket())
    check_forward(out[-3:], tail, w, None, "rms", no.keep_mask(3, d, 0.1, TICKET, 1, first_row=n - 3), 0.1, F16)
    g = torch.zeros_like(h)
    gt = rows(3, d, 43, F16)
    g[-3:] = gt.cuda()
    gh, _, gw, _ = ops.norm_backward(g, None, h, w.cuda(), stats, kind="rms", p=0.1, ticket=ticket(), want_bias=False)
    check_backward((gh[-3:], None, gw, None), gt, tail, w, "rms", no.keep_mask(3, d, 0.1, TICKET, 1, first_row=n - 3), 0.1)
    assert float(gh[:-3].abs().max()) == 0.0


# ---- backward -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,d", SHAPES)
@pytest.mark.parametrize("dtype,out,wdtype,kind", [(F32, F32, F32, "layer"), (F32, F32, F32, "rms"), (BF16, BF16, F32, "layer"),
                                                   (BF16, F32, BF16, "rms"), (F16, F16, F16, "layer"), (F16, F32, F32, "rms")])
def test_norm_backward(n, d, dtype, out, wdtype, kind):
    from t5vqvae_amd import ops
    h, g, w = rows(n, d, 51, dtype, 3.0, 0.7), rows(n, d, 52, out), rows(1, d, 53, wdtype)[0]
    stats = ops.norm_forward(h.cuda(), w.cuda(), None, kind=kind, eps=EPS)[2]
    for p in (0.0, 0.1):
        keep = no.keep_mask(n, d, p, TICKET, 1)
        got = ops.norm_backward(g.cuda(), None, h.cuda(), w.cuda(), stats, kind=kind, p=p, ticket=ticket() if p else None)
        assert got[0].dtype == dtype and got[1] is None and got[2].dtype == wdtype and got[3].dtype == wdtype
        check_backward(got, g, h, w, kind, keep, p)
        again = ops.norm_backward(g.cuda(), None, h.cuda(), w.cuda(), stats, kind=kind, p=p, ticket=ticket() if p else None)
        assert all(torch.equal(x, y) for x, y in zip(got, again) if x is not None)      # no atomics
        only = ops.norm_backward(g.cuda(), None, h.cuda(), w.cuda(), stats, kind=kind, p=p, ticket=ticket() if p else None,
                                 want_weight=False, want_bias=False)
        assert torch.equal(only[0], got[0]) and only[2] is None and only[3] is None


@pytest.mark.parametrize("n,d", SHAPES)
@pytest.mark.parametrize("hidden,branch,out,wdtype,kind", [
    (F32, F32, F32, F32, "rms"), (F32, BF16, F32, F32, "layer"), (F32, F16, F32, F32, "rms"), (BF16, BF16, BF16, BF16, "layer"),
    (BF16, BF16, F32, F32, "rms"), (F16, F16, F16, F32, "layer"), (F16, F16, F32, F16, "rms")])
def test_add_norm_backward(n, d, hidden, branch, out, wdtype, kind):
    from t5vqvae_amd import ops
    h, g, gs, w = rows(n, d, 61, hidden, 3.0, 0.7), rows(n, d, 62, out), rows(n, d, 63, hidden), rows(1, d, 64, wdtype)[0]
    stats = ops.norm_forward(h.cuda(), w.cuda(), None, kind=kind, eps=EPS)[2]
    p0, p1 = 0.2, 0.1
    keep0, keep1 = no.keep_mask(n, d, p0, TICKET, 0), no.keep_mask(n, d, p1, TICKET, 1)
    for s in (gs, None):
        got = ops.norm_backward(g.cuda(), None if s is None else s.cuda(), h.cuda(), w.cuda(), stats, kind=kind, branch_p=p0,
                                p=p1, ticket=ticket(), branch_dtype=branch)
        assert got[1].dtype == branch
        check_backward(got, g, h, w, kind, keep1, p1, s, keep0, p0)


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_gradients_are_the_slopes_of_the_forward(kind):
    """Directional differences of the oracle's forward in 64 bits, along directions in the input and in the parameters,
    against the kernel's gradients: the difference quotient is off by O(step^2), far below the fp32 gradients' bounds."""
    from t5vqvae_amd import norms
    n, d, p0, p1 = 6, 90, 0.2, 0.3
    h, br, w, b = rows(n, d, 71, F32, 2.0, 0.5), rows(n, d, 72), rows(1, d, 73)[0] + 1.0, rows(1, d, 74)[0]
    g, gs = rows(n, d, 75), rows(n, d, 76)
    leaves = [t.cuda().requires_grad_(True) for t in (h, br, w, b)]
    out, total = norms.add_norm(*leaves, kind=kind, eps=EPS, branch_p=p0, p=p1, ticket=ticket())
    grads = torch.autograd.grad((out, total), leaves, (g.cuda(), gs.cuda()))
    keep0, keep1 = no.keep_mask(n, d, p0, TICKET, 0), no.keep_mask(n, d, p1, TICKET, 1)

    def f(h, br, w, b):
        s = h + no.drop(br, keep0, p0)
        return float((no.norm(s, w, b, kind, EPS, keep1, p1) * g.double()).sum() + (s * gs.double()).sum())
    x = [t.double() for t in (h, br, w, b)]
    step = 1e-4
    for i in range(4):
        v = rows(*(x[i].shape if x[i].dim() == 2 else (1, d)), 80 + i).double().reshape(x[i].shape)
        up, down = ([t + (s * v if j == i else 0) for j, t in enumerate(x)] for s in (step, -step))
        slope = (f(*up) - f(*down)) / (2 * step)
        got = float((grads[i].cpu().double() * v).sum())
        size = float((grads[i].cpu().double() * v).abs().sum())
        # each gradient element is off by (C + 16) u times a few of its terms at most; the quotient by about step^2
        assert abs(got - slope) <= 1e-5 * size, (i, got, slope)


@pytest.mark.parametrize("n,d", [(5, 4097), (3, 5120), (9, 6144), (4, 6145), (300, 8192), (5, 8193), (4, 10241), (600, 12288),
                                 (5, 12289), (7, 16383), (6, 16384), (3, 16385), (70001, 3), (1030, 2), (300, 1)])
@pytest.mark.parametrize("hidden,branch,out,wdtype,kind", [
    (F32, F32, F32, F32, "layer"), (F32, BF16, F32, F32, "rms"), (BF16, BF16, BF16, BF16, "layer"), (F16, F16, F32, F32, "rms")])
def test_long_and_short_rows(n, d, hidden, branch, out, wdtype, kind):
    """Where a row's lanes and chunks change, up to where registers do not hold it, and rows of less than one group: both
    norms forward and backward."""
    from t5vqvae_amd import ops
    p, bp = 0.2, 0.3
    h, br, w, b = rows(n, d, 401, hidden), rows(n, d, 402, branch), rows(1, d, 403, wdtype)[0], rows(1, d, 404, wdtype)[0]
    g, gs = rows(n, d, 405, out).cuda(), rows(n, d, 406, hidden).cuda()
    keep0, keep1 = no.keep_mask(n, d, bp, TICKET, 0), no.keep_mask(n, d, p, TICKET, 1)
    y, total, stats, _, _ = ops.norm_forward(h.cuda(), w.cuda(), b.cuda(), kind=kind, eps=EPS, branch=br.cuda(), branch_p=bp,
                                             p=p, ticket=ticket(), out_dtype=out)
    assert torch.equal(total, ops.dropout_add(br.cuda(), bp, h.cuda(), ticket())[0])
    check_forward(y, total, w, b, kind, keep1, p, out)
    plain = ops.norm_forward(total, w.cuda(), b.cuda(), kind=kind, eps=EPS, p=p, ticket=ticket(), out_dtype=out)
    assert torch.equal(plain[0], y) and torch.equal(plain[2], stats)
    got = ops.norm_backward(g, gs, total, w.cuda(), stats, kind=kind, branch_p=bp, p=p, ticket=ticket(), branch_dtype=branch)
    check_backward(got, g, total, w, kind, keep1, p, gs, keep0, bp)
    got = ops.norm_backward(g, None, total, w.cuda(), stats, kind=kind, p=p, ticket=ticket())
    check_backward(got, g, total, w, kind, keep1, p)


@pytest.mark.parametrize("n,d,dtype", [(65541, 768, F32), (131083, 768, BF16), (800005, 64, F32), (50003, 1024, F16),
                                       (25003, 2048, F32), (10003, 6144, F32), (7003, 8192, F32)])
def test_large_calls_equal_their_parts(n, d, dtype):
    """Calls that go past the caches (192 MB and more) against the same rows in small calls, bit for bit, and the oracle's
    masks on the last rows; the parameters' gradients against float64 sums."""
    from t5vqvae_amd import ops
    g = torch.Generator(device="cuda").manual_seed(n)
    h, br, go, gs = (torch.randn(n, d, generator=g, device="cuda").to(dtype) for _ in range(4))
    w, b = torch.randn(d, generator=g, device="cuda"), torch.randn(d, generator=g, device="cuda")
    last = [(0, 37), (n // 2, 61), (n - 29, 29)]
    out, total, stats, _, _ = ops.norm_forward(h, w, b, kind="layer", eps=EPS, branch=br)
    got = ops.norm_backward(go, gs, total, w, stats, kind="layer", branch_dtype=dtype)
    res = ops.dropout_add(br, 0.0, h)[0]
    assert torch.equal(res, total)
    for first, count in last:
        part = slice(first, first + count)
        o, t, s, _, _ = ops.norm_forward(h[part], w, b, kind="layer", eps=EPS, branch=br[part])
        assert torch.equal(o, out[part]) and torch.equal(t, total[part]) and torch.equal(s, stats[part])
        x = ops.norm_backward(go[part], gs[part], t, w, s, kind="layer", branch_dtype=dtype)
        assert torch.equal(x[0], got[0][part]) and torch.equal(x[1], got[1][part])
    unit = (total.double() - stats[:, :1].double()) * stats[:, 1:].double()
    # n is off by 2 u |n| (a subtraction and a product); a column's chain: a wave's rows (n / 2048 at least three), 16 waves,
    # the tree over up to 512 slices
    chain_rows = n / 2048 + 64
    for grad, terms in ((got[2], go.double() * unit), (got[3], go.double())):
        want, size = terms.sum(0), terms.abs().sum(0)
        assert bool(((grad.double() - want).abs() <= (chain_rows + 4) * U * size).all())
    del unit, terms, res, total, got, out
    p = 0.25
    y = ops.dropout_add(torch.ones_like(h), p, None, ticket())[0]
    o, t, s, _, _ = ops.norm_forward(h, w, b, kind="rms", eps=EPS, branch=br, branch_p=p, p=p, ticket=ticket())
    gh, gb, _, _ = ops.norm_backward(go, gs, t, w, s, kind="rms", branch_p=p, p=p, ticket=ticket(), branch_dtype=dtype)
    for first, count in last:
        keep0 = no.keep_mask(count, d, p, TICKET, 0, first_row=first)
        keep1 = no.keep_mask(count, d, p, TICKET, 1, first_row=first)
        part = slice(first, first + count)
        assert torch.equal(y[part].cpu() != 0, keep0)
        check_forward(o[part], t[part], w, b, "rms", keep1, p, dtype)
        check_backward((gh[part], gb[part], None, None), go[part], t[part], w, "rms", keep1, p, gs[part], keep0, p)


@pytest.mark.parametrize("n,d", [(37, 768), (50, 64), (9, 2048), (3, 20000), (40, 2), (70000, 768)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_views_that_start_at_any_element(n, d, dtype):
    """Dense views one element behind an allocation's start (and parameters likewise) give what aligned copies give."""
    from t5vqvae_amd import ops

    def views(m, seed):
        t = torch.randn(m * d + 1, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)[1:]
        t = t.view(m, d) if m > 1 else t
        return t, t.clone()
    h, br, g, gs, w, b = (views(m, 300 + i) for i, m in enumerate((n, n, n, n, 1, 1)))
    res = []
    for k in range(2):
        y = ops.dropout_add(br[k], 0.3, h[k], ticket())[0]
        only = ops.dropout_add(br[k], 0.3, None, ticket())[0]
        out, total, stats, _, _ = ops.norm_forward(h[k], w[k], b[k], branch=br[k], branch_p=0.3, p=0.1, ticket=ticket())
        res.append((y, only, out, total, stats) + tuple(
            ops.norm_backward(g[k], gs[k], h[k], w[k], stats, branch_p=0.3, p=0.1, ticket=ticket(), branch_dtype=dtype)))
    assert h[0].data_ptr() % 16 and not h[1].data_ptr() % 16
    for x, y in zip(*res):
        assert torch.equal(x, y)


# ---- outputs for the searches --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,d", [(1, 64), (45, 768), (130, 2048), (33, 100), (257, 1024), (64, 1536), (31, 192), (50, 256), (7, 140),
                                 (9, 300), (12, 512), (5, 640)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_row_norms_and_image_are_those_of_the_searches(n, d, dtype):
    from t5vqvae_amd import ops
    h, br, w, b = rows(n, d, 91, dtype, 2.0), rows(n, d, 92, dtype), rows(1, d, 93)[0], rows(1, d, 94)[0]
    img = ops.token_image(n, d, "cuda").zero_()
    out, total, _, xx, _ = ops.norm_forward(h.cuda(), w.cuda(), b.cuda(), kind="layer", eps=EPS, branch=br.cuda(), branch_p=0.1,
                                            p=0.1, ticket=ticket(), out_dtype=F32, want_row_norms=True, token_image=img)
    bare = ops.norm_forward(total, w.cuda(), b.cuda(), kind="layer", eps=EPS, p=0.1, ticket=ticket(), out_dtype=F32)[0]
    assert torch.equal(out, bare)
    assert torch.equal(xx, ops.row_sqnorms(out, None)[0])
    if d % 64 == 0:
        codes = rows(500, d, 95).cuda()
        _, ee = ops.row_sqnorms(None, codes)
        keys = ops.dist_argmin_filtered(out, codes, xx, ee, token_image=img)
        assert torch.equal(keys, ops.dist_argmin_filtered(out, codes, xx, ee))
        assert torch.equal(keys, ops.dist_argmin(out, codes, xx, ee))


# ---- the functions and modules ----------------------------------------------------------------------------------------------
def test_gradients_reach_what_asks_for_them():
    """Every subset of inputs that require a gradient gives the same values; outputs that nobody used; gradients that are
    not contiguous; inputs that are views of other shapes."""
    from t5vqvae_amd import norms
    shape, p = (3, 7, 100), 0.2
    base = [rows(21, 100, 101).view(shape), rows(21, 100, 102).view(shape), rows(1, 100, 103)[0], rows(1, 100, 104)[0]]
    g, gs = rows(21, 100, 105).view(shape).cuda(), rows(21, 100, 106).view(shape).cuda()

    def run(mask, use_out=True, use_sum=True, strided=False):
        x = [t.cuda().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate(base)]
        out, total = norms.add_norm(*x, kind="layer", eps=EPS, branch_p=p, p=p, ticket=ticket())
        assert out.shape == total.shape == shape
        loss = 0
        if strided:
            loss = loss + (out.transpose(0, 1) * g.transpose(0, 1).contiguous()).sum() + (total.flip(0) * gs.flip(0)).sum()
        else:
            loss = (loss + (out * g).sum()) if use_out else loss
            loss = (loss + (total * gs).sum()) if use_sum else loss
        loss.backward()
        return [t.grad for t in x]
    full = run(15)
    for mask in range(1, 15):
        got = run(mask, use_sum=bool(mask & 3))                # the sum does not depend on the parameters
        for i in range(4):
            assert (got[i] is None) == (not mask >> i & 1)
            if got[i] is not None:
                assert torch.equal(got[i], full[i]), (mask, i)
    for a, b in zip(run(15, strided=True), full):
        assert torch.equal(a, b)
    only_sum = run(15, use_out=False)
    assert only_sum[2] is None and only_sum[3] is None
    keep = no.keep_mask(21, 100, p, TICKET, 0).view(shape)
    assert torch.equal(only_sum[0], gs) and bool((only_sum[1].cpu()[~keep] == 0).all())
    only_out = run(15, use_sum=False)
    assert torch.equal(only_out[2], full[2]) and not torch.equal(only_out[0], full[0])


def test_broadcast_and_shared_inputs():
    from t5vqvae_amd import norms
    row = rows(1, 64, 111).cuda().requires_grad_(True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    out, total = norms.add_norm(row.expand(9, 64), row.expand(9, 64), w, kind="rms", eps=EPS)
    (out.sum() + total.sum()).backward()
    one = row.detach().clone().requires_grad_(True)
    o1, t1 = norms.add_norm(one, one, w.detach(), kind="rms", eps=EPS)
    (o1.sum() + t1.sum()).backward()
    assert torch.allclose(row.grad, 9 * one.grad, rtol=1e-5, atol=1e-5)
    assert w.grad.shape == (64,)


def test_empty_inputs():
    from t5vqvae_amd import norms, ops
    x = torch.empty(0, 5, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    b = torch.ones(16, device="cuda", requires_grad=True)
    out, total = norms.add_norm(x, x, w, b, branch_p=0.1, p=0.1)
    assert out.shape == total.shape == (0, 5, 16)
    (out.sum() + total.sum()).backward()
    assert x.grad.shape == x.shape and bool((w.grad == 0).all()) and bool((b.grad == 0).all())
    y = norms.dropout(x, 0.5, x)
    assert y.shape == x.shape
    y.sum().backward()
    assert ops.norm_forward(torch.empty(0, 16, device="cuda"), w.detach(), want_row_norms=True)[3].shape == (0,)


def test_refusals_on_the_device():
    from t5vqvae_amd import norms, ops
    x, w = torch.zeros(4, 16, device="cuda"), torch.ones(16, device="cuda")
    t = ticket()
    st = torch.zeros(4, 2, device="cuda")
    for call in (lambda: ops.dropout_add(x.double(), 0.1), lambda: ops.dropout_add(x, 1.5), lambda: ops.dropout_add(x[:, ::2], 0.1),
                 lambda: ops.dropout_add(x.bfloat16(), 0.1, x.half()), lambda: ops.dropout_add(x, 0.1, x[:2]),
                 lambda: ops.dropout_add(x, 0.1, None, t[:1]), lambda: ops.dropout_add(x, 0.1, None, t.int()),
                 lambda: ops.dropout_add(x, 0.1, None, t.cpu()), lambda: ops.dropout_backward(x, 0.1, None),
                 lambda: ops.norm_forward(x, w.double()), lambda: ops.norm_forward(x, w[:8]), lambda: ops.norm_forward(x, w.cpu()),
                 lambda: ops.norm_forward(x, w, w.half()), lambda: ops.norm_forward(x, w, out_dtype=BF16),
                 lambda: ops.norm_forward(x.bfloat16(), w, branch=x), lambda: ops.norm_forward(x, w, kind="group"),
                 lambda: ops.norm_forward(x, w, eps=-1.0), lambda: ops.norm_forward(x.bfloat16(), w, want_row_norms=True),
                 lambda: ops.norm_forward(x, w, token_image=torch.empty(8, dtype=torch.uint8, device="cuda")),
                 lambda: ops.norm_backward(x, None, x, w, st, p=0.1), lambda: ops.norm_backward(x, x.half(), x, w, st),
                 lambda: ops.norm_backward(x, None, x, w, st[:2]), lambda: ops.norm_backward(x.half(), None, x, w, st),
                 lambda: ops.norm_backward(x, None, x, w, st, branch_p=0.1, branch_dtype=F32),
                 lambda: norms.add_norm(x, x[:2], w), lambda: norms.norm(torch.zeros(4, 0, device="cuda"), w),
                 lambda: norms.norm(torch.zeros((), device="cuda"), w)):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(TypeError):
        norms.dropout([1.0])
    y = norms.norm(x.requires_grad_(True), w)
    (gx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gx.sum(), x)
    import torch.autograd.forward_ad as fwd
    plain = torch.zeros(4, 16, device="cuda")
    with fwd.dual_level():
        dual = fwd.make_dual(plain, torch.ones_like(plain))
        for call in (lambda: norms.dropout(dual, 0.1), lambda: norms.dropout(plain, 0.1, dual), lambda: norms.norm(dual, w),
                     lambda: norms.norm(plain, fwd.make_dual(w, w)), lambda: norms.add_norm(plain, dual, w),
                     lambda: torch.autograd.grad(y, x, dual, retain_graph=True)):
            with pytest.raises(RuntimeError):
                call()
    for kind in (2, -1, 1 << 32):
        with pytest.raises(RuntimeError):
            torch.ops.t5vq.norm(plain, None, w, None, kind, EPS, 0.0, 0.0)
        with pytest.raises(RuntimeError):
            torch.ops.t5vq.norm_backward(plain, None, plain, w, st, kind, 0.0, 0.0, None, None, True, True)


# ---- random numbers ---------------------------------------------------------------------------------------------------------
def test_torch_generator_drives_the_masks():
    from t5vqvae_amd import norms, ops
    x = torch.ones(64, 96, device="cuda")
    torch.manual_seed(5)
    y1, t1 = ops.dropout_add(x, 0.5)
    y2, t2 = ops.dropout_add(x, 0.5)
    assert t1.tolist()[0] == 5 and t2.tolist() == [5, t1.tolist()[1] + 8] and not torch.equal(y1, y2)
    assert torch.equal(y1.cpu() != 0, no.keep_mask(64, 96, 0.5, t1.tolist(), 0))
    torch.manual_seed(5)
    assert torch.equal(ops.dropout_add(x, 0.5)[0], y1)
    assert torch.equal(ops.dropout_add(x, 0.5, None, t2)[0], y2)
    state = torch.cuda.get_rng_state()
    ops.dropout_add(x, 0.0)                                       # nothing drawn: the generator stays
    ops.dropout_add(x, 0.5, None, t1)
    assert torch.equal(torch.cuda.get_rng_state(), state)
    # the two sites of one call, and torch's own dropout in between, share nothing
    torch.manual_seed(5)
    ones = torch.ones(64, 96, device="cuda")
    zeros, w0, b1 = torch.zeros_like(ones), torch.zeros(96, device="cuda"), torch.ones(96, device="cuda")
    out, total = norms.add_norm(zeros, ones, w0, b1, branch_p=0.5, p=0.5)
    agree = float(((out != 0) == (total != 0)).float().mean())
    assert 0.45 < agree < 0.55                                    # 6144 fair coins: five standard deviations are 0.032
    # activation checkpointing restores the generator, so the recomputed masks are the first ones
    from torch.utils.checkpoint import checkpoint
    g = rows(64, 96, 121).cuda()
    grads = []
    for recompute in (False, True):
        torch.manual_seed(9)
        h = rows(64, 96, 122).cuda().requires_grad_(True)
        f = (lambda t: norms.norm(norms.dropout(t, 0.3), b1, p=0.4))
        y = checkpoint(f, h, use_reentrant=False) if recompute else f(h)
        (y * g).sum().backward()
        grads.append(h.grad)
    assert torch.equal(*grads)


def test_masks_are_fair_coins():
    """Counts of kept elements over rows, columns and sites stay within six standard deviations."""
    from t5vqvae_amd import ops
    n, d, p = 4096, 512, 0.1
    torch.manual_seed(11)
    x = torch.ones(n, d, device="cuda")
    a, b = (ops.dropout_add(x, p)[0] != 0 for _ in range(2))
    q = no.keep_count(p) / 65536.0
    for m in (a, b):
        assert abs(float(m.double().mean()) - q) <= 6 * (q * (1 - q) / (n * d)) ** 0.5
        assert float((m.double().mean(0) - q).abs().max()) <= 6 * (q * (1 - q) / n) ** 0.5
        assert float((m.double().mean(1) - q).abs().max()) <= 6 * (q * (1 - q) / d) ** 0.5
    both = float((a & b).double().mean())
    assert abs(both - q * q) <= 6 * (q * q * (1 - q * q) / (n * d)) ** 0.5


def test_captured_steps_draw_anew_and_match_their_tickets():
    """A whole step (forward and backward) in a graph, replayed with the program's own eager work between the replays:
    every replay's outputs and gradients equal the eager ones of the ticket it drew, and no two replays share a mask."""
    from t5vqvae_amd import ops
    n, d, p = 300, 768, 0.1
    h, br, w, b, g, gs = (rows(n, d, 131).cuda(), rows(n, d, 132).cuda(), rows(1, d, 133)[0].cuda(), rows(1, d, 134)[0].cuda(),
                          rows(n, d, 135).cuda(), rows(n, d, 136).cuda())

    def step(t=None):
        out, total, stats, _, drawn = ops.norm_forward(h, w, b, branch=br, branch_p=p, p=p, ticket=t)
        t = drawn if t is None else t
        return (t, out, total) + tuple(ops.norm_backward(g, gs, total, w, stats, branch_p=p, p=p, ticket=t, branch_dtype=F32))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    seen = set()
    for k in range(4):
        h.copy_(rows(n, d, 140 + k))
        graph.replay()
        torch.cuda.synchronize()
        drawn = tuple(res[0].tolist())
        assert drawn not in seen
        seen.add(drawn)
        eager = step(res[0].clone())
        for x, y in zip(res[1:], eager[1:]):
            assert torch.equal(x, y)
        assert torch.equal(res[2].cpu(), (h.cpu() + torch.where(no.keep_mask(n, d, p, drawn, 0),
                                                                br.cpu() * np.float32(no.scale_of(p)), torch.zeros(()))))


def test_first_call_of_a_kernel_inside_a_capture():
    """No warm-up: a kernel's first call (which asks how many workgroups the card holds) may be a captured one."""
    from t5vqvae_amd import ops
    h, g, w = rows(40, 5000, 201, F16).cuda(), rows(40, 5000, 202, F16).cuda(), rows(1, 5000, 203, F16)[0].cuda()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _, stats, _, _ = ops.norm_forward(h, w, kind="rms", eps=EPS)
        back = ops.norm_backward(g, None, h, w, stats, kind="rms", want_bias=False)
        drop = ops.dropout_add(h, 0.5, None, None)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        check_forward(out, h, w, None, "rms", None, 0.0, F16)
        check_backward(back, g, h, w, "rms", None, 0.0)
        keep = no.keep_mask(40, 5000, 0.5, drop[1].tolist(), 0)
        assert torch.equal(drop[0].cpu(), torch.where(keep, h.cpu() * 2, torch.zeros((), dtype=F16)))


def test_captured_autograd_steps_follow_their_ticket():
    """Forward and backward through autograd in one graph; the ticket's words change between replays."""
    from t5vqvae_amd import norms
    h, br, g, gs = (rows(200, 768, 211 + k).cuda() for k in range(4))
    w, b = rows(1, 768, 215)[0].cuda(), rows(1, 768, 216)[0].cuda()
    words = ticket()

    def step():
        x = [t.detach().requires_grad_(True) for t in (h, br, w, b)]
        out, total = norms.add_norm(*x, eps=EPS, branch_p=0.1, p=0.1, ticket=words)
        y = norms.dropout(out, 0.2, total, ticket=words)
        return (y.detach(),) + torch.autograd.grad((y, total), x, (g, gs))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    last = None
    for k in range(4):
        words.copy_(torch.tensor([77 + k, 8 * k]))
        graph.replay()
        torch.cuda.synchronize()
        assert last is None or not torch.equal(res[0], last)
        last = res[0].clone()
        for x, y in zip(res, step()):
            assert torch.equal(x, y)


def test_captured_backward_beside_a_living_eager_graph_is_refused():
    """Leaves whose accumulators an eager graph on the default stream keeps: the capture's backward raises before it records
    anything; once the eager graph is gone the same capture works."""
    from t5vqvae_amd import norms
    h, g = rows(50, 64, 221).cuda(), rows(50, 64, 222).cuda()
    w = rows(1, 64, 223)[0].cuda().requires_grad_(True)
    eager = norms.norm(h, w, eps=EPS)
    (want,) = torch.autograd.grad(eager, w, g, retain_graph=True)
    x, t = h.clone().requires_grad_(True), ticket()
    dropped = norms.dropout(x, 0.5, ticket=t)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = h * 2.0                                           # the graph is not empty
        out = norms.norm(h, w, eps=EPS)
        with pytest.raises(RuntimeError, match="eager graph"):
            torch.autograd.grad(out, w, g)
        with pytest.raises(RuntimeError, match="eager graph"):
            norms.dropout(x, 0.5, ticket=t).backward(g)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, h * 2.0) and x.grad is None and w.grad is None
    del eager, dropped, out
    again = torch.cuda.CUDAGraph()
    with torch.cuda.graph(again):
        (got,) = torch.autograd.grad(norms.norm(h, w, eps=EPS), w, g)
    for _ in range(3):
        again.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_two_graphs_of_the_same_operators_replay_beside_each_other():
    """Two graphs captured from the same call, replayed in turn on two streams: no shared workspace."""
    from t5vqvae_amd import ops
    n, d = 2880, 768
    w = rows(1, d, 151)[0].cuda()
    sets = []
    for k in range(2):
        h, g = rows(n, d, 152 + k).cuda(), rows(n, d, 154 + k).cuda()
        stats = ops.norm_forward(h, w)[2]
        eager = ops.norm_backward(g, None, h, w, stats)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = ops.norm_backward(g, None, h, w, stats)
        sets.append((graph, res, eager, (h, g, stats)))         # a graph reads its inputs where they were: they live as long
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (graph, *_) in zip(streams, sets):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for _, res, eager, _ in sets:
        for x, y in zip(res, eager):
            assert (x is None and y is None) or torch.equal(x, y)


def test_other_streams():
    from t5vqvae_amd import ops
    h, w = rows(2880, 768, 161).cuda(), rows(1, 768, 162)[0].cuda()
    want = ops.norm_forward(h, w, kind="rms", p=0.1, ticket=ticket())[0]
    t = ticket()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        h2 = h * 1.0
        got = ops.norm_forward(h2, w, kind="rms", p=0.1, ticket=t)[0]
    side.synchronize()
    assert torch.equal(got, want)


# ---- on the way to the quantizer ------------------------------------------------------------------------------------------
def make_vq(k, d, seed=171):
    from t5vqvae_amd import VectorQuantizerEMA
    m = VectorQuantizerEMA(k, d, 0.25, decay=0.99).cuda()
    with torch.no_grad():
        m._embedding.weight.copy_(rows(k, d, seed))
        m._ema_w.copy_(rows(k, d, seed + 1))
    m.encodings = "indices"
    return m


def test_tail_with_a_counter_equals_the_tail_with_that_mask_stored():
    from t5vqvae_amd import norms
    from t5vqvae_amd.encoder_tail import EncoderTailVQ
    b, s, d, k = 8, 45, 768, 1000
    a, c = EncoderTailVQ(make_vq(k, d), d, dropout="counter").cuda(), EncoderTailVQ(make_vq(k, d), d).cuda()
    gamma = rows(1, d, 173)[0].abs() + 0.5
    with torch.no_grad():
        a.weight.copy_(gamma), c.weight.copy_(gamma)
    h, gq = rows(b * s, d, 174, F32, 2.0).view(b, s, d), rows(b * s, d, 175).view(b, s, d).cuda()
    keep = no.keep_mask(b * s, d, 0.1, TICKET, 1).view(b, s, d).to(torch.uint8).cuda()
    c.dropout_rate = 1.0 - no.keep_count(0.1) / 65536.0          # the stored form scales by the p it is told
    ha, hc = h.cuda().requires_grad_(True), h.cuda().requires_grad_(True)
    la, qa, pa, ia = a(ha, ticket=ticket())
    lc, qc, pc, ic = c(hc, keep_mask=keep)
    mism = int((ia != ic).sum())
    assert mism <= 2                                             # x differs by roundings between the two: near-ties only
    (la * 1.3 + (qa * gq).sum()).backward()
    (lc * 1.3 + (qc * gq).sum()).backward()

    def rel(x, y):
        return float((x.double() - y.double()).norm() / y.double().norm())
    assert rel(la, lc) <= 1e-5
    if mism == 0:
        assert rel(qa, qc) <= 1e-6 and rel(ha.grad, hc.grad) <= 1e-5 and rel(a.weight.grad, c.weight.grad) <= 1e-5
        assert rel(a.vq._embedding.weight, c.vq._embedding.weight) <= 1e-5
    a.eval(), c.eval()
    with torch.no_grad():
        ia, ic = a(h.cuda())[3], c(h.cuda())[3]
    assert int((ia != ic).sum()) <= 2


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sublayer_norm_dropout_and_quantizer_in_one_run(dtype):
    """The last sublayer of an encoder on its way to the quantizer -- dropout and residual sum of one sublayer, then
    EncoderTailVQ(norm="layer") with a branch -- against the same chain made of the single operators: same bits, same
    indices, same gradients."""
    from t5vqvae_amd import norms, ops
    from t5vqvae_amd.encoder_tail import EncoderTailVQ
    b, s, d, k, p = 4, 33, 256, 300, 0.1
    n = b * s
    x0, y0, y1 = (rows(n, d, 180 + i, dtype, 2.0).view(b, s, d) for i in range(3))
    w, bias = rows(1, d, 184)[0] * 0.2 + 1.0, rows(1, d, 185)[0] * 0.2
    gq = rows(n, d, 186).view(b, s, d).cuda()
    t0, t1 = ticket(3, 0), ticket(3, 8)
    tail = EncoderTailVQ(make_vq(k, d), d, dropout_rate=p, norm="layer", dropout="counter").cuda()
    vq = copy.deepcopy(tail.vq)
    with torch.no_grad():
        tail.weight.copy_(w), tail.bias.copy_(bias)
    drop = norms.Dropout(p)
    leaves = [t.cuda().requires_grad_(True) for t in (x0, y0, y1)]
    loss, q, ppl, idx = tail(drop(leaves[1], leaves[0], ticket=t0), branch=leaves[2], ticket=t1)
    (loss + (q * gq).sum()).backward()

    chain = [t.cuda().requires_grad_(True) for t in (x0, y0, y1)]
    wl, bl = w.cuda().requires_grad_(True), bias.cuda().requires_grad_(True)
    h = norms.dropout(chain[1], p, chain[0], ticket=t0)
    h = norms.dropout(chain[2], p, h, ticket=t1)
    x = norms.norm(h, wl, bl, kind="layer", eps=1e-6, p=p, ticket=t1, out_dtype=F32)
    loss2, q2, ppl2, idx2 = vq(x)
    (loss2 + (q2 * gq).sum()).backward()
    assert torch.equal(idx, idx2) and torch.equal(q, q2) and torch.equal(loss, loss2)
    # the chain rounds the gradient of the sum to the stream's type before the branch's dropout scales it; the one pass
    # scales first: one half step for the one pass, two for the chain, in the second branch's gradient
    for u, v, halves in ((leaves[0], chain[0], 0), (leaves[1], chain[1], 0), (leaves[2], chain[2], 0 if dtype == F32 else 3)):
        off = (u.grad.double() - v.grad.double()).abs()
        assert bool((off <= halves * half_step(dtype) * 1.02 * v.grad.double().abs()).all())
    assert torch.equal(tail.weight.grad, wl.grad) and torch.equal(tail.bias.grad, bl.grad)
    vq.eval(), tail.vq.eval()
    torch.manual_seed(1)
    with torch.no_grad():
        out = tail(x0.cuda(), branch=y1.cuda())[1]               # no ticket: torch's generator
    torch.manual_seed(1)
    with torch.no_grad():
        again = tail(x0.cuda(), branch=y1.cuda())[1]
    assert out.shape == (b, s, d) and out.dtype == F32 and torch.equal(out, again)
