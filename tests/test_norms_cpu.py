"""The dropout / norm operators without a GPU: the oracle's own known answers, refusals that come before any launch (C ABI,
extension, modules), and that the oracle's gradients are those of its forward."""
import ctypes
import math

import pytest
import torch

from oracle import norm_oracle as no


def test_oracle_philox_known_answers():
    """Known-answer vectors published with the generator (counter, key -> words)."""
    assert no.philox4x32_10((0, 0, 0, 0), (0, 0)) == (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)
    assert no.philox4x32_10((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0)) == \
        (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)


def test_oracle_draws_are_the_blocks_of_the_generator():
    seed, offset = 0x123456789ABCDEF0, (1 << 40) + 8
    d = no.draws(3, 21, (seed, offset), site=1, first_row=5)
    where = offset // 4 + 1
    for row in range(3):
        for col in range(21):
            w = no.philox4x32_10((where & no.LOW, where >> 32, col // 8, row + 5), (seed & no.LOW, seed >> 32))
            j = col % 8
            assert int(d[row, col]) == (w[j // 2] >> (16 * (j % 2))) & 0xFFFF


@pytest.mark.parametrize("p", [0.0, 2.0 ** -18, 0.1, 0.5, 1.0 / 3, 0.999999, 1.0])
def test_keep_count(p):
    from t5vqvae_amd import _lib, ops
    assert ops.dropout_keep_count(p) == no.keep_count(p) == round((1.0 - p) * 65536)
    lib = _lib.load()
    for bad in (-0.1, 1.1, float("nan"), float("inf")):
        assert lib.t5vq_dropout_keep_count(bad) == -1
        with pytest.raises(RuntimeError, match="p must be in"):
            ops.dropout_keep_count(bad)


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_oracle_gradients_are_those_of_its_forward(kind):
    g = torch.Generator().manual_seed(3)
    n, d, p = 5, 13, 0.3
    h = torch.randn(n, d, generator=g, dtype=torch.float64).requires_grad_(True)
    w = torch.randn(d, generator=g, dtype=torch.float64).requires_grad_(True)
    b = torch.randn(d, generator=g, dtype=torch.float64).requires_grad_(True)
    keep = no.keep_mask(n, d, p, (7, 16), 1)
    go = torch.randn(n, d, generator=g, dtype=torch.float64)
    no.norm(h, w, b, kind, 1e-6, keep, p).backward(go)
    gh, _, gw, gb = no.norm_backward(go, h.detach(), w.detach(), kind, 1e-6, keep, p)
    for got, want in ((gh, h.grad), (gw, w.grad), (gb, b.grad)):
        assert torch.allclose(got, want, rtol=1e-12, atol=1e-12)


def test_c_abi_refuses_bad_calls_before_any_launch():
    from t5vqvae_amd import _lib
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.c_void_p((ctypes.addressof(buf) + 255) // 256 * 256)
    odd, y_, z_ = (ctypes.c_void_p(p.value + k) for k in (1, 512, 1024))
    F32, BF16, F16, LAYER, RMS = 0, 1, 2, 0, 1

    def drop(x=p, xt=F32, res=None, n=4, d=8, prob=0.1, y=y_, yt=F32, sd=None, od=None, to=None):
        return lib.t5vq_dropout_add(x, xt, res, n, d, prob, 1, 0, sd, od, to, y, yt, None)

    for call in (dict(x=None), dict(y=None), dict(xt=3), dict(yt=-1), dict(xt=BF16, yt=F16), dict(n=0), dict(n=1 << 32),
                 dict(d=0), dict(d=(1 << 30) + 1), dict(n=(1 << 32) - 1, d=16), dict(prob=-0.1), dict(prob=1.5),
                 dict(prob=math.nan), dict(x=odd), dict(y=odd), dict(res=odd),
                 dict(y=p), dict(res=y_), dict(sd=z_, to=z_), dict(od=z_, to=z_)):
        assert drop(**call) == 1, call
        assert lib.t5vq_last_error()

    def fwd(h=p, ht=F32, b=None, bt=F32, w=p, bias=None, wt=F32, kind=LAYER, eps=1e-6, n=4, d=8, bp=0.0, prob=0.0, out=y_,
            ot=F32, total=None, xx=None, img=None, sd=None, to=None):
        return lib.t5vq_norm_forward(h, ht, b, bt, w, bias, wt, kind, eps, n, d, bp, prob, 1, 0, sd, None, to, out, ot,
                                     total, None, xx, img, None)

    for call in (dict(h=None), dict(w=None), dict(out=None), dict(b=p), dict(ht=7), dict(wt=7), dict(ot=7),
                 dict(ht=F32, ot=BF16), dict(ht=BF16, ot=F16), dict(ht=BF16, ot=BF16, b=p, bt=F32, total=z_),
                 dict(b=p, bt=5, total=z_), dict(kind=2), dict(eps=-1e-6), dict(eps=math.nan), dict(n=0), dict(n=1 << 32),
                 dict(d=0), dict(bp=1.5), dict(prob=-0.5), dict(prob=math.nan), dict(h=odd), dict(w=odd), dict(out=odd),
                 dict(bias=odd), dict(b=odd, total=z_), dict(b=p, total=odd), dict(out=p), dict(b=p, total=p), dict(b=p, total=y_),
                 dict(b=y_, total=z_), dict(sd=z_, to=z_), dict(xx=p, d=6), dict(xx=p, d=4096),
                 dict(xx=p, ht=BF16, ot=BF16), dict(img=odd)):
        assert fwd(**call) == 1, call
        assert lib.t5vq_last_error()

    def back(g=p, ot=F32, gs=None, h=p, ht=F32, w=p, wt=F32, kind=LAYER, st=p, n=4, d=8, bp=0.0, prob=0.0, ticket=None, gh=y_,
             gb=None, bt=F32, gw=None, gbias=None, ws=None, wsb=0):
        return lib.t5vq_norm_backward(g, ot, gs, h, ht, w, wt, kind, st, n, d, bp, prob, ticket, gh, gb, bt, gw, gbias, ws,
                                      wsb, None)

    need = lib.t5vq_norm_backward_workspace_bytes(4000, 8)
    assert need > 0 and lib.t5vq_norm_backward_workspace_bytes(0, 8) == 0 and lib.t5vq_norm_backward_workspace_bytes(4, 8) == 0
    for call in (dict(g=None), dict(h=None), dict(w=None), dict(st=None), dict(gh=None), dict(ot=BF16), dict(ht=9),
                 dict(ht=BF16, ot=BF16, gb=z_, bt=F32), dict(kind=-1), dict(n=0), dict(d=0), dict(prob=0.1),
                 dict(gb=z_, bp=0.1), dict(gh=p), dict(gb=p), dict(gb=y_), dict(gs=y_), dict(prob=2.0, ticket=p),
                 dict(gw=p, n=4000), dict(gbias=p, ws=p, wsb=need - 1, n=4000), dict(gw=p, ws=odd, wsb=need, n=4000),
                 dict(g=odd), dict(h=odd), dict(gs=odd), dict(gh=odd), dict(gb=odd), dict(gw=odd, ws=p, wsb=need)):
        assert back(**call) == 1, call
        assert lib.t5vq_last_error()


def test_extension_and_functions_refuse_cpu_tensors():
    from t5vqvae_amd import _lib, norms
    ops = _lib.load_torch_ops()
    x, w, t = torch.zeros(2, 8), torch.ones(8), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: ops.dropout_add(x, None, 0.1), lambda: ops.dropout_backward(x, 0.1, t),
                 lambda: ops.norm_forward(x, None, w, None, 0, 1e-6, 0.0, 0.0, None, None, True),
                 lambda: ops.norm_backward(x, None, x, w, torch.zeros(2, 2), 0, 0.0, 0.0, None, None, True, False),
                 lambda: norms.dropout(x), lambda: norms.norm(x, w), lambda: norms.add_norm(x, x, w),
                 lambda: norms.Dropout(0.1)(x), lambda: norms.Norm(8)(x)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_modules_check_their_arguments():
    from t5vqvae_amd import VectorQuantizerEMA, norms
    from t5vqvae_amd.encoder_tail import EncoderTailVQ
    with pytest.raises(RuntimeError, match="p must be in"):
        norms.Dropout(1.5)
    with pytest.raises(RuntimeError, match="kind must be one of"):
        norms.Norm(8, kind="batch")
    with pytest.raises(RuntimeError, match="p must be in"):
        norms.Norm(8, dropout_rate=-1.0)
    assert set(norms.Norm(8).state_dict()) == {"weight", "bias"} and set(norms.Norm(8, "rms").state_dict()) == {"weight"}
    assert set(norms.Norm(8, bias=False).state_dict()) == {"weight"}
    vq = VectorQuantizerEMA(16, 8, 0.25, decay=0.99)
    for bad in (dict(dropout="none"), dict(norm="batch", dropout="counter"), dict(norm="layer"),
                dict(branch_dropout_rate=0.1), dict(bias=torch.nn.Parameter(torch.zeros(8)))):
        with pytest.raises(ValueError):
            EncoderTailVQ(vq, 8, **bad)
    plain, layer = EncoderTailVQ(vq, 8), EncoderTailVQ(vq, 8, norm="layer", dropout="counter")
    assert "bias" not in plain.state_dict() and "bias" in layer.state_dict()
    shared = torch.nn.Parameter(torch.ones(8))
    assert EncoderTailVQ(vq, 8, norm="layer", dropout="counter", bias=shared).bias is shared
    assert EncoderTailVQ(vq, 8, norm="layer", dropout="counter", bias=False).bias is None
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="counter"):
        plain(x, branch=x)
    with pytest.raises(RuntimeError, match="stored"):
        layer(x, keep_mask=x)
    with pytest.raises(RuntimeError, match="no CPU path"):
        layer(x)
