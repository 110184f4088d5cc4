"""The operators around the quantizer's input, as they are measured: dropout from a counter-based generator, layer / RMS
norm with that dropout on its output, and the sum of a residual stream with a dropped-out branch followed by the norm --
each forward, backward, and as one training step (forward and the gradients of all inputs).

The random numbers come from a ticket, int64 {seed, offset}: element (row, col) of site s is kept iff a 16-bit word of
Philox4x32-10 with the counter (offset / 4 + s, col / 8, row) and the key `seed` lies below round((1 - p) * 65536)."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6
MOST = 65536 * 768                    # elements of the largest listed case


def _case(name, op, direction, rows, cols, hidden="f32", branch=None, weights="f32", out=None, kind="rms", bias=False,
          p=0.1, residual=True):
    c = {"op": op, "direction": direction, "rows": rows, "cols": cols, "hidden": hidden, "p": p}
    if op == "dropout":
        c.update(residual=residual)
    else:
        c.update(weights=weights, out=out or hidden, kind=kind, bias=bias)
        if op == "add_norm":
            c.update(branch=branch or hidden)
    return dict(c, name=name) if name else c


def listed():
    return [
        # serving, one token at a time: the norm alone, and the norm behind a sublayer's residual sum
        _case("norm-token", "norm", "forward", 1, 768, kind="layer", bias=True, p=0.0),
        _case("add-norm-token", "add_norm", "forward", 1, 1024, "bf16", weights="bf16", p=0.0),
        # a sublayer's dropout and residual sum on a ragged half-precision batch, and on a large one
        _case("dropout-odd", "dropout", "step", 1003, 771, "f16"),
        _case("dropout-large", "dropout", "forward", 65536, 768, "bf16"),
        # training on 64 sentences of 45 tokens: the encoder's last norm with its dropout, alone and with the sum before it
        _case("norm-batch", "norm", "step", 2880, 768, kind="layer", bias=True),
        _case("add-norm-batch", "add_norm", "step", 2880, 768),
        # a wide encoder in half precision under fp32 weights: backward with both parameter gradients
        _case("norm-wide-backward", "norm", "backward", 4096, 2048, "bf16", kind="layer", bias=True),
        # large batches: forward in half precision, backward in fp32
        _case("norm-large", "norm", "forward", 65536, 768, "bf16", kind="layer", bias=True),
        _case("norm-large-backward", "norm", "backward", 65536, 768),
        # autocast: an fp32 residual stream, the branch straight from a bf16 product
        _case("add-norm-autocast", "add_norm", "forward", 16384, 1024, "f32", branch="bf16", kind="layer", bias=True),
        # rows of an odd length, and the largest step
        _case("add-norm-odd", "add_norm", "backward", 33333, 513, "f16", weights="f16", kind="layer", bias=True),
        _case("add-norm-large", "add_norm", "step", 65536, 768),
    ]


def draw(rng):
    op = rng.choice(("dropout", "norm", "add_norm", "norm", "add_norm"))
    direction = rng.choice(("forward", "backward", "step"))
    cols = int(round(math.exp(rng.uniform(math.log(32), math.log(4096)))))
    if rng.random() < 0.5:
        cols = max(32, cols // 64 * 64)
    rows = max(1, int(math.exp(rng.uniform(0.0, math.log(min(65536, MOST // cols))))))
    hidden = rng.choice(("f32", "bf16", "f16"))
    p = rng.choice((0.0, 0.1, round(rng.uniform(0.01, 0.5), 3)))
    if op == "dropout":
        return _case("", op, direction, rows, cols, hidden, p=p or 0.1, residual=rng.random() < 0.6)
    kind = rng.choice(("layer", "rms"))
    weights = rng.choice(("f32", hidden))
    out, branch = hidden, hidden
    if op == "norm" and rng.random() < 0.3:
        out = "f32"
    if op == "add_norm":
        if hidden == "f32":
            branch = rng.choice(("f32", "bf16", "f16"))
        elif direction == "step":
            weights = hidden
    return _case("", op, direction, rows, cols, hidden, branch, weights, out, kind, kind == "layer" or rng.random() < 0.2, p)


# ---- inputs ---------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, d = case["rows"], case["cols"]
    hidden = TYPES[case["hidden"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    s = dict(case)
    s["ticket"] = torch.randint(0, 1 << 62, (2,), generator=g, device="cuda") // 4 * 4
    # a residual stream: channels of different size and offset, a few of them far larger than the rest
    size = torch.exp(0.5 * normal(d)) * torch.where(torch.rand(d, generator=g, device="cuda") < 0.01, 12.0, 2.0)
    h = (normal(n, d) * size + 0.5 * normal(d)).to(hidden)
    if case["op"] == "dropout":
        if case["direction"] != "backward":
            s["x"] = h
            s["res"] = (3.0 * normal(n, d)).to(hidden) if case["residual"] else None
        if case["direction"] != "forward":
            s["g"] = normal(n, d).to(hidden)
        if case["direction"] == "step":
            for name in ("x", "res"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
        return s
    weights, out = TYPES[case["weights"]], TYPES[case["out"]]
    s["weight"] = (1.0 + 0.2 * normal(d)).to(weights)
    s["bias"] = (0.2 * normal(d)).to(weights) if case["bias"] else None
    if case["direction"] == "backward":                      # what the forward pass left: the normed rows and their statistics
        s["h"] = h
        mean = h.double().mean(1) if case["kind"] == "layer" else torch.zeros(n, dtype=torch.float64, device="cuda")
        r = (h.double() - mean[:, None]).square().mean(1).add(EPS).rsqrt()
        s["stats"] = torch.stack((mean, r), 1).float()
    else:
        s["hidden_rows"] = h
        if case["op"] == "add_norm":
            s["branch_rows"] = normal(n, d).to(TYPES[case["branch"]])
    if case["direction"] != "forward":
        s["g"] = normal(n, d).to(out)
        s["g_sum"] = normal(n, d).to(hidden) if case["op"] == "add_norm" else None
    if case["direction"] == "step":
        for name in ("hidden_rows", "branch_rows", "weight", "bias"):
            if s.get(name) is not None:
                s[name].requires_grad_(True)
    return s


# ---- the plain form ---------------------------------------------------------------------------------------------------
_LOW = 0xFFFFFFFF


def _words(ticket, site, rows, blocks):
    """Four 32-bit words (in int64) for each (row, block of eight columns): Philox4x32-10."""
    where = (ticket[1] >> 2) + site
    a, b = where & _LOW, (where >> 32) & _LOW
    c = torch.arange(blocks, device=ticket.device)
    d = torch.arange(rows, device=ticket.device)[:, None]
    k0, k1 = ticket[0] & _LOW, (ticket[0] >> 32) & _LOW
    for _ in range(10):
        u, v = a * 0xD2511F53, c * 0xCD9E8D57               # 64-bit products, modulo 2^64
        a, b, c, d = ((v >> 32) & _LOW) ^ b ^ k0, v & _LOW, ((u >> 32) & _LOW) ^ d ^ k1, u & _LOW
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    return torch.broadcast_tensors(a, b, c, d)


def _kept(p):
    return round((1.0 - p) * 65536.0)


def _scale(p):
    return float(torch.tensor(65536.0 / _kept(p), dtype=torch.float32)) if _kept(p) else 0.0


def _keep(ticket, site, rows, cols, p):
    blocks = (cols + 7) // 8
    w = torch.stack(_words(ticket, site, rows, blocks), -1)
    halves = torch.stack((w & 0xFFFF, w >> 16), -1)
    return halves.reshape(rows, blocks * 8)[:, :cols] < _kept(p)


def _drop(x, s, site, p):
    if _kept(p) == 65536:
        return x
    return torch.where(_keep(s["ticket"], site, x.shape[0], x.shape[1], p), x * _scale(p), 0.0)


def _plain_norm(h, s):
    if s["kind"] == "layer":
        mean = h.mean(1, keepdim=True)
        r = 1.0 / torch.sqrt((h - mean).square().mean(1, keepdim=True) + EPS)
        return (h - mean) * r, r
    r = 1.0 / torch.sqrt(h.square().mean(1, keepdim=True) + EPS)
    return h * r, r


def _plain_out(n, s):
    y = n * s["weight"].detach().float()
    if s["bias"] is not None:
        y = y + s["bias"].detach().float()
    return _drop(y, s, 1, s["p"]).to(TYPES[s["out"]])


def _plain_backward(n, r, s):
    """Gradients from the normalised rows n and 1 / deviation r."""
    gy = _drop(s["g"].float(), s, 1, s["p"])
    a = gy * s["weight"].detach().float()
    g = a - n * (a * n).mean(1, keepdim=True)
    if s["kind"] == "layer":
        g = g - a.mean(1, keepdim=True)
    g = g * r
    if s["op"] == "add_norm":
        g = g + s["g_sum"].float()
    hidden = TYPES[s["hidden"]]
    got = {"hidden": g.to(hidden)}
    if s["op"] == "add_norm":
        got["branch"] = _drop(g, s, 0, s["p"]).to(TYPES[s["branch"]])
    got["weight"] = (gy * n).sum(0).to(s["weight"].dtype)
    if s["bias"] is not None:
        got["bias"] = gy.sum(0).to(s["weight"].dtype)
    return got


def _plain(s):
    hidden = TYPES[s["hidden"]]
    if s["op"] == "dropout":
        got = {}
        if s["direction"] != "backward":
            y = _drop(s["x"].detach().float(), s, 0, s["p"])
            if s["res"] is not None:
                y = s["res"].detach().float() + y
            got["out"] = y.to(hidden)
        if s["direction"] != "forward":
            got["x"] = _drop(s["g"].float(), s, 0, s["p"]).to(hidden)
            if s["direction"] == "step" and s["res"] is not None:
                got["res"] = s["g"]
        return got
    if s["direction"] == "backward":
        mean, r = s["stats"][:, :1], s["stats"][:, 1:]
        return _plain_backward((s["h"].float() - mean) * r, r, s)
    h = s["hidden_rows"].detach()
    got = {}
    if s["op"] == "add_norm":
        h = (h.float() + _drop(s["branch_rows"].detach().float(), s, 0, s["p"])).to(hidden)   # the stream, in its own type
        got["sum"] = h
    n, r = _plain_norm(h.float(), s)
    got["out"] = _plain_out(n, s)
    if s["direction"] == "step":
        got["grads"] = _plain_backward(n, r, s)
    return got


# ---- the framework's kernels ----------------------------------------------------------------------------------------------
def _own(s):
    from t5vqvae_amd import norms, ops
    if s["op"] == "dropout":
        if s["direction"] == "backward":
            return {"x": ops.dropout_backward(s["g"], s["p"], s["ticket"])}
        if s["direction"] == "forward":
            return {"out": norms.dropout(s["x"], s["p"], s["res"], ticket=s["ticket"])}
        out = norms.dropout(s["x"], s["p"], s["res"], ticket=s["ticket"])
        if s["res"] is None:
            return {"out": out.detach(), "x": torch.autograd.grad(out, s["x"], s["g"])[0]}
        gx, gr = torch.autograd.grad(out, (s["x"], s["res"]), s["g"])
        return {"out": out.detach(), "x": gx, "res": gr}
    p = s["p"]
    if s["direction"] == "backward":
        with_branch = s["op"] == "add_norm"
        gh, gb, gw, gbias = ops.norm_backward(s["g"], s["g_sum"], s["h"], s["weight"], s["stats"], kind=s["kind"],
                                              branch_p=p if with_branch else 0.0, p=p, ticket=s["ticket"],
                                              branch_dtype=TYPES[s["branch"]] if with_branch else None,
                                              want_weight=True, want_bias=s["bias"] is not None)
        got = {"hidden": gh, "weight": gw}
        if with_branch:
            got["branch"] = gb
        if s["bias"] is not None:
            got["bias"] = gbias
        return got
    got = {}
    if s["op"] == "add_norm":
        out, total = norms.add_norm(s["hidden_rows"], s["branch_rows"], s["weight"], s["bias"], kind=s["kind"], eps=EPS,
                                    branch_p=p, p=p, ticket=s["ticket"])
        got["sum"] = total.detach()
    else:
        out = norms.norm(s["hidden_rows"], s["weight"], s["bias"], kind=s["kind"], eps=EPS, p=p, ticket=s["ticket"],
                         out_dtype=TYPES[s["out"]])
    got["out"] = out.detach()
    if s["direction"] == "step":
        names = [k for k in ("hidden_rows", "branch_rows", "weight", "bias") if s.get(k) is not None]
        outs, gs = ((out, total), (s["g"], s["g_sum"])) if s["op"] == "add_norm" else ((out,), (s["g"],))
        grads = torch.autograd.grad(outs, [s[k] for k in names], gs)
        got["grads"] = {k.replace("_rows", ""): v for k, v in zip(names, grads)}
    return got


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------
def work(case):
    n, d = case["rows"], case["cols"]
    size = {k: (4 if k == "f32" else 2) for k in TYPES}
    h, e = size[case["hidden"]], n * d
    way = case["direction"]
    if case["op"] == "dropout":
        b = f = 0
        if way != "backward":
            b, f = b + e * h * (3 if case["residual"] else 2), f + 2 * e
        if way != "forward":
            b, f = b + 2 * e * h, f + e
        return {"bytes": b, "flops": f}
    o, w = size[case["out"]], size[case["weights"]]
    br = size[case["branch"]] if case["op"] == "add_norm" else 0
    params = d * w * (2 if case["bias"] else 1)
    b, f = params, 0
    if way != "backward":                                     # read the stream (and the branch), write the output (and the sum)
        b, f = b + e * (h + o) + (e * (br + h) if br else 0), f + 8 * e
    if way != "forward":                                      # read gradients (and the normed rows), write gradients
        b, f = b + e * (o + h) + params + (e * (h + br) if br else 0), f + 14 * e
        if way == "backward":
            b += e * h + 8 * n
    return {"bytes": b, "flops": f}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------
def _mulhilo(m, x):
    """(high, low) 32 bits of m * x from 16-bit halves: every product and sum stays far below 2^63."""
    m0, m1, x0, x1 = m % 65536, m // 65536, x % 65536, x // 65536
    low = m0 * x0
    mid = m1 * x0 + low // 65536
    other = m0 * x1 + mid % 65536
    return m1 * x1 + mid // 65536 + other // 65536, other % 65536 * 65536 + low % 65536


def _exact_mask(case, s, site):
    n, d, k = case["rows"], case["cols"], round((1.0 - case["p"]) * 65536.0)
    seed, offset = (int(v) for v in s["ticket"].tolist())
    where = offset // 4 + site
    col = torch.arange(d, device="cuda")
    nblk = -(-d // 8)
    ctr = [torch.full((n, nblk), where % 2 ** 32, device="cuda"), torch.full((n, nblk), where // 2 ** 32 % 2 ** 32, device="cuda"),
           torch.arange(nblk, device="cuda").repeat(n, 1), torch.arange(n, device="cuda")[:, None].repeat(1, nblk)]
    key = [seed % 2 ** 32, seed // 2 ** 32 % 2 ** 32]
    for i in range(10):
        h0, l0 = _mulhilo(0xD2511F53, ctr[0])
        h1, l1 = _mulhilo(0xCD9E8D57, ctr[2])
        r0 = (key[0] + i * 0x9E3779B9) % 2 ** 32
        r1 = (key[1] + i * 0xBB67AE85) % 2 ** 32
        ctr = [h1 ^ ctr[1] ^ r0, l1, h0 ^ ctr[3] ^ r1, l0]
    keep = torch.empty(n, d, dtype=torch.bool, device="cuda")
    for j in range(8):
        part = ctr[j // 2] // 65536 if j % 2 else ctr[j // 2] % 65536
        keep[:, col % 8 == j] = part[:, : (d - j + 7) // 8] < k
    return keep, (65536.0 / k if k else 0.0)


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    p = case["p"]

    def drop(v, site):
        if round((1.0 - p) * 65536.0) == 65536:
            return v
        keep, scale = _exact_mask(case, s, site)
        return torch.where(keep, v * scale, torch.zeros((), dtype=f64, device="cuda"))

    def wide(name):
        return s[name].detach().to(f64)

    got = {}
    if case["op"] == "dropout":
        if case["direction"] != "backward":
            y = drop(wide("x"), 0)
            got["out"] = y + wide("res") if s["res"] is not None else y
        if case["direction"] != "forward":
            got["x"] = drop(wide("g"), 0)
            if case["direction"] == "step" and s["res"] is not None:
                got["res"] = wide("g")
        return got
    layer, add = case["kind"] == "layer", case["op"] == "add_norm"
    if case["direction"] == "backward":
        h = wide("h")
        mu, r = wide("stats")[:, 0:1], wide("stats")[:, 1:2]
    else:
        h = wide("hidden_rows")
        if add:
            total = h + drop(wide("branch_rows"), 0)
            got["sum"] = total
            h = total.to(TYPES[case["hidden"]]).to(f64) if case["hidden"] != "f32" else total
        mu = torch.sum(h, 1, keepdim=True) / case["cols"] if layer else torch.zeros(case["rows"], 1, dtype=f64, device="cuda")
        r = torch.pow(torch.sum(torch.pow(h - mu, 2), 1, keepdim=True) / case["cols"] + EPS, -0.5)
    unit = (h - mu) * r
    w = wide("weight")
    if case["direction"] != "backward":
        y = w * unit + (wide("bias") if s["bias"] is not None else 0.0)
        got["out"] = drop(y, 1)
        if case["direction"] == "forward":
            return got
    up = drop(wide("g"), 1)
    back = up * w
    inner = torch.sum(back * unit, 1, keepdim=True) / case["cols"]
    shift = torch.sum(back, 1, keepdim=True) / case["cols"] if layer else 0.0
    gh = (back - shift - unit * inner) * r + (wide("g_sum") if add else 0.0)
    grads = {"hidden": gh, "weight": torch.sum(up * unit, 0)}
    if add:
        grads["branch"] = drop(gh, 0)
    if s["bias"] is not None:
        grads["bias"] = torch.sum(up, 0)
    if case["direction"] == "backward":
        return grads
    got["grads"] = grads
    return got
