"""Plain 64-bit restatement of the dropout / norm operators of include/t5vq.h -- TEST INFRASTRUCTURE ONLY (CPU, numpy and
torch float64).  Masks are exact; everything else is the formula, unrounded."""
import numpy as np
import torch

M0, M1, W0, W1, LOW = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85, 0xFFFFFFFF


def philox4x32_10(counter, key):
    """One block on Python integers (Salmon et al., SC 2011): four counter words and two key words to four words."""
    a, b, c, d = counter
    k0, k1 = key
    for _ in range(10):
        u, v = a * M0, c * M1
        a, b, c, d = (v >> 32) ^ b ^ k0, v & LOW, (u >> 32) ^ d ^ k1, u & LOW
        k0, k1 = (k0 + W0) & LOW, (k1 + W1) & LOW
    return a, b, c, d


def keep_count(p):
    return int(np.rint((1.0 - p) * 65536.0))


def scale_of(p):
    k = keep_count(p)
    return 65536.0 / k if k else 0.0


def draws(rows, cols, ticket, site, first_row=0):
    """uint16 [rows, cols]: the 16 bits of every element (rows counted from first_row)."""
    seed, offset = (int(v) & 0xFFFFFFFFFFFFFFFF for v in ticket)
    blocks = (cols + 7) // 8
    u64 = np.uint64
    where = (offset // 4 + site) & 0xFFFFFFFFFFFFFFFF
    a = np.full((rows, blocks), where & LOW, u64)
    b = np.full((rows, blocks), where >> 32, u64)
    c = np.broadcast_to(np.arange(blocks, dtype=u64), (rows, blocks)).copy()
    d = np.broadcast_to((np.arange(rows, dtype=u64) + u64(first_row))[:, None] & u64(LOW), (rows, blocks)).copy()
    k0, k1 = seed & LOW, seed >> 32
    s32, low = u64(32), u64(LOW)
    for _ in range(10):
        u, v = a * u64(M0), c * u64(M1)
        a, b, c, d = (v >> s32) ^ b ^ u64(k0), v & low, (u >> s32) ^ d ^ u64(k1), u & low
        k0, k1 = (k0 + W0) & LOW, (k1 + W1) & LOW
    words = np.stack((a, b, c, d), -1)
    halves = np.stack((words & u64(0xFFFF), words >> u64(16)), -1).astype(np.uint16)
    return halves.reshape(rows, blocks * 8)[:, :cols]


def keep_mask(rows, cols, p, ticket, site, first_row=0):
    if keep_count(p) == 65536:
        return torch.ones(rows, cols, dtype=torch.bool)
    return torch.from_numpy(draws(rows, cols, ticket, site, first_row).astype(np.int64) < keep_count(p))


def drop(v, keep, p):
    return torch.where(keep, v * scale_of(p), torch.zeros((), dtype=v.dtype))


def stats(h, kind, eps):
    mean = h.mean(1, keepdim=True) if kind == "layer" else torch.zeros(h.shape[0], 1, dtype=h.dtype)
    return mean, 1.0 / torch.sqrt(((h - mean) ** 2).mean(1, keepdim=True) + eps)


def norm(h, weight, bias, kind, eps, keep=None, p=0.0):
    mean, r = stats(h, kind, eps)
    y = (h - mean) * r * weight
    if bias is not None:
        y = y + bias
    return y if keep is None else drop(y, keep, p)


def norm_backward(g, h, weight, kind, eps, keep=None, p=0.0, g_sum=None, branch_keep=None, branch_p=0.0):
    """(grad_hidden, grad_branch, grad_weight, grad_bias)"""
    mean, r = stats(h, kind, eps)
    n = (h - mean) * r
    gy = g if keep is None else drop(g, keep, p)
    a = gy * weight
    gh = a - n * (a * n).mean(1, keepdim=True)
    if kind == "layer":
        gh = gh - a.mean(1, keepdim=True)
    gh = gh * r
    if g_sum is not None:
        gh = gh + g_sum
    gb = gh if branch_keep is None else drop(gh, branch_keep, branch_p)
    return gh, gb, (gy * n).sum(0), gy.sum(0)
