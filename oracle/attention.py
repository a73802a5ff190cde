"""The attention operators over atoms from their definitions, in float64 on the CPU."""
from __future__ import annotations

import numpy as np
import torch


def embedding(ids, table, scale):
    return scale * table[ids]


def embedding_grad(ids, grad, rows, scale):
    out = torch.zeros(rows, grad.shape[-1], dtype=torch.float64)
    ok = (ids >= 0) & (ids < rows)
    return scale * out.index_add(0, ids[ok].reshape(-1), grad[ok].reshape(-1, grad.shape[-1]))


def philox(counter, key):
    """Philox4x32-10 (Salmon, Moraes, Dror and Shaw, SC 2011): four uint32 words."""
    c, k = [int(x) for x in counter], [int(x) for x in key]
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & 0xFFFFFFFF, (p0 >> 32) ^ c[3] ^ k[1], p0 & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def keep_mask(first, n, drop, seed, offset):
    """keep(e) of elements ``first`` to ``first + n``."""
    out, m = np.empty(n, dtype=bool), 0xFFFFFFFF
    block, words = None, None
    for j in range(n):
        e = first + j
        if e // 8 != block:
            block = e // 8
            words = philox((block & m, block >> 32, offset & m, (offset >> 32) & m),
                           (seed & m, (seed >> 32) & m))
        out[j] = ((words[e % 8 // 2] >> (16 * (e % 2))) & 0xFFFF) >= drop
    return torch.from_numpy(out)


def norm_rotate(x, weight, cos, sin, eps, interleaved):
    """One of queries and keys (T, heads, D) with a row of the tables a token."""
    R = 2 * cos.shape[1]
    u = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight
    if R == 0:
        return u
    c, s = cos[:, None, :], sin[:, None, :]
    if interleaved:
        a, b = u[..., 0:R:2], u[..., 1:R:2]
        turned = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    else:
        a, b = u[..., :R // 2], u[..., R // 2:R]
        turned = torch.cat((a * c - b * s, a * s + b * c), -1)
    return torch.cat((turned, u[..., R:]), -1)


def attention(q, k, v, counts, mask=None, scale=None, grad=None):
    """``(out, dq, dk, dv, bounds)``: the attention of each structure's atoms over its kept atoms and,
    with ``grad``, the gradients by their formulas. ``bounds(eps, u, w)`` are the errors of float32
    arithmetic (spacing ``eps``) with outputs rounded to unit ``u`` and probabilities to ``w``."""
    T, H, D = q.shape
    K = k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    mask = torch.ones(T, dtype=torch.bool) if mask is None else mask
    names = ("out", "dq", "dk", "dv")
    value = {n: torch.zeros(T, K if n in ("dk", "dv") else H, D, dtype=torch.float64) for n in names}
    # error terms: of float32 arithmetic, of the weights' rounding, of the stored out in delta
    arith, rounded, stored = ({n: torch.zeros_like(value[n]) for n in names} for _ in range(3))
    start = 0
    for n in counts:
        rows = torch.arange(start, start + n)
        start += n
        keys = rows[mask[rows]]
        if len(keys) == 0:
            continue
        for h in range(H):
            c = h // (H // K)
            a, b, x = q[rows, h], k[keys, c], v[keys, c]
            s = scale * a @ b.T
            L = torch.logsumexp(s, 1, keepdim=True)
            p = torch.exp(s - L)
            o = p @ x
            value["out"][rows, h] = o
            # a score is a sum of D products, scaled; it and L enter an exponential; then n terms
            size = (scale * a.abs() @ b.abs().T).amax(1, keepdim=True)
            rho = 2 * ((D + 4) * size + L.abs() + 4) + n + 8
            arith["out"][rows, h] = rho * (p @ x.abs())
            rounded["out"][rows, h] = p @ x.abs()
            if grad is None:
                continue
            g = grad[rows, h]
            dp, delta = g @ x.T, (g * o).sum(1, keepdim=True)
            ds = p * (dp - delta)
            value["dv"][keys, c] += p.T @ g
            value["dq"][rows, h] = scale * ds @ b
            value["dk"][keys, c] += scale * ds.T @ a
            arith["dv"][keys, c] += (p * rho).T @ g.abs()
            rounded["dv"][keys, c] += p.T @ g.abs()
            e = p * (rho * (dp - delta).abs() + (D + 4) * (g.abs() @ x.abs().T)
                     + (g.abs() * (arith["out"][rows, h] + (D + 4) * o.abs())).sum(1, keepdim=True))
            arith["dq"][rows, h] = scale * (e + n * ds.abs()) @ b.abs()
            arith["dk"][keys, c] += scale * (e + n * ds.abs()).T @ a.abs()
            rounded["dq"][rows, h] = scale * ds.abs() @ b.abs()
            rounded["dk"][keys, c] += scale * ds.abs().T @ a.abs()
            far = p * (g.abs() * (o.abs() + p @ x.abs())).sum(1, keepdim=True)
            stored["dq"][rows, h] = scale * far @ b.abs()
            stored["dk"][keys, c] += scale * far.T @ a.abs()

    def bounds(eps, u, w):
        return tuple(eps * arith[n] + w * rounded[n] + max(u, w) * stored[n] + u * value[n].abs()
                     for n in names)
    return (*(value[n] for n in names), bounds)
