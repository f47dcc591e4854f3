"""Plain 64-bit forms of the paged serving operators (include/mimo_moe_paged.h), for the tests."""
import numpy as np
import torch


def plan(lens, new, table, free, n_free, P, T):
    """Token by token: a token that opens a page takes the last free one.  Returns (cu, lens', n_free', pos, slots,
    table')."""
    table = [list(r) for r in table]
    cu, pos, slots = [0], [], []
    for r, (h, n) in enumerate(zip(lens, new)):
        for p in range(h, h + n):
            if p % P == 0:
                n_free -= 1
                table[r][p // P] = free[n_free]
            pos.append(p)
            slots.append(table[r][p // P] * P + p % P)
        cu.append(cu[-1] + n)
    pad = [-1] * (T - cu[-1])
    return cu, [h + n for h, n in zip(lens, new)], n_free, pos + pad, slots + pad, table


def rope(x, pos, rot, theta):
    """x [T, heads, d] float64 -> (rotated, |x1| + |x2| of each output: what its rounding errors are relative to)."""
    half = rot // 2
    ang = pos[:, None] * np.exp(-2.0 * np.arange(half) / rot * np.log(float(np.float32(theta)))) if rot else pos[:, None][:, :0]
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    y, mag = x.copy(), np.abs(x)
    a, b = x[..., :half], x[..., half:rot]
    y[..., :half], y[..., half:rot] = a * c - b * s, a * s + b * c
    mag[..., :half] = mag[..., half:rot] = np.abs(a) + np.abs(b)
    return y, mag


def attention(q, K, V, first_pos, scale, window=0, keep=0, sinks=None):
    """q [n, nq, d] at positions first_pos.., K [L, nkv, d], V [L, nkv, dv] (float64).  Returns (out [n, nq, dv], the
    same with |V|: the weight every rounding of a probability has)."""
    n, nq, _ = q.shape
    L, nkv, dv = V.shape
    at, key = first_pos + np.arange(n)[:, None], np.arange(L)[None, :]
    seen = key <= at
    if window:
        seen &= (key > at - window) | (key < keep)
    out, mag = np.zeros((n, nq, dv)), np.zeros((n, nq, dv))
    for h in range(nq):
        hk = h * nkv // nq
        s = np.where(seen, q[:, h] @ K[:, hk].T * scale, -np.inf)
        m = s.max(1) if sinks is None else np.maximum(s.max(1), sinks[h])
        p = np.exp(s - m[:, None])
        den = p.sum(1) + (0.0 if sinks is None else np.exp(sinks[h] - m))
        out[:, h] = p @ V[:, hk] / den[:, None]
        mag[:, h] = p @ np.abs(V[:, hk]) / den[:, None]
    return out, mag


def f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().double().cpu().numpy()
