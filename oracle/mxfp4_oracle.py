"""MXFP4 and the experts' operators in numpy, 64 bits -- TEST INFRASTRUCTURE ONLY.

Written from the format's definition (OCP Microscaling, 4 bits): a block of 32 values is
``code * 2^(e - 127)``, ``e = max(floor(log2 max|v|) - 2 + 127, 0)``, each code the nearest E2M1 value
(ties to the even code, above 6 to 6); a block with a NaN or an infinity has ``e = 255``.  Storage as
``mx4.cuh`` states it.  Only ``tests/`` imports this module.
"""

from __future__ import annotations

import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)


def quantize(x):
    """x [.., K] -> (codes [.., B, 32] of 0..15, exponents [.., B]); values past K are zero."""
    x = np.asarray(x, dtype=np.float64)
    k = x.shape[-1]
    pad = -k % 32
    x = np.concatenate([x, np.zeros((*x.shape[:-1], pad))], axis=-1) if pad else x
    x = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    finite = np.isfinite(x).all(-1)
    amax = np.abs(np.where(finite[..., None], x, 0)).max(-1)
    e = np.full(amax.shape, 0)
    nz = amax > 0
    e[nz] = np.maximum(np.frexp(amax[nz])[1] - 1 - 2 + 127, 0)
    e = np.where(finite, e, 255)
    a = np.abs(x) / np.exp2(np.where(finite, e, 127) - 127.0)[..., None]
    # distance to each code, the even one first among equals
    d = np.abs(a[..., None] - GRID)
    with np.errstate(invalid="ignore"):
        order = np.array([0, 2, 4, 6, 1, 3, 5, 7])
        code = order[np.argmin(np.where(np.isnan(d), np.inf, d)[..., order], axis=-1)]
    return code + 8 * (x < 0), e


def values(code, e, k=None):
    """What codes and exponents stand for: [.., K]."""
    v = np.where(code >= 8, -GRID[code & 7], GRID[code & 7])
    s = np.where(e == 255, np.nan, np.exp2(e - 127.0))
    v = (v * s[..., None]).reshape(*code.shape[:-2], code.shape[-2] * 32)
    return v if k is None else v[..., :k]


def rounded(x):
    """x's rows as MXFP4 holds them."""
    return values(*quantize(x), np.asarray(x).shape[-1])


def unpack(codes, scales, rows):
    """Stored codes [.., R, B * 16] and scales [.., tr, tk, 32, 16] -> (codes [.., R, B, 32], e [.., R, B])."""
    blocks = codes.shape[-1] // 16
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], blocks, 32)
    r = np.arange(rows)[:, None]
    b = np.arange(blocks)[None, :]
    e = scales[..., r // 128, b // 4, r % 32, (r % 128) // 32 * 4 + b % 4]
    return c.astype(np.int64), e.astype(np.int64)


def product(a, b, bias=None):
    """(a b^T + bias, |a| |b|^T) of values in 64 bits: the second bounds the sums' rounding."""
    y = a @ b.T
    s = np.abs(a) @ np.abs(b).T
    if bias is not None:
        y, s = y + bias, s + np.abs(bias)
    return y, s


def sort(ids, experts):
    """(order, positions, offsets, scale_rows, tiles) of ids [T, k]."""
    flat = np.asarray(ids).reshape(-1).astype(np.int64)
    key = np.where((flat >= 0) & (flat < experts), flat, experts)
    order = np.argsort(key, kind="stable")
    positions = np.empty_like(order)
    positions[order] = np.arange(order.size)
    counts = np.bincount(key, minlength=experts + 1)[:experts]
    offsets = np.concatenate([[0], np.cumsum(counts)])
    tiles = np.concatenate([[0], np.cumsum(-(-counts // 128))])
    taken = key < experts
    scale_rows = np.where(taken, tiles[np.where(taken, key, 0)] * 128
                          + positions - offsets[np.where(taken, key, 0)], -1)
    return order, positions.reshape(np.shape(ids)), offsets, scale_rows.reshape(np.shape(ids)), tiles


def gather(x, ids, experts):
    order, _, offsets, _, _ = sort(ids, experts)
    out = x[order // np.shape(ids)[1]].copy()
    out[offsets[-1]:] = 0
    return out


def combine(y, weights, ids, experts):
    _, positions, offsets, _, _ = sort(ids, experts)
    taken = (positions < offsets[-1])[..., None]
    return np.where(taken, y[positions] * weights[..., None], 0).sum(1)


def combine_grad(dy, y, weights, ids, experts):
    """(gradient of y, gradient of the weights)."""
    order, positions, offsets, _, _ = sort(ids, experts)
    top = np.shape(ids)[1]
    gy = weights.reshape(-1)[order][:, None] * dy[order // top]
    gy[offsets[-1]:] = 0
    taken = positions < offsets[-1]
    gw = np.where(taken, (np.where(taken[..., None], y[positions], 0) * dy[:, None]).sum(-1), 0)
    return gy, gw
