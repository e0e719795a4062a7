"""Classifier-head oracle: dropout's counter-based mask and the linear softmax cross entropy, in 64 bits (numpy).

Test infrastructure; written from the definitions in include/wino.h, independent of the kernels.
"""
import numpy as np

_M32 = np.uint64(0xFFFFFFFF)
_S32 = np.uint64(32)


def philox4x32_10(counter, key):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011).  counter: (..., 4), key: two ints; returns (..., 4) uint32."""
    c = [np.asarray(counter[..., i], dtype=np.uint64) for i in range(4)]
    k = [int(key[0]), int(key[1])]
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> _S32) ^ c[1] ^ np.uint64(k[0]), p1 & _M32, (p0 >> _S32) ^ c[3] ^ np.uint64(k[1]), p0 & _M32]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, -1).astype(np.uint32)


def dropout_threshold(p):
    return int(np.floor(float(np.float32(p)) * 65536.0 + 0.5))


def dropout_keep(first, count, p, seed, offset):
    """Keep flags of elements first ... first + count - 1."""
    e = np.arange(first, first + count, dtype=np.uint64)
    g = e // np.uint64(8)
    groups, back = np.unique(g, return_inverse=True)
    ctr = np.stack([groups & _M32, groups >> _S32, np.full_like(groups, offset & 0xFFFFFFFF), np.full_like(groups, offset >> 32)], -1)
    r = philox4x32_10(ctr, (seed & 0xFFFFFFFF, seed >> 32))
    lanes = np.stack([r & 0xFFFF, r >> 16], -1).reshape(len(groups), 8)
    return lanes[back, (e % np.uint64(8)).astype(np.int64)] >= dropout_threshold(p)


def dropout(x, p, seed, offset=0):
    t = dropout_threshold(p)
    keep = dropout_keep(0, x.size, p, seed, offset).reshape(x.shape)
    scale = 65536.0 / (65536 - t) if t < 65536 else 0.0
    return np.where(keep, x.astype(np.float64) * scale, 0.0)


def xent(x, w, target, bias=None, reduction="mean", ignore_index=None, smoothing=0.0, dloss=None):
    """loss, lse, dx, dw, db of the linear softmax cross entropy; all arguments and results float64 (numpy)."""
    n, v = x.shape[0], w.shape[0]
    counts = np.ones(n, dtype=bool) if ignore_index is None else target != ignore_index
    x = np.where(counts[:, None], x, 0.0)
    t = np.where(counts, target, 0)
    z = x @ w.T + (0.0 if bias is None else bias)
    m = z.max(1)
    ref = np.where(np.isfinite(m), m, 0.0)
    lse = ref + np.log(np.exp(z - ref[:, None]).sum(1))
    q = np.full((n, v), smoothing / v)
    q[np.arange(n), t] += 1 - smoothing
    loss = lse - (1 - smoothing) * z[np.arange(n), t]
    if smoothing > 0:
        loss = loss - smoothing / v * z.sum(1)
    loss = np.where(counts, loss, 0.0)
    g = counts.astype(np.float64) * (1.0 if dloss is None else dloss)
    total = max(1, int(counts.sum()))
    if reduction == "mean":
        loss, g = loss.sum() / total, g / total
    elif reduction == "sum":
        loss = loss.sum()
    dz = g[:, None] * (np.exp(z - lse[:, None]) - q)
    dz[~counts] = 0.0
    return {"loss": loss, "lse": np.where(counts, lse, 0.0), "dx": dz @ w, "dw": dz.T @ x, "db": dz.sum(0), "dz": dz, "z": z}
