"""The operators of the classifier head, as they are measured: dropout and the linear softmax cross entropy.

`run` computes one pass of a case, in elementary torch operations (own = False) or by the framework's entry points
(own = True), from what `prepare` put on the GPU.  `exact` is the same pass from the definition in 64 bits.
"""
import math

import torch

own = False

# Smallest to largest: what a fine-tuning or evaluation program over the convolution stack's features calls.  4096 features
# and 1000 classes are the classifier tail's own sizes, 25088 = 512 * 7 * 7 the flattened output of the stack, 512 its
# pooled output; the larger class counts are generic.
_LISTED = [
    # dropout after a fully connected layer, a small batch: launch latency
    {"name": "dropout_fwd_bf16_32x4096", "op": "dropout", "back": False, "dtype": "bf16", "rows": 32, "cols": 4096, "pitch": 4096, "p": 0.5},
    # dropout of the flattened features of a large batch: bandwidth
    {"name": "dropout_fwd_bf16_8192x25088", "op": "dropout", "back": False, "dtype": "bf16", "rows": 8192, "cols": 25088, "pitch": 25088, "p": 0.5},
    # gradient through dropout, odd rows inside a wider buffer, single precision
    {"name": "dropout_bwd_fp32_1000x4099", "op": "dropout", "back": True, "dtype": "fp32", "rows": 1000, "cols": 4099, "pitch": 4107, "p": 0.1},
    # validation loss of one small batch on the tail's last layer: latency, few rows
    {"name": "xent_fwd_bf16_16x4096_v1000", "op": "xent", "grad": False, "dtype": "bf16", "n": 16, "d": 4096, "v": 1000,
     "bias": True, "reduction": "mean", "ignored": 0.0, "smoothing": 0.0},
    # validation loss in single precision, ragged rows
    {"name": "xent_fwd_fp32_777x4096_v1000", "op": "xent", "grad": False, "dtype": "fp32", "n": 777, "d": 4096, "v": 1000,
     "bias": True, "reduction": "none", "ignored": 0.0, "smoothing": 0.0},
    # evaluation over a large vocabulary, no logits kept
    {"name": "xent_fwd_bf16_8192x2048_v65536", "op": "xent", "grad": False, "dtype": "bf16", "n": 8192, "d": 2048, "v": 65536,
     "bias": False, "reduction": "mean", "ignored": 0.1, "smoothing": 0.0},
    # the smallest training step: pooled features, ten classes
    {"name": "xent_grad_fp32_32x512_v10", "op": "xent", "grad": True, "dtype": "fp32", "n": 32, "d": 512, "v": 10,
     "bias": True, "reduction": "mean", "ignored": 0.0, "smoothing": 0.0},
    # linear probe on the flattened features: the weight and its gradient dominate
    {"name": "xent_grad_bf16_256x25088_v1000", "op": "xent", "grad": True, "dtype": "bf16", "n": 256, "d": 25088, "v": 1000,
     "bias": True, "reduction": "mean", "ignored": 0.0, "smoothing": 0.1},
    # training step, many classes, odd width, single precision
    {"name": "xent_grad_fp32_1024x1001_v21841", "op": "xent", "grad": True, "dtype": "fp32", "n": 1024, "d": 1001, "v": 21841,
     "bias": True, "reduction": "sum", "ignored": 0.0, "smoothing": 0.1},
    # training step over a vocabulary, padded batch (a tenth of the rows ignored)
    {"name": "xent_grad_bf16_4096x1024_v32000", "op": "xent", "grad": True, "dtype": "bf16", "n": 4096, "d": 1024, "v": 32000,
     "bias": False, "reduction": "mean", "ignored": 0.1, "smoothing": 0.0},
    # the largest training step: ragged vocabulary, wide features
    {"name": "xent_grad_bf16_8192x4096_v50021", "op": "xent", "grad": True, "dtype": "bf16", "n": 8192, "d": 4096, "v": 50021,
     "bias": False, "reduction": "mean", "ignored": 0.0, "smoothing": 0.0},
]

_DTYPE = {"bf16": torch.bfloat16, "fp32": torch.float32}
_IGNORE = -100


def listed():
    return [dict(c) for c in _LISTED]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.3:
        rows, cols = _log_int(rng, 1, 8192), _log_int(rng, 256, 25088)
        return {"op": "dropout", "back": rng.random() < 0.5, "dtype": rng.choice(["bf16", "fp32"]), "rows": rows, "cols": cols,
                "pitch": cols + rng.choice([0, 0, 1, 8, 40]), "p": rng.choice([0.0, 0.1, 0.25, 0.5, 0.9])}
    grad = rng.random() < 0.6
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    budget = 8192 * 4096 * 50021 if dtype == "bf16" else 1024 * 1001 * 21841
    while True:
        n, d, v = _log_int(rng, 1, 8192), _log_int(rng, 32, 25088), _log_int(rng, 2, 65536)
        if rng.random() < 0.5:
            d = (d + 63) // 64 * 64
        if n * d * v <= budget and n * v <= 8192 * 65536 and v * d <= 65536 * 4096:
            break
    return {"op": "xent", "grad": grad, "dtype": dtype, "n": n, "d": d, "v": v, "bias": rng.random() < 0.5,
            "reduction": rng.choice(["mean", "sum", "none"]), "ignored": rng.choice([0.0, 0.0, 0.1, 0.5]) if n >= 64 else 0.0,
            "smoothing": rng.choice([0.0, 0.0, 0.1])}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPE[case["dtype"]]
    st = {"case": case}
    if case["op"] == "dropout":
        rows, cols, pitch = case["rows"], case["cols"], case["pitch"]
        buf = torch.empty((rows, pitch), dtype=dt, device="cuda").normal_(generator=gen)
        x = buf[:, :cols]
        if not case["back"]:
            x.relu_()                       # activations behind a ReLU; gradients stay signed
        st.update(x=x, seed=(1234567 + 982451653 * seed) % 2 ** 63, offset=seed)
        return st
    n, d, v = case["n"], case["d"], case["v"]
    # post-ReLU features and a weight that gives logits a standard deviation of about two; frequent classes come first
    st["x"] = torch.empty((n, d), dtype=dt, device="cuda").normal_(generator=gen).relu_()
    st["w"] = torch.empty((v, d), dtype=dt, device="cuda").normal_(std=2.0 / math.sqrt(0.5 * d), generator=gen)
    st["bias"] = torch.empty(v, device="cuda").normal_(std=0.5, generator=gen) if case["bias"] else None
    u = torch.empty(n, dtype=torch.float64, device="cuda").uniform_(generator=gen)
    t = (u * u * v).long().clamp_(max=v - 1)
    if case["ignored"] > 0:
        t = torch.where(torch.empty(n, device="cuda").uniform_(generator=gen) < case["ignored"], torch.full_like(t, _IGNORE), t)
    st["target"] = t
    if own:
        import cudnntest_b200 as cb
        st["plan"] = cb.LinearXent(n, d, v, dtype="bf16" if case["dtype"] == "bf16" else "fp32x3", bias=case["bias"],
                                   reduction=case["reduction"], ignore_index=_IGNORE if case["ignored"] > 0 else None,
                                   label_smoothing=case["smoothing"], grad=case["grad"])
    return st


def _mulhilo(a, b):
    """Upper and lower 32 bits of a * b for 32-bit values held in 64-bit integers."""
    p0, p1 = (a & 0xFFFF) * b, (a >> 16) * b
    return (p1 + (p0 >> 16)) >> 16, (p0 + (p1 << 16)) & 0xFFFFFFFF


def _plain_dropout(st):
    case, x = st["case"], st["x"]
    rows, cols = case["rows"], case["cols"]
    count = rows * cols
    t16 = int(math.floor(case["p"] * 65536.0 + 0.5))
    g = torch.arange((count + 7) // 8, dtype=torch.int64, device=x.device)
    c = [g & 0xFFFFFFFF, g >> 32, torch.full_like(g, st["offset"] & 0xFFFFFFFF), torch.full_like(g, st["offset"] >> 32)]
    k0, k1 = st["seed"] & 0xFFFFFFFF, st["seed"] >> 32
    for _ in range(10):                     # Philox4x32-10 (Salmon et al. 2011)
        h0, l0 = _mulhilo(c[0], 0xD2511F53)
        h1, l1 = _mulhilo(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    r = torch.stack([h for w in c for h in (w & 0xFFFF, w >> 16)], dim=1).view(-1)[:count].view(rows, cols)
    scale = 65536.0 / (65536 - t16) if t16 < 65536 else 0.0
    return torch.where(r >= t16, x.float() * scale, torch.zeros((), device=x.device)).to(x.dtype)


def _plain_xent(st):
    """Logits in pieces of the vocabulary: a running maximum and sum, then the gradients piece by piece."""
    case, x, w, b, t = st["case"], st["x"], st["w"], st["bias"], st["target"]
    n, d, v, e = case["n"], case["d"], case["v"], case["smoothing"]
    xf = x.float()
    valid = t != _IGNORE
    if case["ignored"] > 0:
        xf = torch.where(valid[:, None], xf, torch.zeros((), device=x.device))
    tc = t.clamp(min=0)
    step = max(1, min(v, (1 << 29) // max(n, d)))
    pieces = [(lo, min(v, lo + step)) for lo in range(0, v, step)]

    def logits(lo, hi):
        z = xf @ w[lo:hi].float().t()
        return z + b[lo:hi] if b is not None else z

    m = torch.full((n,), -math.inf, device=x.device)
    s = torch.zeros(n, device=x.device)
    zt = torch.zeros(n, device=x.device)
    zsum = torch.zeros(n, device=x.device)
    rows = torch.arange(n, device=x.device)
    for lo, hi in pieces:
        z = logits(lo, hi)
        m2 = torch.maximum(m, z.amax(1))
        s = s * torch.exp(m - m2) + torch.exp(z - m2[:, None]).sum(1)
        m = m2
        inside = (tc >= lo) & (tc < hi)
        zt = torch.where(inside, z[rows, (tc - lo).clamp(0, hi - lo - 1)], zt)
        if e > 0:
            zsum = zsum + z.sum(1)
    lse = m + torch.log(s)
    loss = lse - (1 - e) * zt - (e / v) * zsum
    loss = torch.where(valid, loss, torch.zeros((), device=x.device))
    count = valid.sum().float()
    g = valid.float()
    if case["reduction"] == "mean":
        loss = loss.sum() / count.clamp(min=1)
        g = g / count.clamp(min=1)
    elif case["reduction"] == "sum":
        loss = loss.sum()
    if not case["grad"]:
        return {"loss": loss, "lse": torch.where(valid, lse, torch.zeros((), device=x.device))}
    dx = torch.zeros((n, d), device=x.device)
    dw = torch.empty_like(w)
    db = torch.empty(v, device=x.device) if b is not None else None
    for lo, hi in pieces:
        dz = torch.exp(logits(lo, hi) - lse[:, None]) - e / v
        inside = ((tc >= lo) & (tc < hi)).float()
        dz[rows, (tc - lo).clamp(0, hi - lo - 1)] -= (1 - e) * inside
        dz = dz * g[:, None]
        dx += dz @ w[lo:hi].float()
        dw[lo:hi] = (dz.t() @ xf).to(w.dtype)
        if db is not None:
            db[lo:hi] = dz.sum(0)
    out = {"loss": loss, "dx": dx.to(x.dtype), "dw": dw}
    if db is not None:
        out["db"] = db
    return out


def run(state):
    case = state["case"]
    if case["op"] == "dropout":
        if own:
            import cudnntest_b200 as cb
            call = cb.dropout_backward if case["back"] else cb.dropout
            return call(state["x"], case["p"], state["seed"], state["offset"])
        return _plain_dropout(state)
    if not own:
        return _plain_xent(state)
    plan = state["plan"]
    if not case["grad"]:
        loss, lse = plan.forward(state["x"], state["w"], state["target"], state["bias"])
        return {"loss": loss, "lse": lse}
    loss, dx, dw, db = plan.loss_and_grad(state["x"], state["w"], state["target"], state["bias"])
    out = {"loss": loss, "dx": dx, "dw": dw}
    if db is not None:
        out["db"] = db
    return out


def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "dropout":
        count = case["rows"] * case["cols"]
        return {"bytes": 2 * count * es, "flops": count}
    n, d, v = case["n"], case["d"], case["v"]
    loss = 4 * (n if case["reduction"] == "none" else 1) + (0 if case["grad"] else 4 * n)
    bias = 4 * v if case["bias"] else 0
    nbytes = (n * d + v * d) * es + 8 * n + bias + loss
    flops = 2 * n * d * v
    if case["grad"]:
        nbytes += (n * d + v * d) * es + bias
        flops *= 3
    return {"bytes": nbytes, "flops": flops}


def _exact_dropout(case, st):
    import numpy as np
    rows, cols = case["rows"], case["cols"]
    count = rows * cols
    t16 = int(math.floor(case["p"] * 65536.0 + 0.5))
    mask32, sh = np.uint64(0xFFFFFFFF), np.uint64(32)
    keep = np.empty(-(-count // 8) * 8, dtype=bool)
    for lo in range(0, len(keep) // 8, 1 << 17):
        idx = np.arange(lo, min(lo + (1 << 17), len(keep) // 8), dtype=np.uint64)
        ctr = [idx & mask32, idx >> sh, np.full_like(idx, st["offset"] & 0xFFFFFFFF), np.full_like(idx, st["offset"] >> 32)]
        key = [st["seed"] & 0xFFFFFFFF, st["seed"] >> 32]
        for _ in range(10):
            a, b = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
            ctr = [(b >> sh) ^ ctr[1] ^ np.uint64(key[0]), b & mask32, (a >> sh) ^ ctr[3] ^ np.uint64(key[1]), a & mask32]
            key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
        bits = np.stack(ctr, 1).astype("<u4").view("<u2").reshape(-1)
        keep[8 * lo:8 * lo + len(bits)] = bits.astype(np.int64) >= t16
    mask = torch.from_numpy(keep[:count].reshape(rows, cols)).cuda()
    return torch.where(mask, st["x"].double() * (65536.0 / max(1, 65536 - t16)), 0.0)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "dropout":
        return _exact_dropout(case, st)
    n, d, v, e = case["n"], case["d"], case["v"], case["smoothing"]
    t, valid = st["target"], st["target"] >= 0
    x, b = st["x"].double() * valid[:, None], st["bias"]
    count = int(valid.sum())
    weight = valid.double() / (max(1, count) if case["reduction"] == "mean" else 1)
    chunk = max(1, (1 << 28) // v)           # whole rows at a time: the softmax needs no running maximum
    losses, lses, dx = [], [], []
    dw = torch.zeros((v, d), dtype=torch.float64, device=x.device) if case["grad"] else None
    db = torch.zeros(v, dtype=torch.float64, device=x.device)
    wd = st["w"].double()
    for lo in range(0, n, chunk):
        xs, ts, vs = x[lo:lo + chunk], t[lo:lo + chunk].clamp(min=0), valid[lo:lo + chunk]
        z = xs @ wd.T
        if b is not None:
            z += b.double()
        lses.append(torch.logsumexp(z, 1))
        logp = z - lses[-1][:, None]
        losses.append((-(1 - e) * logp.gather(1, ts[:, None])[:, 0] - e / v * logp.sum(1)) * vs)
        if case["grad"]:
            q = torch.full_like(z, e / v).scatter_add_(1, ts[:, None], torch.full((len(ts), 1), 1 - e, dtype=z.dtype, device=z.device))
            dz = (logp.exp() - q) * weight[lo:lo + chunk, None]
            dx.append(dz @ wd)
            dw += dz.T @ xs
            db += dz.sum(0)
    loss = torch.cat(losses)
    if case["reduction"] != "none":
        loss = loss.sum() / (max(1, count) if case["reduction"] == "mean" else 1)
    if not case["grad"]:
        return {"loss": loss, "lse": torch.cat(lses) * valid}
    out = {"loss": loss, "dx": torch.cat(dx), "dw": dw}
    if b is not None:
        out["db"] = db
    return out
