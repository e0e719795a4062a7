"""Classifier head on the GPU, through the public entry points, against the definitions in 64 bits.

Tolerances are element-wise bounds, added up from the roundings that happen, not measured:
  * a rounding to BF16 is off by at most 2^-8 of the value, one to FP32 by 2^-24;
  * a sum of K terms on the tensor cores is off by at most (steps + 16) 2^-23 sum |terms|, one step per 16 terms (one
    truncation of the accumulator, and the alignment of the 16 products); FP32X3 leaves out products below 2^-25 of a term,
    and its six partial products take six times the steps;
  * a sum in FP32 arithmetic by K 2^-24 sum |terms|, one rounding per term;
  * ex2.approx is off by at most 2^-22, and exp(z - lse) by the errors of z and lse on top.
"""
import numpy as np
import pytest

from oracle import head

pytestmark = pytest.mark.gpu

BF, F32 = 2.0 ** -8, 2.0 ** -24


def _torch():
    import torch
    assert torch.cuda.is_available()
    return torch


def _sum_eps(k, dtype):
    """Relative (to the sum of magnitudes) error of a product with contraction length k."""
    steps = max(-(-k // 16) * (1 if dtype == "bf16" else 6), k / 2)
    return (steps + 17) * 2.0 ** -23


class Case:
    def __init__(self, n, d, v, dtype, seed=0, bias=True, ignored=0.0, ldx=0, ldw=0, ignore_index=-100, xscale=1.0):
        torch = _torch()
        self.n, self.d, self.v, self.dtype = n, d, v, dtype
        self.ldx, self.ldw = ldx, ldw
        self.tdt = torch.bfloat16 if dtype == "bf16" else torch.float32
        rng = np.random.default_rng(seed)
        xb = torch.full((n, ldx or d), float("nan"), dtype=self.tdt, device="cuda")
        wb = torch.full((v, ldw or d), float("nan"), dtype=self.tdt, device="cuda")
        self.x, self.w = xb[:, :d], wb[:, :d]
        self.x.copy_(torch.from_numpy(np.maximum(rng.standard_normal((n, d)), 0) * xscale))
        self.w.copy_(torch.from_numpy(rng.standard_normal((v, d)) * (2.0 / np.sqrt(0.5 * d))))
        self.bias = torch.from_numpy(rng.standard_normal(v).astype(np.float32)).cuda() if bias else None
        self.t = rng.integers(0, v, n)
        self.ignore_index = ignore_index if ignored > 0 else None
        if ignored > 0:
            self.t[rng.random(n) < ignored] = ignore_index
        self.target = torch.from_numpy(self.t).cuda()

    def plan(self, **kw):
        import cudnntest_b200 as cb
        return cb.LinearXent(self.n, self.d, self.v, dtype=self.dtype if self.dtype == "bf16" else "fp32x3", bias=self.bias is not None,
                             ignore_index=self.ignore_index, ldx=self.ldx, ldw=self.ldw, **kw)

    def oracle(self, reduction, smoothing=0.0, dloss=None):
        f = lambda a: None if a is None else a.double().cpu().numpy()
        self.xd, self.wd, self.bd = f(self.x), f(self.w), f(self.bias)
        if self.ignore_index is not None:
            self.xd = np.where((self.t == self.ignore_index)[:, None], 0.0, self.xd)
        return head.xent(self.xd, self.wd, self.t, self.bd, reduction, self.ignore_index, smoothing, dloss)

    def z_error(self, ref):
        """Bound on |z - z_exact| per element, on |lse - lse_exact| per row, on the relative error of exp(z - lse)."""
        ax, aw = np.abs(self.xd), np.abs(self.wd)
        ez = _sum_eps(self.d, self.dtype) * (ax @ aw.T) + 2 * F32 * (np.abs(ref["z"]) + (0 if self.bd is None else np.abs(self.bd)))
        # lse: the worst z, the exponentials' own errors, a sum of v of them and the logarithm
        el = ez.max(1) + 2.0 ** -20 + (self.v / 64 + 32) * 2.0 ** -23 + 4 * F32 * np.abs(ref["z"]).max(1)
        ep = ez + el[:, None] + 2.0 ** -20 + 2 * F32 * np.abs(ref["z"] - ref["z"].max(1, keepdims=True))
        return ez, el, ep

    def check(self, got, ref, reduction, g, smoothing=0.0):
        """got: loss, dx, dw, db (db may be None); g: weight of each row in the gradient."""
        loss, dx, dw, db = (None if a is None else a.double().cpu().numpy() for a in got)
        ez, el, ep = self.z_error(ref)
        counts = np.ones(self.n, bool) if self.ignore_index is None else self.t != self.ignore_index
        row = (el + ez.max(1) + 4 * F32 * (np.abs(ref["z"]).max(1) + np.abs(ref["lse"]))) * counts
        bound = row if reduction == "none" else row.sum() / (max(1, counts.sum()) if reduction == "mean" else 1) + 2 * F32 * np.abs(ref["loss"])
        assert (np.abs(loss - ref["loss"]) <= bound + 1e-30).all(), (np.abs(loss - ref["loss"]).max(), np.max(bound))
        # dz: the exponential's error, FP32 arithmetic, then the rounding (or the three parts, 2^-24) of the stored value
        p = np.exp(ref["z"] - np.where(counts, ref["lse"], np.inf)[:, None])
        store = BF if self.dtype == "bf16" else F32
        e32 = np.abs(g)[:, None] * (p * ep * 1.01 + 4 * F32 * (p + smoothing / self.v)) + 4 * F32 * np.abs(ref["dz"])
        e32[np.arange(self.n), np.where(counts, self.t, 0)] += 4 * F32 * np.abs(g)
        e32[~counts] = 0
        # an exponential below 2^-126 is flushed to 0, and so may be a part of a split value: at most 4 * 2^-126 in dz
        # before the row's weight (logits thousands apart make such values, and x of thousands carries them into dW)
        # Without a bias BF16 may hold the exponentials before dz is made of them: one more rounding of p.
        if self.dtype == "bf16" and self.bd is None:
            e32 = e32 + np.abs(g)[:, None] * BF * 1.01 * p * counts[:, None]
        edz = e32 + store * (np.abs(ref["dz"]) + e32) + (np.abs(g) * counts)[:, None] * 2.0 ** -124
        adz = np.abs(ref["dz"]) + edz
        out = BF if self.dtype == "bf16" else F32
        for name, val, eb, mag, k in (("dx", dx, edz @ np.abs(self.wd), adz @ np.abs(self.wd), self.v),
                                      ("dw", dw, edz.T @ np.abs(self.xd), adz.T @ np.abs(self.xd), self.n)):
            if val is None:
                continue
            err, tol = np.abs(val - ref[name]), eb + (_sum_eps(k, self.dtype) + 64 * F32) * mag
            tol = tol + out * (np.abs(ref[name]) + tol) + 1e-37
            assert np.isfinite(val).all(), name
            assert (err <= tol).all(), (name, err.max(), (err / tol).max())
        if db is not None:
            assert (np.abs(db - ref["db"]) <= e32.sum(0) + (self.n / 8 + 40) * F32 * adz.sum(0) + 1e-37).all()


# what each case reaches is in its comment: which kernels, and which ragged edge
CASES = [
    # n, d, v, dtype, extra
    (1, 1, 1, "bf16", {}),                                        # one of everything; loss is 0
    (1, 1, 1, "fp32", {}),
    (1, 4096, 1000, "bf16", {}),                                  # one row, split contraction
    (16, 4096, 1000, "fp32", {}),
    (32, 512, 10, "fp32", {}),                                    # one tile, all operands inside a box
    (33, 65, 257, "bf16", {}),                                    # one past a warp, a slice and a tile; rows not 16-byte multiples
    (129, 63, 255, "fp32", {}),
    (257, 72, 300, "bf16", dict(bias=False)),                     # one past a pair tile
    (300, 200, 1100, "bf16", dict(ldx=208, ldw=216)),             # pitches that TMA takes
    (300, 200, 1100, "bf16", dict(ldx=201, ldw=203)),             # pitches that need repacking
    (300, 201, 1100, "fp32", dict(ldx=204, ldw=201)),
    (2305, 40, 2100, "bf16", {}),                                 # statistics in the epilogue, logits recomputed
    (2305, 40, 2100, "fp32", {}),
    (2304, 1024, 2050, "bf16", {}),                               # logits kept as floats, contraction not split
    (2304, 300, 2050, "fp32", {}),
    (2304, 1024, 2050, "bf16", dict(bias=False)),                 # logits kept as exponentials
    (2500, 24, 2303, "bf16", dict(bias=False)),
    (600, 1100, 9001, "bf16", {}),                                # rows too wide for one kernel: statistics with the product
    (1100, 300, 9000, "fp32", {}),
    (20, 4096, 9001, "bf16", {}),                                 # the same with a split contraction
    (20, 1025, 9002, "fp32", {}),
    (100, 3000, 8000, "bf16", {}),                                # the widest row of the one-kernel path, and narrower ones
    (100, 900, 4000, "fp32", {}),
    (700, 1500, 1900, "bf16", {}),
    (1000, 40, 100, "fp32", {}),                                  # plain FP32 kernels up to their most rows and classes
    (3, 1001, 1024, "bf16", {}),
    (16, 1001, 3000, "fp32", {}),                                 # W split inside the products
    (9, 1001, 3000, "bf16", dict(bias=False)),
    (8, 1002, 3000, "bf16", {}),
    (3, 260, 70001, "fp32", dict(ldx=264, ldw=261)),
    (13, 6001, 130, "fp32", {}),
    (100, 515, 31, "bf16", {}),                                   # logits, softmax and dz in one kernel; ragged widths
    (128, 128, 128, "fp32", {}),
    (9, 2050, 7, "fp32", dict(bias=False, ldx=2053, ldw=2052)),
    (7, 40, 128, "bf16", {}),
    (3000, 3001, 3, "fp32", {}),                                  # few classes: FP32 arithmetic on the caller's matrices
    (2777, 1000, 16, "fp32", dict(ldx=1003, ldw=1001)),
    (9000, 260, 1, "fp32", {}),
    (300, 202, 1100, "bf16", {}),                                 # repacked by pairs
    (300, 600, 70, "bf16", dict(ldx=603, ldw=604)),
    (17, 1001, 3000, "fp32", {}),
    (64, 1001, 3000, "fp32", {}),
    (300, 2200, 700, "bf16", dict(bias=False)),                   # blocks of the contraction: 1024 + 1024 + 152
    (2100, 700, 2400, "fp32", {}),                                # 256 + 256 + 188, logits recomputed below
    (4000, 64, 5, "bf16", {}),                                    # long contraction of dW over rows, few classes
    (5, 48, 20000, "fp32", {}),                                   # long contraction of dx over classes, few rows
]


@pytest.mark.parametrize("n,d,v,dtype,kw", CASES)
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_gradient_against_definition(n, d, v, dtype, kw, reduction):
    torch = _torch()
    c = Case(n, d, v, dtype, seed=n + d + v, **kw)
    up = np.random.default_rng(1).standard_normal(n if reduction == "none" else 1).astype(np.float32)
    dloss = torch.from_numpy(up).cuda()
    ref = c.oracle(reduction, dloss=up.astype(np.float64))
    plan = c.plan(reduction=reduction)
    got = plan.loss_and_grad(c.x, c.w, c.target, c.bias, dloss=dloss)
    g = up.astype(np.float64) * np.ones(n) / (n if reduction == "mean" else 1)
    c.check(got, ref, reduction, g)
    again = plan.loss_and_grad(c.x, c.w, c.target, c.bias, dloss=dloss)
    for a, b in zip(got, again):
        assert (a is None and b is None) or torch.equal(a, b)     # deterministic, and the scratch holds nothing over
    import cudnntest_b200 as cb
    cb.device_status()


@pytest.mark.parametrize("n,d,v,dtype", [(40, 4096, 1000, "bf16"), (300, 96, 700, "fp32"), (2305, 40, 2100, "bf16"), (2305, 40, 2100, "fp32"),
                                         (15, 2300, 700, "fp32"), (7, 2301, 700, "bf16"), (100, 64, 100, "bf16"), (700, 3100, 9, "fp32"), (60, 3000, 100, "fp32"), (5, 700, 4000, "fp32")])
@pytest.mark.parametrize("ignored", [0.3, 1.0])
@pytest.mark.parametrize("ignore_index", [-100, 3, 2 ** 62])
def test_ignored_rows_leave_no_trace(n, d, v, dtype, ignored, ignore_index):
    """Rows with the ignored target may hold NaN; with every row ignored loss and gradients are exactly 0.  The ignored
    index may be a class of its own."""
    torch = _torch()
    c = Case(n, d, v, dtype, seed=3, ignored=ignored, ignore_index=ignore_index)
    off = torch.from_numpy(c.t == ignore_index).cuda()
    c.x[off] = float("nan")
    ref = c.oracle("mean", smoothing=0.1)
    got = c.plan(reduction="mean", label_smoothing=0.1).loss_and_grad(c.x, c.w, c.target, c.bias)
    counts = c.t != ignore_index
    c.check(got, ref, "mean", counts / max(1, counts.sum()), smoothing=0.1)
    assert (got[1][off] == 0).all()
    loss, lse = c.plan(reduction="none", label_smoothing=0.1, grad=False).forward(c.x, c.w, c.target, c.bias)
    assert (loss[off] == 0).all() and (lse[off] == 0).all() and torch.isfinite(loss).all()
    if ignored == 1.0:
        for a in got:
            assert (a == 0).all()


@pytest.mark.parametrize("n,d,v,dtype", [(1, 1, 1, "bf16"), (16, 4096, 1000, "bf16"), (777, 512, 1000, "fp32"), (2305, 40, 2100, "bf16"),
                                         (2305, 40, 2100, "fp32"), (3, 50, 70000, "bf16"),
                                         (500, 96, 33, "fp32"), (8, 512, 10, "bf16"), (500, 2000, 100, "bf16")])
@pytest.mark.parametrize("smoothing", [0.0, 0.2, 1.0])
def test_forward_against_definition(n, d, v, dtype, smoothing):
    c = Case(n, d, v, dtype, seed=11)
    mean = c.plan(reduction="mean", label_smoothing=smoothing, grad=False).forward(c.x, c.w, c.target, c.bias)
    ref = c.oracle("none", smoothing)
    loss, lse = c.plan(reduction="none", label_smoothing=smoothing, grad=False).forward(c.x, c.w, c.target, c.bias)
    ez, el, _ = c.z_error(ref)
    assert (np.abs(lse.double().cpu().numpy() - ref["lse"]) <= el + 2 * F32 * np.abs(ref["lse"])).all()
    row = el + ez.max(1) + (8 + smoothing * v / 64) * F32 * (np.abs(ref["z"]).max(1) + np.abs(ref["lse"]))
    assert (np.abs(loss.double().cpu().numpy() - ref["loss"]) <= row).all()
    assert abs(float(mean[0]) - ref["loss"].mean()) <= row.mean() + 2 * F32 * abs(ref["loss"].mean())
    assert (np.abs(mean[1].double().cpu().numpy() - ref["lse"]) <= el + 2 * F32 * np.abs(ref["lse"])).all()


# The longer float matrix split inside the products: W (one past and up to both widths of a tile of rows), or x with up to 128
# classes; features, classes and rows that end inside a tile, a step of 64 and a block of 256; rows on any boundary; statistics
# in one kernel and in two; more parts than one.  (8 rows: FP32 arithmetic instead.)
LONG_W = [(8, 1001, 3001, {}), (9, 2001, 1000, {}), (17, 4099, 300, {}), (64, 2048, 1000, dict(ldw=2052)), (65, 1023, 2001, dict(ldw=1030, ldx=1027)),
          (65, 1023, 17001, dict(ldw=1030, ldx=1027)), (128, 515, 8201, {}), (128, 2055, 8201, {}), (100, 64, 17000, dict(bias=False)),
          (33, 20001, 130, dict(ldw=20004)), (127, 1000, 17841, dict(ldw=1001)), (128, 128, 8192, {}),
          (3001, 1030, 17, {}), (2777, 1001, 64, dict(ldx=1003)), (1025, 1500, 33, dict(bias=False, ldx=1504)), (17001, 1000, 100, dict(ldw=1001)),
          (8200, 2052, 128, {}), (131, 9001, 70, {})]


@pytest.mark.parametrize("n,d,v,kw", LONG_W)
@pytest.mark.parametrize("ignored,smoothing", [(0.0, 0.0), (0.3, 0.1)])
def test_long_float_weight(n, d, v, kw, ignored, smoothing):
    torch = _torch()
    c = Case(n, d, v, "fp32", seed=101, ignored=ignored, **kw)
    off = torch.from_numpy(c.t == -100).cuda()
    c.x[off] = float("nan")
    ref = c.oracle("mean", smoothing=smoothing)
    plan = c.plan(reduction="mean", label_smoothing=smoothing, lddx=d + 1, lddw=d + 3)
    bx, bw = torch.full((n + 1, d + 1), 5.0, device="cuda"), torch.full((v + 1, d + 3), 5.0, device="cuda")
    got = plan.loss_and_grad(c.x, c.w, c.target, c.bias, dx=bx[:n, :d], dw=bw[:v, :d])
    counts = c.t != -100
    c.check(got, ref, "mean", counts / counts.sum(), smoothing=smoothing)
    assert (bx[n:] == 5).all() and (bx[:, d:] == 5).all() and (bw[v:] == 5).all() and (bw[:, d:] == 5).all()
    again = plan.loss_and_grad(c.x, c.w, c.target, c.bias)
    assert all((a is None and b is None) or torch.equal(a, b) for a, b in zip(got, again))
    only = plan.loss_and_grad(c.x, c.w, c.target, c.bias, need_dw=False)
    assert only[2] is None and torch.equal(only[0], got[0]) and torch.equal(only[1], got[1])
    loss, lse = c.plan(reduction="none", label_smoothing=smoothing, grad=False).forward(c.x, c.w, c.target, c.bias)
    rows = c.oracle("none", smoothing)
    ez, el, _ = c.z_error(rows)
    keep = counts & np.isfinite(rows["lse"])
    row = el + ez.max(1) + (8 + smoothing * v / 64) * F32 * (np.abs(rows["z"]).max(1) + np.abs(rows["lse"]))
    assert (np.abs(loss.double().cpu().numpy() - rows["loss"])[keep] <= row[keep]).all() and (loss[off] == 0).all() and (lse[off] == 0).all()
    import cudnntest_b200 as cb
    cb.device_status()


@pytest.mark.parametrize("n,d,v,ldx,ldw", [(20, 200, 6000, 0, 0), (20, 201, 6000, 0, 0), (6000, 200, 20, 0, 0), (6000, 200, 20, 203, 201)])
def test_long_floats_near_the_largest_float(n, d, v, ldx, ldw):
    """Floats that would round to BF16's infinity, in the matrix that is split inside the products."""
    torch = _torch()
    c = Case(n, d, v, "fp32", seed=111, ldx=ldx, ldw=ldw)
    long, short = (c.w, c.x) if n < v else (c.x, c.w)
    far = torch.tensor([3.4e38, -3.4e38, 3.3961775e38, 1.0], device="cuda")
    long[:, 0] = far[torch.arange(long.shape[0], device="cuda") % 4]
    short[:, 0] = 2.0 ** -100 * (1 + torch.arange(short.shape[0], device="cuda") / 64)
    ref = c.oracle("none")
    assert np.abs(ref["z"]).max() > 2.0 ** 27
    loss, lse = c.plan(reduction="none", grad=False).forward(c.x, c.w, c.target, c.bias)
    ez, el, _ = c.z_error(ref)
    assert (np.abs(lse.double().cpu().numpy() - ref["lse"]) <= el + 2 * F32 * np.abs(ref["lse"])).all()
    row = el + ez.max(1) + 8 * F32 * (np.abs(ref["z"]).max(1) + np.abs(ref["lse"]))
    assert (np.abs(loss.double().cpu().numpy() - ref["loss"]) <= row).all()


@pytest.mark.parametrize("n,d,v", [(40, 600, 3000), (3000, 600, 40)])
def test_long_float_matrix_in_a_graph(n, d, v):
    """A captured call, replayed on other values and beside an eager call on another stream: the same as eager."""
    torch = _torch()
    c = Case(n, d, v, "fp32", seed=121)
    plan, other = c.plan(reduction="mean"), c.plan(reduction="mean")
    plan.loss_and_grad(c.x, c.w, c.target, c.bias)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = plan.loss_and_grad(c.x, c.w, c.target, c.bias)
    for _ in range(2):
        c.x.mul_(0.75)
        c.w.mul_(-1.25)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        g.replay()
        with torch.cuda.stream(side):
            eager = other.loss_and_grad(c.x, c.w, c.target, c.bias)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))
    import cudnntest_b200 as cb
    cb.device_status()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n,d,v,limit", [(700, 130, 3000, 1), (2305, 40, 2100, 2305 * 2 * 600), (600, 1032, 11000, 1 << 20)])
def test_pieces_of_the_vocabulary(dtype, n, d, v, limit):
    """A small scratch limit: the gradient in several pieces, dx added up over them, ragged last piece."""
    c = Case(n, d, v, dtype, seed=21)
    ref = c.oracle("sum", smoothing=0.1)
    got = c.plan(reduction="sum", label_smoothing=0.1, scratch_limit=limit).loss_and_grad(c.x, c.w, c.target, c.bias)
    c.check(got, ref, "sum", np.ones(n), smoothing=0.1)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n,v", [(64, 900), (2305, 2100)])
@pytest.mark.parametrize("low", [-np.inf, -3.4028234663852886e38])
def test_classes_masked_by_the_bias(dtype, n, v, low):
    """Classes with a bias of -inf or of the lowest float: probability 0, no NaN, even where they fill whole tiles."""
    torch = _torch()
    c = Case(n, 48, v, dtype, seed=31)
    mask = np.ones(v, bool)
    mask[600:700] = False
    mask[5] = False
    c.bias[torch.from_numpy(mask).cuda()] = float(low)
    c.t = 600 + c.t % 100
    c.target = torch.from_numpy(c.t).cuda()
    live = ~mask
    loss, dx, dw, db = c.plan(reduction="mean").loss_and_grad(c.x, c.w, c.target, c.bias)
    f = lambda a: a.double().cpu().numpy()
    # the same problem without the masked classes
    sub = Case(n, 48, v, dtype, seed=31)
    sub.w, sub.bias, sub.t, sub.v = c.w[torch.from_numpy(live).cuda()], c.bias[torch.from_numpy(live).cuda()], np.cumsum(live)[c.t] - 1, int(live.sum())
    ref = sub.oracle("mean")
    sub.check((loss, dx, dw[torch.from_numpy(live).cuda()], db[torch.from_numpy(live).cuda()]), ref, "mean", np.full(n, 1.0 / n))
    assert (f(dw)[mask] == 0).all() and (f(db)[mask] == 0).all()


def test_infinite_and_nan_logits_reach_their_row_only():
    torch = _torch()
    for n, v in ((40, 300), (2305, 2100)):
        c = Case(n, 64, v, "bf16", seed=41, bias=False)
        c.x[7, 3] = float("nan")
        loss, lse = c.plan(reduction="none", grad=False).forward(c.x, c.w, c.target)
        bad = torch.isnan(loss)
        assert bad[7] and int(bad.sum()) == 1 and torch.isnan(lse[7])


def test_far_logits():
    """Logits of several thousand: the maximum is taken out before anything is exponentiated."""
    c = Case(50, 256, 700, "fp32", seed=51, xscale=1000.0)
    ref = c.oracle("none")
    assert np.abs(ref["z"]).max() > 3000
    c.check(c.plan(reduction="none").loss_and_grad(c.x, c.w, c.target, c.bias), ref, "none", np.ones(50))


def test_float_operands_near_the_largest_float():
    """Splitting a float into BF16 parts must not overflow where the float does not."""
    torch = _torch()
    c = Case(4, 8, 5, "fp32", seed=61, bias=False)
    c.x.zero_()
    c.x[:, 0] = torch.tensor([3.4e38, -3.4e38, 3.0e38, 1.0], device="cuda")
    c.w.mul_(1e-37)
    ref = c.oracle("none")
    loss, _ = c.plan(reduction="none", grad=False).forward(c.x, c.w, c.target)
    # The weights here are near 2^-122: the third BF16 part of such a float lies below BF16's smallest value, 2^-133, so a
    # weight is off by up to 2^-134, times |x| < 2^128 a logit by up to 2^-6; a loss is the difference of two of them.
    small = 2 * 2.0 ** -6 * np.abs(c.xd).max(1) / 2.0 ** 128
    assert (np.abs(loss.double().cpu().numpy() - ref["loss"]) <= small + 1e-4 * (1 + np.abs(ref["z"]).max())).all()


def test_target_out_of_range_is_reported():
    torch = _torch()
    import cudnntest_b200 as cb
    for bad in (-1, 300, 2 ** 40):
        for n in (40, 2305):
            c = Case(n, 64, 300 if n == 40 else 2100, "bf16", seed=71)
            c.target[3] = bad if n == 40 else (bad if bad != 300 else 2100)
            loss, dx, dw, db = c.plan(reduction="none").loss_and_grad(c.x, c.w, c.target, c.bias)
            assert torch.isnan(loss[3]) and int(torch.isnan(loss).sum()) == 1
            assert (dx[3] == 0).all() and torch.isfinite(dw.float()).all() and torch.isfinite(db).all()
            with pytest.raises(cb.WinoError) as e:
                cb.device_status()
            assert e.value.code == cb._lib.E_BADARG
            cb.device_status()


def test_no_rows():
    torch = _torch()
    import cudnntest_b200 as cb
    for dtype, tdt in (("bf16", torch.bfloat16), ("fp32x3", torch.float32)):
        plan = cb.LinearXent(0, 24, 10, dtype=dtype, bias=True, lddw=40)
        x, w = torch.empty(0, 24, dtype=tdt, device="cuda"), torch.ones(10, 24, dtype=tdt, device="cuda")
        buf = torch.full((10, 40), 7.0, dtype=tdt, device="cuda")
        loss, dx, dw, db = plan.loss_and_grad(x, w, torch.empty(0, dtype=torch.int64, device="cuda"), torch.ones(10, device="cuda"), dw=buf[:, :24])
        assert float(loss) == 0 and dx.shape == (0, 24) and (dw == 0).all() and (db == 0).all() and (buf[:, 24:] == 7).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n,d,v", [(300, 200, 700), (2305, 40, 2100), (14, 301, 7001), (100, 60, 100), (7300, 301, 10), (300, 206, 700)])
@pytest.mark.parametrize("pad", [0, 1, 2, 8])
def test_outputs_stay_inside_their_rows(dtype, n, d, v, pad):
    """dx and dw inside wider buffers with guard rows: nothing but the results is written; left-out products cost nothing."""
    torch = _torch()
    c = Case(n, d, v, dtype, seed=81)
    ref = c.oracle("mean")
    plan = c.plan(reduction="mean", lddx=d + pad, lddw=d + pad)
    bx = torch.full((n + 2, d + pad), 5.0, dtype=c.tdt, device="cuda")
    bw = torch.full((v + 2, d + pad), 5.0, dtype=c.tdt, device="cuda")
    got = plan.loss_and_grad(c.x, c.w, c.target, c.bias, dx=bx[:n, :d], dw=bw[:v, :d])
    c.check(got, ref, "mean", np.full(n, 1.0 / n))
    for b, rows in ((bx, n), (bw, v)):
        assert (b[rows:] == 5).all() and (b[:rows, d:] == 5).all()
    fresh = plan.loss_and_grad(c.x, c.w, c.target, c.bias)                       # allocated by the call
    assert all(torch.equal(a, b) for a, b in zip(fresh, got)) and fresh[1].shape == c.x.shape and (n < 2 or fresh[1].stride(0) == d + pad)
    only = plan.loss_and_grad(c.x, c.w, c.target, c.bias, need_dx=False)
    assert only[1] is None and torch.equal(only[2], got[2]) and torch.equal(only[3], got[3])
    only = plan.loss_and_grad(c.x, c.w, c.target, c.bias, need_dw=False)
    assert only[2] is None and torch.equal(only[1], got[1])


def test_results_have_the_pitch_of_the_plan():
    """Inputs and results of the same wide pitch: what the call allocates is laid out by the plan, not like the input."""
    torch = _torch()
    import cudnntest_b200 as cb
    c = Case(50, 40, 60, "bf16", seed=5, ldx=64, ldw=64)
    got = c.plan(lddx=64, lddw=64, reduction="mean").loss_and_grad(c.x, c.w, c.target, c.bias)
    assert got[1].stride() == (64, 1) and got[2].stride() == (64, 1)
    c.check(got, c.oracle("mean"), "mean", np.full(50, 1.0 / 50))


def test_python_checks():
    torch = _torch()
    import cudnntest_b200 as cb
    c = Case(20, 32, 40, "bf16")
    plan = c.plan()
    args = dict(x=c.x, w=c.w, target=c.target, bias=c.bias)
    for bad in (dict(x=c.x.float()), dict(x=c.x[:10]), dict(x=c.x.t().contiguous().t()), dict(w=c.w[:, :16]), dict(target=c.target.int()),
                dict(target=c.target[:5]), dict(bias=None), dict(bias=c.bias.double()), dict(x=c.x.cpu())):
        with pytest.raises(ValueError):
            plan.loss_and_grad(**{**args, **bad})
    with pytest.raises(ValueError):
        c.plan(grad=False).loss_and_grad(**args)
    with pytest.raises(ValueError):
        plan.loss_and_grad(**args, dloss=torch.ones(20, device="cuda"))
    with pytest.raises(cb.WinoError):                             # a view that starts inside a 16-byte unit
        wide = torch.zeros(20, 40, dtype=torch.bfloat16, device="cuda")
        cb.LinearXent(20, 32, 40, ldx=40).forward(wide[:, 1:33], c.w, c.target)


# ---- dropout ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (257,), (64, 4096), (33, 65), (3, 5, 7), (1000, 3)])
def test_dropout_against_definition(dtype, p, shape):
    """The mask is exact; a kept value is the product with the FP32 scale (off by 2^-24), rounded to the type."""
    torch = _torch()
    import cudnntest_b200 as cb
    tdt = torch.bfloat16 if dtype == "bf16" else torch.float32
    x = torch.randn(shape, generator=torch.Generator().manual_seed(1)).to(tdt).cuda()
    seed, offset = 0x123456789ABCDEF0, 2 ** 40 + 5
    y = cb.dropout(x, p, seed, offset)
    ref = head.dropout(x.double().cpu().numpy(), p, seed, offset)
    got = y.double().cpu().numpy()
    assert ((got == 0) == (ref == 0)).all()
    assert (np.abs(got - ref) <= (2 * F32 + (BF if dtype == "bf16" else F32)) * np.abs(ref)).all()
    assert torch.equal(cb.dropout_backward(x, p, seed, offset), y)
    assert torch.equal(cb.dropout(x.clone(), p, seed, offset - 9, offset_dev=torch.tensor([9], device="cuda")), y)
    inplace = x.clone()
    assert cb.dropout(inplace, p, seed, offset, out=inplace) is inplace and torch.equal(inplace, y)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,cols,ldx,ldy", [(37, 64, 72, 64), (37, 64, 64, 80), (37, 65, 72, 65), (5, 3, 4, 9), (100, 40, 41, 43), (1, 24, 24, 24)])
def test_dropout_strided(dtype, rows, cols, ldx, ldy):
    """The mask belongs to the dense element index, whatever the pitches; gaps are left as they were."""
    torch = _torch()
    import cudnntest_b200 as cb
    tdt = torch.bfloat16 if dtype == "bf16" else torch.float32
    xb = torch.randn((rows, ldx), generator=torch.Generator().manual_seed(2)).to(tdt).cuda()
    yb = torch.full((rows, ldy), 3.0, dtype=tdt, device="cuda")
    x = xb[:, :cols]
    y = cb.dropout(x, 0.3, 99, 1, out=yb[:, :cols])
    assert torch.equal(y, cb.dropout(x.contiguous(), 0.3, 99, 1)) and (yb[:, cols:] == 3).all()
    assert torch.equal(cb.dropout(x, 0.3, 99, 1), y)


def test_dropout_drops_what_is_not_finite():
    torch = _torch()
    import cudnntest_b200 as cb
    for tdt in (torch.bfloat16, torch.float32):
        for count in (4096, 4099):
            x = torch.full((count,), float("nan"), dtype=tdt, device="cuda")
            keep = torch.from_numpy(head.dropout_keep(0, count, 0.5, 5, 0)).cuda()
            y = cb.dropout(x, 0.5, 5)
            assert (y[~keep] == 0).all() and torch.isnan(y[keep]).all()


def test_dropout_far_offsets():
    """Elements past 2^32: the group index keeps its upper half."""
    torch = _torch()
    import cudnntest_b200 as cb
    count = 2 ** 32 + 64
    x = torch.ones(count, dtype=torch.bfloat16, device="cuda")
    y = cb.dropout(x, 0.5, 77, 3, out=x)
    for first in (0, 2 ** 31 - 32, 2 ** 32 - 64):
        keep = head.dropout_keep(first, 128, 0.5, 77, 3)
        assert ((y[first:first + 128].float().cpu().numpy() != 0) == keep).all()


def test_dropout_in_a_graph_draws_again():
    torch = _torch()
    import cudnntest_b200 as cb
    x = torch.ones(64, 256, device="cuda")
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    y = torch.empty_like(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cb.dropout(x, 0.5, 11, offset_dev=step, out=y)
        step.add_(1)
    for i in range(3):
        g.replay()
        assert torch.equal(y, cb.dropout(x, 0.5, 11, i))


# ---- together --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_training_step_of_a_head(dtype):
    """features -> dropout -> linear + cross entropy -> gradients -> dropout backward, eagerly, on a side stream and as a
    replayed graph: the same bits; and against the definition, composed."""
    torch = _torch()
    import cudnntest_b200 as cb
    c = Case(200, 512, 100, dtype, seed=91, ignored=0.1)
    plan = c.plan(reduction="mean")

    def step():
        h = cb.dropout(c.x, 0.5, 17, 4)
        loss, dh, dw, db = plan.loss_and_grad(h, c.w, c.target, c.bias)
        return h, loss, cb.dropout_backward(dh, 0.5, 17, 4), dh, dw, db
    eager = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = step()
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    for a, b, d in zip(eager, other, captured):
        assert torch.equal(a, b) and torch.equal(a, d)
    h, loss, dx, dh, dw, db = eager
    feats = c.x
    c.x = h
    ref = c.oracle("mean")
    counts = c.t != -100
    c.check((loss, dh, dw, db), ref, "mean", counts / counts.sum())
    keep = head.dropout_keep(0, feats.numel(), 0.5, 17, 4).reshape(feats.shape)
    assert np.array_equal(dx.float().cpu().numpy(), np.where(keep, dh.float().cpu().numpy() * 2, 0))


def test_two_plans_in_two_graphs_share_nothing():
    torch = _torch()
    a, b = Case(40, 256, 300, "bf16", seed=1), Case(2305, 40, 2100, "bf16", seed=2)
    pa, pb = a.plan(), b.plan()
    want = pa.loss_and_grad(a.x, a.w, a.target, a.bias), pb.loss_and_grad(b.x, b.w, b.target, b.bias)
    graphs, outs = [], []
    for c, p in ((a, pa), (b, pb)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(p.loss_and_grad(c.x, c.w, c.target, c.bias))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        for x, y in zip(w, o):
            assert torch.equal(x, y)


@pytest.mark.parametrize("n,d,v", [(6, 40, 9), (300, 64, 20)])
def test_gradient_against_differences(n, d, v):
    """Central differences of the library's own loss along random directions (FP32X3, one loss per row).

    With step h along a unit direction u: truncation is below h^2 / 6 |third derivative| <= h^2 (2 max|W u|)^3, each loss is
    off by at most its own bound, so the quotient by (sum of row bounds) / h."""
    torch = _torch()
    c = Case(n, d, v, "fp32", seed=101)
    plan = c.plan(reduction="none")
    loss, dx, dw, db = plan.loss_and_grad(c.x, c.w, c.target, c.bias)
    ref = c.oracle("none")
    ez, el, _ = c.z_error(ref)
    row = (el + ez.max(1) + 4 * F32 * (np.abs(ref["z"]).max(1) + np.abs(ref["lse"]))).sum() * 1.1
    gen = torch.Generator(device="cuda").manual_seed(7)
    h = 2.0 ** -5
    for which, grad in (("x", dx), ("w", dw), ("bias", db)):
        base = getattr(c, which)
        u = torch.randn(base.shape, generator=gen, device="cuda")
        u /= u.norm()
        vals = []
        for sign in (1, -1):
            moved = {k: getattr(c, k) for k in ("x", "w", "bias")}
            moved[which] = (base + sign * h * u).contiguous()
            vals.append(plan.loss_and_grad(moved["x"], moved["w"], c.target, moved["bias"])[0].double().sum().item())
            step = (moved[which] - base).abs().max()
        got = (vals[0] - vals[1]) / (2 * h)
        want = (grad.double() * u.double()).sum().item()
        f = lambda a: a.double().cpu().numpy()
        zu = np.abs({"x": lambda: f(u) @ c.wd.T, "w": lambda: c.xd @ f(u).T, "bias": lambda: np.tile(f(u), (n, 1))}[which]())
        third = ((2 * zu.max(1)) ** 3).sum()
        moved_rounding = 2 * F32 * float(base.abs().max()) / h * float(grad.abs().sum())
        assert abs(got - want) <= h * h * third + row / h + moved_rounding + 1e-5 * abs(want), which


# ---- where the framework itself calls them -----------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "fp32x3"])
@pytest.mark.parametrize("layout", ["NHWC", "NCHW"])
def test_classifier_head_on_the_convolution_stack(dtype, layout):
    """The stack's features through the head: loss and gradients against the definition on those features; the mask of a
    call follows from its number."""
    torch = _torch()
    from cudnntest_b200 import vgg
    layers = [(3, 64, 16, False), (64, 64, 16, True), (64, 128, 8, True)]
    stack = vgg.VGG16ConvStack(20, layout=layout, dtype=dtype, layers=layers)
    head_ = vgg.ClassifierHead(20, 128 * 4 * 4, 30, dtype=dtype, ignore_index=-1, label_smoothing=0.1)
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(stack.in_shape, generator=gen, device="cuda").to(stack.io_dtype)
    feats = stack(x).clone()
    target = torch.arange(20, device="cuda")
    target[4] = -1
    plain = head_.loss(feats, target)
    for step in range(2):
        loss, dx, dw, db = head_.loss_and_grad(feats, target, need_dx=True)
        keep = head.dropout_keep(0, feats.numel(), 0.5, head_.seed, step).reshape(20, -1)
        flat = feats.reshape(20, -1)
        c = Case.__new__(Case)
        c.n, c.d, c.v, c.dtype, c.ignore_index = 20, 2048, 30, "bf16" if dtype == "bf16" else "fp32", -1
        c.t = target.cpu().numpy()
        c.x = flat * torch.from_numpy(keep).cuda() * 2
        c.w, c.bias = head_.weight, head_.bias
        counts = c.t != -1
        ref = c.oracle("mean", smoothing=0.1)
        dh = dx.reshape(20, -1).double() / 2                     # exact: dropout's factor at p = 1/2
        back = torch.from_numpy(keep).cuda()
        assert (dh[~back] == 0).all()
        ref_dx = ref["dx"]
        ref["dx"] = np.where(keep, ref_dx, 0.0)
        c.check((loss, dh, dw, db), ref, "mean", counts / counts.sum(), smoothing=0.1)
    assert head_.steps == 2 and torch.isfinite(plain)
    assert head_.loss_and_grad(feats, target)[1] is None
    with pytest.raises(ValueError):
        head_.loss(feats[:, :1], target)


def test_net_test_reports_the_cross_entropy():
    """netTest tail=1: the batch's cross entropy from the library agrees with the harness's restatement in double."""
    import json
    import os
    import subprocess
    exe = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cudnntest_b200", "harness", "bin", "netTest")
    out = subprocess.run([exe, "set", "batch=3", "mode=1", "dtype=bf16", "rounds=1", "tail=1"], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "classifier tail error" not in out.stdout, out.stdout + out.stderr
    s = json.loads([l for l in out.stdout.splitlines() if l.startswith("{")][-1])
    assert s["tail_loss"] > 0 and s["tail_loss_max_err"] <= 1e-4
