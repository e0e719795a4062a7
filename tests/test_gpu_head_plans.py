"""Calls of the classifier head that go across plans, sizes and streams, against the definitions in 64 bits.

Cases, bounds and their derivation are those of test_gpu_head.py.
"""
import numpy as np
import pytest

from test_gpu_head import F32, Case, _torch

pytestmark = pytest.mark.gpu


def _check_forward(c, plan, reduction, smoothing=0.0):
    """forward of a plan with reduction "mean", "sum" or "none" against the definition, element by element."""
    loss, lse = (a.double().cpu().numpy() for a in plan.forward(c.x, c.w, c.target, c.bias))
    ref = c.oracle("none", smoothing)
    ez, el, _ = c.z_error(ref)
    counts = np.ones(c.n, bool) if c.ignore_index is None else c.t != c.ignore_index
    assert (np.abs(lse - ref["lse"]) <= (el + 2 * F32 * np.abs(ref["lse"])) * counts).all()
    row = (el + ez.max(1) + (8 + smoothing * c.v / 64) * F32 * (np.abs(ref["z"]).max(1) + np.abs(ref["lse"]))) * counts
    if reduction == "none":
        assert (np.abs(loss - ref["loss"]) <= row).all()
    else:
        rows = max(1, counts.sum()) if reduction == "mean" else 1
        want = ref["loss"].sum() / rows
        assert abs(loss - want) <= row.sum() / rows + 2 * F32 * abs(want)


@pytest.mark.parametrize("n,d,v,dtype,kw", [
    (677, 1500, 1383, "bf16", dict(label_smoothing=0.1, scratch_limit=4 << 20)),  # forward keeps logits, the gradient does not
    (1457, 1, 7119, "bf16", {}),                                                  # forward in the plain kernels
    (58, 5, 4892, "fp32", dict(scratch_limit=1)),
    (100, 2000, 300, "fp32", {}), (3, 40, 9, "bf16", {}),
])
def test_forward_of_a_plan_with_gradients(n, d, v, dtype, kw):
    """Both calls on one plan, in either order: the loss alone, then with gradients, then alone again."""
    torch = _torch()
    c = Case(n, d, v, dtype, seed=131)
    plan = c.plan(reduction="mean", **kw)
    smoothing = kw.get("label_smoothing", 0.0)
    first = plan.forward(c.x, c.w, c.target, c.bias)
    got = plan.loss_and_grad(c.x, c.w, c.target, c.bias)
    c.check(got, c.oracle("mean", smoothing), "mean", np.full(n, 1.0 / n), smoothing=smoothing)
    again = plan.forward(c.x, c.w, c.target, c.bias)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    _check_forward(c, plan, "mean", smoothing)


@pytest.mark.parametrize("n,d,v", [(600000, 9, 3), (524281, 2, 1), (1 << 20, 1, 15), (1025, 16, 9), (1024, 16, 64), (40, 16, 1700), (600000, 2, 9)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_loss_of_many_rows_with_few_products(n, d, v, dtype, reduction):
    """Few products however many rows there are: to both sides of what the plain kernels take."""
    c = Case(n, d, v, dtype, seed=141)
    _check_forward(c, c.plan(reduction=reduction, grad=False), reduction)


@pytest.mark.parametrize("n,d,v,limit", [(1, 1, 1, 1), (7, 40, 9, 1), (128, 16, 64, 1), (100, 1001, 128, 1), (64, 16, 1000, 1000), (1, 1 << 14, 15, 100),
                                         (8, 1000, 3000, 1000), (3000, 1000, 8, 1000), (100, 1030, 2000, 1 << 16)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_few_products_within_a_small_scratch(n, d, v, dtype, limit):
    """A limit below what the plain kernels, those of few rows or classes, and the split inside take."""
    c = Case(n, d, v, dtype, seed=151)
    plan = c.plan(reduction="sum", scratch_limit=limit)
    c.check(plan.loss_and_grad(c.x, c.w, c.target, c.bias), c.oracle("sum"), "sum", np.ones(n))
    _check_forward(c, c.plan(reduction="mean", scratch_limit=limit, grad=False), "mean")


@pytest.mark.parametrize("n,d,v,dtype,limit", [(1000, 1024, 9000, "bf16", 1000 * 9000 * 6), (2304, 300, 2050, "fp32", 2304 * 2052 * 10)])
def test_kept_logits_at_the_edge_of_the_scratch(n, d, v, dtype, limit):
    """Room for the logits and dz but not for dbias's column sums, and one with room for all three: the same gradient."""
    c = Case(n, d, v, dtype, seed=161)
    ref = c.oracle("mean")
    for more in (0, 64 << 20):
        got = c.plan(reduction="mean", scratch_limit=limit + more).loss_and_grad(c.x, c.w, c.target, c.bias)
        c.check(got, ref, "mean", np.full(n, 1.0 / n))


@pytest.mark.parametrize("grad", [True, False])
def test_plan_dropped_while_a_side_stream_uses_it(grad):
    """The scratch of a plan whose call still waits on a side stream is not handed out again before that call is over."""
    torch = _torch()
    c = Case(300, 512, 1000, "bf16", seed=171)
    plan = c.plan(reduction="mean", grad=grad)

    def call():
        return plan.loss_and_grad(c.x, c.w, c.target, c.bias) if grad else plan.forward(c.x, c.w, c.target, c.bias)
    want = call()
    torch.cuda.synchronize()
    at, size = plan.workspace.data_ptr(), plan.workspace.numel()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(800_000_000)                            # less than half a second
        got = call()
    del plan
    others = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(3)]
    early = not side.query()
    if early:
        assert all(o.data_ptr() + size <= at or at + size <= o.data_ptr() for o in others)
    for o in others:
        o.fill_(255)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    if not early:
        pytest.skip("the host was held up until the call was over: nothing to see")


def test_classifier_head_of_no_images():
    torch = _torch()
    from cudnntest_b200 import vgg
    head_ = vgg.ClassifierHead(0, 16, 10)
    feats = torch.empty((0, 2, 2, 4), dtype=torch.bfloat16, device="cuda")
    target = torch.empty(0, dtype=torch.int64, device="cuda")
    assert float(head_.loss(feats, target)) == 0
    loss, dx, dw, db = head_.loss_and_grad(feats, target, need_dx=True)
    assert float(loss) == 0 and dx.shape == feats.shape and (dw == 0).all() and (db == 0).all()


def test_captured_classifier_step_draws_a_mask_per_replay():
    """Every replay has the mask of its number, as eager calls before and after it do."""
    torch = _torch()
    from cudnntest_b200 import vgg
    from oracle import head
    head_ = vgg.ClassifierHead(20, 512, 30, dtype="fp32x3")
    feats = torch.rand((20, 512), device="cuda") + 0.5
    target = torch.arange(20, device="cuda")

    def mask(step):
        return torch.from_numpy(head.dropout_keep(0, feats.numel(), 0.5, head_.seed, step).reshape(20, 512)).cuda()

    assert torch.equal(head_.loss_and_grad(feats, target, need_dx=True)[1] != 0, mask(0))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = head_.loss_and_grad(feats, target, need_dx=True)
    for step in (1, 2, 3):
        g.replay()
        assert torch.equal(got[1] != 0, mask(step))
        plain = vgg.ClassifierHead(20, 512, 30, dtype="fp32x3")
        plain.steps = step
        assert all(torch.equal(a, b) for a, b in zip(got, plain.loss_and_grad(feats, target, need_dx=True)))
    assert head_.steps == 4
    assert torch.equal(head_.loss_and_grad(feats, target, need_dx=True)[1] != 0, mask(4))


def test_classifier_head_on_features_inside_wider_rows():
    torch = _torch()
    from cudnntest_b200 import vgg
    wide = torch.randn((20, 40), device="cuda", dtype=torch.bfloat16)
    target = torch.arange(20, device="cuda")
    a, b = (vgg.ClassifierHead(20, 32, 30) for _ in range(2))
    x = wide[:, :32]
    assert torch.equal(a.loss(x, target), b.loss(x.clone(), target))
    for got, want in zip(a.loss_and_grad(x, target, need_dx=True), b.loss_and_grad(x.clone(), target, need_dx=True)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("n,v,limit", [(512, 9000, 0), (500, 1003, 1 << 20), (512, 9001, 0)])
@pytest.mark.parametrize("spread", [2.0, 16.0])
def test_probabilities_kept_in_16_bits(n, v, limit, spread):
    """BF16 without a bias: exp(z - maximum) waits in 16 bits for the rows' sums.  With x the identity dW is dz itself, one element each,
    rounded once to BF16 (2^-8); what was kept before is off by at most 2^-10, the exponentials and the sum by 2^-14 together
    (ex2 2^-22 each, |z - max| below 256 rounded to 2^-24 of itself, a sum of v terms in float pairs)."""
    torch = _torch()
    import cudnntest_b200 as cb
    d = 512
    x = torch.eye(n, d, dtype=torch.bfloat16, device="cuda")
    w = (torch.randn((v, d), generator=torch.Generator().manual_seed(5)) * spread).to(torch.bfloat16).cuda()
    target = torch.arange(n, device="cuda") * 7 % v
    loss, dx, dw, _ = cb.LinearXent(n, d, v, reduction="sum", scratch_limit=limit).loss_and_grad(x, w, target)
    p = torch.softmax(w[:, :n].double().t(), 1)
    want = p.clone()
    want[torch.arange(n, device="cuda"), target] -= 1
    got = dw.double()[:, :n].t()
    off = torch.ones_like(p, dtype=torch.bool)
    off[torch.arange(n, device="cuda"), target] = False
    err, tol = (got - want).abs(), p * (2.0 ** -8 + 2.0 ** -10 + 2.0 ** -14) + 2.0 ** -124
    assert (err <= tol)[off].all(), float((err / tol)[off].max())
    # the target's own value comes from its logit in FP32
    assert (err <= want.abs() * 2.0 ** -8 + p * 2.0 ** -14 + 2.0 ** -22)[~off].all()
    assert (dw[:, n:] == 0).all()


@pytest.mark.parametrize("n,d,v,ldx,ldw", [(300, 200, 1100, 0, 0), (300, 201, 1100, 203, 202), (20, 200, 6000, 0, 0), (6000, 201, 20, 0, 0), (5, 513, 5000, 0, 0)])
@pytest.mark.parametrize("which", ["x", "w"])
def test_floats_near_the_largest_float_on_tensor_cores(n, d, v, ldx, ldw, which):
    """Floats that would round to BF16's infinity, in either matrix: split beforehand, or inside the products."""
    torch = _torch()
    c = Case(n, d, v, "fp32", seed=181, ldx=ldx, ldw=ldw)
    large, other = (c.x, c.w) if which == "x" else (c.w, c.x)
    far = torch.tensor([3.4e38, -3.4e38, 3.3961775e38, 1.0], device="cuda")
    large[:, 0] = far[torch.arange(large.shape[0], device="cuda") % 4]
    other[:, 0] = 2.0 ** -100 * (1 + (torch.arange(other.shape[0], device="cuda") % 64) / 64)
    ref = c.oracle("none")
    assert np.abs(ref["z"]).max() > 2.0 ** 27
    loss, lse = c.plan(reduction="none", grad=False).forward(c.x, c.w, c.target, c.bias)
    ez, el, _ = c.z_error(ref)
    assert (np.abs(lse.double().cpu().numpy() - ref["lse"]) <= el + 2 * F32 * np.abs(ref["lse"])).all()
    row = el + ez.max(1) + 8 * F32 * (np.abs(ref["z"]).max(1) + np.abs(ref["lse"]))
    assert (np.abs(loss.double().cpu().numpy() - ref["loss"]) <= row).all()


@pytest.mark.parametrize("bias,limit", [(False, 8 << 30), (True, 20 << 30), (True, 0)])
def test_more_than_2_31_logits(bias, limit):
    """Offsets past 32 bits in kept exponentials, kept floats and pieces: some rows of dx, some classes of dW, against 64 bits.

    dz is off by its own rounding (2^-8), by that of a kept exponential (2^-10) and by less than 2^-12 in the exponentials, the sums and
    the products; the result by one rounding more."""
    torch = _torch()
    import cudnntest_b200 as cb
    n, d, v = 40000, 1024, 60001
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((n, d), generator=gen, device="cuda").relu_().to(torch.bfloat16)
    w = (torch.randn((v, d), generator=gen, device="cuda") * 2 / (0.5 * d) ** 0.5).to(torch.bfloat16)
    b = torch.randn(v, generator=gen, device="cuda") if bias else None
    target = torch.randint(0, v, (n,), generator=gen, device="cuda")
    target[-1] = v - 1
    plan = cb.LinearXent(n, d, v, bias=bias, reduction="sum", scratch_limit=limit)
    loss, dx, dw, db = plan.loss_and_grad(x, w, target, b)
    lse = plan.forward(x, w, target, b)[1].double()
    dz_eps = 2.0 ** -8 + 2.0 ** -10 + 2.0 ** -12

    def check(got, want, mag):
        assert ((got.double() - want).abs() <= mag * dz_eps + want.abs() * 2.0 ** -8).all(), ((got.double() - want).abs() / mag).max()
    rows = torch.tensor([0, 1, 17777, 35791, 35792, n - 2, n - 1], device="cuda")
    z = x[rows].double() @ w.double().t() + (b.double() if bias else 0)
    assert ((lse[rows] - torch.logsumexp(z, 1)).abs() <= 2.0 ** -14).all()
    dz = torch.softmax(z, 1)
    dz[torch.arange(len(rows), device="cuda"), target[rows]] -= 1
    check(dx[rows], dz @ w.double(), dz.abs() @ w.double().abs())
    classes = torch.cat([torch.tensor([0, 1, 30000, 53687, v - 2, v - 1], device="cuda"), target[[0, n // 2, n - 1]]])
    zt = x.double() @ w[classes].double().t() + (b[classes].double() if bias else 0)
    dz = torch.exp(zt - lse[:, None]) - (target[:, None] == classes).double()
    check(dw[classes], dz.t() @ x.double(), dz.abs().t() @ x.double().abs())
    if bias:
        assert ((db[classes].double() - dz.sum(0)).abs() <= dz.abs().sum(0) * 2.0 ** -12).all()
