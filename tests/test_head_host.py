"""CPU-side checks of the classifier head: the oracle against published vectors and differences, descriptor checks,
scratch sizes, refusals - nothing here needs a GPU."""
import ctypes

import numpy as np
import pytest

import cudnntest_b200 as cb
from oracle import head


@pytest.mark.parametrize("ctr,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0), (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_oracle_generator_known_answers(ctr, key, want):
    """The published known-answer vectors of Philox4x32-10."""
    assert tuple(int(v) for v in head.philox4x32_10(np.array([ctr], dtype=np.uint64), key)[0]) == want


def test_oracle_mask_rate_and_independence():
    """Keep rate within five standard deviations; other offsets and seeds give other masks; p = 0 and 1 are exact."""
    count = 1 << 16
    for p in (0.1, 0.5, 0.9):
        k = head.dropout_keep(0, count, p, 7, 3)
        assert abs(k.mean() - (1 - p)) <= 5 * np.sqrt(p * (1 - p) / count)
    a, b, c = (head.dropout_keep(0, count, 0.5, s, o) for s, o in ((7, 3), (7, 4), (8, 3)))
    for other in (b, c):
        assert abs((a ^ other).mean() - 0.5) <= 5 * 0.5 / np.sqrt(count)
    assert head.dropout_keep(0, 64, 0.0, 1, 1).all() and not head.dropout_keep(0, 64, 1.0, 1, 1).any()
    assert (head.dropout_keep(1000, 100, 0.5, 7, 3) == head.dropout_keep(0, 1100, 0.5, 7, 3)[1000:]).all()


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("smoothing", [0.0, 0.1])
def test_oracle_gradient_against_differences(reduction, smoothing):
    """Central differences of the oracle's own loss: step 1e-5 leaves an error of order step^2 and 2^-53 / step."""
    rng = np.random.default_rng(5)
    n, d, v = 5, 7, 6
    x, w, b = rng.standard_normal((n, d)), rng.standard_normal((v, d)), rng.standard_normal(v)
    t = np.array([0, 5, -100, 2, 2])
    up = rng.standard_normal(n) if reduction == "none" else rng.standard_normal()
    kw = dict(reduction=reduction, ignore_index=-100, smoothing=smoothing)
    ref = head.xent(x, w, t, b, dloss=up, **kw)

    def f(x, w, b):
        return float(np.sum(head.xent(x, w, t, b, **kw)["loss"] * up))
    h = 1e-5
    for k, (arr, grad) in enumerate(((x, ref["dx"]), (w, ref["dw"]), (b, ref["db"]))):
        for i in np.ndindex(arr.shape):
            args = [x.copy(), w.copy(), b.copy()]
            args[k][i] += h
            hi = f(*args)
            args[k][i] -= 2 * h
            assert abs((hi - f(*args)) / (2 * h) - grad[i]) <= 1e-8


def _desc(**kw):
    s = cb.XentDesc()
    s.n, s.d, s.v, s.dtype = 64, 96, 40, cb.BF16
    for k, v in kw.items():
        setattr(s, k, v)
    return s


@pytest.mark.parametrize("field,value", [("n", -1), ("d", 0), ("v", 0), ("d", -5), ("dtype", cb.FP32), ("dtype", cb.TF32), ("dtype", 9),
                                         ("has_bias", 2), ("has_ignore", -1), ("reduction", 3), ("label_smoothing", -0.1),
                                         ("label_smoothing", 1.5), ("label_smoothing", float("nan")), ("ldx", 95), ("ldw", 1),
                                         ("lddx", 95), ("lddw", -96), ("scratch_limit", -1), ("n", (1 << 30) + 1)])
def test_xent_descriptor_refusals(field, value):
    L = cb.lib()
    for grad in (0, 1):
        assert L.wino_xent_workspace_bytes(ctypes.byref(_desc()), grad) > 0
        assert L.wino_xent_workspace_bytes(ctypes.byref(_desc(**{field: value})), grad) == 0
        assert b"xent" in L.wino_last_error_string()
    assert L.wino_xent_workspace_bytes(None, 0) == 0


@pytest.mark.parametrize("n,d,v", [(0, 1, 1), (0, 4096, 1000), (1, 1, 1), (1, 1 << 30, 1), (1 << 30, 1, 1), (1, 1, 1 << 30), (1 << 16, 1 << 12, 1 << 18)])
@pytest.mark.parametrize("dtype", [cb.BF16, cb.FP32X3])
def test_xent_plans_of_extreme_sizes(n, d, v, dtype):
    L = cb.lib()
    for grad in (0, 1):
        for limit in (0, 1, 1 << 62):
            s = _desc(n=n, d=d, v=v, dtype=dtype, scratch_limit=limit, has_bias=1, has_ignore=1, label_smoothing=0.1)
            assert L.wino_xent_workspace_bytes(ctypes.byref(s), grad) > 0


def test_xent_scratch_is_bounded():
    """The part that grows with n * v stays within scratch_limit (or 256 classes): statistics, row vectors and the float
    parts of dx aside.  dx is split into parts only while tiles * parts stays within the 74 CTA pairs, so its parts take
    at most 74 tiles of 256 x 256 floats."""
    L = cb.lib()
    s = _desc(n=4096, d=512, v=65536, scratch_limit=64 << 20)
    small = L.wino_xent_workspace_bytes(ctypes.byref(s), 1)
    stats = 65536 // 128 * 4096 * 8
    assert small <= (64 << 20) + stats + 5 * 4096 * 4 + 74 * 256 * 256 * 4 + (1 << 16)
    s.scratch_limit = 0
    assert L.wino_xent_workspace_bytes(ctypes.byref(s), 1) > small
    assert L.wino_xent_workspace_bytes(ctypes.byref(s), 0) < small


def _grad_args(L, s, **kw):
    """A call's arguments; the pointers are never followed, every case below is refused before a launch."""
    a = dict(x=1 << 20, w=1 << 21, bias=None, target=1 << 22, dloss=None, loss=1 << 23, lse=None, dx=1 << 24, dw=1 << 25, db=None,
             ws=1 << 26, bytes=L.wino_xent_workspace_bytes(ctypes.byref(s), 1))
    a.update(kw)
    return [ctypes.byref(s)] + list(a.values()) + [None]


@pytest.mark.parametrize("kw,code", [
    (dict(x=None), cb._lib.E_BADARG), (dict(w=None), cb._lib.E_BADARG), (dict(target=None), cb._lib.E_BADARG), (dict(loss=None), cb._lib.E_BADARG),
    (dict(x=(1 << 20) + 2), cb._lib.E_BADARG), (dict(dx=(1 << 24) + 8), cb._lib.E_BADARG), (dict(dw=(1 << 24) + 8), cb._lib.E_BADARG),
    (dict(target=(1 << 22) + 4), cb._lib.E_BADARG), (dict(loss=(1 << 23) + 2), cb._lib.E_BADARG), (dict(db=1 << 27), cb._lib.E_BADARG),
    (dict(dx=1 << 20), cb._lib.E_BADARG), (dict(dw=1 << 21), cb._lib.E_BADARG), (dict(dw=1 << 24), cb._lib.E_BADARG),
    (dict(ws=None), cb._lib.E_WORKSPACE), (dict(bytes=1000), cb._lib.E_WORKSPACE), (dict(ws=(1 << 26) + 4), cb._lib.E_BADARG),
])
def test_xent_call_refusals(kw, code):
    L = cb.lib()
    assert L.wino_xent_grad(*_grad_args(L, _desc(), **kw)) == code
    assert L.wino_xent_grad(*_grad_args(L, _desc(has_bias=1), **kw)) != 0      # and a missing bias


@pytest.mark.parametrize("kw", [dict(dtype=cb.TF32), dict(rows=-1), dict(cols=-3), dict(ldx=7), dict(ldy=7), dict(p=-0.1), dict(p=1.1),
                                dict(p=float("nan")), dict(x=None), dict(y=None), dict(x=(1 << 20) + 2), dict(offset_dev=(1 << 22) + 4),
                                dict(y=1 << 20, ldy=16), dict(rows=1 << 62, cols=8)])
@pytest.mark.parametrize("name", ["wino_dropout_forward", "wino_dropout_backward"])
def test_dropout_refusals(name, kw):
    L = cb.lib()
    a = dict(dtype=cb.FP32, rows=4, cols=8, ldx=8, ldy=8, p=0.5, seed=1, offset=2, offset_dev=None, x=1 << 20, y=1 << 21, stream=None)
    a.update(kw)
    assert getattr(L, name)(*a.values()) == cb._lib.E_BADARG
    assert b"dropout" in L.wino_last_error_string()
    a.update(dtype=cb.FP32, rows=0, cols=8, ldx=8, ldy=8, p=0.5, offset_dev=None, x=None, y=None)
    assert getattr(L, name)(*a.values()) == 0                                   # nothing to do


def test_python_refusals():
    import torch
    with pytest.raises(cb.WinoError):
        cb.LinearXent(8, 0, 10, device="cpu")
    plan = cb.LinearXent(8, 16, 10, device="cpu")
    x, w, t = torch.zeros(8, 16, dtype=torch.bfloat16), torch.zeros(10, 16, dtype=torch.bfloat16), torch.zeros(8, dtype=torch.int64)
    with pytest.raises(ValueError):
        plan.forward(x, w, t)                                                   # CPU tensors
    for bad in (dict(p=1.5), dict(p=-0.5), dict(seed=-1), dict(offset=1 << 64)):
        with pytest.raises(ValueError):
            cb.dropout(x, **{**dict(p=0.5, seed=0, offset=0), **bad})
    with pytest.raises(ValueError):
        cb.dropout(x.double(), 0.5, 0)
    with pytest.raises(ValueError):
        cb.dropout(x, 0.5, 0)
