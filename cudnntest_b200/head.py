"""Classifier-head operators over the C ABI: dropout and the linear softmax cross entropy with its gradient.

They sit behind the convolution stack's features: a program that fits or evaluates a classifier on them runs
``dropout`` -> ``LinearXent.loss_and_grad`` -> ``dropout_backward``.  PyTorch is used for device memory and streams only.
Every call runs on the current stream of its tensors' device.
"""
import ctypes

import torch

from . import _lib
from ._lib import DTYPE_CODES, REDUCTION_CODES, XentDesc, check, lib
from .conv import _TORCH_DTYPE, _code, _ptr


def _rows(t, what):
    """(rows, cols, pitch) of a CUDA matrix whose rows are contiguous; any contiguous tensor counts as one long row."""
    if not t.is_cuda:
        raise ValueError("libwino needs CUDA tensors (%s)" % what)
    if t.is_contiguous():
        return 1, t.numel(), t.numel()
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= t.shape[1]:
        return t.shape[0], t.shape[1], t.stride(0)
    raise ValueError("%s must be contiguous, or a matrix with contiguous rows" % what)


def _dropout(name, x, p, seed, offset, offset_dev, out):
    dt = {torch.float32: _lib.FP32, torch.bfloat16: _lib.BF16}.get(x.dtype)
    if dt is None:
        raise ValueError("dropout takes float32 or bfloat16, not %s" % x.dtype)
    if not (0.0 <= p <= 1.0):
        raise ValueError("p must lie in [0, 1]")
    if not (0 <= seed < 2 ** 64 and 0 <= offset < 2 ** 64):
        raise ValueError("seed and offset are unsigned 64-bit integers")
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    elif out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError("out must have the input's shape, dtype and device")
    if offset_dev is not None and (offset_dev.dtype != torch.int64 or offset_dev.numel() != 1 or offset_dev.device != x.device):
        raise ValueError("offset_dev must be one int64 on the input's device")
    rows, cols, ldx = _rows(x, "input")
    orows, ocols, ldy = _rows(out, "output")
    if (rows, cols) != (orows, ocols):      # one of the two is a strided matrix: take both by rows
        rows, cols = x.shape
        ldx, ldy = (t.stride(0) if not t.is_contiguous() else cols for t in (x, out))
    with torch.cuda.device(x.device):
        check(getattr(lib(), name)(dt, rows, cols, ldx, ldy, p, seed, offset, _ptr(offset_dev), _ptr(x), _ptr(out),
                                   ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    return out


def dropout(x, p, seed, offset=0, offset_dev=None, out=None):
    """y = x / (1 - p) where kept, 0 where dropped; the mask follows from (seed, offset, element index) and is not stored.

    p is met to 2^-17 (``include/wino.h``: T = round(65536 p), scale 65536 / (65536 - T)).  The element index is that of
    the dense tensor, whatever its strides or type.  Draw another mask with another offset; ``offset_dev`` (one int64 on
    the device, added to offset when the kernel runs) does that for a captured graph.  ``out`` may be x."""
    return _dropout("wino_dropout_forward", x, p, seed, offset, offset_dev, out)


def dropout_backward(dy, p, seed, offset=0, offset_dev=None, out=None):
    """Gradient through ``dropout`` with the same p, seed and offset."""
    return _dropout("wino_dropout_backward", dy, p, seed, offset, offset_dev, out)


class LinearXent:
    """loss = cross entropy of softmax(x W^T + bias) against class numbers, and its gradient, without an (n, v) tensor of
    logits in the caller's memory.

    x: (n, d), w: (v, d), both bfloat16 (dtype "bf16") or both float32 (dtype "fp32x3": operands split into three
    bfloat16 parts, FP32-level accuracy); bias: v float32; target: n int64.  reduction "mean" (over the rows that count),
    "sum" or "none"; ignore_index: rows with that target leave no trace, whatever they hold.  The scratch is owned here
    (or handed in as ``workspace``); ``scratch_limit`` bounds the part that grows with n * v.  grad=False plans for
    ``forward`` alone.  Calls that share a plan share its scratch: keep them on one stream or otherwise serialised.
    """

    def __init__(self, n, d, v, dtype="bf16", bias=False, reduction="mean", ignore_index=None, label_smoothing=0.0,
                 grad=True, ldx=0, ldw=0, lddx=0, lddw=0, scratch_limit=0, device="cuda", workspace=None):
        s = XentDesc()
        s.n, s.d, s.v = n, d, v
        s.dtype, s.reduction = _code(DTYPE_CODES, dtype), _code(REDUCTION_CODES, reduction)
        s.has_bias, s.has_ignore = int(bias), int(ignore_index is not None)
        s.ignore_index = 0 if ignore_index is None else ignore_index
        s.label_smoothing = label_smoothing
        s.ldx, s.ldw, s.lddx, s.lddw, s.scratch_limit = ldx, ldw, lddx, lddw, scratch_limit
        self.desc, self.grad, self.device = s, bool(grad), torch.device(device)
        self.ws_bytes = lib().wino_xent_workspace_bytes(ctypes.byref(s), int(self.grad))
        if self.ws_bytes == 0:
            raise _lib.WinoError(_lib.E_BADARG, lib().wino_last_error_string().decode())
        self.io_dtype = _TORCH_DTYPE[s.dtype]
        if workspace is not None and workspace.numel() * workspace.element_size() >= self.ws_bytes:
            self.workspace = workspace
        else:
            self.workspace = torch.empty(self.ws_bytes, dtype=torch.uint8, device=self.device)

    def _matrix(self, t, what, rows, ld, dtype=None):
        d = self.desc.d
        if not t.is_cuda or t.device != self.workspace.device:
            raise ValueError("%s must be on the plan's device" % what)
        if t.dtype != self.io_dtype:
            raise ValueError("%s dtype %s, expected %s" % (what, t.dtype, self.io_dtype))
        if tuple(t.shape) != (rows, d) or (d > 1 and t.stride(1) != 1) or (rows > 1 and t.stride(0) != (ld or d)):
            raise ValueError("%s must be (%d, %d) with rows %d elements apart" % (what, rows, d, ld or d))
        return t

    def _vector(self, t, what, count, dtype):
        if not t.is_cuda or t.device != self.workspace.device or t.dtype != dtype or t.numel() != count or not t.is_contiguous():
            raise ValueError("%s must be %d contiguous %s values on the plan's device" % (what, count, dtype))
        return t

    def _inputs(self, x, w, target, bias):
        s = self.desc
        self._matrix(x, "x", s.n, s.ldx)
        self._matrix(w, "w", s.v, s.ldw)
        self._vector(target, "target", s.n, torch.int64)
        if bool(s.has_bias) != (bias is not None):
            raise ValueError("the plan was made with bias=%s" % bool(s.has_bias))
        if bias is not None:
            self._vector(bias, "bias", s.v, torch.float32)

    def _losses(self, device):
        s = self.desc
        return torch.empty((s.n,) if s.reduction == _lib.NONE else (), dtype=torch.float32, device=device)

    def forward(self, x, w, target, bias=None):
        """(loss, lse): loss is a scalar (or n values), lse_i = log sum_j exp z_ij (0 for an ignored row)."""
        self._inputs(x, w, target, bias)
        loss, lse = self._losses(x.device), torch.empty(self.desc.n, dtype=torch.float32, device=x.device)
        with torch.cuda.device(x.device):
            check(lib().wino_xent_forward(ctypes.byref(self.desc), _ptr(x), _ptr(w), _ptr(bias), _ptr(target), _ptr(loss),
                                          _ptr(lse), _ptr(self.workspace), self.workspace.numel() * self.workspace.element_size(),
                                          ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
        return loss, lse

    def loss_and_grad(self, x, w, target, bias=None, dloss=None, dx=None, dw=None, need_dx=True, need_dw=True):
        """(loss, dx, dw, dbias) in one call; dloss: upstream gradient (one float32 value, n for reduction "none").

        dx and dw may be handed in; need_dx / need_dw = False leaves a product out (its result is None).  dbias is None
        without a bias."""
        s = self.desc
        if not self.grad:
            raise ValueError("the plan was made for forward alone (grad=False)")
        self._inputs(x, w, target, bias)
        if dloss is not None:
            self._vector(dloss, "dloss", s.n if s.reduction == _lib.NONE else 1, torch.float32)

        def result(t, need, what, rows, ld):
            if not need:
                return None
            if t is None:
                t = torch.empty((rows, ld or s.d), dtype=self.io_dtype, device=x.device)[:, :s.d]
            return self._matrix(t, what, rows, ld)

        dx = result(dx, need_dx, "dx", s.n, s.lddx)
        dw = result(dw, need_dw, "dw", s.v, s.lddw)
        db = torch.empty(s.v, dtype=torch.float32, device=x.device) if s.has_bias else None
        loss = self._losses(x.device)
        with torch.cuda.device(x.device):
            check(lib().wino_xent_grad(ctypes.byref(s), _ptr(x), _ptr(w), _ptr(bias), _ptr(target), _ptr(dloss), _ptr(loss), None,
                                       _ptr(dx), _ptr(dw), _ptr(db), _ptr(self.workspace),
                                       self.workspace.numel() * self.workspace.element_size(),
                                       ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
        return loss, dx, dw, db
