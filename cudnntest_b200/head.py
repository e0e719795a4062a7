"""Classifier-head operators over the C ABI: dropout and the linear softmax cross entropy with its gradient.

They sit behind the convolution stack's features: a program that fits or evaluates a classifier on them runs
``dropout`` -> ``LinearXent.loss_and_grad`` -> ``dropout_backward``.  PyTorch is used for device memory and streams only.
Every call runs on the current stream of its tensors' device.
"""
import ctypes

import torch

from . import _lib
from ._lib import DTYPE_CODES, REDUCTION_CODES, XentDesc, check, lib
from .conv import _TORCH_DTYPE, _code


# The current stream's handle by device index.  torch.cuda.current_stream builds a Stream object first, 2 to 3 us of a call
# that otherwise costs about 8; this is what it asks.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(fn, device_index, *args):
    """fn(*args, stream) with the tensors' device current and that device's current stream."""
    if torch.cuda.current_device() == device_index:
        return check(fn(*args, _raw_stream(device_index)))
    with torch.cuda.device(device_index):
        return check(fn(*args, _raw_stream(device_index)))


def _rows(t, what):
    """(rows, cols, pitch) of a matrix whose rows are contiguous; any contiguous tensor counts as one long row."""
    if t.is_contiguous():
        n = t.numel()
        return 1, n, n
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= t.shape[1]:
        return t.shape[0], t.shape[1], t.stride(0)
    raise ValueError("%s must be contiguous, or a matrix with contiguous rows" % what)


_DROPOUT_DTYPE = {torch.float32: _lib.FP32, torch.bfloat16: _lib.BF16}


def _dropout(fn, x, p, seed, offset, offset_dev, out):
    dt = _DROPOUT_DTYPE.get(x.dtype)
    if dt is None:
        raise ValueError("dropout takes float32 or bfloat16, not %s" % x.dtype)
    if not x.is_cuda:
        raise ValueError("libwino needs CUDA tensors")
    if not (0.0 <= p <= 1.0):
        raise ValueError("p must lie in [0, 1]")
    if not (0 <= seed < 2 ** 64 and 0 <= offset < 2 ** 64):
        raise ValueError("seed and offset are unsigned 64-bit integers")
    rows, cols, ldx = _rows(x, "input")
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    elif out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError("out must have the input's shape, dtype and device")
    if offset_dev is not None and (offset_dev.dtype != torch.int64 or offset_dev.numel() != 1 or offset_dev.device != x.device):
        raise ValueError("offset_dev must be one int64 on the input's device")
    orows, ocols, ldy = _rows(out, "output")
    if rows != orows or cols != ocols:      # one of the two is a strided matrix: take both by rows
        rows, cols = x.shape
        ldx, ldy = (t.stride(0) if not t.is_contiguous() else cols for t in (x, out))
    _call(fn, x.get_device(), dt, rows, cols, ldx, ldy, p, seed, offset, None if offset_dev is None else offset_dev.data_ptr(),
          x.data_ptr(), out.data_ptr())
    return out


def dropout(x, p, seed, offset=0, offset_dev=None, out=None):
    """y = x / (1 - p) where kept, 0 where dropped; the mask follows from (seed, offset, element index) and is not stored.

    p is met to 2^-17 (``include/wino.h``: T = round(65536 p), scale 65536 / (65536 - T)).  The element index is that of
    the dense tensor, whatever its strides or type.  Draw another mask with another offset; ``offset_dev`` (one int64 on
    the device, added to offset when the kernel runs) does that for a captured graph.  ``out`` may be x."""
    return _dropout(lib().wino_dropout_forward, x, p, seed, offset, offset_dev, out)


def dropout_backward(dy, p, seed, offset=0, offset_dev=None, out=None):
    """Gradient through ``dropout`` with the same p, seed and offset."""
    return _dropout(lib().wino_dropout_backward, dy, p, seed, offset, offset_dev, out)


class LinearXent:
    """loss = cross entropy of softmax(x W^T + bias) against class numbers, and its gradient, in one call; an (n, v) matrix
    exists at most in the scratch, as far as ``scratch_limit`` (0: 1 GiB) allows.

    x: (n, d), w: (v, d), both bfloat16 (dtype "bf16") or both float32 (dtype "fp32x3": operands split into three
    bfloat16 parts, FP32-level accuracy); bias: v float32; target: n int64.  reduction "mean" (over the rows that count),
    "sum" or "none"; ignore_index: rows with that target leave no trace, whatever they hold.  The scratch is owned here
    (or handed in as ``workspace``); ``scratch_limit`` bounds the part that grows with n * v.  grad=False plans for
    ``forward`` alone, grad=True for both calls.  Calls that share a plan share its scratch: keep them on one stream or
    otherwise serialised.  A graph that holds a call needs the plan for as long as it is replayed.
    """

    def __init__(self, n, d, v, dtype="bf16", bias=False, reduction="mean", ignore_index=None, label_smoothing=0.0,
                 grad=True, ldx=0, ldw=0, lddx=0, lddw=0, scratch_limit=0, device="cuda", workspace=None):
        s = XentDesc()
        fields = dict(n=n, d=d, v=v, dtype=_code(DTYPE_CODES, dtype), reduction=_code(REDUCTION_CODES, reduction), has_bias=int(bias),
                      has_ignore=int(ignore_index is not None), ignore_index=0 if ignore_index is None else ignore_index,
                      ldx=ldx, ldw=ldw, lddx=lddx, lddw=lddw, scratch_limit=scratch_limit)
        for name, value in fields.items():
            setattr(s, name, value)
            if getattr(s, name) != value:       # ctypes keeps the lower bits without a word
                raise ValueError("%s = %d does not fit wino_xent_desc" % (name, value))
        s.label_smoothing = label_smoothing
        self.desc, self.grad, self.device = s, bool(grad), torch.device(device)
        # forward plans for itself, and may need more than the gradient (whose dz counts against scratch_limit too)
        needs = [lib().wino_xent_workspace_bytes(ctypes.byref(s), g) for g in ((0, 1) if self.grad else (0,))]
        if 0 in needs:
            raise _lib.WinoError(_lib.E_BADARG, lib().wino_last_error_string().decode())
        self.ws_bytes = max(needs)
        self.io_dtype = _TORCH_DTYPE[s.dtype]
        if workspace is not None and not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous")
        if workspace is not None and workspace.numel() * workspace.element_size() >= self.ws_bytes:
            self.workspace = workspace
        else:
            self.workspace = torch.empty(self.ws_bytes, dtype=torch.uint8, device=self.device)
        self._desc_ref, self._ws_size = ctypes.byref(s), self.workspace.numel() * self.workspace.element_size()
        self._index = self.workspace.get_device()
        self._made_on = _raw_stream(self._index) if self._index >= 0 else None
        self._forms = [(torch.Size((rows, d)), (ld or d, 1)) for rows, ld in ((n, ldx), (v, ldw), (n, lddx), (v, lddw))]
        # what results are allocated like
        self._lse_like = torch.empty(n, dtype=torch.float32, device=self.workspace.device)
        self._loss_like = self._lse_like if s.reduction == _lib.NONE else torch.empty((), dtype=torch.float32, device=self.workspace.device)

    def _matrix(self, t, what, form):
        """Device address of a matrix of the plan's rows and pitch; form: (shape, strides)."""
        if t.shape == form[0] and t.stride() == form[1] and t.dtype == self.io_dtype and t.get_device() == self._index:
            return t.data_ptr()
        (rows, d), (ld, _) = form
        if t.get_device() != self._index:
            raise ValueError("%s must be on the plan's device" % what)
        if t.dtype != self.io_dtype:
            raise ValueError("%s dtype %s, expected %s" % (what, t.dtype, self.io_dtype))
        # the pitch of a single row and the step of a single column mean nothing
        if tuple(t.shape) != (rows, d) or (d > 1 and t.stride(1) != 1) or (rows > 1 and t.stride(0) != ld):
            raise ValueError("%s must be (%d, %d) with rows %d elements apart" % (what, rows, d, ld))
        return t.data_ptr()

    def _vector(self, t, what, count, dtype):
        if t.get_device() != self._index or t.dtype != dtype or t.numel() != count or not t.is_contiguous():
            raise ValueError("%s must be %d contiguous %s values on the plan's device" % (what, count, dtype))
        return t.data_ptr()

    def _keep(self, *tensors):
        """The allocator keeps them for the current stream's work, even if their owner is dropped."""
        if self._index >= 0 and _raw_stream(self._index) != self._made_on:
            stream = torch.cuda.current_stream(self._index)
            for t in tensors:
                t.record_stream(stream)

    def _scratch(self):
        self._keep(self.workspace)
        return self.workspace.data_ptr(), self._ws_size

    def _inputs(self, x, w, target, bias):
        s = self.desc
        if self._index < 0:
            raise ValueError("libwino needs CUDA tensors")
        if bool(s.has_bias) != (bias is not None):
            raise ValueError("the plan was made with bias=%s" % bool(s.has_bias))
        return (self._matrix(x, "x", self._forms[0]), self._matrix(w, "w", self._forms[1]),
                None if bias is None else self._vector(bias, "bias", s.v, torch.float32), self._vector(target, "target", s.n, torch.int64))

    def forward(self, x, w, target, bias=None):
        """(loss, lse): loss is a scalar (or n values), lse_i = log sum_j exp z_ij (0 for an ignored row)."""
        args = self._inputs(x, w, target, bias)
        loss, lse = torch.empty_like(self._loss_like), torch.empty_like(self._lse_like)
        _call(lib().wino_xent_forward, self._index, self._desc_ref, *args, loss.data_ptr(), lse.data_ptr(), *self._scratch())
        return loss, lse

    def loss_and_grad(self, x, w, target, bias=None, dloss=None, dx=None, dw=None, need_dx=True, need_dw=True):
        """(loss, dx, dw, dbias) in one call; dloss: upstream gradient (one float32 value, n for reduction "none").

        dx and dw may be handed in; need_dx / need_dw = False leaves a product out (its result is None).  dbias is None
        without a bias."""
        s = self.desc
        if not self.grad:
            raise ValueError("the plan was made for forward alone (grad=False)")
        args = self._inputs(x, w, target, bias)
        if dloss is not None:
            dloss = self._vector(dloss, "dloss", s.n if s.reduction == _lib.NONE else 1, torch.float32)

        def result(t, need, what, like, form):
            if not need:
                return None, None
            if t is not None:
                return t, self._matrix(t, what, form)
            if form[1][0] == s.d and like.stride() == form[1]:       # both dense
                t = torch.empty_like(like)
            else:
                t = like.new_empty((form[0][0], form[1][0]))[:, :s.d]
            return t, t.data_ptr()

        dx, dx_ptr = result(dx, need_dx, "dx", x, self._forms[2])
        dw, dw_ptr = result(dw, need_dw, "dw", w, self._forms[3])
        db = torch.empty_like(bias) if s.has_bias else None
        loss = torch.empty_like(self._loss_like)
        _call(lib().wino_xent_grad, self._index, self._desc_ref, *args, dloss, loss.data_ptr(), None, dx_ptr, dw_ptr,
              None if db is None else db.data_ptr(), *self._scratch())
        return loss, dx, dw, db
