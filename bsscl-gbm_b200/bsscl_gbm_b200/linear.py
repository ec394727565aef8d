"""Device operators for leaf-wise linear models (gbm_softmax_xent,
gbm_leaf_linear, gbm_grad_clip of include/gbm_b200.h) on torch CUDA tensors.

The reference's leaves hold constants and its multi-class loss keeps F for
every row and class (E:2989-3008); these operators are the training step of a
model whose leaves hold linear maps under a softmax head of many classes:

    y = leaf_linear(x, w, offsets)                       rows lie leaf after leaf
    loss, lse = softmax_xent(y, head, target)
    dy, dhead = softmax_xent_grad(y, head, target, lse, grad_loss)
    dx, dw = leaf_linear_grad(x, w, offsets, dy)
    norm = GradClip([dw, dhead]).clip(1.0)

Every call runs on the current stream of its tensors' device, whatever the
current device is, waits for nothing, and may be captured into a CUDA graph.
There is no CPU path.  Wrong types, shapes, strides and devices raise
ValueError before anything is launched.
"""

from __future__ import annotations

import ctypes as C

from ._lib import ERRORS, GBM_OK, lib

_TYPES = None


def _torch():
    import torch
    return torch


def _types():
    """torch dtype -> GBM_TYPE_* code."""
    global _TYPES
    if _TYPES is None:
        t = _torch()
        _TYPES = {t.float32: 0, t.bfloat16: 2, t.float16: 3}
    return _TYPES


def _call(name, device, *args):
    """One library call on `device`'s current stream."""
    t = _torch()
    err = C.create_string_buffer(256)
    with t.cuda.device(device):
        rc = getattr(lib(), name)(*args, t.cuda.current_stream().cuda_stream, err, 256)
    if rc == GBM_OK:
        return
    msg = f"{err.value.decode(errors='replace')} ({ERRORS.get(rc, rc)})"
    raise ValueError(msg) if rc in (1, 7) else RuntimeError(msg)


def _matrix(a, name, cols=None, like=None, rows=None):
    """Row stride of a 2-D bf16/f16 CUDA tensor whose rows are contiguous."""
    t = _torch()
    if not isinstance(a, t.Tensor) or not a.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if a.dtype not in (t.bfloat16, t.float16):
        raise ValueError(f"{name} must be bfloat16 or float16, got {a.dtype}")
    if a.dim() != 2:
        raise ValueError(f"{name} must be 2-D, got shape {tuple(a.shape)}")
    if like is not None and (a.dtype != like.dtype or a.device != like.device):
        raise ValueError(f"{name} must have the type and device of the other operands "
                         f"({like.dtype}, {like.device}), got {a.dtype}, {a.device}")
    if cols is not None and a.shape[1] != cols:
        raise ValueError(f"{name} must have {cols} columns, got shape {tuple(a.shape)}")
    if rows is not None and a.shape[0] != rows:
        raise ValueError(f"{name} must have {rows} rows, got shape {tuple(a.shape)}")
    n, d = a.shape
    if d == 0:
        raise ValueError(f"{name} has no columns")
    if d > 1 and a.stride(1) != 1:
        raise ValueError(f"{name}: the elements of a row must be contiguous (strides {a.stride()})")
    if n <= 1:
        return d
    if a.stride(0) < d:
        raise ValueError(f"{name}: rows overlap (strides {a.stride()})")
    return a.stride(0)


def _vector(a, name, dtype, n, like):
    t = _torch()
    if not isinstance(a, t.Tensor) or a.dtype != dtype or a.device != like.device or tuple(a.shape) != (n,):
        raise ValueError(f"{name} must be a {dtype} tensor of shape ({n},) on {like.device}")
    if n > 1 and a.stride(0) != 1:
        raise ValueError(f"{name} must be contiguous")


def _in_place(*operands):
    """1 where every operand's rows start on 16-byte boundaries."""
    return int(all(a.data_ptr() % 16 == 0 and ld % 8 == 0 for a, ld in operands))


def _workspace(size, like):
    if size < 0:
        raise ValueError("a size is out of range")
    t = _torch()
    # of the current stream's pool, so calls on two streams (and two captured graphs) never share one
    with t.cuda.device(like.device):
        return t.empty(max(size, 1), dtype=t.uint8, device=like.device)


def softmax_xent(x, w, target):
    """Softmax cross entropy of the linear head ``x @ w.T`` without keeping
    the logits: ``(loss, lse)``, float32 [n].  x [n, d] and w [v, d] bfloat16
    or float16 (rows contiguous, any row stride), target int64 [n].  A row
    whose target is outside 0..v-1 is ignored: its loss is 0."""
    t = _torch()
    ldx = _matrix(x, "x")
    ldw = _matrix(w, "w", cols=x.shape[1], like=x)
    n, d, v = x.shape[0], x.shape[1], w.shape[0]
    _vector(target, "target", t.int64, n, x)
    loss = t.empty(n, dtype=t.float32, device=x.device)
    lse = t.empty(n, dtype=t.float32, device=x.device)
    size = lib().gbm_softmax_xent_workspace(n, d, v, 0, _in_place((x, ldx), (w, ldw)))
    ws = _workspace(size, x)
    _call("gbm_softmax_xent", x.device, x.data_ptr(), ldx, w.data_ptr(), ldw, _types()[x.dtype], n, d, v,
          target.data_ptr(), loss.data_ptr(), lse.data_ptr(), ws.data_ptr(), size)
    return loss, lse


def softmax_xent_grad(x, w, target, lse, grad_loss, want_dx=True, want_dw=True):
    """Gradients ``(dx, dw)`` of ``sum(grad_loss * loss)`` in the operands'
    type; lse as :func:`softmax_xent` returned it, grad_loss float32 [n].
    Ignored rows get dx = 0 and add nothing to dw.  ``want_dx=False`` /
    ``want_dw=False`` give None in that place and save its product."""
    t = _torch()
    ldx = _matrix(x, "x")
    ldw = _matrix(w, "w", cols=x.shape[1], like=x)
    n, d, v = x.shape[0], x.shape[1], w.shape[0]
    _vector(target, "target", t.int64, n, x)
    _vector(lse, "lse", t.float32, n, x)
    _vector(grad_loss, "grad_loss", t.float32, n, x)
    if not (want_dx or want_dw):
        raise ValueError("neither dx nor dw is wanted")
    dx = t.empty(n, d, dtype=x.dtype, device=x.device) if want_dx else None
    dw = t.empty(v, d, dtype=x.dtype, device=x.device) if want_dw else None
    size = lib().gbm_softmax_xent_workspace(n, d, v, 1, _in_place((x, ldx), (w, ldw)))
    ws = _workspace(size, x)
    if n == 0 and not want_dw:
        return dx, dw
    _call("gbm_softmax_xent_grad", x.device, x.data_ptr(), ldx, w.data_ptr(), ldw, _types()[x.dtype], n, d, v,
          target.data_ptr(), lse.data_ptr(), grad_loss.data_ptr(), dx.data_ptr() if want_dx and n else None, d,
          dw.data_ptr() if want_dw else None, d, ws.data_ptr(), size)
    return dx, dw


def _leaf_args(x, w, offsets, name):
    t = _torch()
    if not isinstance(w, t.Tensor) or w.dim() != 3 or not w.is_contiguous() or 0 in w.shape:
        raise ValueError("w must be a contiguous tensor [leaves, dout, din]")
    if w.dtype != x.dtype or w.device != x.device:
        raise ValueError(f"w must have {name}'s type and device ({x.dtype}, {x.device}), got {w.dtype}, {w.device}")
    if not isinstance(offsets, t.Tensor):
        raise ValueError("offsets must be a tensor")
    _vector(offsets, "offsets", t.int32, w.shape[0] + 1, x)


def _output(out, rows, cols, like, name):
    t = _torch()
    if out is None:
        return t.empty(rows, cols, dtype=like.dtype, device=like.device), cols, 1
    return out, _matrix(out, name, cols=cols, like=like, rows=rows), 0


def leaf_linear(x, w, offsets, out=None):
    """Products grouped by leaf: row r of leaf g, offsets[g] <= r <
    offsets[g+1], gives ``y[r] = w[g] @ x[r]``.  x [t, din] (rows contiguous,
    any row stride), w [leaves, dout, din] contiguous, both bfloat16 or
    float16; offsets int32 [leaves + 1] on the device, non-decreasing within
    0..t.  Rows that no leaf has (before offsets[0], from offsets[-1] on) are 0 in a new y and left as they
    were in ``out``."""
    ldx = _matrix(x, "x")
    _leaf_args(x, w, offsets, "x")
    e, dout, din = w.shape
    if x.shape[1] != din:
        raise ValueError(f"x must have {din} columns, got shape {tuple(x.shape)}")
    n = x.shape[0]
    y, ldy, rest = _output(out, n, dout, x, "out")
    if n == 0:
        return y
    size = lib().gbm_leaf_linear_workspace(n, e, din, dout, 0, _in_place((x, ldx), (w, din)))
    ws = _workspace(size, x)
    _call("gbm_leaf_linear", x.device, x.data_ptr(), ldx, w.data_ptr(), offsets.data_ptr(), _types()[x.dtype], n, e,
          din, dout, y.data_ptr(), ldy, rest, ws.data_ptr(), size)
    return y


def leaf_linear_grad(x, w, offsets, dy, want_dx=True, want_dw=True):
    """Gradients ``(dx, dw)`` of :func:`leaf_linear` in the operands' type:
    ``dx[r] = w[g].T @ dy[r]`` (0 in rows that no leaf has) and ``dw[g]`` the
    sum of ``outer(dy[r], x[r])`` over leaf g's rows (0 for an empty leaf)."""
    t = _torch()
    ldx = _matrix(x, "x")
    _leaf_args(x, w, offsets, "x")
    e, dout, din = w.shape
    n = x.shape[0]
    if x.shape[1] != din:
        raise ValueError(f"x must have {din} columns, got shape {tuple(x.shape)}")
    lddy = _matrix(dy, "dy", cols=dout, like=x, rows=n)
    if not (want_dx or want_dw):
        raise ValueError("neither dx nor dw is wanted")
    dx = t.empty(n, din, dtype=x.dtype, device=x.device) if want_dx else None
    dw = t.empty(e, dout, din, dtype=x.dtype, device=x.device) if want_dw else None
    if n == 0 and not want_dw:
        return dx, dw
    size = lib().gbm_leaf_linear_workspace(n, e, din, dout, 1, _in_place((x, ldx), (w, din), (dy, lddy)))
    ws = _workspace(size, x)
    _call("gbm_leaf_linear_grad", x.device, x.data_ptr(), ldx, w.data_ptr(), offsets.data_ptr(), dy.data_ptr(), lddy,
          _types()[x.dtype], n, e, din, dout, dx.data_ptr() if want_dx and n else None, din, 1,
          dw.data_ptr() if want_dw else None, ws.data_ptr(), size)
    return dx, dw


class GradClip:
    """The global 2-norm of many gradients, and clipping to it.

    Made once for the gradients of a model (a list of CUDA tensors of one
    device; float32, bfloat16 or float16, each dense), whose buffers it keeps; ``out`` (default: the gradients themselves) takes the
    clipped values.  No two buffers may overlap, but out[i] may be grads[i].
    """

    def __init__(self, grads, out=None):
        t = _torch()
        grads = list(grads)
        out = grads if out is None else list(out)
        if not grads:
            raise ValueError("no gradients")
        if len(out) != len(grads):
            raise ValueError(f"{len(grads)} gradients but {len(out)} outputs")
        types = _types()
        for i, (g, o) in enumerate(zip(grads, out)):
            for a, name in ((g, "gradient"), (o, "output")):
                if not isinstance(a, t.Tensor) or not a.is_cuda or a.dtype not in types:
                    raise ValueError(f"{name} {i} must be a float32, bfloat16 or float16 CUDA tensor")
                if a.device != grads[0].device:
                    raise ValueError(f"{name} {i} is on {a.device}, gradient 0 on {grads[0].device}")
            if o.dtype != g.dtype or o.shape != g.shape or o.stride() != g.stride():
                raise ValueError(f"output {i} must have its gradient's type, shape and strides")
            if not _dense(g):
                raise ValueError(f"gradient {i} is not dense (shape {tuple(g.shape)}, strides {g.stride()})")
        n = len(grads)
        self.device = grads[0].device
        self._keep = (grads, out)
        sizes = (C.c_int64 * n)(*(g.numel() for g in grads))
        L = lib()
        size = L.gbm_grad_clip_plan_bytes(sizes, n)
        if size < 0:
            raise ValueError("a gradient is too large")
        self._plan = C.create_string_buffer(size)
        err = C.create_string_buffer(256)
        rc = L.gbm_grad_clip_plan((C.c_void_p * n)(*(g.data_ptr() for g in grads)),
                                  (C.c_void_p * n)(*(o.data_ptr() for o in out)), sizes,
                                  (C.c_int32 * n)(*(types[g.dtype] for g in grads)), n, self._plan, size, err, 256)
        if rc != GBM_OK:
            raise ValueError(err.value.decode(errors="replace"))
        # a copy that waits: the plan may be used on any stream from here on
        self._plan_dev = t.frombuffer(bytearray(self._plan.raw), dtype=t.uint8).to(self.device)
        self._ws = L.gbm_grad_clip_workspace(self._plan)

    def clip(self, max_norm):
        """``out = grad * min(1, max_norm / (norm + 1e-6))`` for every
        gradient; returns the norm before clipping, a float32 scalar tensor
        (nothing is read back to the host)."""
        t = _torch()
        norm = t.empty((), dtype=t.float32, device=self.device)
        with t.cuda.device(self.device):
            ws = t.empty(self._ws, dtype=t.uint8, device=self.device)
        _call("gbm_grad_clip", self.device, self._plan, self._plan_dev.data_ptr(), float(max_norm), norm.data_ptr(),
              ws.data_ptr(), self._ws)
        return norm


def _dense(a):
    """Whether the tensor's elements fill one contiguous range, each once."""
    want = 1
    for stride, size in sorted((st, n) for st, n in zip(a.stride(), a.shape) if n != 1):
        if stride != want:
            return a.numel() == 0
        want *= size
    return True


def status(device=None):
    """Waits for the current stream and raises RuntimeError when a bounded
    wait inside one of these operators ran out on `device` since the last
    call, or an asynchronous error occurred."""
    t = _torch()
    _call("gbm_ops_status", t.device("cuda", t.cuda.current_device()) if device is None else t.device(device))
