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
import threading

import torch

from ._lib import ERRORS, GBM_OK, lib

_TYPES = {torch.float32: 0, torch.bfloat16: 2, torch.float16: 3}     # GBM_TYPE_*
_local = threading.local()
_stream_of = torch._C._cuda_getCurrentRawStream    # current_stream(i).cuda_stream without its wrapper object (3 us)
_current = torch._C._cuda_getDevice


def _call(fn, device, *args):
    """One library call on `device`'s current stream."""
    try:
        err = _local.err
    except AttributeError:
        err = _local.err = C.create_string_buffer(256)
    i = device.index
    if i == _current():
        rc = fn(*args, _stream_of(i), err, 256)
    else:
        with torch.cuda.device(i):
            rc = fn(*args, _stream_of(i), err, 256)
    if rc != GBM_OK:
        msg = f"{err.value.decode(errors='replace')} ({ERRORS.get(rc, rc)})"
        raise ValueError(msg) if rc in (1, 7) else RuntimeError(msg)


def _matrix(a, name, like=None):
    """(rows, columns, row stride) of a 2-D bf16/f16 CUDA tensor whose rows are contiguous."""
    if not isinstance(a, torch.Tensor) or not a.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    t = a.dtype
    if t is not torch.bfloat16 and t is not torch.float16:
        raise ValueError(f"{name} must be bfloat16 or float16, got {t}")
    if a.dim() != 2:
        raise ValueError(f"{name} must be 2-D, got shape {tuple(a.shape)}")
    if like is not None and (t is not like.dtype or a.device != like.device):
        raise ValueError(f"{name} must have the type and device of the other operands "
                         f"({like.dtype}, {like.device}), got {t}, {a.device}")
    n, d = a.shape
    ld, one = a.stride()
    if d == 0:
        raise ValueError(f"{name} has no columns")
    if one != 1 and d > 1:
        raise ValueError(f"{name}: the elements of a row must be contiguous (strides {a.stride()})")
    if n <= 1:
        return n, d, d
    if ld < d:
        raise ValueError(f"{name}: rows overlap (strides {a.stride()})")
    return n, d, ld


def _vector(a, name, dtype, n, like):
    """Address of a contiguous 1-D tensor of n elements."""
    if not isinstance(a, torch.Tensor) or a.dtype is not dtype or a.dim() != 1 or a.shape[0] != n or a.device != like.device:
        raise ValueError(f"{name} must be a {dtype} tensor of shape ({n},) on {like.device}")
    if n > 1 and a.stride(0) != 1:
        raise ValueError(f"{name} must be contiguous")
    return a.data_ptr()


def _in_place(p, ldp, q, ldq):
    """1 where both operands' rows start on 16-byte boundaries."""
    return 0 if (p | q) & 15 or (ldp | ldq) & 7 else 1


def _empty_like(a, contiguous):
    """An uninitialised contiguous tensor of a's shape and type (empty_like takes half of empty's time)."""
    return torch.empty_like(a) if contiguous else a.new_empty(a.shape)


def _workspace(size, device):
    """Workspace of the current stream's pool, so that calls on two streams
    (and two captured graphs) never share one."""
    if size < 0:
        raise ValueError("a size is out of range")
    return torch.empty(size or 1, dtype=torch.uint8, device=device)


def softmax_xent(x, w, target):
    """Softmax cross entropy of the linear head ``x @ w.T`` without keeping
    the logits: ``(loss, lse)``, float32 [n].  x [n, d] and w [v, d] bfloat16
    or float16 (rows contiguous, any row stride), target int64 [n].  A row
    whose target is outside 0..v-1 is ignored: its loss is 0."""
    n, d, ldx = _matrix(x, "x")
    v, dw, ldw = _matrix(w, "w", x)
    if d != dw:
        raise ValueError(f"x has {d} columns and w {dw}")
    y = _vector(target, "target", torch.int64, n, x)
    px, pw, device = x.data_ptr(), w.data_ptr(), x.device
    loss = torch.empty(n, dtype=torch.float32, device=device)
    lse = torch.empty_like(loss)
    L = lib()
    size = L.gbm_softmax_xent_workspace(n, d, v, 0, _in_place(px, ldx, pw, ldw))
    ws = _workspace(size, device) if size else None
    _call(L.gbm_softmax_xent, device, px, ldx, pw, ldw, _TYPES[x.dtype], n, d, v, y, loss.data_ptr(), lse.data_ptr(), ws.data_ptr() if size else None, size)
    return loss, lse


def softmax_xent_grad(x, w, target, lse, grad_loss, want_dx=True, want_dw=True, dw_out=None):
    """Gradients ``(dx, dw)`` of ``sum(grad_loss * loss)`` in the operands'
    type; lse as :func:`softmax_xent` returned it, grad_loss float32 [n].
    Ignored rows get dx = 0 and add nothing to dw.  ``want_dx=False`` /
    ``want_dw=False`` give None in that place and save its product;
    ``dw_out`` (of w's shape and type, rows contiguous) takes dw, so that a :class:`GradClip`
    made once for it stays good."""
    n, d, ldx = _matrix(x, "x")
    v, dw, ldw = _matrix(w, "w", x)
    if d != dw:
        raise ValueError(f"x has {d} columns and w {dw}")
    y = _vector(target, "target", torch.int64, n, x)
    z = _vector(lse, "lse", torch.float32, n, x)
    c = _vector(grad_loss, "grad_loss", torch.float32, n, x)
    if not (want_dx or want_dw):
        raise ValueError("neither dx nor dw is wanted")
    px, pw, device = x.data_ptr(), w.data_ptr(), x.device
    dx = _empty_like(x, ldx == d) if want_dx else None
    lddw = d
    if not want_dw:
        dw = None
    elif dw_out is None:
        dw = _empty_like(w, ldw == d)
    else:
        dw = dw_out
        rows, cols, lddw = _matrix(dw, "dw_out", x)
        if (rows, cols) != (v, d):
            raise ValueError(f"dw_out must have shape ({v}, {d}), got ({rows}, {cols})")
    if n == 0 and not want_dw:
        return dx, dw
    L = lib()
    size = L.gbm_softmax_xent_workspace(n, d, v, 1, _in_place(px, ldx, pw, ldw))
    ws = _workspace(size, device)
    _call(L.gbm_softmax_xent_grad, device, px, ldx, pw, ldw, _TYPES[x.dtype], n, d, v, y, z, c, dx.data_ptr() if want_dx and n else None, d,
          dw.data_ptr() if want_dw else None, lddw, ws.data_ptr(), size)
    return dx, dw


def _leaf_args(x, w, offsets):
    """(rows, x's row stride, leaves, dout, din, offsets' address) of a grouped product."""
    n, d, ldx = _matrix(x, "x")
    if not isinstance(w, torch.Tensor) or w.dim() != 3 or not w.is_contiguous() or 0 in w.shape:
        raise ValueError("w must be a contiguous tensor [leaves, dout, din]")
    if w.dtype is not x.dtype or w.device != x.device:
        raise ValueError(f"w must have x's type and device ({x.dtype}, {x.device}), got {w.dtype}, {w.device}")
    e, dout, din = w.shape
    if d != din:
        raise ValueError(f"x must have {din} columns, got {d}")
    return n, ldx, e, dout, din, _vector(offsets, "offsets", torch.int32, e + 1, x)


def leaf_linear(x, w, offsets, out=None):
    """Products grouped by leaf: row r of leaf g, offsets[g] <= r <
    offsets[g+1], gives ``y[r] = w[g] @ x[r]``.  x [t, din] (rows contiguous,
    any row stride), w [leaves, dout, din] contiguous, both bfloat16 or
    float16; offsets int32 [leaves + 1] on the device, non-decreasing within
    0..t.  Rows that no leaf has (before offsets[0], from offsets[-1] on) are
    0 in a new y and left as they were in ``out``."""
    n, ldx, e, dout, din, off = _leaf_args(x, w, offsets)
    px, pw, device = x.data_ptr(), w.data_ptr(), x.device
    if out is None:
        y, ldy = x.new_empty((n, dout)), dout
    else:
        y = out
        rows, cols, ldy = _matrix(out, "out", x)
        if (rows, cols) != (n, dout):
            raise ValueError(f"out must have shape ({n}, {dout}), got ({rows}, {cols})")
    if n == 0:
        return y
    L = lib()
    size, ws = 0, None
    if not _in_place(px, ldx, pw, din):
        size = L.gbm_leaf_linear_workspace(n, e, din, dout, 0, 0)
        ws = _workspace(size, device)
    _call(L.gbm_leaf_linear, device, px, ldx, pw, off, _TYPES[x.dtype], n, e, din, dout, y.data_ptr(), ldy, int(out is None),
          ws.data_ptr() if size else None, size)
    return y


def leaf_linear_grad(x, w, offsets, dy, want_dx=True, want_dw=True, dw_out=None):
    """Gradients ``(dx, dw)`` of :func:`leaf_linear` in the operands' type:
    ``dx[r] = w[g].T @ dy[r]`` (0 in rows that no leaf has) and ``dw[g]`` the
    sum of ``outer(dy[r], x[r])`` over leaf g's rows (0 for an empty leaf).
    ``dw_out`` (contiguous, of w's shape and type) takes dw."""
    n, ldx, e, dout, din, off = _leaf_args(x, w, offsets)
    rows, cols, lddy = _matrix(dy, "dy", x)
    if (rows, cols) != (n, dout):
        raise ValueError(f"dy must have shape ({n}, {dout}), got ({rows}, {cols})")
    if not (want_dx or want_dw):
        raise ValueError("neither dx nor dw is wanted")
    px, pw, pg, device = x.data_ptr(), w.data_ptr(), dy.data_ptr(), x.device
    dx = _empty_like(x, ldx == din) if want_dx else None
    if not want_dw:
        dw = None
    elif dw_out is None:
        dw = torch.empty_like(w)
    else:
        dw = dw_out
        if not isinstance(dw, torch.Tensor) or dw.shape != w.shape or dw.dtype is not w.dtype or dw.device != w.device or not dw.is_contiguous():
            raise ValueError("dw_out must be contiguous and have w's shape, type and device")
    if n == 0 and not want_dw:
        return dx, dw
    L = lib()
    size = L.gbm_leaf_linear_workspace(n, e, din, dout, 1, _in_place(px, ldx, pw, din) and _in_place(pg, lddy, 0, 0))
    ws = _workspace(size, device) if size else None
    _call(L.gbm_leaf_linear_grad, device, px, ldx, pw, off, pg, lddy, _TYPES[x.dtype], n, e, din, dout, dx.data_ptr() if want_dx and n else None,
          din, 1, dw.data_ptr() if want_dw else None, ws.data_ptr() if size else None, size)
    return dx, dw


class GradClip:
    """The global 2-norm of many gradients, and clipping to it.

    Made once for the gradients of a model (a list of CUDA tensors of one
    device; float32, bfloat16 or float16, each dense), whose buffers it keeps; ``out`` (default: the gradients themselves) takes the
    clipped values.  No two buffers may overlap, but out[i] may be grads[i].
    """

    def __init__(self, grads, out=None):
        grads = list(grads)
        out = grads if out is None else list(out)
        if not grads:
            raise ValueError("no gradients")
        if len(out) != len(grads):
            raise ValueError(f"{len(grads)} gradients but {len(out)} outputs")
        types = _TYPES
        for i, (g, o) in enumerate(zip(grads, out)):
            for a, name in ((g, "gradient"), (o, "output")):
                if not isinstance(a, torch.Tensor) or not a.is_cuda or a.dtype not in types:
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
        self._plan_dev = torch.frombuffer(bytearray(self._plan.raw), dtype=torch.uint8).to(self.device)
        self._ws = L.gbm_grad_clip_workspace(self._plan)
        self._plan_at, self._plan_to, self._clip = C.addressof(self._plan), self._plan_dev.data_ptr(), L.gbm_grad_clip

    def clip(self, max_norm):
        """``out = grad * min(1, max_norm / (norm + 1e-6))`` for every
        gradient; returns the norm before clipping, a float32 scalar tensor
        (nothing is read back to the host)."""
        norm = torch.empty((), dtype=torch.float32, device=self.device)
        ws = _workspace(self._ws, self.device)
        _call(self._clip, self.device, self._plan_at, self._plan_to, float(max_norm), norm.data_ptr(), ws.data_ptr(), self._ws)
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
    device = torch.device("cuda" if device is None else device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    _call(lib().gbm_ops_status, device)
