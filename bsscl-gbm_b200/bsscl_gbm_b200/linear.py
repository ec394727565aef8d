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
There is no CPU path.  The operators know no autograd: tensors that require
gradients are taken as they are, results require none, and the gradients are
what the ``_grad`` calls return (``backward()`` finds nothing behind a
result).  Wrong types, shapes, strides and devices, and a given output that
overlaps what its call reads, raise ValueError before anything is launched.
"""

from __future__ import annotations

import ctypes as C

import torch

from ._lib import ERRORS, GBM_OK, lib

lib()     # a missing library is reported by name, before the module that links it
try:
    from . import _torch_ops as _ops
except ImportError as e:
    raise RuntimeError(f"_torch_ops.so cannot be loaded ({e}); build it with `make -C bsscl-gbm_b200/csrc` for this torch") from e

_TYPES = {torch.float32: 0, torch.bfloat16: 2, torch.float16: 3}     # GBM_TYPE_*


def softmax_xent(x, w, target):
    """Softmax cross entropy of the linear head ``x @ w.T`` without keeping
    the logits: ``(loss, lse)``, float32 [n] and computed in 32 bits.  x [n, d]
    and w [v, d] bfloat16 or float16 (rows contiguous, any row stride that keeps
    them apart), target int64 [n].  A row whose target is outside 0..v-1 is
    ignored: its loss is 0."""
    return _ops.softmax_xent(x, w, target)


def softmax_xent_grad(x, w, target, lse, grad_loss, want_dx=True, want_dw=True, dw_out=None):
    """Gradients ``(dx, dw)`` of ``sum(grad_loss * loss)`` in the operands'
    type; lse as :func:`softmax_xent` returned it, grad_loss float32 [n].
    Ignored rows get dx = 0 and add nothing to dw.  The rows x classes matrix
    between them is rounded to the operands' type once (up to 256 rows it is
    kept in two parts), in float16 relative to the largest ``|grad_loss|`` (down
    to 2^-39 of it); products are summed in 32 bits.  ``want_dx=False`` /
    ``want_dw=False`` give None in that place and save its product;
    ``dw_out`` (of w's shape and type, rows contiguous) takes dw, so that a
    :class:`GradClip` made once for it stays good."""
    return _ops.softmax_xent_grad(x, w, target, lse, grad_loss, want_dx, want_dw, dw_out)


def leaf_linear(x, w, offsets, out=None):
    """Products grouped by leaf: row r of leaf g, offsets[g] <= r <
    offsets[g+1], gives ``y[r] = w[g] @ x[r]``.  x [t, din] (rows as
    :func:`softmax_xent`'s), w [leaves, dout, din] contiguous, both bfloat16 or
    float16; offsets int32 [leaves + 1] on the device, non-decreasing within
    0..t.  Rows that no leaf has (before offsets[0], from offsets[-1] on) are
    0 in a new y and left as they were in ``out``."""
    return _ops.leaf_linear(x, w, offsets, out)


def leaf_linear_grad(x, w, offsets, dy, want_dx=True, want_dw=True, dw_out=None):
    """Gradients ``(dx, dw)`` of :func:`leaf_linear` in the operands' type:
    ``dx[r] = w[g].T @ dy[r]`` (0 in rows that no leaf has) and ``dw[g]`` the
    sum of ``outer(dy[r], x[r])`` over leaf g's rows (0 for an empty leaf).
    ``dw_out`` (contiguous, of w's shape and type) takes dw."""
    return _ops.leaf_linear_grad(x, w, offsets, dy, want_dx, want_dw, dw_out)


class GradClip:
    """The global 2-norm of many gradients, and clipping to it.

    Made once for the gradients of a model (a list of CUDA tensors of one
    device; float32, bfloat16 or float16, each dense), whose buffers it keeps;
    ``out`` (default: the gradients themselves) takes the clipped values.  Making
    it takes some 40 us for 5 gradients and 0.9 ms for 300 (checks, and a copy
    that waits): keep it, and the gradients in their buffers, from step to step.  No
    two buffers may overlap, but out[i] may be grads[i], and calls on two
    streams at once would write the same outputs: wait between them.  A CUDA
    graph that holds its calls needs the object as long as it is replayed.
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
        self._plan_at = C.addressof(self._plan)

    def clip(self, max_norm):
        """``out = grad * min(1, max_norm / (norm + 1e-6))`` for every
        gradient; returns the norm before clipping, a float32 scalar tensor
        (nothing is read back to the host)."""
        return _ops.grad_clip(self._plan_at, self._plan_dev, max_norm)


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
    call, or an asynchronous error occurred.  After a wait that ran out the
    products do nothing until this has told it.  There is one answer a device:
    with several streams at work, wait for all of them and ask once."""
    err = C.create_string_buffer(256)
    with torch.cuda.device(device):
        rc = lib().gbm_ops_status(torch.cuda.current_stream().cuda_stream, err, 256)
    if rc != GBM_OK:
        raise RuntimeError(f"{err.value.decode(errors='replace')} ({ERRORS.get(rc, rc)})")
