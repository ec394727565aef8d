"""Linear models in a tree's leaves under one softmax head.

The reference's leaves hold constants (E:517-823) and its multi-class fit
grows a tree per class and round (E:2949-3065; the engine takes up to 64
classes).  :class:`LeafLinearClassifier` lets one trained tree route the rows,
gives every leaf a linear map of its own and classifies with a head shared by
all leaves, over any number of classes.  Its training step is made of the
device operators of :mod:`bsscl_gbm_b200.linear`.
"""

from __future__ import annotations

import math
import os

import numpy as np

from .estimator import _device_index, _dist


def leaf_of_rows(model, X, tree=0, class_index=0):
    """Index (0 .. leaves-1, in node order) of the leaf that each row of X
    reaches in tree ``tree`` of a fitted estimator (of class ``class_index``'s
    trees for a multi-class one), and the number of leaves.  The rows are
    binned on the GPU with the model's edges and walked like predict_batch_jit
    (E:843-861)."""
    X = model._prep_X(X)
    t = (model.mc_trees[class_index] if model._is_multiclass else model.trees)[tree]
    tf, tt, _, tl, tr, nc = t[:6]
    tf, tt, tl, tr = (np.asarray(a)[:nc] for a in (tf, tt, tl, tr))
    nan_right = None
    if not model._is_multiclass and tree < len(model._tree_nan_right):
        nan_right = model._tree_nan_right[tree]
    xb = model._get_engine().bin_features(X, model.bin_edges, model.feature_bin_counts, model._nan_bin_id)
    node, rows = np.zeros(len(X), np.int64), np.arange(len(X))
    while True:
        f = tf[node]
        inner = f >= 0
        if not inner.any():
            break
        b = xb[rows, np.where(inner, f, 0)].astype(np.int64)
        left = b <= tt[node]
        if nan_right is not None:
            left &= ~((nan_right[node] != 0) & (b == 0))
        node = np.where(inner, np.where(left, tl[node], tr[node]), node)
    leaves = np.flatnonzero(tf < 0)
    return np.searchsorted(leaves, node).astype(np.int32), len(leaves)


class LeafLinearClassifier:
    """Softmax classifier whose hidden rows are linear in the features, with a
    map of their own in every leaf of a routing tree: for a row x of leaf g,
    ``logits = head @ (w[g] @ [x, 1])``.

    router: a fitted HybridHistGBMNumbaV1_0_1 (binary, multi-class or
    regression) whose tree ``tree`` routes the rows; None = one leaf.  Trained
    by stochastic gradient descent on the class-weighted log-loss
    (class_weight as the estimator's), the gradients clipped to ``max_norm``.
    Weights are kept in float32 and multiplied in ``dtype``; in float16 each
    step's loss is scaled so that the gradients fill the type's range.  Features
    are standardised; a missing or infinite value counts as the mean.
    random_state None starts from another state at each fit.
    """

    def __init__(self, router=None, tree=0, n_hidden=64, learning_rate=0.5, max_norm=1.0, n_epochs=10, batch_size=8192,
                 class_weight='balanced_sqrt', dtype='bfloat16', random_state=0, device='b200'):
        if dtype not in ('bfloat16', 'float16'):
            raise ValueError(f"dtype must be 'bfloat16' or 'float16', got {dtype!r}")
        if n_hidden < 1 or n_epochs < 1 or batch_size < 1:
            raise ValueError("n_hidden, n_epochs and batch_size must be at least 1")
        _device_index(device)
        self.router, self.tree, self.n_hidden = router, tree, int(n_hidden)
        self.learning_rate, self.max_norm = float(learning_rate), float(max_norm)
        self.n_epochs, self.batch_size = int(n_epochs), int(batch_size)
        self.class_weight, self.dtype, self.random_state, self.device = class_weight, dtype, random_state, device
        self.loss_history_ = []

    # -- data ---------------------------------------------------------------
    def _device(self):
        import torch
        index = _device_index(self.device)
        if index is None:      # the GPU that the routing estimator takes
            index = int(os.environ.get("LOCAL_RANK", 0)) if _dist() is not None else 0
        return torch.device("cuda", index)

    def _routes(self, X):
        if self.router is None:
            return np.zeros(len(X), np.int32), 1
        return leaf_of_rows(self.router, X, self.tree)

    def _features(self, X):
        """Standardised features and a column of ones, on the device."""
        import torch
        Z = np.nan_to_num((np.asarray(X, np.float64) - self._mean) / self._std, nan=0.0, posinf=0.0, neginf=0.0)
        Z = np.column_stack([Z, np.ones(len(Z))]).astype(np.float32)
        return torch.from_numpy(Z).to(self._device()).to(getattr(torch, self.dtype))

    def _by_leaf(self, rows, leaf):
        """The rows in order of their leaves, and the leaves' offsets."""
        import torch
        order = torch.argsort(leaf[rows], stable=True)
        rows = rows[order]
        count = torch.bincount(leaf[rows], minlength=self.n_leaves_)
        offsets = torch.zeros(self.n_leaves_ + 1, dtype=torch.int32, device=rows.device)
        offsets[1:] = torch.cumsum(count, 0)
        return rows, offsets

    def _check(self, X):
        X = np.asarray(X)
        if X.ndim != 2 or len(X) == 0:
            raise ValueError(f"X must be 2-D with rows, got shape {X.shape}")
        return X

    # -- training -----------------------------------------------------------
    @staticmethod
    def _loss_scale(h, head, x_top):
        """The factor that takes a float16 step's gradients to at most 2^15, on
        the device.  A row's share of the loss is about 1 / rows, so that its
        dh would lie among the type's subnormals or below.  With the rows'
        weights c summing to 1 and sum_v |G_iv| <= 2 c_i: |dhead| <= max |h|,
        |dh| and |dw| <= 2 max |head| max |x| (x has a column of ones)."""
        import torch
        h_top, head_top = (torch.linalg.vector_norm(a, math.inf, dtype=torch.float32) for a in (h, head))
        return 2.0 ** 15 / torch.maximum(h_top, head_top * (2.0 * x_top)).add_(2.0 ** -14)

    def fit(self, X, y):
        import torch

        from . import linear
        X, y = self._check(X), np.asarray(y)
        if len(y) != len(X):
            raise ValueError(f"X has {len(X)} rows but y has {len(y)}")
        if not self.max_norm >= 0:
            raise ValueError(f"max_norm must not be negative, got {self.max_norm}")
        classes, index = np.unique(y, return_inverse=True)
        if len(classes) < 2:
            raise ValueError("y holds a single class")
        self.__dict__.pop('_w', None)      # not fitted until the operators' results are known to be valid
        self.classes_, self.n_features_in_, K = classes, X.shape[1], len(classes)
        finite = np.where(np.isfinite(X), X, np.nan).astype(np.float64)
        seen = np.isfinite(finite).sum(0) > 0
        self._mean, self._std = np.zeros(X.shape[1]), np.ones(X.shape[1])
        self._mean[seen], self._std[seen] = np.nanmean(finite[:, seen], 0), np.nanstd(finite[:, seen], 0)
        self._std[self._std == 0] = 1.0
        weight = np.ones(K)
        if self.class_weight in ('balanced', 'balanced_sqrt'):   # E:2570-2603
            weight = len(y) / (K * np.bincount(index, minlength=K))
            if self.class_weight == 'balanced_sqrt':
                weight = weight ** 0.35
        route, self.n_leaves_ = self._routes(X)
        dev, dt = self._device(), getattr(torch, self.dtype)
        x, leaf = self._features(X), torch.from_numpy(route.astype(np.int64)).to(dev)
        target = torch.from_numpy(index.astype(np.int64).reshape(-1)).to(dev)
        weight = torch.from_numpy(weight).to(dev, torch.float32)
        g = torch.Generator(device=dev).manual_seed(
            int.from_bytes(os.urandom(7), 'little') if self.random_state is None else int(self.random_state))
        p = x.shape[1]
        # one start for all leaves: they part where their rows differ
        first = torch.randn(1, self.n_hidden, p, generator=g, device=dev) * p ** -0.5
        w32 = first.expand(self.n_leaves_, -1, -1).contiguous()
        head32 = torch.randn(K, self.n_hidden, generator=g, device=dev) * 0.1 * self.n_hidden ** -0.5
        w, head = w32.to(dt), head32.to(dt)
        dw, dhead = torch.empty_like(w), torch.empty_like(head)
        clip = linear.GradClip([dw, dhead])
        self.loss_history_ = []
        half = dt == torch.float16
        x_top = float(x.abs().amax()) if half else None
        for _ in range(self.n_epochs):
            total = torch.zeros((), dtype=torch.float64, device=dev)
            shuffled = torch.randperm(len(x), generator=g, device=dev)
            for at in range(0, len(x), self.batch_size):
                rows, offsets = self._by_leaf(shuffled[at:at + self.batch_size], leaf)
                xb, yb = x[rows], target[rows]
                c = weight[yb]
                c = c / c.sum()
                h = linear.leaf_linear(xb, w, offsets)
                loss, lse = linear.softmax_xent(h, head, yb)
                if half:
                    scale = self._loss_scale(h, head, x_top)
                    c = c * scale
                dh, _ = linear.softmax_xent_grad(h, head, yb, lse, c, dw_out=dhead)
                linear.leaf_linear_grad(xb, w, offsets, dh, want_dx=False, dw_out=dw)
                norm = clip.clip(math.inf if half else self.max_norm)
                if half:      # clipped where they are scaled back, in float32
                    step = torch.minimum(self.max_norm / torch.add(norm, scale, alpha=1e-6), 1.0 / scale)
                for master, copy, grad in ((w32, w, dw), (head32, head, dhead)):
                    if half:
                        master.addcmul_(grad.float(), step, value=-self.learning_rate)
                    else:
                        master.add_(grad.float(), alpha=-self.learning_rate)
                    copy.copy_(master)
                total += loss.sum(dtype=torch.float64)
            linear.status(dev)
            self.loss_history_.append(float(total) / len(x))
        self._w, self._head = w32, head32
        return self

    # -- answers ------------------------------------------------------------
    def _hidden(self, X, rows=1 << 16):
        """Blocks of (rows of X, their hidden rows), `rows` at a time.  Raises
        at the end when a wait of the operators that the blocks went through
        ran out."""
        import torch

        from . import linear
        if not hasattr(self, '_w'):
            raise ValueError("This LeafLinearClassifier instance is not fitted yet.")
        X = self._check(X)
        if X.shape[1] != self.n_features_in_:
            raise ValueError(f"X has {X.shape[1]} features; the model has {self.n_features_in_}")
        route, _ = self._routes(X)
        w = self._w.to(getattr(torch, self.dtype))
        for at in range(0, len(X), rows):
            x = self._features(X[at:at + rows])
            leaf = torch.from_numpy(route[at:at + rows].astype(np.int64)).to(x.device)
            order, offsets = self._by_leaf(torch.arange(len(x), device=x.device), leaf)
            yield at + order, linear.leaf_linear(x[order], w, offsets)
        linear.status(self._device())

    def _probabilities(self, X):
        """Blocks of (rows of X, their probabilities in float64 on the device),
        of at most 2^26 values."""
        import torch
        classes = len(self.classes_) if hasattr(self, 'classes_') else 1
        for rows, h in self._hidden(X, max(1, min(1 << 16, (1 << 26) // classes))):
            yield rows, torch.softmax(h.double() @ self._head.to(h.dtype).double().T, 1)

    def predict_proba(self, X):
        """Class probabilities [n, classes] (float64)."""
        out = np.empty((len(X), len(self.classes_) if hasattr(self, 'classes_') else 0))
        for rows, p in self._probabilities(X):
            out[rows.cpu().numpy()] = p.cpu().numpy()
            del p      # before the next block is computed
        return out

    def predict(self, X):
        """The most probable class of each row, without the n x classes matrix."""
        best = np.empty(len(X), np.int64)
        for rows, p in self._probabilities(X):
            best[rows.cpu().numpy()] = p.argmax(1).cpu().numpy()
            del p
        return self.classes_[best]

    def log_loss(self, X, y):
        """Mean log-loss of the labels, without the n x classes matrix of
        probabilities; labels that fit() did not see raise KeyError."""
        import torch

        from . import linear
        y = np.asarray(y)
        if len(y) != len(X):
            raise ValueError(f"X has {len(X)} rows but y has {len(y)}")
        total = 0.0
        for rows, h in self._hidden(X):
            labels = y[rows.cpu().numpy()]
            index = np.minimum(np.searchsorted(self.classes_, labels), len(self.classes_) - 1)
            if np.any(self.classes_[index] != labels):
                raise KeyError("y holds a label that fit() did not see")
            loss, _ = linear.softmax_xent(h, self._head.to(h.dtype), torch.from_numpy(index.astype(np.int64)).to(h.device))
            total += float(loss.sum(dtype=torch.float64))
        return total / len(y)
