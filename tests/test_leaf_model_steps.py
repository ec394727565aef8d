"""LeafLinearClassifier on the CPU, its operators replaced by their formulas
(results rounded to the operands' type, as the operators round them)."""
import numpy as np
import pytest

pytest.importorskip("torch")
import torch


class _Clip:
    def __init__(self, grads, out=None):
        self.grads, self.outs = grads, grads if out is None else out

    def clip(self, limit):
        norm = torch.stack([g.double().square().sum() for g in self.grads]).sum().sqrt()
        c = torch.clamp(limit / (norm + 1e-6), max=1.0).float()
        for g, o in zip(self.grads, self.outs):
            o.copy_(g.float() * c)
        return norm.float()


def _leaves(x, offsets):
    return torch.searchsorted(offsets.long(), torch.arange(len(x)), right=True) - 1


def _leaf_linear(x, w, offsets, out=None):
    return torch.einsum("ni,noi->no", x.double(), w.double()[_leaves(x, offsets)]).to(x.dtype)


def _leaf_linear_grad(x, w, offsets, dy, want_dx=True, want_dw=True, dw_out=None):
    leaf = _leaves(x, offsets)
    dw = torch.zeros(w.shape, dtype=torch.float64).index_add_(0, leaf, dy.double()[:, :, None] * x.double()[:, None, :]).to(w.dtype)
    if dw_out is not None:
        dw = dw_out.copy_(dw)
    return torch.einsum("no,noi->ni", dy.double(), w.double()[leaf]).to(x.dtype) if want_dx else None, dw


def _softmax_xent(x, w, target):
    l = x.double() @ w.double().T
    lse = torch.logsumexp(l, 1)
    return (lse - l.gather(1, target[:, None])[:, 0]).float(), lse.float()


def _softmax_xent_grad(x, w, target, lse, grad_loss, want_dx=True, want_dw=True, dw_out=None):
    g = torch.softmax(x.double() @ w.double().T, 1)
    g[torch.arange(len(x)), target] -= 1.0
    g *= grad_loss.double()[:, None]
    dw = (g.T @ x.double()).to(w.dtype)
    return (g @ w.double()).to(x.dtype), dw if dw_out is None else dw_out.copy_(dw)


@pytest.fixture
def on_cpu(monkeypatch, built_lib):
    """The operators' stand-ins; a list to which the test may put errors that linear.status() is to report."""
    from bsscl_gbm_b200 import LeafLinearClassifier, linear
    for f in (_leaf_linear, _leaf_linear_grad, _softmax_xent, _softmax_xent_grad):
        monkeypatch.setattr(linear, f.__name__[1:], f)
    monkeypatch.setattr(linear, "GradClip", _Clip)
    monkeypatch.setattr(LeafLinearClassifier, "_device", lambda self: torch.device("cpu"))
    late = []

    def status(device=None):
        if late:
            raise RuntimeError(late.pop())

    monkeypatch.setattr(linear, "status", status)
    return late


def _data(n=400, p=6, classes=7, seed=0):
    rng = np.random.default_rng(seed)
    X, y = rng.standard_normal((n, p)), rng.integers(0, classes, n)
    y[:classes] = np.arange(classes)
    return X, y


def test_answers_ask_whether_a_wait_ran_out(on_cpu):
    """Weights and answers of operators that say they are not valid are not handed out."""
    from bsscl_gbm_b200 import LeafLinearClassifier
    X, y = _data()
    kw = dict(n_hidden=4, n_epochs=2, batch_size=128)
    m = LeafLinearClassifier(**kw).fit(X, y)
    for ask in (lambda: m.predict_proba(X), lambda: m.predict(X), lambda: m.log_loss(X, y)):
        on_cpu.append("a wait ran out")
        with pytest.raises(RuntimeError, match="ran out"):
            ask()
        assert not on_cpu
        ask()
    on_cpu.append("a wait ran out")
    with pytest.raises(RuntimeError, match="ran out"):
        m.fit(X, y)
    assert not on_cpu
    with pytest.raises(ValueError, match="not fitted"):      # neither the weights of that fit nor the last one's
        m.predict(X)


def test_a_refused_fit_leaves_the_model_as_it_was(on_cpu):
    from bsscl_gbm_b200 import LeafLinearClassifier
    X, y = _data()
    m = LeafLinearClassifier(n_hidden=4, n_epochs=1, batch_size=128).fit(X, y)
    P, best = m.predict_proba(X), m.predict(X)
    for bad in ((X, np.zeros(len(X))), (X, y[:-1]), (X[0], y)):
        with pytest.raises(ValueError):
            m.fit(*bad)
        assert np.array_equal(m.predict_proba(X), P) and np.array_equal(m.predict(X), best)


def _check_step(n, classes, n_hidden, seed, max_norm, few_of_a_class=None):
    """One full-batch float16 step moves the weights by -lr times the 64-bit gradient, clipped.  Features, weights and
    hidden rows are rounded once (the first two in the formula too), dh and the gradients once more: 2^-11 of a value each,
    and of the logits, whose shift is under 2^-11 |h| |head| < 2^-9.  Under 1 % norm-wise in all, for the leaf maps alone and
    for the head alone."""
    from bsscl_gbm_b200 import LeafLinearClassifier
    X, y = _data(n, 5, classes, seed)
    if few_of_a_class:
        y[classes * few_of_a_class:] = 0
        y[:classes * few_of_a_class] = np.arange(classes * few_of_a_class) % classes
    kw = dict(n_hidden=n_hidden, n_epochs=1, batch_size=n, max_norm=max_norm, random_state=1, dtype="float16", class_weight="balanced")
    start = LeafLinearClassifier(learning_rate=0.0, **kw).fit(X, y)
    done = LeafLinearClassifier(learning_rate=1.0, **kw).fit(X, y)
    dev = start._device()
    x, index = start._features(X).double(), torch.from_numpy(np.searchsorted(start.classes_, y)).to(dev)
    w, head = (a.to(torch.float16).double().requires_grad_() for a in (start._w, start._head))
    c = n / (classes * torch.bincount(index, minlength=classes).double())
    loss = torch.nn.functional.cross_entropy(x @ w[0].T @ head.T, index, reduction="none")
    (loss * c[index] / c[index].sum()).sum().backward()
    norm = float((w.grad.square().sum() + head.grad.square().sum()).sqrt())
    clipped = min(1.0, max_norm / (norm + 1e-6))
    for a, b, g in ((start._w, done._w, w.grad), (start._head, done._head, head.grad)):
        moved = (a - b).double()
        assert float((moved - clipped * g).norm() / (clipped * g).norm()) < 0.01
    return norm


STEPS = [(262_144, 30, 8, None), (65_536, 90, 64, None), (8192, 90, 64, 1), (300, 7, 16, None)]


@pytest.mark.parametrize("n,classes,n_hidden,few", STEPS)
def test_half_precision_step(on_cpu, n, classes, n_hidden, few):
    """Many rows a step, and rows of a class that is 99 % of the table: dh of float16 without a scale was 0 for most."""
    norm = _check_step(n, classes, n_hidden, 2, 1e9, few)
    _check_step(n, classes, n_hidden, 2, norm / 3, few)


@pytest.mark.parametrize("h,head,x_top", [(4.0, 0.05, 6.0), (300.0, 2.0, 50.0), (0.0, 0.0, 1.0), (60000.0, 3.0, 1e4), (1.0, 1e-7, 1.0)])
@pytest.mark.parametrize("kind", [torch.float16, torch.float32])
def test_half_precision_scale_fills_the_range(h, head, x_top, kind):
    from bsscl_gbm_b200 import LeafLinearClassifier
    scale = float(LeafLinearClassifier._loss_scale(torch.tensor([[h, -h / 2]], dtype=kind), torch.tensor([[head / 3, -head]], dtype=kind), x_top))
    most = max(h, 2 * head * x_top)
    assert 0 < scale <= 2.0 ** 29 and scale * most <= 2.0 ** 15 * 1.001
    assert most < 2.0 ** -13 or scale * most > 2.0 ** 14


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("max_norm", [-1.0, float("nan")])
def test_a_negative_norm_is_refused(on_cpu, dtype, max_norm):
    """In either type, before anything is learnt; 0 and infinity are limits like others."""
    from bsscl_gbm_b200 import LeafLinearClassifier
    X, y = _data()
    kw = dict(n_hidden=4, n_epochs=1, batch_size=128, dtype=dtype)
    with pytest.raises(ValueError, match="max_norm"):
        LeafLinearClassifier(max_norm=max_norm, **kw).fit(X, y)
    still, free = (LeafLinearClassifier(max_norm=m, **kw).fit(X, y) for m in (0.0, float("inf")))
    start = LeafLinearClassifier(learning_rate=0.0, **kw).fit(X, y)
    assert torch.equal(still._w, start._w) and torch.equal(still._head, start._head)
    assert torch.isfinite(free._w).all() and not torch.equal(free._w, start._w)


def test_a_fit_without_a_random_state(on_cpu):
    from bsscl_gbm_b200 import LeafLinearClassifier
    X, y = _data()
    a, b = (LeafLinearClassifier(n_hidden=4, n_epochs=1, batch_size=128, random_state=None).fit(X, y) for _ in range(2))
    assert torch.isfinite(a._w).all() and not torch.equal(a._w, b._w)


def test_each_rank_takes_its_own_gpu(monkeypatch):
    """As the routing estimator does: LOCAL_RANK's in a process group, the first one elsewhere, a named one always."""
    from bsscl_gbm_b200 import LeafLinearClassifier, leaf_model
    monkeypatch.setenv("LOCAL_RANK", "3")
    assert LeafLinearClassifier()._device() == torch.device("cuda", 0)
    monkeypatch.setattr(leaf_model, "_dist", lambda: object())
    assert LeafLinearClassifier()._device() == torch.device("cuda", 3)
    assert LeafLinearClassifier(device="cuda:1")._device() == torch.device("cuda", 1)


def test_answers_take_classes_in_blocks(on_cpu, monkeypatch):
    """200,000 classes: probabilities of at most 2^26 values at a time, and none of the n x classes matrix for predict."""
    from bsscl_gbm_b200 import LeafLinearClassifier
    X, y = _data(900)
    m = LeafLinearClassifier(n_hidden=4, n_epochs=1, batch_size=900).fit(X, y)
    small = m.predict_proba(X)
    assert np.array_equal(m.predict(X), m.classes_[small.argmax(1)])
    m.classes_, m._head = np.arange(200_000) * 2, torch.randn(200_000, 4, generator=torch.Generator().manual_seed(0))
    softmax, sizes = torch.softmax, []

    def seen(a, dim):
        sizes.append(a.numel())
        return softmax(a, dim)

    monkeypatch.setattr(torch, "softmax", seen)
    monkeypatch.setattr(LeafLinearClassifier, "predict_proba", None)
    best = m.predict(X)
    assert len(sizes) > 1 and max(sizes) <= 1 << 26 and sum(sizes) == 900 * 200_000
    h = torch.cat([h[torch.argsort(rows)] for rows, h in m._hidden(X)]).double()
    at = (h @ m._head.to(torch.bfloat16).double().T).argmax(1).numpy()
    assert np.array_equal(best, m.classes_[at])


@pytest.mark.gpu
def test_predict_of_many_classes_keeps_its_memory():
    from bsscl_gbm_b200 import LeafLinearClassifier
    X, y = _data(20_000, 5, 15_000)
    m = LeafLinearClassifier(n_hidden=16, n_epochs=1).fit(X, y)
    torch.cuda.empty_cache()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    best = m.predict(X)
    assert torch.cuda.max_memory_allocated() - before < 3 * 8 * 2 ** 26       # a block's logits and probabilities, and the head
    assert np.array_equal(best[:700], m.classes_[m.predict_proba(X[:700]).argmax(1)])


@pytest.mark.gpu
@pytest.mark.parametrize("n,classes,n_hidden,few", STEPS)
def test_half_precision_step_on_the_device(n, classes, n_hidden, few):
    norm = _check_step(n, classes, n_hidden, 2, 1e9, few)
    _check_step(n, classes, n_hidden, 2, norm / 3, few)
