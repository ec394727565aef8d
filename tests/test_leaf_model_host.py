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
