"""LeafLinearClassifier: rows routed by a trained tree, a linear map in every
leaf, one softmax head; its answers against the formula in 64 bits."""
import numpy as np
import pytest

pytest.importorskip("torch")


def _data(n=3000, p=11, seed=0, classes=90):
    rng = np.random.default_rng(seed)
    X = rng.standard_normal((n, p))
    X[rng.random((n, p)) < 0.05] = np.nan
    y = rng.integers(0, classes, n)
    y[:classes] = np.arange(classes)
    return X, y


def _router(X, seed=0):
    from bsscl_gbm_b200 import HybridHistGBMNumbaV1_0_1
    z = (np.nan_to_num(X[:, 0]) * np.nan_to_num(X[:, 1]) > 0.1).astype(int)
    return HybridHistGBMNumbaV1_0_1(n_estimators=3, max_depth=4, random_state=seed, verbose=False).fit(X, z)


def test_refusals_need_no_gpu():
    from bsscl_gbm_b200 import LeafLinearClassifier
    for kw in ({"dtype": "float32"}, {"n_hidden": 0}, {"batch_size": 0}, {"n_epochs": 0}, {"device": "cpu"}):
        with pytest.raises(ValueError):
            LeafLinearClassifier(**kw)
    m = LeafLinearClassifier()
    with pytest.raises(ValueError, match="single class"):
        m.fit(np.zeros((4, 2)), np.zeros(4))
    with pytest.raises(ValueError, match="rows"):
        m.fit(np.zeros((4, 2)), np.zeros(3))
    with pytest.raises(ValueError, match="not fitted"):
        m.predict_proba(np.zeros((4, 2)))


def test_every_answer_of_an_unfitted_model_says_so(built_lib):
    from bsscl_gbm_b200 import LeafLinearClassifier
    X = np.zeros((3, 2))
    for ask in (LeafLinearClassifier().predict, LeafLinearClassifier().predict_proba):
        with pytest.raises(ValueError, match="not fitted"):
            ask(X)


@pytest.mark.gpu
def test_leaf_of_rows_follows_the_tree():
    from bsscl_gbm_b200 import leaf_of_rows
    X, _ = _data()
    router = _router(X)
    for k in range(3):
        leaf, count = leaf_of_rows(router, X, k)
        tf, _, tv, _, _, nc, _ = router.trees[k]
        values = np.asarray(tv)[:nc][np.asarray(tf)[:nc] < 0]
        assert count == len(values) and leaf.min() >= 0 and leaf.max() < count
        # one tree's value of each row, as the single-tree predict has it
        from bsscl_gbm_b200.estimator import _predict_tree_host
        xb = router._get_engine().bin_features(router._prep_X(X), router.bin_edges, router.feature_bin_counts, router._nan_bin_id)
        assert np.array_equal(values[leaf], _predict_tree_host(xb, router.trees[k]))


@pytest.mark.gpu
def test_routers_of_other_kinds():
    """A multi-class, a regression and a NaN-direction model's trees route rows too."""
    from bsscl_gbm_b200 import HybridHistGBMNumbaV1_0_1, HybridHistGBMRegressorV1_0_1, LeafLinearClassifier, leaf_of_rows
    X, y = _data(n=1200, classes=70)
    z = np.nan_to_num(X[:, 0]) + np.nan_to_num(X[:, 1])
    kw = dict(n_estimators=2, max_depth=3, random_state=0, verbose=False)
    for model, labels in ((HybridHistGBMNumbaV1_0_1(**kw), np.digitize(z, [-0.5, 0.5])), (HybridHistGBMRegressorV1_0_1(**kw), z),
                          (HybridHistGBMNumbaV1_0_1(nan_direction='learn', **kw), (z > 0).astype(int))):
        model.fit(X, labels)
        leaf, count = leaf_of_rows(model, X, 1)
        assert count > 1 and set(np.unique(leaf)) <= set(range(count)) and len(np.unique(leaf)) > 1
        m = LeafLinearClassifier(model, tree=1, n_hidden=8, n_epochs=1).fit(X, y)
        assert m.n_leaves_ == count and np.isfinite(m.predict_proba(X[:50])).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("routed", [False, True])
def test_fit_and_answers(routed, dtype):
    from bsscl_gbm_b200 import LeafLinearClassifier, leaf_of_rows
    X, y = _data()
    y = y * 3 - 7
    router = _router(X) if routed else None
    m = LeafLinearClassifier(router, n_hidden=24, n_epochs=2, batch_size=700, dtype=dtype, random_state=3).fit(X, y)
    assert len(m.classes_) == 90 and len(m.loss_history_) == 2 and np.isfinite(m.loss_history_).all()
    assert m.n_leaves_ == (leaf_of_rows(router, X)[1] if routed else 1)
    P = m.predict_proba(X)
    assert P.shape == (3000, 90) and np.abs(P.sum(1) - 1).max() < 1e-12
    assert np.array_equal(m.predict(X), m.classes_[P.argmax(1)])
    # the answers from the weights, in 64 bits with the hidden rows rounded once: one rounding that falls the other way
    # moves a logit by eps |h| |head|, well under the 1 % taken here
    leaf = leaf_of_rows(router, X)[0] if routed else np.zeros(3000, int)
    import torch
    dt = getattr(torch, dtype)
    x = m._features(X).double().cpu()
    w, head = m._w.to(dt).double().cpu(), m._head.to(dt).double().cpu()
    h = torch.einsum("ni,noi->no", x, w[torch.from_numpy(leaf.astype(np.int64))]).to(dt).double()
    want = torch.softmax(h @ head.T, 1).numpy()
    assert np.abs(P / want - 1).max() < 0.01
    # the mean of -log of the labels' probabilities, both computed from the same hidden rows
    ll = -np.log(P[np.arange(3000), np.searchsorted(m.classes_, y)]).mean()
    assert abs(m.log_loss(X, y) - ll) < 1e-5
    with pytest.raises(KeyError):
        m.log_loss(X[:2], np.array([0, 1]))
    with pytest.raises(ValueError, match="features"):
        m.predict(X[:, :5])
    # the same seed gives the same model
    again = LeafLinearClassifier(router, n_hidden=24, n_epochs=2, batch_size=700, dtype=dtype, random_state=3).fit(X, y)
    assert again.loss_history_ == m.loss_history_ and np.array_equal(again.predict_proba(X), P)


@pytest.mark.gpu
def test_one_step_is_the_formulas_gradient():
    """One full-batch step without clipping moves the weights by -lr times the 64-bit gradient of the weighted log-loss.
    Hidden rows, G and the gradients are rounded once each (bf16: 2^-8 of a value), the hidden rows' rounding moves the
    logits by under 1 %: 4 % norm-wise in all."""
    import torch

    from bsscl_gbm_b200 import LeafLinearClassifier, leaf_of_rows
    X, y = _data(n=1500, classes=70)
    router = _router(X)
    kw = dict(n_hidden=16, n_epochs=1, batch_size=1500, max_norm=1e9, random_state=1)
    start = LeafLinearClassifier(router, learning_rate=0.0, **kw).fit(X, y)
    done = LeafLinearClassifier(router, learning_rate=1.0, **kw).fit(X, y)
    leaf = torch.from_numpy(leaf_of_rows(router, X)[0].astype(np.int64)).cuda()
    x = start._features(X).double()
    w, head = (a.to(torch.bfloat16).double().requires_grad_() for a in (start._w, start._head))
    index = torch.from_numpy(np.searchsorted(start.classes_, y)).cuda()
    c = (1500 / (70 * torch.bincount(index, minlength=70).double())) ** 0.35
    logits = torch.einsum("ni,noi->no", x, w[leaf]) @ head.T
    loss = torch.nn.functional.cross_entropy(logits, index, reduction="none")
    (loss * c[index] / c[index].sum()).sum().backward()
    for a, b, g in ((start._w, done._w, w.grad), (start._head, done._head, head.grad)):
        moved = (a - b).double()
        assert float((moved - g).norm() / g.norm()) < 0.04
