"""The device operators for leaf-wise linear models against their definitions
in 64 bits: softmax cross entropy of a linear head with its gradients,
products grouped by leaf with theirs, the global norm and clipping.

Tolerances, element by element, with u = finfo(type).eps / 2 (one rounding):
- a sum of K products in 32 bits, in any order and with truncating adds:
  K 2^-23 sum |a b|  =: eps_K;
- a logit: eps_d; a sum of v exponentials: v 2^-23 of itself; exp and log:
  2^-20 of the value and absolute, so |lse - lse64| <= eps_d + v 2^-23 + 2^-20
  + |lse| 2^-23 and the loss takes one eps_d more;
- G = c (p - [k = y]) : |c| p (e^(both errors) - 1 + 2^-20) before it is
  rounded once (u |G|, in half precision at least 2^-40 of the largest |c|,
  its power-of-two scale); dx and dw sum these errors over |w| and |x|, then
  round (u, and 2^-25 where half precision runs out of exponents).
"""
import ctypes as C

import numpy as np
import pytest

pytest.importorskip("torch")
import torch

gpu = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _u(t):
    return torch.finfo(t).eps / 2


def _tiny(t):
    return 2.0 ** -25 if t == torch.float16 else 2.0 ** -130


def _near(got, want, tol, what):
    got = got.double()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} values off, worst "
                           f"{float(((got - want).abs() / tol).nan_to_num(nan=float('inf')).max()):.3g} x the tolerance")


def _rand(shape, t, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(t)


def _targets(n, v, ignored, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    y = torch.randint(0, v, (n,), generator=g, device="cuda")
    y[torch.rand(n, generator=g, device="cuda") < ignored] = -1
    return y


# ---------------------------------------------------------------------------
# softmax cross entropy
# ---------------------------------------------------------------------------

def _xent64(x, w, y, c):
    """loss, lse, dx, dw and their tolerances, from the definition in 64 bits."""
    t, (n, d), v = x.dtype, x.shape, w.shape[0]
    has = (y >= 0) & (y < v)
    X, W = x.double(), w.double()
    X = torch.where(has[:, None], X, 0.0) if not torch.isfinite(X).all() else X
    l = X @ W.T
    size = X.abs() @ W.abs().T                                # sum |x w| of each logit
    el = d * 2.0 ** -23 * size.max(1).values                  # of every logit of the row
    lse = torch.logsumexp(l, 1)
    tz = el + v * 2.0 ** -23 + 2.0 ** -20 + lse.abs() * 2.0 ** -23
    at = y.clamp(0, v - 1)[:, None]
    ly = l.gather(1, at)[:, 0]
    loss = torch.where(has, lse - ly, 0.0)
    tl = torch.where(has, tz + el + (lse.abs() + ly.abs()) * 2.0 ** -23, 0.0)
    p = torch.exp(l - lse[:, None])
    cc = torch.where(has, c.double(), 0.0)[:, None]
    g = cc * (p - torch.zeros_like(p).scatter_(1, at, 1.0))
    eg = cc.abs() * p * (torch.expm1(el + tz) + 2.0 ** -20)[:, None] + _u(t) * g.abs() \
        + cc.abs() * 2.0 ** -22 * (g.abs() > 0)
    if t == torch.float16:
        eg = eg + cc.abs().max() * 2.0 ** -40
    Xz = torch.where(has[:, None], X, 0.0)
    dx, dw = g @ W, g.T @ Xz
    tdx = eg @ W.abs() + v * 2.0 ** -23 * (g.abs() @ W.abs())
    tdw = eg.T @ Xz.abs() + n * 2.0 ** -23 * (g.abs().T @ Xz.abs())
    return (loss, lse, dx, dw), (tl + 1e-30, tz, tdx + _u(t) * dx.abs() + _tiny(t), tdw + _u(t) * dw.abs() + _tiny(t))


def _check_xent(x, w, y, c):
    from bsscl_gbm_b200 import linear
    loss, lse = linear.softmax_xent(x, w, y)
    dx, dw = linear.softmax_xent_grad(x, w, y, lse, c)
    linear.status()
    want, tol = _xent64(x, w, y, c)
    for got, a, b, name in zip((loss, lse, dx, dw), want, tol, ("loss", "lse", "dx", "dw")):
        _near(got, a, b, name)
    return loss, lse, dx, dw


XENT = [(1, 1, 1), (1, 8, 2), (1, 64, 1000), (2, 30, 3), (3, 100, 64), (7, 64, 65), (64, 64, 64), (65, 100, 129),
        (127, 200, 255), (128, 256, 256), (129, 72, 257), (255, 1024, 300), (256, 65, 1000), (300, 128, 5000),
        (1000, 100, 1501), (33, 2048, 70), (513, 264, 513), (2000, 40, 2000),
        # few rows against many classes, features that end inside a step
        (1, 72, 9001), (5, 1000, 20011), (8, 264, 9000), (9, 520, 30000), (16, 104, 20000), (17, 1024, 9999), (32, 8, 40001)]


@gpu
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("n,d,v", XENT)
def test_xent_sizes(n, d, v, kind):
    t = TYPES[kind]
    x, w = _rand((n, d), t, n + d), _rand((v, d), t, v, 2.0 / d ** 0.5)
    y = _targets(n, v, 0.2, 5)
    c = torch.rand(n, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda") + 0.25
    _check_xent(x, w, y, c)


@gpu
@pytest.mark.parametrize("n,d,v", [(2100, 24, 131073), (19100, 16, 14849)])
def test_xent_pieces(n, d, v):
    """More than 512 MB of G: two pieces of classes, dx summed over them (the first case with split sums as well)."""
    t = torch.bfloat16
    x, w = _rand((n, d), t, 1), _rand((v, d), t, 2, 2.0 / d ** 0.5)
    c = torch.rand(n, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda") + 0.25
    _check_xent(x, w, _targets(n, v, 0.2, 5), c)
    torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_xent_strides(kind):
    """Rows of a wider table, at offsets that are not 16-byte aligned."""
    t = TYPES[kind]
    for off, d, pitch in ((0, 96, 136), (1, 96, 131), (3, 50, 77), (8, 64, 65)):
        x = _rand((150, pitch), t, 1)[:, off:off + d]
        w = _rand((333, pitch), t, 2, 2.0 / d ** 0.5)[:, off:off + d]
        c = torch.linspace(-1.0, 2.0, 150, device="cuda")
        _check_xent(x, w, _targets(150, 333, 0.1, 3), c)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_xent_rows_without_a_target(kind):
    t = TYPES[kind]
    x, w = _rand((140, 64), t, 1), _rand((300, 64), t, 2, 0.25)
    c = torch.ones(140, device="cuda")
    # every row ignored; targets beyond both ends
    y = torch.full((140,), -100, device="cuda")
    y[::3] = 300
    y[1::3] = -2 ** 62
    loss, lse, dx, dw = _check_xent(x, w, y, c)
    assert not loss.any() and not dx.any() and not dw.any()
    # NaN and infinities in ignored rows' features reach neither dw nor other rows
    y = _targets(140, 300, 0.0, 4)
    x[5], x[77], y[5], y[77] = float("nan"), float("inf"), -1, 300
    from bsscl_gbm_b200 import linear
    loss, lse = linear.softmax_xent(x, w, y)
    dx, dw = linear.softmax_xent_grad(x, w, y, lse, c)
    want, tol = _xent64(x, w, y, c)
    keep = torch.ones(140, dtype=torch.bool, device="cuda")
    keep[[5, 77]] = False
    _near(loss, want[0], tol[0], "loss")
    _near(lse[keep], want[1][keep], tol[1][keep], "lse")
    _near(dx, want[2], tol[2], "dx")
    _near(dw, want[3], tol[3], "dw")
    # with few rows too, against classes enough for many blocks
    few, many = x[:8].contiguous(), _rand((9000, 64), t, 7, 0.25)
    z = linear.softmax_xent(few, many, y[:8])[1]
    assert torch.isnan(z[5]) and torch.isfinite(z[[0, 1, 2, 3, 4, 6, 7]]).all()
    # NaN in a row that counts stays in that row's loss
    y[5] = 3
    loss = linear.softmax_xent(x, w, y)[0]
    assert torch.isnan(loss[5]) and torch.isfinite(loss[keep]).all()


@gpu
def test_xent_wide_logits():
    """Logits of hundreds: the maximum carries the row; a class far below it gives a probability of 0."""
    x, w = _rand((70, 128), torch.bfloat16, 1, 8.0), _rand((500, 128), torch.bfloat16, 2, 4.0)
    _check_xent(x, w, _targets(70, 500, 0.0, 3), torch.ones(70, device="cuda"))


@gpu
@pytest.mark.parametrize("size", [2.0 ** -12, 1.0, 2.0 ** 10])
def test_xent_half_gradients_keep_their_bits(size):
    """Half precision holds 5 exponent bits: the upstream gradient's size must not cost the probabilities theirs."""
    x, w = _rand((256, 64), torch.float16, 1), _rand((4096, 64), torch.float16, 2, 0.1)
    _check_xent(x, w, _targets(256, 4096, 0.0, 3), torch.full((256,), size, device="cuda"))


@gpu
def test_xent_empty_and_partial():
    from bsscl_gbm_b200 import linear
    w = _rand((50, 16), torch.float16, 2)
    x = torch.empty(0, 16, dtype=torch.float16, device="cuda")
    y = torch.empty(0, dtype=torch.int64, device="cuda")
    f = torch.empty(0, device="cuda")
    loss, lse = linear.softmax_xent(x, w, y)
    assert loss.shape == lse.shape == (0,)
    dx, dw = linear.softmax_xent_grad(x, w, y, f, f)
    assert dx.shape == (0, 16) and not dw.any()
    x, y, c = _rand((40, 16), torch.float16, 3), _targets(40, 50, 0.1, 4), torch.ones(40, device="cuda")
    lse = linear.softmax_xent(x, w, y)[1]
    both = linear.softmax_xent_grad(x, w, y, lse, c)
    one = linear.softmax_xent_grad(x, w, y, lse, c, want_dw=False)
    two = linear.softmax_xent_grad(x, w, y, lse, c, want_dx=False)
    assert one[1] is None and two[0] is None
    assert torch.equal(one[0], both[0]) and torch.equal(two[1], both[1])


@gpu
def test_xent_gradient_against_differences():
    """The loss summed in 64 bits over the operator's rows, moved along a direction, against the operator's gradients.
    The features take steps of 2^-4 that bf16 holds exactly (values on a 2^-4 grid below 8), so the difference's error is
    its third-order term, h^2/6 |f'''| <= h^2/6 sum_i c_i 4 max|l'|^3, and the losses' tolerance over 2h."""
    from bsscl_gbm_b200 import linear
    n, d, v, h = 40, 24, 100, 2.0 ** -4
    g = torch.Generator(device="cuda").manual_seed(1)
    x = (torch.randint(-32, 33, (n, d), generator=g, device="cuda") * 2.0 ** -4).to(torch.bfloat16)
    w = _rand((v, d), torch.bfloat16, 2, 0.2)
    y, c = _targets(n, v, 0.1, 3), torch.rand(n, generator=g, device="cuda") + 0.5
    step = torch.zeros(n, d, device="cuda")
    step[:, 5] = torch.randint(0, 2, (n,), generator=g, device="cuda") * 2.0 - 1.0
    lse = linear.softmax_xent(x, w, y)[1]
    dx, _ = linear.softmax_xent_grad(x, w, y, lse, c)
    f = [(linear.softmax_xent((x.float() + s * h * step).to(torch.bfloat16), w, y)[0].double() * c).sum() for s in (1, -1)]
    want = (f[0] - f[1]) / (2 * h)
    got = (dx.double() * step).sum()
    (_, tol) = _xent64(x, w, y, c)
    slope = w[:, 5].double().abs().max()
    bound = h * h / 6 * c.sum() * 4 * slope ** 3 + (tol[0] * c).sum() / h + (tol[2] * step.abs()).sum()
    assert abs(float(got - want)) <= float(bound)


# ---------------------------------------------------------------------------
# products grouped by leaf
# ---------------------------------------------------------------------------

def _offsets(counts, first=0):
    return torch.tensor(np.concatenate([[first], first + np.cumsum(counts)]), dtype=torch.int32, device="cuda")


def _check_leaf(x, w, off, dy, t_rows=None):
    from bsscl_gbm_b200 import linear
    t, (e, dout, din), n = x.dtype, w.shape, x.shape[0]
    y = linear.leaf_linear(x, w, off)
    dx, dw = linear.leaf_linear_grad(x, w, off, dy)
    linear.status()
    edge = [min(max(int(o), 0), n) for o in off.tolist()]
    Y, DX, DW = (torch.zeros(s, dtype=torch.float64, device="cuda") for s in ((n, dout), (n, din), (e, dout, din)))
    TY, TX, TW = (torch.zeros_like(a) for a in (Y, DX, DW))
    for k in range(e):
        lo, hi = edge[k], max(edge[k], edge[k + 1])
        a, b, m = x[lo:hi].double(), dy[lo:hi].double(), w[k].double()
        Y[lo:hi], TY[lo:hi] = a @ m.T, din * 2.0 ** -23 * (a.abs() @ m.abs().T)
        DX[lo:hi], TX[lo:hi] = b @ m, dout * 2.0 ** -23 * (b.abs() @ m.abs())
        DW[k], TW[k] = b.T @ a, (hi - lo) * 2.0 ** -23 * (b.abs().T @ a.abs())
    for got, want, tol, name in ((y, Y, TY, "y"), (dx, DX, TX, "dx"), (dw, DW, TW, "dw")):
        _near(got, want, tol + _u(t) * want.abs() + _tiny(t) * (want != 0), name)
    return y, dx, dw


# a few rows in most leaves, a block of them in one; then
# many short leaves: one stage of rows a tile, each with its tail, many tiles a cluster
LEAF = [([1, 0, 2] * 20 + [70], 1032, 40), ([0] * 9 + [40], 264, 17), ([3, 1, 7, 63, 2, 65] * 40, 264, 520), ([1], 1, 1), ([1], 8, 8), ([0, 3, 0], 30, 20), ([5, 0, 64, 1], 64, 64), ([63, 65, 127, 129], 100, 61),
        ([0, 0, 0], 16, 24), ([256, 255, 257, 1, 0, 2], 128, 256), ([700], 264, 136), ([1] * 40, 72, 300),
        ([33, 0, 500, 7], 1000, 50), ([64] * 8, 256, 512), ([3, 1000, 0, 20], 40, 520)]


@gpu
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("counts,din,dout", LEAF)
def test_leaf_sizes(counts, din, dout, kind):
    t, n, e = TYPES[kind], sum(counts), len(counts)
    x, dy = _rand((n, din), t, 1), _rand((n, dout), t, 2)
    w = _rand((e, dout, din), t, 3, din ** -0.5)
    _check_leaf(x, w, _offsets(counts), dy)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_leaf_strides_and_rows_outside(kind):
    """Rows before the first and behind the last leaf, NaN in them; row strides and offsets that are not 16-byte aligned."""
    from bsscl_gbm_b200 import linear
    t, counts = TYPES[kind], [70, 0, 130, 9]
    n = sum(counts) + 40
    off = _offsets(counts, 13)
    for at, din, dout, pitch in ((0, 64, 64, 96), (1, 64, 72, 99), (5, 33, 17, 61)):
        x, dy = _rand((n, pitch), t, 1)[:, at:at + din], _rand((n, 2 * pitch), t, 2)[:, at:at + dout]
        w = _rand((4, dout, din), t, 3, din ** -0.5)
        x[:13], x[n - 27:] = float("nan"), float("inf")
        dy[:13], dy[n - 27:] = float("nan"), float("inf")
        y, dx, dw = _check_leaf(x, w, off, dy)
        assert not y[:13].any() and not y[n - 27:].any() and not dx[:13].any() and not dx[n - 27:].any()
        # an output of the caller's keeps what those rows held, and what lies between its rows
        hold = torch.full((n, dout + 7), 5.0, dtype=t, device="cuda")
        out = linear.leaf_linear(x, w, off, out=hold[:, 2:2 + dout])
        assert out.data_ptr() == hold[:, 2:].data_ptr()
        assert torch.equal(out[13:n - 27], y[13:n - 27])
        assert (hold[:13] == 5).all() and (hold[n - 27:] == 5).all()
        assert (hold[:, :2] == 5).all() and (hold[:, 2 + dout:] == 5).all()


@gpu
def test_leaf_nan_stays_in_its_leaf():
    """NaN in one leaf's rows or weights does not reach its neighbours, whose rows share tiles with it."""
    from bsscl_gbm_b200 import linear
    t, counts = torch.bfloat16, [10, 20, 30]
    x, dy, w = _rand((60, 72), t, 1), _rand((60, 40), t, 2), _rand((3, 40, 72), t, 3, 0.1)
    x[10:30], dy[12], w[1] = float("nan"), float("inf"), float("nan")
    off = _offsets(counts)
    y = linear.leaf_linear(x, w, off)
    dx, dw = linear.leaf_linear_grad(x, w, off, dy)
    for a in (y[:10], y[30:], dx[:10], dx[30:], dw[0], dw[2]):
        assert torch.isfinite(a).all()
    assert torch.isnan(y[10:30]).all() and torch.isnan(dw[1]).all()


@gpu
def test_leaf_bad_offsets_stay_inside():
    """Offsets out of order or out of range are clamped: nothing outside the arrays is touched."""
    from bsscl_gbm_b200 import linear
    t = torch.float16
    x, dy, w = _rand((100, 64), t, 1), _rand((100, 32), t, 2), _rand((4, 32, 64), t, 3, 0.1)
    off = torch.tensor([-5, 40, 20, 60, 1000], dtype=torch.int32, device="cuda")
    hold = torch.full((140, 32), 5.0, dtype=t, device="cuda")
    linear.leaf_linear(x, w, off, out=hold[20:120])
    dx, dw = linear.leaf_linear_grad(x, w, off, dy)
    linear.status()
    assert (hold[:20] == 5).all() and (hold[120:] == 5).all()
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all()
    want = x[60:].double() @ w[3].double().T
    _near(hold[80:120], want, 64 * 2.0 ** -23 * (x[60:].double().abs() @ w[3].double().abs().T) + _u(t) * want.abs() + _tiny(t), "y")
    assert not dw[1].any()


@gpu
def test_leaf_many_leaves():
    """Thousands of leaves, most of them empty: more than one look at 32 of them, and than the 2048 that are sorted."""
    for e in (100, 3000):
        counts = np.random.default_rng(e).integers(0, 3, e) * (np.random.default_rng(1).random(e) < 0.3)
        counts[-1] = 5
        n = int(counts.sum())
        x, dy, w = _rand((n, 40), torch.bfloat16, 1), _rand((n, 24), torch.bfloat16, 2), _rand((e, 24, 40), torch.bfloat16, 3, 0.2)
        _check_leaf(x, w, _offsets(counts), dy)


@gpu
def test_offsets_beyond_32_bits():
    """More than 2^31 elements in one operand: the last rows are where they belong."""
    from bsscl_gbm_b200 import linear
    t, n, wide = torch.bfloat16, 140_000, 16_384
    assert n * wide > 2 ** 31
    x, w = _rand((n, 8), t, 1), _rand((2, wide, 8), t, 2)
    off = _offsets([n - 300, 300])
    y = linear.leaf_linear(x, w, off)
    for lo, hi, k in ((0, 200, 0), (n - 400, n - 300, 0), (n - 300, n, 1)):
        want = x[lo:hi].double() @ w[k].double().T
        _near(y[lo:hi], want, 8 * 2.0 ** -23 * (x[lo:hi].double().abs() @ w[k].double().abs().T) + _u(t) * want.abs(), "y")
    dx, dw = linear.leaf_linear_grad(x, w, off, y)
    last = y[n - 300:].double()
    want = last @ w[1].double()
    _near(dx[n - 300:], want, wide * 2.0 ** -23 * (last.abs() @ w[1].double().abs()) + _u(t) * want.abs(), "dx")
    want = last.T @ x[n - 300:].double()
    _near(dw[1], want, 300 * 2.0 ** -23 * (last.abs().T @ x[n - 300:].double().abs()) + _u(t) * want.abs(), "dw")
    head = _rand((50, wide), t, 4, 0.01)
    target = _targets(n, 50, 0.0, 5)
    loss, lse = linear.softmax_xent(y, head, target)
    l = last @ head.double().T
    el = wide * 2.0 ** -23 * (last.abs() @ head.double().abs().T).max(1).values
    want = torch.logsumexp(l, 1)
    _near(lse[n - 300:], want, el + 2.0 ** -18 + want.abs() * 2.0 ** -23, "lse")
    dy, dhead = linear.softmax_xent_grad(y, head, target, lse, torch.ones(n, device="cuda"))
    linear.status()
    g = torch.exp(l - want[:, None])
    g[torch.arange(300, device="cuda"), target[n - 300:]] -= 1.0
    want = g @ head.double()
    # G's error: its rounding, and the logits' and lse's
    eg = g.abs() * (_u(t) + 2.0 ** -18) + (torch.expm1(2 * el) + 2.0 ** -17)[:, None]
    _near(dy[n - 300:], want, eg @ head.double().abs() + _u(t) * want.abs() + 50 * 2.0 ** -23 * (g.abs() @ head.double().abs()), "dy")
    del x, w, y, dx, dw, dy, last
    torch.cuda.empty_cache()


@gpu
def test_leaf_partial_and_empty():
    from bsscl_gbm_b200 import linear
    t = torch.bfloat16
    x, dy, w, off = _rand((90, 64), t, 1), _rand((90, 32), t, 2), _rand((3, 32, 64), t, 3), _offsets([30, 30, 30])
    both = linear.leaf_linear_grad(x, w, off, dy)
    one = linear.leaf_linear_grad(x, w, off, dy, want_dw=False)
    two = linear.leaf_linear_grad(x, w, off, dy, want_dx=False)
    assert one[1] is None and two[0] is None and torch.equal(one[0], both[0]) and torch.equal(two[1], both[1])
    off = torch.zeros(4, dtype=torch.int32, device="cuda")
    assert linear.leaf_linear(x[:0], w, off).shape == (0, 32)
    dx, dw = linear.leaf_linear_grad(x[:0], w, off, dy[:0])
    assert dx.shape == (0, 64) and dw.shape == w.shape and not dw.any()


# ---------------------------------------------------------------------------
# norm and clipping
# ---------------------------------------------------------------------------

def _check_clip(grads, outs, limit):
    from bsscl_gbm_b200 import linear
    src = [g.clone() for g in grads]
    norm = linear.GradClip(grads, out=outs).clip(limit)
    want = torch.stack([(g.double() ** 2).sum() for g in src]).sum().sqrt()
    _near(norm, want, want * (2.0 ** -24 + 1e-12), "norm")
    c = torch.clamp(limit / (want + 1e-6), max=1.0)
    for g, o in zip(src, outs if outs is not None else grads):
        r = g.double() * c
        # the factor's rounding, the product's, the result's
        u = _u(g.dtype)
        low = 2.0 ** -149 if g.dtype == torch.float32 else 2.0 ** -133 if g.dtype == torch.bfloat16 else 2.0 ** -25
        _near(o, r, r.abs() * (2 * 2.0 ** -24 + 1e-12 + u) * (1 + 2.0 ** -7) + low, f"gradient of {g.numel()}")
    return norm


@gpu
@pytest.mark.parametrize("limit", [0.0, 1e-3, 1.0, 1e9])
def test_clip_types_and_sizes(limit):
    f, b, h = torch.float32, torch.bfloat16, torch.float16
    shapes = [((1,), f), ((0,), f), ((3, 5), b), ((1001,), h), ((257, 129), f), ((65536,), b), ((65537,), f),
              ((300_001,), h), ((7, 3, 11), f), ((131072 + 8,), b)]
    grads = [_rand(s, t, i, 0.1) for i, (s, t) in enumerate(shapes)]
    _check_clip(grads, [torch.empty_like(g) for g in grads], limit)
    _check_clip(grads, None, limit)


@gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16, torch.float16])
def test_clip_views_that_are_not_aligned(kind):
    flat, to = _rand((70_000,), kind, 1), torch.full((70_000,), 7.0, dtype=kind, device="cuda")
    cuts = [0, 1, 2, 5, 13, 4000, 4001, 69_999]
    grads, outs = ([a[i + 1:j] for i, j in zip(cuts, cuts[1:])] for a in (flat, to))
    _check_clip(grads, outs, 0.5)
    assert all(float(to[i]) == 7.0 for i in cuts)
    # a transposed matrix is dense: it is scaled in its own order
    a = _rand((40, 60), kind, 3).T
    _check_clip([a], [torch.empty_strided(a.shape, a.stride(), dtype=kind, device="cuda")], 0.5)


@gpu
def test_clip_large_small_and_not_finite():
    from bsscl_gbm_b200 import linear
    big = torch.full((1000,), 1e30, device="cuda")      # squares beyond 32 bits
    _check_clip([big], [torch.empty_like(big)], 1.0)
    low = torch.full((1000,), 1e-30, device="cuda")     # squares below them
    _check_clip([low], [torch.empty_like(low)], 1e-40)
    zero = torch.zeros(33, device="cuda")
    assert float(_check_clip([zero], None, 1.0)) == 0.0
    inf, one = torch.tensor([float("inf"), 1.0], device="cuda"), torch.ones(5, device="cuda")
    norm = linear.GradClip([inf, one]).clip(1.0)
    assert torch.isinf(norm) and torch.isnan(inf[0]) and float(inf[1]) == 0.0 and not one.any()
    nan, one = torch.tensor([float("nan"), 1.0], device="cuda"), torch.ones(5, device="cuda")
    norm = linear.GradClip([nan, one]).clip(1.0)
    assert torch.isnan(norm) and torch.isnan(nan).all() and torch.isnan(one).all()


@gpu
def test_clip_same_at_every_call():
    from bsscl_gbm_b200 import linear
    grads = [_rand((n,), torch.float32, n) for n in (10_000_001, 333, 70_000)]
    clip = linear.GradClip(grads, out=[torch.empty_like(g) for g in grads])
    assert len({float(clip.clip(1.0)) for _ in range(5)}) == 1


@gpu
def test_clip_refusals():
    from bsscl_gbm_b200 import linear
    a = torch.ones(100, device="cuda")
    for grads, out, word in (([], None, "no gradients"), ([a, a], None, "overlaps"), ([a[:60], a[50:]], None, "overlaps"),
                             ([a[:50], a[50:]], [a[50:], a[:50]], "overlaps"), ([a[::2]], None, "not dense"),
                             ([a.expand(3, 100)], None, "not dense"), ([a], [a[:50]], "must have"),
                             ([a.double()], None, "float32"), ([a.cpu()], None, "CUDA"), ([a], [], "outputs")):
        with pytest.raises(ValueError, match=word):
            linear.GradClip(grads, out=out)
    with pytest.raises(ValueError, match="max_norm"):
        linear.GradClip([a]).clip(float("nan"))
    with pytest.raises(ValueError, match="max_norm"):
        linear.GradClip([a]).clip(-1.0)
    assert (a == 1).all()


# ---------------------------------------------------------------------------
# together, streams, graphs
# ---------------------------------------------------------------------------

def _step(s, clip=True):
    from bsscl_gbm_b200 import linear
    y = linear.leaf_linear(s["x"], s["w"], s["off"])
    loss, lse = linear.softmax_xent(y, s["head"], s["target"])
    dy, dhead = linear.softmax_xent_grad(y, s["head"], s["target"], lse, s["c"])
    dx, dw = linear.leaf_linear_grad(s["x"], s["w"], s["off"], dy)
    norm = linear.GradClip([dw, dhead]).clip(0.5) if clip else None
    return y, loss, dy, dhead, dx, dw, norm


def _problem(seed, n=500, din=60, hid=72, v=700, e=5, t=torch.bfloat16):
    counts = np.random.default_rng(seed).multinomial(n, np.ones(e) / e)
    return {"x": _rand((n, din), t, seed), "w": _rand((e, hid, din), t, seed + 1, din ** -0.5),
            "head": _rand((v, hid), t, seed + 2, 2 * hid ** -0.5), "off": _offsets(counts),
            "target": _targets(n, v, 0.1, seed + 3), "c": torch.full((n,), 1.0 / n, device="cuda")}


@gpu
def test_training_step_against_64_bits():
    """The step's gradients against 64-bit autograd of the whole step.  Norm-wise: the hidden rows are rounded once (u),
    which moves every later value by about u of its norm; G once more, and every output once: 4 u in all, and the
    logits' shift (u |y| |head|, under 4 u here) on the probabilities."""
    s = _problem(1)
    y, loss, dy, dhead, dx, dw, norm = _step(s)
    X, W, H = (s[k].double().requires_grad_() for k in ("x", "w", "head"))
    leaf = torch.searchsorted(s["off"].long(), torch.arange(500, device="cuda"), right=True) - 1
    Y = torch.einsum("ni,noi->no", X, W[leaf])
    full = torch.nn.functional.cross_entropy(Y @ H.T, s["target"], ignore_index=-1, reduction="none")
    (full * s["c"].double()).sum().backward()
    n64 = (W.grad.square().sum() + H.grad.square().sum()).sqrt()
    scale = min(1.0, 0.5 / (float(n64) + 1e-6))
    u = 2.0 ** -8
    for got, want, name in ((loss, full.detach(), "loss"), (dx, X.grad, "dx"), (dw, W.grad * scale, "dw"),
                            (dhead, H.grad * scale, "dhead"), (norm, n64, "norm")):
        assert float((got.double() - want).norm() / want.norm()) <= 8 * u, name


@gpu
def test_other_stream_and_overlap():
    """The same step on two side streams at once equals the one on the default stream, bit for bit."""
    a, b = _problem(2), _problem(7, n=900, v=3000)
    want = [_step(a), _step(b)]
    torch.cuda.synchronize()
    st = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(3):
        got = []
        for s, q in zip((a, b), st):
            with torch.cuda.stream(q):
                got.append(_step(s))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for p, q in zip(g, w):
            assert torch.equal(p, q)


@gpu
def test_captured_step_follows_its_inputs():
    """A captured step replayed on new inputs, and two graphs replayed at once on two streams."""
    s = _problem(3)
    _step(s, clip=False)
    torch.cuda.synchronize()
    graphs = []
    for seed in (3, 4):
        p = _problem(seed)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _step(p, clip=False)
        graphs.append((g, p, out))
    new = [_problem(11), _problem(12)]
    want = [_step(p, clip=False) for p in new]
    for (g, p, out), q in zip(graphs, new):
        for k in ("x", "w", "head", "off", "target", "c"):
            p[k].copy_(q[k])
    torch.cuda.synchronize()
    st = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for (g, p, out), q in zip(graphs, st):
            with torch.cuda.stream(q):
                g.replay()
    torch.cuda.synchronize()
    for (g, p, out), w in zip(graphs, want):
        for a, b in zip(out[:6], w[:6]):
            assert torch.equal(a, b)


@gpu
def test_captured_clip_follows_its_gradients():
    from bsscl_gbm_b200 import linear
    grads = [_rand((n,), torch.bfloat16, n) for n in (5000, 70_001, 3)]
    clip = linear.GradClip(grads, out=[torch.empty_like(g) for g in grads])
    clip.clip(1.0)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        norm = clip.clip(1.0)
    for k in range(2):
        for a in grads:
            a.mul_(3.0)
        g.replay()
        want = torch.stack([(a.double() ** 2).sum() for a in grads]).sum().sqrt()
        _near(norm, want, want * (2.0 ** -24 + 1e-12), "norm")


@gpu
def test_two_threads_at_once():
    """Calls from two host threads on streams of their own."""
    import threading
    problems, want, got = [_problem(21), _problem(22, n=700, v=2500)], [], [None, None]
    for p in problems:
        want.append(_step(p, clip=False))
    torch.cuda.synchronize()

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[k] = _step(problems[k], clip=False)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g[:6], w[:6]))


@gpu
def test_a_wait_that_runs_out_is_reported_once():
    from bsscl_gbm_b200 import lib, linear
    linear.status()
    err = C.create_string_buffer(256)
    assert lib().gbm_test_ops_wait(20, None, err, 256) == 6 and b"ran out" in err.value
    linear.status()                                    # told once, and the context is usable
    assert lib().gbm_test_ops_wait(0, None, err, 256) == ARG
    s = _problem(1)
    assert torch.isfinite(_step(s)[1]).all()


@gpu
def test_leaves_of_a_graph_and_long_features():
    """Parameters that require gradients, and more features than a product has stages many times over."""
    from bsscl_gbm_b200 import linear
    s = _problem(9)
    w = s["w"].clone().requires_grad_()
    y = linear.leaf_linear(s["x"], w, s["off"])
    assert not y.requires_grad and torch.equal(y, linear.leaf_linear(s["x"], s["w"], s["off"]))
    x, head = _rand((5, 70_001), torch.bfloat16, 1), _rand((9, 70_001), torch.bfloat16, 2, 0.005)
    _check_xent(x, head, _targets(5, 9, 0.0, 3), torch.ones(5, device="cuda"))


# ---------------------------------------------------------------------------
# refusals (no GPU: nothing is launched)
# ---------------------------------------------------------------------------

BF16, F16, F32 = 2, 3, 0
OK, ARG, UNSUPPORTED = 0, 1, 7
PTR = 1 << 20     # an aligned address nobody reads


@pytest.fixture(scope="module")
def L(built_lib):
    from bsscl_gbm_b200 import lib
    return lib()


def _rc(f, *a):
    err = C.create_string_buffer(256)
    rc = f(*a, None, err, 256)
    return rc, err.value.decode()


def test_xent_refusals(L):
    assert L.gbm_softmax_xent_workspace(10, 16, 20, 0, 1) == 0      # few classes: no parts to join
    need = L.gbm_softmax_xent_workspace(10, 16, 100000, 0, 1)
    good = [PTR, 16, PTR, 16, BF16, 10, 16, 100000, PTR, PTR, PTR, PTR, need]
    for at, value, rc, word in ((0, None, ARG, "null"), (1, 15, ARG, "stride"), (2, None, ARG, "null"), (3, 8, ARG, "stride"),
                                (4, F32, UNSUPPORTED, "type"), (4, 9, UNSUPPORTED, "type"), (5, -1, ARG, "sizes"), (6, 0, ARG, "sizes"),
                                (7, 0, ARG, "sizes"), (7, 1 << 31, ARG, "sizes"), (8, None, ARG, "null"), (9, None, ARG, "null"),
                                (10, PTR + 2, ARG, "aligned"), (0, PTR + 1, ARG, "aligned"), (11, PTR + 8, ARG, "aligned"), (11, None, ARG, "workspace"),
                                (12, need - 1, ARG, "workspace")):
        a = list(good)
        a[at] = value
        got, msg = _rc(L.gbm_softmax_xent, *a)
        assert got == rc and word in msg and "gbm_softmax_xent" in msg, (at, value, got, msg)
    assert _rc(L.gbm_softmax_xent, None, 16, PTR, 16, BF16, 0, 16, 20, None, None, None, PTR, 1 << 30)[0] == OK   # no rows
    need = L.gbm_softmax_xent_workspace(10, 16, 20, 1, 1)
    good = [PTR, 16, PTR, 16, F16, 10, 16, 20, PTR, PTR, PTR, PTR, 16, PTR, 16, PTR, need]
    for at, value, rc, word in ((9, None, ARG, "null"), (10, None, ARG, "null"), (12, 15, ARG, "stride"), (14, 15, ARG, "stride"),
                                (11, PTR + 1, ARG, "unaligned"), (16, need - 1, ARG, "workspace"), (4, 1, UNSUPPORTED, "type")):
        a = list(good)
        a[at] = value
        got, msg = _rc(L.gbm_softmax_xent_grad, *a)
        assert got == rc and word in msg, (at, value, got, msg)
    a = list(good)
    a[11] = a[13] = None
    assert _rc(L.gbm_softmax_xent_grad, *a)[0] == ARG
    assert L.gbm_softmax_xent_workspace((1 << 31) - 600, 1, (1 << 31) - 600, 1, 1) == -1      # counts of bytes stay within 64 bits
    assert L.gbm_leaf_linear_workspace(10, 65535, 1, 1 << 20, 1, 1) == -1
    assert L.gbm_softmax_xent_workspace(-1, 1, 1, 0, 0) == -1 and L.gbm_softmax_xent_workspace(1, 1, 1 << 31, 1, 1) == -1


def test_leaf_refusals(L):
    need = max(L.gbm_leaf_linear_workspace(10, 3, 16, 24, g, 0) for g in (0, 1))
    good = [PTR, 16, PTR, PTR, BF16, 10, 3, 16, 24, PTR, 24, 1, PTR, need]
    for at, value, rc in ((0, None, ARG), (1, 15, ARG), (2, None, ARG), (3, None, ARG), (4, F32, UNSUPPORTED), (5, -1, ARG), (6, 0, ARG),
                          (6, 65536, ARG), (7, 0, ARG), (8, 0, ARG), (9, None, ARG), (10, 23, ARG), (9, PTR + 1, ARG), (3, PTR + 2, ARG)):
        a = list(good)
        a[at] = value
        got, msg = _rc(L.gbm_leaf_linear, *a)
        assert got == rc and "gbm_leaf_linear" in msg, (at, value, got, msg)
    assert _rc(L.gbm_leaf_linear, None, 16, PTR, PTR, BF16, 0, 3, 16, 24, None, 24, 1, PTR, need)[0] == OK
    good = [PTR, 16, PTR, PTR, PTR, 24, F16, 10, 3, 16, 24, PTR, 16, 1, PTR, PTR, need]
    for at, value, rc in ((0, None, ARG), (2, None, ARG), (4, None, ARG), (5, 23, ARG), (1, 15, ARG), (12, 15, ARG), (6, 1, UNSUPPORTED),
                          (14, PTR + 1, ARG)):
        a = list(good)
        a[at] = value
        got, msg = _rc(L.gbm_leaf_linear_grad, *a)
        assert got == rc, (at, value, got, msg)
    a = list(good)
    a[11] = a[14] = None
    assert _rc(L.gbm_leaf_linear_grad, *a)[0] == ARG


def _plan(L, src, dst, sizes, types):
    n = len(src)
    size = (C.c_int64 * n)(*sizes)
    need = L.gbm_grad_clip_plan_bytes(size, n)
    buf = C.create_string_buffer(max(need, 1))
    err = C.create_string_buffer(256)
    rc = L.gbm_grad_clip_plan((C.c_void_p * n)(*src), (C.c_void_p * n)(*dst), size, (C.c_int32 * n)(*types), n, buf, need, err, 256)
    return rc, err.value.decode(), buf


def test_clip_plan_refusals(L):
    K = 1 << 20
    assert _plan(L, [PTR, PTR + K], [PTR, PTR + K], [100, 200], [F32, BF16])[0] == OK
    assert _plan(L, [PTR, PTR + 400], [PTR, PTR + 400], [100, 200], [F32, BF16])[0] == OK        # neighbours
    assert _plan(L, [PTR, PTR], [PTR + K, PTR + 2 * K], [100, 100], [F32, F32])[0] == OK          # read twice, written apart
    for src, dst, sizes, types, rc, word in (
            ([PTR, PTR + 399], [PTR, PTR + 399], [100, 200], [F32, F16], ARG, "unaligned"),
            ([PTR, PTR + 398], [PTR, PTR + 398], [100, 200], [F32, F16], ARG, "overlaps"),
            ([PTR], [PTR + 4], [100], [F32], ARG, "overlaps"),
            ([PTR, PTR + K], [PTR + K, PTR], [100, 100], [F32, F32], ARG, "overlaps"),
            ([PTR, PTR], [PTR + K, PTR + K], [100, 100], [F32, F32], ARG, "overlaps"),
            ([PTR, PTR + 64], [PTR, PTR + 2 * K], [1000, 8], [F32, F32], ARG, "overlaps"),
            ([None], [PTR], [1], [F32], ARG, "null"), ([PTR + 2], [PTR + 2], [1], [F32], ARG, "unaligned"),
            ([PTR], [PTR], [1], [1], UNSUPPORTED, "type"), ([PTR], [PTR], [-1], [F32], ARG, "size")):
        got, msg, _ = _plan(L, src, dst, sizes, types)
        assert got == rc and word in msg, (got, msg, word)
    rc, _, plan = _plan(L, [PTR, None], [PTR, None], [70000, 0], [F32, F16])
    assert rc == OK
    need = L.gbm_grad_clip_workspace(plan)
    for a, word in (((plan, None, 1.0, PTR, PTR, need), "null"), ((plan, PTR, 1.0, None, PTR, need), "null"),
                    ((plan, PTR, 1.0, PTR, PTR, need - 1), "workspace"), ((plan, PTR, 1.0, PTR, PTR + 8, need), "unaligned"),
                    ((plan, PTR, -1.0, PTR, PTR, need), "max_norm"), ((plan, PTR, float("nan"), PTR, PTR, need), "max_norm"),
                    ((C.create_string_buffer(64), PTR, 1.0, PTR, PTR, need), "not a plan")):
        rc, msg = _rc(L.gbm_grad_clip, *a)
        assert rc == ARG and word in msg, (rc, msg)
    assert L.gbm_grad_clip_workspace(C.create_string_buffer(64)) == -1


def test_python_refusals_need_no_gpu(built_lib):
    from bsscl_gbm_b200 import linear
    x = torch.zeros(4, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        linear.softmax_xent(x, x, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        linear.leaf_linear(x, x[None], torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        linear.GradClip([x])


@gpu
def test_gradients_into_the_callers_buffers():
    from bsscl_gbm_b200 import linear
    s = _problem(5)
    y = linear.leaf_linear(s["x"], s["w"], s["off"])
    _, lse = linear.softmax_xent(y, s["head"], s["target"])
    want = linear.softmax_xent_grad(y, s["head"], s["target"], lse, s["c"])
    hold = torch.full((700, 80), 3.0, dtype=torch.bfloat16, device="cuda")
    got = linear.softmax_xent_grad(y, s["head"], s["target"], lse, s["c"], dw_out=hold[:, 4:76])
    assert torch.equal(got[0], want[0]) and torch.equal(hold[:, 4:76], want[1]) and (hold[:, :4] == 3).all() and (hold[:, 76:] == 3).all()
    want = linear.leaf_linear_grad(s["x"], s["w"], s["off"], want[0])
    dw = torch.empty_like(s["w"])
    got = linear.leaf_linear_grad(s["x"], s["w"], s["off"], got[0], want_dx=False, dw_out=dw)
    assert got[0] is None and got[1] is dw and torch.equal(dw, want[1])
    with pytest.raises(ValueError, match="dw_out"):
        linear.leaf_linear_grad(s["x"], s["w"], s["off"], y, dw_out=dw[:2])
    with pytest.raises(ValueError, match="dw_out"):
        linear.softmax_xent_grad(y, s["head"], s["target"], lse, s["c"], dw_out=hold)


@gpu
def test_python_refusals():
    from bsscl_gbm_b200 import linear
    t = torch.bfloat16
    x, w, y = _rand((6, 16), t, 1), _rand((9, 16), t, 2), torch.zeros(6, dtype=torch.int64, device="cuda")
    f = torch.zeros(6, device="cuda")
    for a in ((x.float(), w, y), (x, w.half(), y), (x.T, w, y), (x, w[:, :8], y), (x, w, y.int()), (x, w, y[:5]), (x, w, y.cpu()),
              (x[0], w, y), (x[:1].expand(6, 16), w, y), (x[:, :0], w[:, :0], y), (x, w[:0], y)):
        with pytest.raises(ValueError):
            linear.softmax_xent(*a)
    for a in ((x, w, y, f.double(), f), (x, w, y, f, f[:3]), (x, w, y, f.cpu(), f)):
        with pytest.raises(ValueError):
            linear.softmax_xent_grad(*a)
    with pytest.raises(ValueError):
        linear.softmax_xent_grad(x, w, y, f, f, want_dx=False, want_dw=False)
    lw, off, dy = _rand((2, 5, 16), t, 3), _offsets([2, 4]), _rand((6, 5), t, 4)
    for a in ((x, lw[:, :, :8], off), (x, lw, off.long()), (x, lw, off[:2]), (x, lw[0], off), (x, lw.half(), off), (x, lw.transpose(1, 2), off),
              (x[:, :8], lw, off), (x, lw, off.cpu())):
        with pytest.raises(ValueError):
            linear.leaf_linear(*a)
    with pytest.raises(ValueError):
        linear.leaf_linear(x, lw, off, out=torch.empty(6, 4, dtype=t, device="cuda"))
    with pytest.raises(ValueError):
        linear.leaf_linear(x, lw, off, out=torch.empty(5, 5, dtype=t, device="cuda"))
    for a in ((x, lw, off, dy[:5]), (x, lw, off, dy[:, :4]), (x, lw, off, dy.half())):
        with pytest.raises(ValueError):
            linear.leaf_linear_grad(*a)


@gpu
def test_outputs_that_overlap_inputs():
    """The caller's output may lie beside an operand, never on it."""
    from bsscl_gbm_b200 import linear
    t = torch.bfloat16
    hold = _rand((40, 48), t, 1)
    lw, off = _rand((2, 16, 16), t, 2), _offsets([19, 20])
    x = hold[:, :16]
    want = linear.leaf_linear(x, lw, off)
    for out in (x, hold[:, 8:24], hold[:, 15:31], hold.view(-1)[:640].view(40, 16)):
        with pytest.raises(ValueError, match="overlaps"):
            linear.leaf_linear(x, lw, off, out=out)
    with pytest.raises(ValueError, match="overlaps"):
        linear.leaf_linear(hold[:, 32:], lw, off, out=hold[:, 24:40])
    with pytest.raises(ValueError, match="overlaps"):
        linear.leaf_linear(x[:16], lw, _offsets([9, 7]), out=lw[1])
    before = hold[:, 32:].clone()
    got = linear.leaf_linear(x, lw, off, out=hold[:, 16:32])
    assert torch.equal(got[:39], want[:39]) and torch.equal(hold[:, 32:], before)
    got = linear.leaf_linear(hold[:, 32:], lw, off, out=hold[:, 16:32])      # to the left of what it reads
    assert torch.equal(got[:39], linear.leaf_linear(before, lw, off)[:39])
    dy = _rand((40, 16), t, 3)
    for dw in (lw, dy[:32].view(2, 16, 16)):
        with pytest.raises(ValueError, match="overlaps"):
            linear.leaf_linear_grad(x, lw, off, dy, dw_out=dw)
    head, target = _rand((9, 16), t, 4), torch.arange(40, device="cuda") % 9
    c = torch.ones(40, device="cuda")
    _, lse = linear.softmax_xent(dy, head, target)
    for dw in (head, dy[3:12], dy[31:]):
        with pytest.raises(ValueError, match="overlaps"):
            linear.softmax_xent_grad(dy, head, target, lse, c, dw_out=dw)
