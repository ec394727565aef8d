"""The tensor-core frame under the operators for leaf-wise linear models: what
its roles wait for.  Its protocol is read from the source and run on the CPU;
on the GPU the launches that follow one another run many times over."""
import ctypes as C
import os
import random
import re
import subprocess
import time

import numpy as np
import pytest

pytest.importorskip("torch")
import torch

from conftest import ROOT

gpu = pytest.mark.gpu


def _source():
    with open(os.path.join(ROOT, "bsscl-gbm_b200", "csrc", "linear_tc.cuh")) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def _frame():
    text = _source()
    return text[text.index("k_tc(const"):text.index("k_wait(")]


def test_tensor_memory_is_taken_and_freed_while_both_ctas_are_there():
    """The cluster meets, the launch in front is over, tensor memory is allocated, the cluster meets (the fetching warp, which
    does not touch it, at the end of its role); at the end it meets, frees, and meets again before either CTA leaves.  A
    launch that does nothing meets once more and leaves before it allocates."""
    order = re.findall(r"cluster_(?:sync|arrive|wait)\(\)|depend\(\)|return;|tcgen05\.alloc|tcgen05\.dealloc|op\.epilogue|if \(warp\) ", _frame())
    assert order == ["cluster_sync()", "depend()", "cluster_sync()", "return;", "tcgen05.alloc", "cluster_arrive()", "if (warp) ", "cluster_wait()",
                     "cluster_wait()", "op.epilogue", "cluster_sync()", "tcgen05.dealloc", "cluster_sync()"]


class _Bar:
    """An mbarrier: phases that end with `count` arrivals and all expected bytes."""

    def __init__(self, count):
        self.count, self.left, self.bytes, self.phase = count, count, 0, 0

    def move(self, arrive=0, bytes_=0):
        self.left -= arrive
        self.bytes += bytes_
        if self.left == 0 and self.bytes == 0:
            self.left, self.phase = self.count, self.phase + 1

    def passed(self, parity):
        return self.phase % 2 != parity


def _run_ring(count, second_arrives, boxes, laps, rng):
    """Both CTAs' fetching threads and the products over `laps` rounds of six stages, in a random order of their steps (the
    second CTA a slow one); boxes = what the second CTA brings of a stage.  None, or what went wrong."""
    n = 6
    full, empty = [_Bar(count) for _ in range(n)], [[_Bar(1) for _ in range(n)] for _ in range(2)]
    at, total = {"first": 0, "second": 0, "products": 0}, n * laps
    late = []                                     # bytes and arrivals on their way
    pace = {"first": 1.0, "second": rng.choice([0.02, 0.2, 1.0]), "products": 1.0}
    while at["second"] < total or at["products"] < total:
        moved = False
        for who in ("first", "second", "products"):
            k = at[who]
            if k == total or rng.random() > pace[who]:
                moved |= k < total and pace[who] < 1.0
                continue
            s, lap = k % n, k // n
            if who == "products":
                if full[s].passed(lap % 2):
                    late += [(empty[0][s], 1, 0), (empty[1][s], 1, 0)]
                    at[who], moved = k + 1, True
                continue
            cta = who == "second"
            if not empty[cta][s].passed(lap % 2 ^ 1):
                continue
            if empty[cta][s].phase != lap:
                return f"the {who} CTA's wait stands for lap {empty[cta][s].phase}, not {lap}"
            if cta:
                full[s].move(arrive=int(second_arrives))
                late += [(full[s], 0, -1)] * boxes
            else:
                full[s].move(arrive=1, bytes_=1 + boxes)
                late += [(full[s], 0, -1)]
            at[who], moved = k + 1, True
        if late and rng.random() < 0.8:
            bar, arrive, bytes_ = late.pop(0)
            bar.move(arrive, bytes_)
            moved = True
        if not moved and not late:
            return f"stuck at {at}"
    return None


def test_a_cta_that_fetches_nothing_is_held_in_step():
    """The barriers of the ring as the source has them, in random orders: no wait ever stands for another lap's phase."""
    text = _source()
    count = int(re.search(r"mbar_init\(full \+ 8 \* lane, (\d)\)", text).group(1))
    fetch = re.sub(r"\s+", " ", text[text.index("bool fetch("):text.index("void multiply_stage")])
    arrives = "if (rank == 0) mbar_expect(bar, bytes); else mbar_arrive_at<false>(bar, 0);" in fetch
    rng = random.Random(1)
    for _ in range(300):
        for boxes in (0, 1, 2):
            assert _run_ring(count, arrives, boxes, 8, rng) is None
    # the model tells: without the second CTA's arrival it is lapped where it fetches nothing
    assert any(_run_ring(1, False, 0, 8, rng) for _ in range(300))
    assert not any(_run_ring(1, False, 1, 8, rng) for _ in range(300))


def test_build_needs_no_torch_with_cuda(tmp_path):
    """The engine's library is built beside a torch that has no CUDA, without the torch binding."""
    csrc = os.path.join(ROOT, "bsscl-gbm_b200", "csrc")

    def plan():
        return subprocess.run(["make", "-n", "-B", "-C", csrc, f"TORCH={tmp_path}"], check=True, capture_output=True, text=True).stdout

    (tmp_path / "lib").mkdir()
    assert "libgbm_b200.so" in plan() and "torch_ops.cpp" not in plan()
    (tmp_path / "lib" / "libc10_cuda.so").touch()
    assert "torch_ops.cpp" in plan()


def _rand(shape, t, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(t)


@gpu
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16])
def test_training_steps_that_follow_one_another(kind):
    """Launches of the frame on all SMs, one directly behind the other, hundreds of times: the same bits each time."""
    from bsscl_gbm_b200 import linear
    n, d, v = 4096, 512, 16384
    x, w = _rand((n, d), kind, 1), _rand((v, d), kind, 2, 2.0 / d ** 0.5)
    g = torch.Generator(device="cuda").manual_seed(3)
    y, c = torch.randint(-1, v, (n,), generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda") + 0.5

    def step():
        loss, lse = linear.softmax_xent(x, w, y)
        return (loss, lse) + linear.softmax_xent_grad(x, w, y, lse, c)

    want, bad = step(), torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(400):
        for a, b in zip(step(), want):
            bad += (a != b).sum()
    linear.status()
    assert int(bad) == 0


@gpu
def test_leaf_products_that_follow_one_another():
    from bsscl_gbm_b200 import linear
    t, n, e = torch.bfloat16, 40_000, 7
    off = torch.tensor([0, 9000, 9000, 9100, 20_001, 30_000, 39_999, n], dtype=torch.int32, device="cuda")
    x, dy, w = _rand((n, 256), t, 1), _rand((n, 512), t, 2), _rand((e, 512, 256), t, 3, 0.06)
    want = (linear.leaf_linear(x, w, off),) + linear.leaf_linear_grad(x, w, off, dy)
    for _ in range(500):
        got = linear.leaf_linear(x, w, off), linear.leaf_linear(x, w, off)
    grad = [linear.leaf_linear_grad(x, w, off, dy) for _ in range(100)][-1]
    linear.status()
    for a, b in zip(got + grad, (want[0],) + want):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("classes,hidden", [(128, 32), (100, 32), (65, 24), (128, 8), (20, 30), (1, 1)])
def test_tiles_of_which_the_second_cta_has_nothing(classes, hidden):
    """At most 128 rows and 32 columns of a result, over 64 and more stages: every product of the frame."""
    from bsscl_gbm_b200 import linear
    t, n = torch.bfloat16, 6000                       # dw's k axis: 94 stages of rows
    x, w = _rand((n, hidden), t, 1), _rand((classes, hidden), t, 2, 0.2)
    y, c = torch.arange(n, device="cuda") % classes, torch.ones(n, device="cuda")
    l = x.double() @ w.double().T
    lse64 = torch.logsumexp(l, 1)
    for _ in range(20):
        loss, lse = linear.softmax_xent(x, w, y)
        dx, dw = linear.softmax_xent_grad(x, w, y, lse, c)
    # logits and few rows: the k axis is the features'
    wide, rows = _rand((classes, 5000), t, 3, 0.02), _rand((hidden, 5000), t, 4)
    for _ in range(20):
        few = linear.softmax_xent(rows, wide, y[:hidden] * 0)[1]
        fx, fw = linear.softmax_xent_grad(rows, wide, y[:hidden] * 0, few, c[:hidden])
    off = torch.tensor([0, n - 100, n], dtype=torch.int32, device="cuda")
    dy, lw = _rand((n, classes), t, 5), _rand((2, classes, hidden), t, 6, 0.2)
    for _ in range(20):
        ly = linear.leaf_linear(x, lw, off)
        lx, ldw = linear.leaf_linear_grad(x, lw, off, dy)
    linear.status()
    u = 2.0 ** -8
    g = torch.exp(l - lse64[:, None])
    g[torch.arange(n, device="cuda"), y] -= 1.0
    # norm-wise: G's rounding and the result's, and 32-bit sums.  G itself is off by the logits' and lse's errors,
    # 2 hidden 2^-23 sum |x w| + 2^-20 < 2^-15 here, which is all there is of it with one class.
    for got, want, size in ((dx, g @ w.double(), w.double().abs().sum(0).expand(n, -1)),
                            (dw, g.T @ x.double(), x.double().abs().sum(0).expand(classes, -1))):
        assert float((got.double() - want).norm()) <= 2 * u * float(want.norm()) + 2.0 ** -15 * float(size.norm())
    for got, want in ((lse, lse64), (few, torch.logsumexp(rows.double() @ wide.double().T, 1)),
                      (ly[:n - 100], x[:n - 100].double() @ lw[0].double().T), (lx[n - 100:], dy[n - 100:].double() @ lw[1].double()),
                      (ldw[0], dy[:n - 100].double().T @ x[:n - 100].double()), (ldw[1], dy[n - 100:].double().T @ x[n - 100:].double())):
        assert float((got.double() - want).norm()) <= 2 * u * float(want.norm()) + 1e-5
    if classes > 1:
        p = torch.softmax(rows.double() @ wide.double().T, 1)
        p[:, 0] -= 1.0
        for got, want in ((fx, p @ wide.double()), (fw, p.T @ rows.double())):
            assert float((got.double() - want).norm()) <= 2 * u * float(want.norm()) + 1e-5


@gpu
def test_launches_behind_a_wait_that_ran_out_do_nothing():
    """Hundreds of calls after one that ran out: none waits for itself, none writes, and the first to ask is told once."""
    from bsscl_gbm_b200 import lib, linear
    t = torch.bfloat16
    x, w = _rand((300, 64), t, 1), _rand((2, 128, 64), t, 2, 0.1)
    off = torch.tensor([0, 100, 300], dtype=torch.int32, device="cuda")
    want = linear.leaf_linear(x, w, off)
    linear.status()
    err = C.create_string_buffer(256)
    stream = torch.cuda.current_stream().cuda_stream
    assert lib().gbm_test_ops_expire(20, stream, err, 256) == 0
    torch.cuda.synchronize()
    out = torch.full_like(want, 5.0)
    began = time.monotonic()
    for _ in range(300):
        linear.leaf_linear(x, w, off, out=out)
    torch.cuda.synchronize()
    assert time.monotonic() - began < 1.0 and (out == 5).all()
    with pytest.raises(RuntimeError, match="ran out"):
        linear.status()
    linear.status()
    assert torch.equal(linear.leaf_linear(x, w, off, out=out), want)
    assert lib().gbm_test_ops_expire(0, stream, err, 256) == 1 and b"expire" in err.value


@gpu
def test_a_tile_that_takes_longer_than_the_shortest_limit():
    """One row of 2^31 - 600 features: 33 million stages in one tile.  Ones in a few places, the last one among them: exact."""
    from bsscl_gbm_b200 import linear
    d = 2 ** 31 - 600
    x, w = torch.zeros(1, d, dtype=torch.bfloat16, device="cuda"), torch.ones(1, d, dtype=torch.bfloat16, device="cuda")
    x[0, [0, 77, 1 << 30, d - 1]] = 1.0
    loss, lse = linear.softmax_xent(x, w, torch.zeros(1, dtype=torch.int64, device="cuda"))
    linear.status()
    assert float(lse) == 4.0 and float(loss) == 0.0
    del x, w
    torch.cuda.empty_cache()


@gpu
def test_another_calls_error_is_not_the_operators():
    """An engine call that found too little memory has told so; the operators behind it succeed."""
    from bsscl_gbm_b200 import Engine, lib, linear
    x, w = _rand((40, 64), torch.bfloat16, 1), _rand((30, 64), torch.bfloat16, 2)
    y = torch.zeros(40, dtype=torch.int64, device="cuda")
    want = linear.softmax_xent(x, w, y)
    eng = Engine(0)
    try:
        one = C.create_string_buffer(64)
        assert lib().gbm_predict_upload(eng._h, one, 1 << 40, 1000) == 2         # 2^50 bytes: nothing is read
        assert "cudaMalloc" in eng.last_error()
        got = linear.softmax_xent(x, w, y)
        dx, dw = linear.softmax_xent_grad(x, w, y, got[1], torch.ones(40, device="cuda"))
        assert lib().gbm_predict_upload(eng._h, one, 1 << 40, 1000) == 2
        linear.leaf_linear(x, w[None], torch.tensor([0, 40], dtype=torch.int32, device="cuda"))
    finally:
        eng.close()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,d,v", [(8, 64, 9000), (13, 72, 20_000), (70, 64, 300), (300, 100, 5000), (2000, 64, 16_000)])
def test_infinite_logits(n, d, v, kind):
    """log sum exp of a row with a logit of +inf is +inf, of -inf beside finite ones finite; its loss follows, and its neighbours
    are as they are without it."""
    from bsscl_gbm_b200 import linear
    x, w = _rand((n, d), kind, 1), _rand((v, d), kind, 2, 0.1)
    w[:, 0] = 0.0
    y = torch.arange(n, device="cuda") % v
    want, lse = linear.softmax_xent(x, w, y)
    x[3], x[5] = 0.0, 0.0
    x[3, 0], x[5, 0] = float("inf"), 1.0
    w[:, 0], w[v // 2, 0] = -1.0, 1.0            # one class of +inf in row 3
    x[:3, 0], x[4, 0], x[6:, 0] = 0.0, 0.0, 0.0
    y[3] = 7
    loss, got = linear.softmax_xent(x, w, y)
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[[3, 5]] = False
    assert torch.equal(loss[keep], want[keep]) and torch.equal(got[keep], lse[keep])
    assert float(got[3]) == float("inf") and float(loss[3]) == float("inf")
    e = (v - 1) * 2.718281828459045 ** -1 + 2.718281828459045
    assert abs(float(got[5]) - float(torch.log(torch.tensor(e, dtype=torch.float64)))) < 1e-5
    y[3] = v // 2                                # inf - inf
    loss, got = linear.softmax_xent(x, w, y)
    assert torch.isnan(loss[3]) and float(got[3]) == float("inf")
    w[:, 0] = -1.0                               # every logit -inf
    assert float(linear.softmax_xent(x, w, y)[1][3]) == float("-inf")
    w[::2, 0] = 1.0                              # half of them +inf
    assert float(linear.softmax_xent(x, w, y)[1][3]) == float("inf")
    w[1] = float("nan")                          # and a NaN among them
    assert torch.isnan(linear.softmax_xent(x, w, y)[1]).all()
    linear.status()


@gpu
@pytest.mark.parametrize("n", [400, 2000])
@pytest.mark.parametrize("top", [2.0 ** 14, 1.9 * 2.0 ** 14])
def test_half_gradients_of_rows_of_very_different_weights(n, top):
    """Two classes and upstream gradients over ten decades (the largest one's row is near its target, so that its dx fits): what half precision's subnormals round away of G is at most
    2^-39 of the largest upstream gradient (a power of two takes that to 2^14 at least, half a subnormal step is 2^-25),
    beside one rounding of G and one of dx, and |c| p 2^-19 for p's own error (16 products, exp and log in 32 bits)."""
    from bsscl_gbm_b200 import linear
    x, w = _rand((n, 16), torch.float16, 1, 2.0 ** -12), _rand((2, 16), torch.float16, 2, 400.0)
    y = torch.arange(n, device="cuda") % 2
    apart = w[0].double() - w[1].double()
    x[0] = (20.0 * apart / apart.square().sum()).half()
    c = torch.exp2(-14.0 - (torch.arange(n, device="cuda") % 11)).float() * 1.37
    c[0] = top
    loss, lse = linear.softmax_xent(x, w, y)
    dx, _ = linear.softmax_xent_grad(x, w, y, lse, c, want_dw=False)
    linear.status()
    p = torch.softmax(x.double() @ w.double().T, 1)
    g = c.double()[:, None] * (p - torch.nn.functional.one_hot(y, 2))
    want, u = g @ w.double(), 2.0 ** -11
    tol = (u * g.abs() + c.double()[:, None] * 2.0 ** -19 + top * 2.0 ** -39) @ w.double().abs() + u * want.abs() + 2.0 ** -25
    assert ((dx.double() - want).abs() <= tol).all(), float(((dx.double() - want).abs() / tol).max())


@gpu
def test_a_clip_that_is_let_go_while_another_stream_runs_it():
    """The plan, made on one stream, is not handed to that stream's next tensors before the other stream has read it."""
    from bsscl_gbm_b200 import linear
    for size in (5, 70_000):
        grads = [_rand((size + k,), torch.float32, k) for k in range(40)]
        outs = [torch.zeros_like(g) for g in grads]
        want = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()
        clip, side = linear.GradClip(grads, out=outs), torch.cuda.Stream()
        room = clip._plan_dev.numel()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(50_000_000)          # some 30 ms
            norm = clip.clip(1.0)
        del clip
        over = [torch.full((room,), 255, dtype=torch.uint8, device="cuda") for _ in range(8)]
        torch.cuda.synchronize()
        assert abs(float(norm) - float(want)) <= 1e-6 * float(want)
        c = float(torch.clamp(1.0 / (want + 1e-6), max=1.0))
        for g, o in zip(grads, outs):
            assert torch.allclose(o.double(), g.double() * c, rtol=1e-6, atol=0)
        del over


@gpu
def test_a_wish_that_is_neither_true_nor_false():
    from bsscl_gbm_b200 import linear
    x, w, off = _rand((6, 16), torch.bfloat16, 1), _rand((1, 9, 16), torch.bfloat16, 2), torch.tensor([0, 6], dtype=torch.int32, device="cuda")
    y, f = torch.zeros(6, dtype=torch.int64, device="cuda"), torch.zeros(6, device="cuda")
    many = np.zeros(2)
    for call in (lambda: linear.softmax_xent_grad(x, w[0], y, f, f, want_dx=many), lambda: linear.softmax_xent_grad(x, w[0], y, f, f, want_dw=many),
                 lambda: linear.leaf_linear_grad(x, w, off, x[:, :9], want_dx=many), lambda: linear.leaf_linear_grad(x, w, off, x[:, :9], want_dw=many)):
        with pytest.raises(ValueError, match="ambiguous"):
            call()


@gpu
def test_calls_behind_copies_fills_and_other_streams():
    """In order behind what another stream, a copy or a fill made: eagerly and captured with a fork and a join."""
    from bsscl_gbm_b200 import linear
    t, n, d, v = torch.bfloat16, 3000, 64, 5000
    src = [_rand((n, d), t, k) for k in range(4)]
    w, y, c = _rand((v, d), t, 9, 0.2), torch.arange(n, device="cuda") % v, torch.ones(n, device="cuda")
    off, lw = torch.tensor([0, 1000, n], dtype=torch.int32, device="cuda"), _rand((2, 48, d), t, 10, 0.1)
    x, side = torch.empty_like(src[0]), torch.cuda.Stream()

    def work():
        loss, lse = linear.softmax_xent(x, w, y)
        return (loss, lse) + linear.softmax_xent_grad(x, w, y, lse, c) + (linear.leaf_linear(x, lw, off),)

    def forked(a):
        """x filled on this stream, then copied over on the side stream, worked on there and here after the join."""
        main = torch.cuda.current_stream()
        x.zero_()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            x.copy_(a)
            there = work()
            for o in there:
                o.record_stream(main)
        main.wait_stream(side)
        here = work()
        x.fill_(1.0)
        return there, here, work()

    want = []
    for a in src:
        x.copy_(a)
        torch.cuda.synchronize()
        want.append(work())
        torch.cuda.synchronize()
    x.fill_(1.0)
    torch.cuda.synchronize()
    ones = work()
    torch.cuda.synchronize()

    def check(got, k):
        torch.cuda.synchronize()
        for g, e in zip(got, (want[k], want[k], ones)):
            for p, q in zip(g, e):
                assert torch.equal(p, q)

    for k, a in enumerate(src):
        check(forked(a), k)
    a, graph = src[0].clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = forked(a)
    for k in (2, 3, 1):
        a.copy_(src[k])
        graph.replay()
        check(got, k)
    linear.status()
