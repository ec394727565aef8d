"""The tensor-core frame under the operators for leaf-wise linear models: what
its roles wait for.  Its protocol is read from the source and run on the CPU;
on the GPU the launches that follow one another run many times over."""
import os
import re

import pytest

pytest.importorskip("torch")
import torch

from conftest import ROOT

gpu = pytest.mark.gpu


def _frame():
    with open(os.path.join(ROOT, "bsscl-gbm_b200", "csrc", "linear_tc.cuh")) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    return text[text.index("k_tc(const"):text.index("k_wait(")]


def test_tensor_memory_is_taken_and_freed_while_both_ctas_are_there():
    """The cluster meets, the launch in front is over, tensor memory is allocated, the cluster meets; at the end it meets,
    frees, and meets again before either CTA leaves."""
    order = re.findall(r"cluster_sync\(\)|depend\(\)|tcgen05\.alloc|tcgen05\.dealloc|op\.epilogue", _frame())
    assert order == ["cluster_sync()", "depend()", "tcgen05.alloc", "cluster_sync()", "op.epilogue",
                     "cluster_sync()", "tcgen05.dealloc", "cluster_sync()"]


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
