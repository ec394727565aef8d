"""The leaves' gradients where their tiles are dealt out longest leaf first: more tiles than clusters, at least 64 stages of
64 rows a cluster (rows / 64 x tiles of one leaf's dw >= 4736), and 2 to 2048 leaves; every value of y, dx and dw."""
import numpy as np
import pytest

pytest.importorskip("torch")
import torch

from test_linear_ops import _check_leaf, _offsets, _rand

gpu = pytest.mark.gpu


def _counts(kind, leaves, rows, seed=0):
    r = np.random.default_rng(seed)
    if kind == "equal":
        counts = np.full(leaves, rows // leaves)
    elif kind == "uneven":                      # ties and empty leaves among them
        share = np.exp(r.normal(0.0, 1.5, leaves))
        counts = (rows * share / share.sum()).astype(int) // 50 * 50
        counts[::7] = 0
    else:                                       # one leaf holds nearly all, the others one row or none
        counts = np.arange(leaves) % 2
        counts[leaves // 2] = 0
    counts[leaves // 2] += max(0, rows - counts.sum())
    return counts


@gpu
@pytest.mark.parametrize("kind", ["equal", "uneven", "one"])
@pytest.mark.parametrize("leaves,rows,din,dout", [(63, 20_011, 1024, 1024), (6, 19_500, 1000, 1024), (1500, 303_200, 256, 256),
                                                  (2048, 303_200, 256, 200), (2049, 303_200, 256, 256), (1025, 155_000, 264, 256)])
def test_longest_leaf_first(leaves, rows, din, dout, kind):
    tiles = -(-din // 256) * -(-dout // 256)
    counts = _counts(kind, leaves, rows)
    n, t = int(counts.sum()) + 17, torch.bfloat16
    assert leaves * tiles > 74 and n // 64 * tiles >= 4736
    x, dy, w = _rand((n, din), t, 1), _rand((n, dout), t, 2), _rand((leaves, dout, din), t, 3, din ** -0.5)
    _check_leaf(x, w, _offsets(counts, 9), dy)
    torch.cuda.empty_cache()
