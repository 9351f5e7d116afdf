"""GPU: partial sums of decode steps whose keys are split, beside prompts and in batches by shares, against the plain form
in 64 bits (kv_ref.py)."""
import numpy as np
import pytest

from kv_ref import Batch
from test_gpu_kv import check_attn, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group", [1, 3, 4, 16, 20])
@pytest.mark.parametrize("lens", [
    [(1, 19000), (40, 300)],                                    # more ranges than a wave joins at once
    [(70, 500), (1, 5000), (0, 10), (3, 2500), (2, 0), (1, 4097)],
    [(5, 18000), (33, 40), (1, 17000)],
])
def test_decode_steps_beside_prompts(kq4, torch_dev, lens, group, dim):
    rng = np.random.default_rng(dim + group)
    b = Batch(rng, lens, 2, dim, 64, dim, pad=2)
    b.fill(rng, upto="all", spread=1.0)
    check_attn(kq4, torch_dev, b, rand(rng, b.n, 2 * group, dim), 2 * group)


@pytest.mark.parametrize("lens,tile,split", [
    ([(1, 3000), (40, 2000), (4, 2500)], 0, 3), ([(1, 3000), (40, 2000), (4, 2500)], 0, 30),
    ([(1, 3000), (4, 2000), (3, 2500)], 16, 20), ([(1, 3000), (9, 2000), (4, 2500)], 16, 3),
])
def test_given_numbers_of_ranges(kq4, torch_dev, lens, tile, split):
    """Also of sequences with more rows than a tile of the 16-row form."""
    rng = np.random.default_rng(split)
    b = Batch(rng, lens, 2, 128, 32, 128, pad=1)
    b.fill(rng, upto="all", spread=1.0)
    x = rand(rng, b.n, 8, 128)
    with kq4.options(attn_tile=tile, attn_split=split):
        check_attn(kq4, torch_dev, b, x, 8)
        check_attn(kq4, torch_dev, b, x, 8, window=900)


@pytest.mark.parametrize("kv_heads,lens", [
    (2, [(1, 5000)]), (1, [(1, 2000), (1, 1), (0, 700), (1, 0), (2, 900)]),     # more than 16 ranges: the join of many
    (2, [(1, 300 + 31 * i) for i in range(40)]), (8, [(1, 2000), (1, 5), (1, 700)] * 4),   # up to 16: that of few
    (2, [(9, 600), (1, 1500), (5, 40)]),                       # more rows than the bound says: those stay whole
])
@pytest.mark.parametrize("window", [0, 333])
@pytest.mark.parametrize("dim", [64, 128])
def test_shares_of_all_keys(kq4, torch_dev, lens, kv_heads, window, dim):
    """A bound far above the lengths, so that ranges go by the keys that are there, of both head sizes."""
    rng = np.random.default_rng(dim + len(lens))
    b = Batch(rng, lens, kv_heads, dim, 64, dim, pad=1)
    b.fill(rng, upto="all", spread=1.0)
    check_attn(kq4, torch_dev, b, rand(rng, b.n, 4 * kv_heads, dim), 4 * kv_heads, window=window, max_q=1, max_kv=1000000)
