"""GPU: the attention where a row's numbers lie far apart, against the plain form in 64 bits (kv_ref.py)."""
import numpy as np
import pytest

from kv_ref import F32, Batch
from test_gpu_kv import check_attn, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tile,split", [(0, 0), (16, 1), (16, 2), (128, 1), (128, 2), (256, 1)])
@pytest.mark.parametrize("q", [1, 5])
@pytest.mark.parametrize("values", ["zeros then some", "least scale"])
def test_many_keys_of_the_least_value_scale(kq4, torch_dev, tile, split, q, values):
    """100000 keys; those after the first 1024 score 5 (7.2 in powers of 2, less than the running maximum is raised for)
    above them, so the row's sum is 2^16.6 times 2^(6 + 7.2) over a value scale of 2^-100: past fp32 unless it is held
    lower. Of the values either 60 % are zeros as they are appended and the others ordinary, or all are of the least
    scale."""
    rng, n = np.random.default_rng(31), 100000
    b = Batch(rng, [(q, n)], 1, 64, 64, 0)
    keys, vals, none = np.full((64, 16), 0), np.full((64, 16), 0), np.zeros((64, 16), np.int64)
    keys[0] = 127
    vals[:] = np.where(np.arange(64) % 2, 50, 100)[:, None]
    for g0 in range(0, n, 16):
        p, g, _ = b.place(0, g0)
        some = values == "least scale" or g0 >= 60000
        b.put_group(p, 0, g, np.stack([keys if g0 >= 1024 else none, vals if some else none]))
        b.scales[p, 0, g] = 5 / 127, 1 / 64 if some and values != "least scale" else 2.0 ** -100
    x = np.zeros((q, 4, 64), F32)
    x[:, :, 0] = 1
    with kq4.options(attn_tile=tile, attn_split=split):
        check_attn(kq4, torch_dev, b, x, 4, scale=1.0)


@pytest.mark.parametrize("tile,split", [(0, 0), (16, 1), (16, 2), (16, 30), (128, 1), (128, 2), (256, 1)])
def test_a_late_key_keeps_the_share_of_zeros_before_it(kq4, torch_dev, tile, split):
    """60000 keys of zero values (scale 2^-100), then one of value scale 1 whose weight is 2^27 times theirs: together they
    have 4.5e-4 of the row, though the running maximum rises by 2^127. The one output is off by its own weight's two
    halves (2^-22) and a few roundings of 2^-24; the share itself, right to 2^-16, moves it by less: 2^-20 in all."""
    rng, n = np.random.default_rng(32), 60001
    b = Batch(rng, [(1, n)], 1, 64, 64, 0)
    none = np.zeros((64, 16), np.int64)
    for g0 in range(0, n, 16):
        p, g, _ = b.place(0, g0)
        b.put_group(p, 0, g, np.stack([none, none]))
        b.scales[p, 0, g] = 1 / 127, 2.0 ** -100
    c = np.zeros((2, 64, 16), np.int64)
    c[0, 0, (n - 1) % 16], c[1, :, (n - 1) % 16] = 127, rng.integers(50, 128, 64)
    b.put_group(p, 0, g, c)
    b.scales[p, 0, g] = 27 * np.log(2) / 127, 1.0
    x = np.zeros((1, 4, 64), F32)
    x[:, :, 0] = 1
    with kq4.options(attn_tile=tile, attn_split=split):
        got = check_attn(kq4, torch_dev, b, x, 4, scale=1.0)
    want = b.attention(x, 4, 1.0)[0]
    assert (np.abs(got - want) <= 2.0 ** -20 * np.abs(want)).all()
