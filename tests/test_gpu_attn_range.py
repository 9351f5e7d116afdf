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
