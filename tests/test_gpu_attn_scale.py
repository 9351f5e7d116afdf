"""GPU: attention of queries and keys whose magnitudes lie at the ends of fp32, their products where scores are."""
import numpy as np
import pytest

from kv_ref import F32
from test_attn_accuracy import BOUND, batch, measure

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tile", [16, 128, 256])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("by", [-124, -116, -108, 60, 90])
def test_queries_far_from_one(kq4, torch_dev, tile, dim, by):
    """Queries times 2^by, key scales times 2^-by: the same scores, exactly."""
    torch = torch_dev
    b, q = batch([(30, 200), (1, 70)], 1, dim, 42)
    b.rope, b.rope_dim = None, 0
    q[np.abs(q) < 2.0 ** -2] = 0                              # (no subnormal query: each stays what it was)
    want = b.attention(q, 4, float(F32(dim ** -0.5)))[0]
    q = np.ldexp(q, by).astype(F32)
    b.scales[..., 0] = np.ldexp(b.scales[..., 0], -by)
    out = torch.empty((b.n, 4 * dim), device="cuda")
    with kq4.options(attn_tile=tile):
        kq4.attn_dev(out, torch.from_numpy(q.reshape(b.n, -1)).cuda(), b.device(torch, kq4), 4, dim ** -0.5, max_q=30,
                     max_kv=200)
    assert measure(out.cpu().numpy().astype(np.float64).reshape(want.shape), want) <= BOUND
