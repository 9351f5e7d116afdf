"""The attention's workspace without a GPU: partial sums of a decode step's long key axis are kept for its rows alone, not
for those of the prompts beside it, and their bytes stay within a bound."""
import pytest

from test_serving_host import SETUP
from test_workspace_routes import standin  # noqa: F401

HEADS, KV, DIM = 32, 8, 128
MIB = 1 << 20


@pytest.mark.parametrize("n_tok,n_seq,max_q,max_kv,most", [
    (2049, 2, 2048, 131072, 64 * MIB),       # a decode step beside a chunk
    (8193, 2, 8192, 131072, 64 * MIB),
    (8192 + 63, 64, 8192, 131072, 256 * MIB),
    (16384, 64, 4096, 131072, 256 * MIB),
    (4096, 1, 1, 131072, 64 * MIB),          # a prompt where a bound says that there is none
    (2049, 2, 2048, (1 << 31) - 1, 256 * MIB),
    (64, 64, 1, (1 << 31) - 1, 256 * MIB),
    (4096, 4096, 1, 131072, 256 * MIB),
])
def test_partial_sums_stay_small(kq4_cpu, n_tok, n_seq, max_q, max_kv, most):
    assert kq4_cpu.attn_workspace_bytes(n_tok, n_seq, HEADS, KV, DIM, max_q, max_kv) <= most


def test_joins_of_the_short_sequences_alone(standin):  # noqa: F811
    """Decode steps over long caches beside a chunk: the join of many ranges is as large as the steps' rows."""
    res = standin(SETUP + """
hip.standin_clear()
rc = attn(kv(n_seq=2, n_tok=8193), out=at(20), max_q=8192, max_kv=131072)
result = [rc] + [s for s in hip.standin_log().decode().split("\\n")[:-1] if "join" in s]
""")
    assert res[0] == 0 and len(res) == 2, res
    grid = int(res[1].split(" ")[-2])
    assert grid == 2 * KV * 16 * (DIM // 32)


@pytest.mark.parametrize("tile,split", [(-1, -1), (-1, 3), (16, -1), (16, 40), (128, -1), (256, 5)])
@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (8, 1), (20, 1), (12, 4), (64, 64)])
def test_a_reservation_holds_every_smaller_batch(standin, heads, kv_heads, tile, split):  # noqa: F811
    """The size for a largest batch is enough for any of fewer tokens, sequences and lower bounds: captured calls, which
    cannot grow the workspace, all run."""
    res = standin(SETUP + """
import random
rng = random.Random(heads * 100 + tile + split)
assert k.kq4_set_option(b"attn_tile", tile) == 0 and k.kq4_set_option(b"attn_split", split) == 0
log = lambda n: max(0, int(round((n + 1) ** rng.random())) - rng.randint(0, 1))
result = []
for n_seq, max_q, max_kv, window in [(1, 1, 1000, 0), (64, 1, 8192, 0), (33, 1, 200000, 0), (300, 2, 5000, 0), (8, 4, 70000, 0),
                                     (4, 2048, 16384, 0), (70, 600, 131072, 0), (9, 300, 100000, 1500), (1, 1, 700, 0),
                                     (1, 8192, 8192, 0)]:
    n_tok = max(n_seq, min(n_seq * max_q, 9000))
    need = k.kq4_attn_workspace_bytes(n_tok, n_seq, heads, kv_heads, 128, window, max_q, max_kv)
    hip.standin_capture(0)
    assert k.kq4_shutdown() is None and k.kq4_init(0) == 0
    reserve_exactly(need)
    hip.standin_capture(1)
    for i in range(400):
        s = n_seq if i % 3 == 0 else max(1, min(n_seq, log(n_seq)))
        q, m = min(max_q, log(max_q)), min(max_kv, log(max_kv) if i % 2 else rng.randint(max_kv // 2, max_kv))
        t = max(1, min(n_tok, rng.choice([s, s * q, log(n_tok), n_tok])))
        c = kv(n_seq=s, n_tok=t, kv_heads=kv_heads)
        rc = attn(c, out=at(30), q=at(20), ldq=heads * 128, heads=heads, window=window, max_q=q, max_kv=m)
        if rc:
            result.append((n_seq, max_q, max_kv, window, s, q, m, t, rc, kq4.last_error()))
""", heads=heads, kv_heads=kv_heads, tile=tile, split=split)
    assert res == []
