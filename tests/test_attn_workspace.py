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
