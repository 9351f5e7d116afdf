"""Calls whose launches would pass 2^32 threads are refused before anything is launched (on the stand-in for the HIP
runtime, tests/c/hip_standin.c)."""
import pytest

from test_serving_host import SETUP
from test_workspace_routes import standin  # noqa: F401


@pytest.mark.parametrize("call,want", [
    ("logprobs(n=(1 << 24) - 1, vocab=5)", [0, 2]), ("logprobs(n=1 << 24, vocab=5)", [-1, 0]),
    ("logprobs(n=1 << 23, vocab=8193, ld=8193)", [-1, 0]), ("logprobs(n=1 << 20, vocab=8193, ld=8193)", [0, 2]),
    ("attn(kv(n_seq=1 << 20, n_tok=1 << 20), out=at(60), max_q=1, max_kv=200)", [0, 1]),
    ("attn(kv(n_seq=1 << 22, n_tok=1 << 22), out=at(60), max_q=1, max_kv=200)", [-1, 0]),
    ("attn(kv(n_seq=1, n_tok=1 << 24), heads=8, ldq=1024, out=at(60), max_q=1 << 24, max_kv=1 << 24)", [0, 1]),
    ("attn(kv(n_seq=1 << 23, n_tok=1 << 23), heads=8, ldq=1024, out=at(60), max_q=40, max_kv=40)", [-1, 0]),
])
def test_launches_that_fit(standin, call, want):  # noqa: F811
    assert standin(SETUP + f"result = launched(lambda: {call})") == want


def test_sizes_of_refused_rows(kq4_cpu):
    assert kq4_cpu.logprobs_workspace_bytes((1 << 24) - 1, 5, 1) > 0 == kq4_cpu.logprobs_workspace_bytes(1 << 24, 5, 1)


def test_scales_past_the_exponent(standin):  # noqa: F811
    """The scale times log2(e) has to be a number."""
    assert standin(SETUP + "result = [launched(lambda: attn(kv(), max_kv=100, scale=s)) for s in (1.9e38, 2.5e38)]") == \
        [[0, 1], [-1, 0]]
