"""The host side of the cache, attention and log probability calls without a GPU, on the stand-in for the HIP
runtime (tests/c/hip_standin.c): what they refuse, launch and ask of the workspace; and the binding's refusals."""
import pytest

from test_workspace_routes import standin  # noqa: F401

SETUP = """
class KV(kq4.KV):
    pass

def kv(**more):
    f = dict(codes=at(1), scales=at(2), n_pages=100, page_tokens=64, kv_heads=8, head_dim=128, block_table=at(3),
             table_pages=50, q_start=at(4), kv_len=at(5), n_seq=3, n_tok=7, rope=at(6), rope_rows=4096, rope_dim=128,
             rope_pos=None)
    f.update(more)
    return KV(**f)

def append(c, k=at(7), ldk=1024, v=at(8), ldv=1024):
    return k_.kq4_kv_append_dev(ctypes.byref(c) if c else None, k, ldk, v, ldv, None)

def attn(c, out=at(9), q=at(10), ldq=4096, heads=32, scale=0.1, window=0, max_q=3, max_kv=3000):
    return k_.kq4_attn_dev(out, ctypes.byref(c) if c else None, q, ldq, heads, scale, window, max_q, max_kv, None)

def logprobs(lp=at(1), ent=at(2), tlp=at(3), tid=at(4), x=at(5), ld=1000, token=at(6), n=4, vocab=1000, top=5):
    return k_.kq4_logprobs_dev(lp, ent, tlp, tid, x, ld, token, n, vocab, top, None)

def launched(f):
    hip.standin_clear()
    rc = f()
    return rc, len(hip.standin_log().decode().split("\\n")) - 1

k_ = k
"""

CACHE = [dict(n_pages=0), dict(page_tokens=48), dict(page_tokens=8), dict(page_tokens=8192), dict(kv_heads=0),
         dict(head_dim=96), dict(head_dim=256), dict(codes=None), dict(codes="at(1) + 8"), dict(scales="at(2) + 4"),
         dict(scales=None), dict(block_table=None), dict(q_start=None), dict(kv_len=None), dict(kv_len="at(5) + 2"),
         dict(n_seq=-1), dict(n_tok=-1), dict(table_pages=0), dict(table_pages=1 << 26), dict(rope_dim=0),
         dict(rope=None), dict(rope_dim=144), dict(rope_dim=160), dict(rope_dim=20), dict(rope_rows=0),
         dict(rope="at(6) + 8"), dict(rope_pos="at(6) + 1")]


def args(d):
    return ", ".join(f"{n}={v if isinstance(v, str) else repr(v)}" for n, v in d.items())


def test_cache_refusals(standin):  # noqa: F811
    lines = "".join(f"c = kv({args(d)})\nresult.append([launched(lambda: append(c)), launched(lambda: attn(c))])\n"
                    for d in CACHE)
    res = standin(SETUP + "result = []\n" + lines)
    for d, r in zip(CACHE, res):
        assert r == [[-1, 0], [-1, 0]], d


@pytest.mark.parametrize("call", [
    "append(None)", "append(kv(), k=None)", "append(kv(), v=None)", "append(kv(), k=at(7) + 4)", "append(kv(), ldk=1023)",
    "append(kv(), ldk=1020)", "append(kv(), ldv=1026)", "append(kv(), ldv=-1024)",
    "attn(None)", "attn(kv(), out=None)", "attn(kv(), q=None)", "attn(kv(), heads=0)", "attn(kv(), heads=12)",
    "attn(kv(), heads=-8)", "attn(kv(), scale=0.0)", "attn(kv(), scale=-1.0)", "attn(kv(), scale=float('nan'))",
    "attn(kv(), scale=float('inf'))", "attn(kv(), window=-1)", "attn(kv(), max_q=-1)", "attn(kv(), max_kv=-1)",
    "attn(kv(), ldq=4095)", "attn(kv(), ldq=4092)", "attn(kv(), q=at(10) + 8)", "attn(kv(), out=at(9) + 4)",
    "attn(kv(), out=at(10))", "attn(kv(), out=at(10) + 16 * 4096)", "attn(kv(), q=at(9) + 4)",
    "logprobs(n=-1)", "logprobs(vocab=0)", "logprobs(vocab=1001)", "logprobs(vocab=(1 << 20) + 1, ld=1 << 21)",
    "logprobs(top=33)", "logprobs(top=-1)", "logprobs(vocab=4, top=5)", "logprobs(x=None)", "logprobs(token=None)",
    "logprobs(tlp=None)", "logprobs(tid=None)", "logprobs(top=0)", "logprobs(lp=None, ent=None, tlp=None, tid=None, top=0)",
    "logprobs(x=at(5) + 2)", "logprobs(lp=at(1) + 1)", "logprobs(n=(1 << 31) - 1, vocab=1 << 20, ld=1 << 20)",
])
def test_argument_refusals(standin, call):  # noqa: F811
    assert standin(SETUP + f"result = launched(lambda: {call})") == [-1, 0]


def test_nothing_to_do_launches_nothing(standin):  # noqa: F811
    calls = ["append(kv(n_tok=0))", "append(kv(n_seq=0))", "attn(kv(n_tok=0))", "attn(kv(n_seq=0))", "logprobs(n=0)"]
    body = "result = [" + ", ".join(f"launched(lambda: {c})" for c in calls) + "]"
    assert standin(SETUP + body) == [[0, 0]] * len(calls)


def test_workspace_of_captured_calls(standin):  # noqa: F811
    """A split attention and the log probabilities need the workspace: refused on a capturing stream that cannot
    grow it, done after a reservation of the bytes they name."""
    res = standin(SETUP + """
calls = [lambda: attn(kv(), max_q=1, max_kv=100000), lambda: logprobs()]
need = [k.kq4_attn_workspace_bytes(7, 3, 32, 8, 128, 0, 1, 100000), k.kq4_logprobs_workspace_bytes(4, 1000, 5)]
hip.standin_capture(1)
before = [launched(f) for f in calls]
hip.standin_capture(0)
assert k.kq4_workspace_reserve(max(need)) == 0
hip.standin_capture(1)
after = [launched(f) for f in calls]
result = [need, before, after]
""")
    need, before, after = res
    assert min(need) > 0
    assert before == [[-1, 0], [-1, 0]]
    assert after == [[0, 2], [0, 2]]


@pytest.mark.parametrize("batch,want", [
    (dict(n_seq=1, n_tok=1, max_q=1, max_kv=800), ["rows16", "join_few"]),          # short: 4 waves, split
    (dict(n_seq=1, n_tok=1, max_q=1, max_kv=200), ["rows16"]),
    (dict(n_seq=64, n_tok=64, max_q=1, max_kv=4000), ["rows16"]),                    # a workgroup a CU without splits
    (dict(n_seq=1, n_tok=1, max_q=1, max_kv=131072), ["rows16", "join"]),
    (dict(n_seq=64, n_tok=64, max_q=1, max_kv=131072), ["rows16", "join_few"]),      # however long one may be
    (dict(n_seq=32, n_tok=32, max_q=1, max_kv=8192), ["rows16", "join_few"]),        # in halves, by length
    (dict(n_seq=64, n_tok=64, max_q=1, max_kv=4100), ["rows16"]),                    # whole, by length
    (dict(n_seq=8, n_tok=8, max_q=1, max_kv=65536), ["rows16", "join_few"]),         # shares of all keys
    (dict(n_seq=1, n_tok=4, max_q=4, max_kv=800), ["rows16", "join_few"]),           # 16 rows per kv head
    (dict(n_seq=1, n_tok=4096, max_q=4096, max_kv=4096), ["rows32"]),
    (dict(n_seq=1, n_tok=128, max_q=128, max_kv=16000), ["rows32", "join_few"]),
    (dict(n_seq=9, n_tok=200, max_q=150, max_kv=150), ["mixed"]),                    # decode steps and a prompt
    (dict(n_seq=9, n_tok=200, max_q=150, max_kv=3000), ["mixed", "join_few"]),
    (dict(n_seq=1, n_tok=1500, max_q=1500, max_kv=1500), ["rows32"]),                   # a split's sums would cost more
    (dict(n_seq=9, n_tok=9000, max_q=8000, max_kv=9000), ["rows32", "rows16", "join_few"]),
    (dict(n_seq=4, n_tok=0, max_q=9, max_kv=9), []),
])
def test_attention_launches(standin, batch, want):  # noqa: F811
    """Which kernels a batch takes (32 query heads, 8 kv heads of 128): the forms, and joins where keys are split."""
    res = standin(SETUP + """
hip.standin_clear()
rc = attn(kv(n_seq=n_seq, n_tok=n_tok), out=at(20), max_q=max_q, max_kv=max_kv)
result = [rc] + [s.split(" ")[0] for s in hip.standin_log().decode().split("\\n")[:-1]]
""", **batch)
    assert res[0] == 0
    names = ["join_few" if "join_few" in s else "join" if "join" in s else "mixed" if "mixed" in s else
             "rows16" if "rows16" in s else "rows32" if "rows32" in s else s for s in res[1:]]
    assert names == want


def test_sizes(kq4_cpu):
    assert kq4_cpu.kv_codes_shape(3, 32, 2, 64) == (3, 2, 2, 2, 1024)
    lib = kq4_cpu.lib()
    assert lib.kq4_kv_codes_bytes(1 << 20, 64, 8, 128) == (1 << 20) * 64 * 8 * 256
    assert lib.kq4_kv_scales_bytes(3, 32, 2, 64) == 3 * 2 * 2 * 2 * 4
    for bad in ((0, 64, 8, 128), (1, 24, 8, 128), (1, 64, 0, 128), (1, 64, 8, 80)):
        assert lib.kq4_kv_codes_bytes(*bad) == 0 and lib.kq4_kv_scales_bytes(*bad) == 0
        with pytest.raises(kq4_cpu.KQ4Error):
            kq4_cpu.kv_codes_shape(*bad)
    assert kq4_cpu.attn_workspace_bytes(0, 1, 8, 8, 128, 1, 100) == 0
    assert kq4_cpu.attn_workspace_bytes(1, 1, 9, 8, 128, 1, 100) == 0
    assert kq4_cpu.logprobs_workspace_bytes(1, 0, 0) == 0


def test_binding_refuses_host_tensors_and_shapes(kq4_cpu):
    import torch
    codes, scales = torch.zeros((4, 2, 1, 2, 1024), dtype=torch.uint8), torch.zeros((4, 2, 1, 2))
    table = torch.zeros((1, 4), dtype=torch.int32)
    start, length = torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(kq4_cpu.KQ4Error, match="device tensor"):
        kq4_cpu.KVBatch(codes, scales, 16, table, start, length, 1)
    with pytest.raises(kq4_cpu.KQ4Error, match="expected"):
        kq4_cpu.KVBatch(codes, scales[:3], 16, table, start, length, 1)
    with pytest.raises(kq4_cpu.KQ4Error, match="expected"):
        kq4_cpu.KVBatch(codes, scales, 32, table, start, length, 1)
    with pytest.raises(kq4_cpu.KQ4Error, match="sequences"):
        kq4_cpu.KVBatch(codes, scales, 16, table, start, torch.zeros(2, dtype=torch.int32), 1)
    with pytest.raises(kq4_cpu.KQ4Error, match="device tensor"):
        kq4_cpu.logprobs_dev(torch.zeros(2, 100), entropy=torch.zeros(2))


def test_rope_table_in_64_bits(kq4_cpu):
    import math
    t = kq4_cpu.rope_table(100001, 64, 1e6, device="cpu")
    assert tuple(t.shape) == (100001, 32, 2)
    a = 100000 * 1e6 ** (-2 / 64)
    assert abs(t[100000, 1, 0].item() - math.cos(a)) < 2.0 ** -24 + 1e-10
    assert abs(t[100000, 1, 1].item() - math.sin(a)) < 2.0 ** -24 + 1e-10
