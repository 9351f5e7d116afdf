"""GPU: appending to the paged int8 key/value cache and the attention over it, against the plain forms in 64 bits
(kv_ref.py). Codes and scales have to be equal byte for byte; attention within the bound that kv_ref derives."""
import numpy as np
import pytest

from kv_ref import F32, Batch

pytestmark = pytest.mark.gpu


def up(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def rand(rng, n, heads, dim):
    x = rng.standard_normal((n, heads, dim)).astype(F32)
    x[:, :, rng.random(dim) < 0.05] *= 6
    return x


def check_append(kq4, torch, b, k, v):
    kv = b.device(torch, kq4)
    kq4.kv_append_dev(kv, up(torch, k.reshape(b.n, -1)), up(torch, v.reshape(b.n, -1)))
    torch.cuda.synchronize()
    b.append(k, v)
    codes, scales = kv.tensors["codes"].cpu().numpy(), kv.tensors["scales"].cpu().numpy()
    np.testing.assert_array_equal(scales, b.scales)           # (NaN where NaN: nothing else was touched)
    np.testing.assert_array_equal(codes, b.codes)


def check_attn(kq4, torch, b, q, heads, window=0, max_q=None, max_kv=None, scale=None):
    scale = scale or b.dim ** -0.5
    want, tol, rows = b.attention(q, heads, float(F32(scale)), window)
    kv = b.device(torch, kq4)
    out = torch.full((b.n, heads * b.dim), 7.5, device="cuda")
    kq4.attn_dev(out, up(torch, q.reshape(b.n, -1)), kv, heads, scale, window=window,
                 max_q=max([q for q, _ in b.lens] + [0]) if max_q is None else max_q,
                 max_kv=max([kv for _, kv in b.lens] + [0]) if max_kv is None else max_kv)
    torch.cuda.synchronize()
    got = out.cpu().numpy().astype(np.float64).reshape(b.n, heads, b.dim)
    assert (got[~rows] == 7.5).all()                          # rows behind the last sequence
    np.testing.assert_array_equal(np.isnan(got[rows]), np.isnan(want[rows]))
    here = rows[:, None, None] & np.isfinite(want)
    err = np.abs(got - want)
    assert (err[here] <= tol[here]).all(), (err[here].max(), (err[here] / np.maximum(tol[here], 1e-300)).max())
    return got


# ---- append ------------------------------------------------------------------------------------

LENS = [
    [(1, 1)], [(1, 16)], [(1, 17)], [(16, 16)], [(17, 17)], [(1, 777)], [(100, 100)], [(33, 90)],
    [(1, 5), (1, 31), (1, 64), (1, 65), (1, 200)],
    [(3, 3), (0, 40), (20, 45), (1, 129), (64, 64), (15, 16)],
]


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("heads,dim,page,rope", [(8, 128, 64, 128), (2, 64, 16, 64), (5, 128, 16, 32),
                                                 (1, 64, 128, 0), (3, 128, 32, 96), (4, 64, 32, 32)])
def test_append(kq4, torch_dev, lens, heads, dim, page, rope):
    rng = np.random.default_rng(len(lens) * 1000 + heads * 10 + page)
    b = Batch(rng, lens, heads, dim, page, rope, pad=2)
    b.fill(rng)
    check_append(kq4, torch_dev, b, rand(rng, b.n, heads, dim), rand(rng, b.n, heads, dim))


def test_append_many_sequences(kq4, torch_dev):
    """More sequences than a wave has lanes, empty ones among them."""
    rng = np.random.default_rng(5)
    lens = [(int(rng.integers(0, 4)), int(rng.integers(4, 60))) for _ in range(150)]
    b = Batch(rng, lens, 2, 64, 16, 64)
    b.fill(rng)
    check_append(kq4, torch_dev, b, rand(rng, b.n, 2, 64), rand(rng, b.n, 2, 64))


def test_append_token_by_token(kq4, torch_dev):
    """The same cache grown one token at a time: scales that grow rewrite the earlier codes, as in the plain form."""
    torch, rng = torch_dev, np.random.default_rng(6)
    lens = [(1, 1), (1, 14)]
    b = Batch(rng, [(1, 40), (1, 53)], 2, 128, 32, 128)
    b.lens, b.kv_len = lens, np.array([1, 14], np.int32)
    b.fill(rng)
    kv = b.device(torch, kq4)
    for step in range(39):
        b.lens = [(1, 1 + step), (1, 14 + step)]
        b.kv_len = np.array([1 + step, 14 + step], np.int32)
        kv.tensors["kv_len"].copy_(up(torch, b.kv_len))
        k, v = rand(rng, 2, 2, 128) * F32(1.2 ** step), rand(rng, 2, 2, 128)
        kq4.kv_append_dev(kv, up(torch, k.reshape(2, -1)), up(torch, v.reshape(2, -1)))
        b.append(k, v)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(kv.tensors["scales"].cpu().numpy(), b.scales)
    np.testing.assert_array_equal(kv.tensors["codes"].cpu().numpy(), b.codes)


def test_append_columns_of_a_fused_tensor(kq4, torch_dev):
    torch, rng = torch_dev, np.random.default_rng(7)
    b = Batch(rng, [(20, 30), (1, 7)], 2, 64, 16, 64)
    b.fill(rng)
    qkv = rng.standard_normal((b.n, 8 * 64)).astype(F32)      # 4 query, 2 key, 2 value heads
    d = up(torch, qkv)
    kv = b.device(torch, kq4)
    kq4.kv_append_dev(kv, d[:, 256:384], d[:, 384:])
    torch.cuda.synchronize()
    b.append(qkv[:, 256:384].reshape(b.n, 2, 64), qkv[:, 384:].reshape(b.n, 2, 64))
    np.testing.assert_array_equal(kv.tensors["codes"].cpu().numpy(), b.codes)


@pytest.mark.parametrize("what", ["zero", "tiny", "huge", "nan", "inf", "old_nan"])
def test_append_values_at_the_ends(kq4, torch_dev, what):
    rng = np.random.default_rng(8)
    b = Batch(rng, [(5, 12), (20, 20)], 2, 64, 16, 0)
    b.fill(rng)
    k, v = rand(rng, b.n, 2, 64), rand(rng, b.n, 2, 64)
    if what == "zero":
        k[:], v[6] = 0, 0
    elif what == "tiny":
        k *= F32(1e-42)
        v *= F32(1e-33)
    elif what == "huge":
        k *= F32(1e36)
    elif what == "nan":
        k[2, 0, 5] = np.nan
        v[10, 1, 63] = np.nan
    elif what == "inf":
        v[3, 1, 0] = np.inf
        k[24, 0, 1] = -np.inf
    else:
        p, g, _ = b.place(0, 3)
        b.scales[p, 1, g, 0] = np.nan
    check_append(kq4, torch_dev, b, k, v)


def test_append_skips_what_has_no_place(kq4, torch_dev):
    """Pages that the cache does not have, positions past the table, tokens before position 0."""
    rng = np.random.default_rng(9)
    b = Batch(rng, [(40, 60), (1, 20), (9, 4), (30, 70)], 2, 64, 16, 64)
    b.fill(rng)
    b.table[0, 2] = b.codes.shape[0]
    b.table[1, 1] = -7
    b.table = np.ascontiguousarray(b.table[:, :4])            # the last sequence's 70 positions pass 64
    check_append(kq4, torch_dev, b, rand(rng, b.n, 2, 64), rand(rng, b.n, 2, 64))


def test_append_rope_positions(kq4, torch_dev):
    """Rows given per token; a row outside the table makes that key, and its group, NaN."""
    rng = np.random.default_rng(10)
    b = Batch(rng, [(40, 40), (3, 50)], 1, 128, 64, 64)
    b.fill(rng)
    b.rope_pos = rng.integers(0, 50, b.n).astype(np.int32)
    b.rope_pos[3], b.rope_pos[41] = 50, -1
    check_append(kq4, torch_dev, b, rand(rng, b.n, 1, 128), rand(rng, b.n, 1, 128))


# ---- attention ---------------------------------------------------------------------------------

@pytest.mark.parametrize("lens", [
    [(1, 1)], [(1, 16)], [(1, 63)], [(1, 64)], [(1, 65)], [(1, 300)], [(1, 1500)],
    [(1, 1), (1, 100), (1, 17), (1, 256), (1, 257)],
    [(2, 2), (5, 64), (3, 129)], [(40, 40)], [(130, 200)],
    [(33, 33), (1, 500), (0, 20), (70, 300), (4, 4)],
])
@pytest.mark.parametrize("heads,kv_heads,dim,page,rope", [(4, 2, 128, 64, 128), (8, 1, 64, 16, 64),
                                                          (3, 3, 128, 16, 32), (10, 2, 64, 128, 0)])
def test_attention(kq4, torch_dev, lens, heads, kv_heads, dim, page, rope):
    rng = np.random.default_rng(sum(kv for _, kv in lens) + heads)
    b = Batch(rng, lens, kv_heads, dim, page, rope, pad=1)
    b.fill(rng, upto="all", spread=1.0)
    check_attn(kq4, torch_dev, b, rand(rng, b.n, heads, dim), heads)


@pytest.mark.parametrize("heads,kv_heads", [(16, 1), (17, 1), (32, 1), (33, 3), (48, 2)])
def test_attention_many_heads_per_key(kq4, torch_dev, heads, kv_heads):
    rng = np.random.default_rng(heads)
    b = Batch(rng, [(1, 90), (3, 33), (2, 2)], kv_heads, 64, 32, 64)
    b.fill(rng, upto="all")
    check_attn(kq4, torch_dev, b, rand(rng, b.n, heads, 64), heads)


@pytest.mark.parametrize("window", [1, 2, 15, 16, 64, 100, 10000])
@pytest.mark.parametrize("lens", [[(1, 700), (1, 3)], [(80, 80), (60, 333), (2, 130)]])
def test_attention_window(kq4, torch_dev, window, lens):
    rng = np.random.default_rng(window)
    b = Batch(rng, lens, 2, 64, 16, 64)
    b.fill(rng, upto="all")
    # groups before the window hold NaN: nothing masked may reach a row
    for i, (q, kv) in enumerate(lens):
        for pos in range(0, max(0, kv - q - window - 15), 16):
            p, g, _ = b.place(i, pos)
            b.scales[p, :, g] = np.nan
    check_attn(kq4, torch_dev, b, rand(rng, b.n, 4, 64), 4, window=window)


@pytest.mark.parametrize("max_q,max_kv", [(0, 0), (1, 1), (1, 300), (64, 64), (500, 100000), (7, 5000)])
def test_attention_bounds_change_no_result(kq4, torch_dev, max_q, max_kv):
    rng = np.random.default_rng(3)
    b = Batch(rng, [(1, 1100), (50, 70), (2, 400)], 2, 128, 32, 128)
    b.fill(rng, upto="all", spread=1.0)
    check_attn(kq4, torch_dev, b, rand(rng, b.n, 8, 128), 8, max_q=max_q, max_kv=max_kv)


@pytest.mark.parametrize("tile", [16, 128, 256])
@pytest.mark.parametrize("split", [1, 2, 5, 20])
def test_attention_forms(kq4, torch_dev, tile, split):
    """Every form and number of splits, also where the planner would take another."""
    rng = np.random.default_rng(tile + split)
    b = Batch(rng, [(1, 1400), (90, 90), (3, 700), (0, 9), (40, 1000)], 2, 64, 32, 64, pad=3)
    b.fill(rng, upto="all", spread=1.0)
    x = rand(rng, b.n, 6, 64)
    with kq4.options(attn_tile=tile, attn_split=split):
        check_attn(kq4, torch_dev, b, x, 6)
        check_attn(kq4, torch_dev, b, x, 6, window=300)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens", [[(1, 9000)], [(1, 7000), (1, 50), (1, 4097)], [(30, 5000)], [(1, 6000), (70, 300)]])
def test_attention_long_contexts(kq4, torch_dev, dim, lens):
    """Many splits of the key axis, sequences that use few of them beside those that use all."""
    rng = np.random.default_rng(dim)
    b = Batch(rng, lens, 1, dim, 64, dim)
    b.fill(rng, upto="all", spread=1.0)
    check_attn(kq4, torch_dev, b, rand(rng, b.n, 4, dim), 4)


@pytest.mark.parametrize("lens", [[(1, 400), (1, 0), (5, 3), (1, 90)], [(70, 60), (64, 400), (1, 0)]])
def test_attention_empty_rows_and_missing_pages(kq4, torch_dev, lens):
    """Sequences without keys, tokens before position 0, pages that the cache does not have, positions past the
    table: rows that see nothing are zeros, others see the rest."""
    rng = np.random.default_rng(4)
    b = Batch(rng, lens, 2, 64, 16, 64)
    b.fill(rng, upto="all")
    at = int(np.argmax(b.kv_len))
    b.table[at, 3] = -1
    b.table[at, 0] = 1 << 30
    b.table = np.ascontiguousarray(b.table[:, :20])           # 320 positions
    check_attn(kq4, torch_dev, b, rand(rng, b.n, 4, 64), 4)


@pytest.mark.parametrize("q", [1, 40])
@pytest.mark.parametrize("what", ["zero_v", "zero_k", "wide_v", "sharp", "tiny_q", "zero_q", "nan_q", "nan_k", "inf_v"])
def test_attention_values_at_the_ends(kq4, torch_dev, what, q):
    rng = np.random.default_rng(11)
    b = Batch(rng, [(q, 200), (q, 77)], 1, 64, 16, 0)
    b.fill(rng, upto="all", spread=1.0)
    x = rand(rng, b.n, 4, 64)
    p, g, _ = b.place(0, 100)
    if what == "zero_v":          # appended zeros: scale 2^-100, codes 0; the group still takes its share
        b.scales[p, 0, g, 1] = 2.0 ** -100
        c = b.group(p, 0, g)
        c[1] = 0
        b.put_group(p, 0, g, c)
    elif what == "zero_k":
        b.scales[p, 0, g, 0] = 2.0 ** -100
    elif what == "wide_v":
        b.scales[p, 0, g, 1] *= 2.0 ** 40
        p2, g2, _ = b.place(1, 20)
        b.scales[p2, 0, g2, 1] *= 2.0 ** -60
    elif what == "sharp":
        x *= 30
    elif what == "tiny_q":
        x *= F32(1e-38)
    elif what == "zero_q":
        x[0] = 0
    elif what == "nan_q":
        x[q, 2, 3] = np.nan
    elif what == "nan_k":
        b.scales[p, 0, g, 0] = np.nan
    elif what == "inf_v":
        b.scales[p, 0, g, 1] = np.inf
    if what in ("nan_k", "inf_v"):                            # every row that sees the group is not finite
        want, _, _ = b.attention(x, 4, 0.125)
        kv = b.device(torch_dev, kq4)
        out = torch_dev.empty((b.n, 256), device="cuda")
        kq4.attn_dev(out, up(torch_dev, x.reshape(b.n, -1)), kv, 4, 0.125, max_q=q, max_kv=200)
        got = out.cpu().numpy().reshape(b.n, 4, 64)
        seen = 200 - q + np.arange(q) >= 96
        assert not np.isfinite(got[:q][seen]).any()
        np.testing.assert_allclose(got[:q][~seen], want[:q][~seen], atol=1e-3)
        assert np.isfinite(got[q:]).all()
        return
    check_attn(kq4, torch_dev, b, x, 4)


def test_attention_rope_positions_and_strides(kq4, torch_dev):
    torch, rng = torch_dev, np.random.default_rng(12)
    b = Batch(rng, [(5, 60), (1, 33)], 2, 128, 64, 128)
    b.fill(rng, upto="all", spread=1.0)
    b.rope_pos = rng.integers(0, 60, b.n).astype(np.int32)
    b.rope_pos[2] = 60                                        # off the table: that row is NaN
    x = rand(rng, b.n, 4, 128)
    got = check_attn(kq4, torch, b, x, 4)
    assert np.isnan(got[2]).all()
    wide = torch.zeros((b.n, 1024), device="cuda")
    wide[:, 256:768] = up(torch, x.reshape(b.n, -1))
    out = torch.empty((b.n, 512), device="cuda")
    kq4.attn_dev(out, wide[:, 256:768], b.device(torch, kq4), 4, 128 ** -0.5, max_q=5, max_kv=60)
    np.testing.assert_array_equal(out.cpu().numpy(), got.reshape(b.n, -1).astype(F32))


def test_cache_past_32_bit_offsets(kq4, torch_dev):
    """Pages whose bytes lie beyond 4 GiB: appended to and read there, nothing at the offsets modulo 2^32."""
    torch, rng = torch_dev, np.random.default_rng(13)
    b = Batch(rng, [(40, 40), (1, 30)], 8, 128, 64, 128, pool=8)
    k, v, x = rand(rng, b.n, 8, 128), rand(rng, b.n, 8, 128), rand(rng, b.n, 8, 128)
    b.fill(rng)
    far = (4 << 30) // (64 * 8 * 128 * 2) + 5                 # first page used, 128 KiB each
    codes = torch.zeros((far + 8, 8, 4, 2, 2048), dtype=torch.uint8, device="cuda")
    scales = torch.zeros((far + 8, 8, 4, 2), device="cuda")
    codes[far:] = up(torch, b.codes)
    scales[far:] = up(torch, b.scales)
    table = np.where(b.table >= 0, b.table + far, -1).astype(np.int32)
    kv = kq4.KVBatch(codes, scales, 64, up(torch, table), up(torch, b.q_start), up(torch, b.kv_len), b.n,
                     rope=up(torch, b.rope))
    kq4.kv_append_dev(kv, up(torch, k.reshape(b.n, -1)), up(torch, v.reshape(b.n, -1)))
    out = torch.empty((b.n, 1024), device="cuda")
    kq4.attn_dev(out, up(torch, x.reshape(b.n, -1)), kv, 8, 128 ** -0.5, max_q=40, max_kv=40)
    torch.cuda.synchronize()
    b.append(k, v)
    np.testing.assert_array_equal(codes[far:].cpu().numpy(), b.codes)
    assert int(codes[:far].count_nonzero()) == 0 and int(scales[:far].count_nonzero()) == 0
    want, tol, _ = b.attention(x, 8, float(F32(128 ** -0.5)))
    assert (np.abs(out.cpu().numpy().reshape(want.shape) - want) <= tol).all()


def test_shared_prefix_pages(kq4, torch_dev):
    """Two sequences read the same first pages and append to pages of their own."""
    rng = np.random.default_rng(14)
    b = Batch(rng, [(3, 40), (1, 50)], 2, 64, 16, 64)
    b.table[1, :2] = b.table[0, :2]                           # positions 0..31
    b.fill(rng, spread=1.0)
    k, v = rand(rng, b.n, 2, 64), rand(rng, b.n, 2, 64)
    check_append(kq4, torch_dev, b, k, v)
    check_attn(kq4, torch_dev, b, rand(rng, b.n, 4, 64), 4)


def test_graph_replays(kq4, torch_dev):
    """Append and a split attention captured once and replayed as the sequence grows, each replay as the eager calls
    on the same contents; eager calls with a workspace of their own in between."""
    torch, rng = torch_dev, np.random.default_rng(15)
    b = Batch(rng, [(1, 900), (1, 400)], 2, 128, 64, 128)
    b.fill(rng, spread=1.0)
    kv, other = b.device(torch, kq4), b.device(torch, kq4)
    b.lens = [(1, 880), (1, 380)]
    k, v, q = (torch.empty((2, w), device="cuda") for w in (256, 256, 512))
    out, want = torch.empty((2, 512), device="cuda"), torch.empty((2, 512), device="cuda")

    def step(c, o, stream=None):
        kq4.kv_append_dev(c, k, v, stream=stream)
        kq4.attn_dev(o, q, c, 4, 128 ** -0.5, max_q=1, max_kv=900, stream=stream)

    kq4.workspace_reserve(kq4.attn_workspace_bytes(2, 2, 4, 2, 128, 1, 900))
    kv.tensors["kv_len"].copy_(torch.tensor([880, 380], dtype=torch.int32))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(kv, out, torch.cuda.current_stream())
    for i in range(5):
        length = torch.tensor([880 + i, 380 + i], dtype=torch.int32)
        for t, w in ((k, 256), (v, 256), (q, 512)):
            t.copy_(up(torch, rng.standard_normal((2, w)).astype(F32)))
        kv.tensors["kv_len"].copy_(length)
        other.tensors["kv_len"].copy_(length)
        graph.replay()
        torch.cuda.synchronize()
        step(other, want)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        assert torch.equal(kv.tensors["codes"], other.tensors["codes"]), i
        assert torch.allclose(kv.tensors["scales"], other.tensors["scales"], rtol=0, atol=0, equal_nan=True)


def test_another_stream(kq4, torch_dev):
    torch, rng = torch_dev, np.random.default_rng(16)
    b = Batch(rng, [(1, 600), (9, 100)], 2, 64, 16, 64)
    b.fill(rng, upto="all", spread=1.0)
    x = up(torch, rand(rng, b.n, 4, 64).reshape(b.n, -1))
    kv = b.device(torch, kq4)
    outs = [torch.empty((b.n, 256), device="cuda") for _ in range(2)]
    kq4.attn_dev(outs[0], x, kv, 4, 0.125, max_q=9, max_kv=600)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        kq4.attn_dev(outs[1], x, kv, 4, 0.125, max_q=9, max_kv=600, stream=s)
    s.synchronize()
    assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("lens,tile,split,hint", [
    ([(1, 300), (1, 90)], 0, 0, 300),                # 16 rows of 4 waves, one range
    ([(1, 300), (1, 90)], 0, 0, 60000),              # of 8 waves, by a bound of the lengths
    ([(100, 200), (3, 700), (1, 64)], 0, 0, 700),    # short and long runs in one launch
    ([(70, 500), (130, 130)], 128, 1, 500), ([(70, 500), (130, 130)], 256, 1, 500),
    ([(70, 500), (130, 130)], 256, 3, 500), ([(9, 1500)], 16, 20, 1500),
    ([(1, 300)] * 70 + [(1, 90)] * 50, 0, 0, 5000),  # halves by length
    ([(1, 90)] * 70 + [(1, 300)] * 70, 0, 0, 5000),  # whole by length
    ([(1, 1900), (1, 90)], 0, 0, 1000000),           # shares of all keys
])
def test_captured_forms(kq4, torch_dev, lens, tile, split, hint):
    """Every form of the attention in a graph, replayed with other queries and lengths, each replay as the eager call
    before it; other library calls that use the workspace in between."""
    torch, rng = torch_dev, np.random.default_rng(17)
    b = Batch(rng, lens, 2, 64, 16, 64)
    b.fill(rng, upto="all", spread=1.0)
    kv, most = b.device(torch, kq4), max(q for q, _ in lens)
    q, out, want = (torch.zeros((b.n, 256), device="cuda") for _ in range(3))
    logits = torch.randn((3, 9000), device="cuda")
    ent = torch.empty(3, device="cuda")

    def attn(o, stream=None):
        kq4.attn_dev(o, q, kv, 4, 0.125, max_q=most, max_kv=hint, stream=stream)

    kq4.set_option("attn_tile", tile)
    kq4.set_option("attn_split", split)
    try:
        attn(want)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            attn(out, torch.cuda.current_stream())
        for i in range(4):
            q.copy_(up(torch, rand(rng, b.n, 4, 64).reshape(b.n, -1)))
            kv.tensors["kv_len"].copy_(torch.tensor([max(n, l - 7 * i) for n, l in lens], dtype=torch.int32))
            attn(want)
            kq4.logprobs_dev(logits, entropy=ent)
            torch.cuda.synchronize()
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), i
    finally:
        kq4.set_option("attn_tile", -1)
        kq4.set_option("attn_split", -1)


@pytest.mark.parametrize("tile", [16, 128, 256])
@pytest.mark.parametrize("dim,rope", [(64, 64), (64, 32), (128, 128), (128, 64), (128, 96), (128, 0)])
def test_attention_rotations(kq4, torch_dev, tile, dim, rope):
    """Whole and partial rotations in every form, a position off the table among the queries."""
    rng = np.random.default_rng(18)
    b = Batch(rng, [(40, 70), (1, 130)], 1, dim, 64, rope)
    b.fill(rng, upto="all", spread=1.0)
    if rope:
        b.rope_pos = rng.integers(0, 130, b.n).astype(np.int32)
        b.rope_pos[7], b.rope_pos[33] = -1, b.rope.shape[0]
    kq4.set_option("attn_tile", tile)
    try:
        got = check_attn(kq4, torch_dev, b, rand(rng, b.n, 3, dim), 3)
    finally:
        kq4.set_option("attn_tile", -1)
    assert np.isnan(got[7]).all() == np.isnan(got[33]).all() == bool(rope)


@pytest.mark.parametrize("tile,split", [(0, 0), (0, 3), (16, 3), (128, 1), (256, 20)])
def test_attention_many_sequences(kq4, torch_dev, tile, split):
    """More sequences than a wave has lanes, empty ones and a long one among them: the search for an item's and a row's
    sequence goes round."""
    rng = np.random.default_rng(19)
    lens = [(int(rng.integers(0, 4)), int(rng.integers(4, 70))) for _ in range(150)]
    lens[77], lens[131] = (30, 600), (20, 20)
    b = Batch(rng, lens, 2, 64, 16, 64, pad=3)
    b.fill(rng, upto="all", spread=1.0)
    kq4.set_option("attn_tile", tile)
    kq4.set_option("attn_split", split)
    try:
        check_attn(kq4, torch_dev, b, rand(rng, b.n, 4, 64), 4)
    finally:
        kq4.set_option("attn_tile", -1)
        kq4.set_option("attn_split", -1)


def test_large_pages(kq4, torch_dev):
    """The largest page, appended to and attended over across its border."""
    rng = np.random.default_rng(20)
    b = Batch(rng, [(40, 4110), (1, 4096)], 1, 64, 4096, 64)
    b.fill(rng, spread=1.0)
    check_append(kq4, torch_dev, b, rand(rng, b.n, 1, 64), rand(rng, b.n, 1, 64))
    check_attn(kq4, torch_dev, b, rand(rng, b.n, 2, 64), 2)


@pytest.mark.parametrize("n_seq", [65, 112, 128, 150, 256])
@pytest.mark.parametrize("heads,dim,window", [(4, 64, 0), (2, 128, 0), (4, 64, 40)])
def test_attention_sequences_by_length(kq4, torch_dev, n_seq, heads, dim, window):
    """Many sequences under a bound of the lengths that makes their order (whole or in halves) go by length: of all
    lengths, equal ones and empty ones among them, one far longer than the others."""
    rng = np.random.default_rng(n_seq)
    lens = [(int(rng.integers(0, 3)), int(rng.choice([0, 1, 60, 255, 256, 257, 300]))) for _ in range(n_seq)]
    lens[n_seq // 3] = (1, 1100)
    b = Batch(rng, lens, 2, dim, 64, 64, pad=1)
    b.fill(rng, upto="all", spread=1.0)
    check_attn(kq4, torch_dev, b, rand(rng, b.n, heads, dim), heads, window=window, max_kv=5000, max_q=2)


@pytest.mark.parametrize("lens", [[(1, 5000)], [(1, 2000), (1, 1), (0, 700), (1, 0), (2, 900)], [(1, 300)] * 60,
                                  [(1, int(n)) for n in np.linspace(1, 900, 64)], [(9, 600), (1, 1500)]])
@pytest.mark.parametrize("kv_heads,window", [(2, 0), (1, 0), (2, 333)])
def test_attention_under_loose_bounds(kq4, torch_dev, lens, kv_heads, window):
    """A bound far above the lengths: ranges by the keys that are there, also where a sequence has more rows than the
    bound says."""
    rng = np.random.default_rng(21)
    b = Batch(rng, lens, kv_heads, 64, 64, 64, pad=1)
    b.fill(rng, upto="all", spread=1.0)
    check_attn(kq4, torch_dev, b, rand(rng, b.n, 4 * kv_heads, 64), 4 * kv_heads, window=window, max_q=1, max_kv=1000000)
