"""GPU: microscaled matrices. Quantisation and packing equal the plain form (mx_ref.py) byte for byte; products and the
gated block lie within the bounds of fp32 sums of their definition in 64 bits; odd sizes, strides, NaN, streams, graphs."""
import numpy as np
import pytest

import mx_ref as R

pytestmark = pytest.mark.gpu
F32 = np.float32


def up(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def packed(kq4, torch, codes, scales, bits=4):
    m = kq4.MX(codes.shape[0], codes.shape[1], bits)
    kq4.mx_pack_dev(m, up(torch, R.row_major(codes, bits)), up(torch, scales))
    return m


def strided(torch, a, pad, fill=np.nan):
    """A device tensor of a's values whose rows lie `pad` floats further apart, and the tensor around it."""
    wide = np.full((a.shape[0], a.shape[1] + pad), fill, F32)
    wide[:, :a.shape[1]] = a
    t = up(torch, wide)
    return t[:, :a.shape[1]], t


# ---- quantisation and packing ----------------------------------------------------------------------

def edges(bits, cols):
    """Blocks at every border: ties, the scale's steps, subnormals, zeros of both signs, NaN and infinities."""
    el = R.elements(bits)
    mid = (el[1:] + el[:-1]) / 2
    both = np.concatenate([mid, np.nextafter(mid.astype(F32), F32(np.inf)), np.nextafter(mid.astype(F32), F32(0)), el]).astype(F32)
    rows = []
    for e in (-149, -140, -127, -120, -3, 0, 5, 118):
        for i in range(0, both.size, 31):
            part = both[i:i + 31] * (-1.0) ** np.arange(both[i:i + 31].size)
            row = np.zeros(32)
            row[:part.size] = part
            row[31] = el[-1]
            rows.append(row * 2.0 ** e)
    top = el[-1]
    for v in (top, 6.99, 7.0, 7.01, 7.4, 7.74, 7.75, 7.76, 7.99, 3.4028235e38, 1e-45, 1e-38):
        rows.append(np.where(np.arange(32) == 9, v, v * 0.3))
    rows += [np.zeros(32), -np.zeros(32), np.full(32, -0.0)]
    for bad in (np.nan, np.inf, -np.inf):
        row = np.arange(32.0)
        row[17] = bad
        rows.append(row)
    with np.errstate(over="ignore"):
        x = np.array(rows).astype(F32)
    x[(np.abs(x) == np.inf) & (np.arange(len(x)) < len(x) - 3)[:, None]] = F32(3.4028235e38)
    reps = -(-x.size // cols)
    return np.resize(x, (reps, cols))


@pytest.mark.parametrize("bits", [4, 6])
@pytest.mark.parametrize("cols", [32, 128, 544])
def test_quantize_at_every_border(kq4, torch_dev, bits, cols):
    x = edges(bits, cols)
    m = kq4.MX(x.shape[0], cols, bits)
    kq4.mx_quantize_dev(m, up(torch_dev, x))
    np.testing.assert_array_equal(m.data.cpu().numpy(), R.matrix(*R.quantize(x, bits), bits))


@pytest.mark.parametrize("bits", [4, 6])
@pytest.mark.parametrize("rows,cols,pad", [(1, 32, 0), (1, 4096, 4), (15, 96, 100), (17, 512, 0), (129, 1056, 12), (300, 640, 0)])
def test_quantize(kq4, torch_dev, rows, cols, pad, bits):
    rng = np.random.default_rng(rows)
    x = R.acts(rng, rows, cols)
    want = R.matrix(*R.quantize(x, bits), bits)
    data = torch_dev.full((want.size + 64,), 0xA5, dtype=torch_dev.uint8, device="cuda")
    m = kq4.MX(rows, cols, bits, data=data)
    kq4.mx_quantize_dev(m, strided(torch_dev, x, pad)[0])
    got = data.cpu().numpy()
    np.testing.assert_array_equal(got[:want.size], want)
    assert (got[want.size:] == 0xA5).all()


@pytest.mark.parametrize("bits", [4, 6])
@pytest.mark.parametrize("rows,cols", [(1, 32), (16, 128), (130, 672), (257, 1536), (5, 2048)])
def test_pack_and_unpack(kq4, torch_dev, rows, cols, bits):
    torch, rng = torch_dev, np.random.default_rng(rows)
    codes = rng.integers(0, 1 << bits, (rows, cols), np.uint8)
    scales = rng.integers(0, 256, (rows, cols // 32)).astype(np.uint8)
    m = packed(kq4, torch, codes, scales, bits)
    np.testing.assert_array_equal(m.data.cpu().numpy(), R.matrix(codes, scales, bits))
    c = torch.full((rows * cols * bits // 8 + 16,), 7, dtype=torch.uint8, device="cuda")
    s = torch.full((rows * cols // 32 + 16,), 7, dtype=torch.uint8, device="cuda")
    kq4.mx_unpack_dev(c, s, m)
    np.testing.assert_array_equal(c.cpu().numpy(), np.append(R.row_major(codes, bits), np.full(16, 7)))
    np.testing.assert_array_equal(s.cpu().numpy(), np.append(scales, np.full(16, 7)))


def test_stacked_matrices(kq4, torch_dev):
    """Whole groups of 128 rows packed as one matrix are their matrices one after the other, part by part."""
    rng = np.random.default_rng(1)
    (c1, s1), (c2, s2) = R.random_weights(rng, 128, 544), R.random_weights(rng, 70, 544)
    m = packed(kq4, torch_dev, np.concatenate([c1, c2]), np.concatenate([s1, s2]))
    np.testing.assert_array_equal(m.data.cpu().numpy(), R.matrix(np.concatenate([c1, c2]), np.concatenate([s1, s2]), 4))


# ---- products ----------------------------------------------------------------------------------------

def check_matmul(kq4, torch, rng, n, rows, cols, act, res, pad_x=0, pad_out=0, quantized=False, stream=None):
    codes, scales = R.random_weights(rng, rows, cols)
    x = R.acts(rng, n, cols)
    w = packed(kq4, torch, codes, scales)
    xv = R.values(*R.quantize(x, act), act)
    r = rng.standard_normal((n, rows)).astype(F32) if res else None
    want, tol = R.product(xv, R.values(codes, scales, 4), r)
    out, wide = strided(torch, r if res == "in place" else np.full((n, rows), np.nan, F32), pad_out, 7.0)
    rt = out if res == "in place" else strided(torch, r, pad_out)[0] if res else None
    if quantized:
        xq = kq4.MX(n, cols, act)
        kq4.mx_quantize_dev(xq, strided(torch, x, pad_x)[0])
        kq4.mx_matmul_q_dev(out, xq, w, residual=rt)
    else:
        kq4.mx_matmul_dev(out, strided(torch, x, pad_x)[0], w, act=act, residual=rt)
    got = wide.cpu().numpy()
    assert (np.abs(got[:, :rows] - want) <= tol).all(), (np.abs(got[:, :rows] - want) / tol).max()
    assert (got[:, rows:] == 7.0).all()


@pytest.mark.parametrize("act", [4, 6])
@pytest.mark.parametrize("n", [1, 2, 3, 15, 16, 17, 33, 64, 65, 129, 300])
@pytest.mark.parametrize("rows,cols", [(1, 32), (16, 128), (33, 544), (130, 1056)])
def test_matmul(kq4, torch_dev, n, rows, cols, act):
    check_matmul(kq4, torch_dev, np.random.default_rng(n * rows), n, rows, cols, act, n % 2)


@pytest.mark.parametrize("act", [4, 6])
@pytest.mark.parametrize("n,rows,cols", [(1, 4099, 512), (7, 2000, 2016), (40, 1030, 4096), (260, 515, 1120), (515, 300, 512),
                                         (1, 64, 12288), (100, 257, 6176)])
@pytest.mark.parametrize("quantized", [False, True])
def test_matmul_of_odd_sizes_and_strides(kq4, torch_dev, n, rows, cols, act, quantized):
    check_matmul(kq4, torch_dev, np.random.default_rng(n), n, rows, cols, act, "in place" if n % 2 else True, pad_x=4 * (n % 5),
                 pad_out=n % 3, quantized=quantized)


@pytest.mark.parametrize("act", [4, 6])
@pytest.mark.parametrize("n,rows,cols", [(1, 130, 544), (16, 300, 2080), (33, 515, 1120), (129, 257, 4096), (300, 600, 1536), (1100, 2100, 544), (2500, 2300, 160), (2700, 2300, 160), (2700, 5000, 96)])
@pytest.mark.parametrize("form,split", [(1, 0), (2, 1), (2, 2), (2, 3), (2, 50)])
def test_every_form(kq4, torch_dev, n, rows, cols, act, form, split):
    """The rows kernel and the GEMM, whole and with K in slices, at sizes of either, with and without a residual."""
    with kq4.options(mx_form=form, mx_split=split):
        check_matmul(kq4, torch_dev, np.random.default_rng(n), n, rows, cols, act, split % 2, pad_x=4, pad_out=1)
        check_gated(kq4, torch_dev, np.random.default_rng(n), n, rows, cols, act)


@pytest.mark.parametrize("act", [4, 6])
@pytest.mark.parametrize("n,rows,cols", [(3, 6500, 2080), (2, 9001, 1120), (5, 17000, 1056), (17, 2100, 1120), (64, 3100, 544),
                                         (64, 4100, 1056), (64, 8200, 544), (100, 4000, 4128), (16, 16500, 1120), (30, 8000, 544), (1500, 260, 4384), (3007, 33, 2848)])
def test_every_tile_of_the_rows_kernel(kq4, torch_dev, n, rows, cols, act):
    """Launches past a tile a CU (256 CUs): activations quantized in workgroups of 8 waves with 4, 2 and 1 of them on a
    tile; tiles of 16 x 16 to 32 x 64, from quantized activations too; activations past an XCD's cache."""
    with kq4.options(mx_form=1):
        check_matmul(kq4, torch_dev, np.random.default_rng(n), n, rows, cols, act, n % 2, pad_x=4, pad_out=1)
        check_matmul(kq4, torch_dev, np.random.default_rng(n), n, rows, cols, act, True, pad_out=2, quantized=True)
        check_gated(kq4, torch_dev, np.random.default_rng(n), n, rows, cols, act)


def test_outputs_past_the_caches(kq4, torch_dev):
    """Outputs of more than 80 MiB, ragged at both edges."""
    rng = np.random.default_rng(4)
    for res in (None, True, "in place"):
        check_matmul(kq4, torch_dev, rng, 1301, 16500, 96, 4 if res else 6, res, pad_out=3)
    check_gated(kq4, torch_dev, rng, 1301, 16500, 64, 6)


@pytest.mark.parametrize("n", [1, 20, 200])
@pytest.mark.parametrize("act", [4, 6])
def test_nan_stays_in_its_token_and_row(kq4, torch_dev, n, act):
    """A NaN or infinity in a token's row, a NaN scale in a weight's row: those outputs are NaN, no other is."""
    torch, rng = torch_dev, np.random.default_rng(n)
    rows, cols = 150, 672
    codes, scales = R.random_weights(rng, rows, cols)
    scales[77, 20] = 255
    x = R.acts(rng, n, cols)
    x[n // 2, 5] = np.nan
    if n > 1:
        x[n - 1, cols - 1] = -np.inf
    xv = R.values(*R.quantize(x, act), act)
    want, tol = R.product(xv, R.values(codes, scales, 4))
    out = torch.empty(n, rows, device="cuda")
    kq4.mx_matmul_dev(out, up(torch, x), packed(kq4, torch, codes, scales), act=act)
    got = out.cpu().numpy()
    nan = np.zeros((n, rows), bool)
    nan[:, 77] = nan[n // 2] = True
    if n > 1:
        nan[n - 1] = True
    np.testing.assert_array_equal(np.isnan(got), nan)
    assert (np.abs(got - want) <= tol)[~nan].all()


@pytest.mark.parametrize("n", [1, 40, 300])
def test_scales_at_their_ends(kq4, torch_dev, n):
    """Scales of 2^-127 and 2^100 in the weights, zeros and tiny rows in the activations."""
    torch, rng = torch_dev, np.random.default_rng(5)
    rows, cols = 64, 512
    codes, scales = R.random_weights(rng, rows, cols)
    scales[::4], scales[1::4], scales[2::4, ::2] = 0, 220, 0
    x = R.acts(rng, n, cols)
    x[0, :256] = 0
    if n > 1:
        x[1], x[2] = 0, x[2] * F32(1e-41)
    xv = R.values(*R.quantize(x, 6), 6)
    want, tol = R.product(xv, R.values(codes, scales, 4))
    out = torch.empty(n, rows, device="cuda")
    kq4.mx_matmul_dev(out, up(torch, x), packed(kq4, torch, codes, scales))
    assert (np.abs(out.cpu().numpy() - want) <= tol).all()


def check_gated(kq4, torch, rng, n, rows, cols, act):
    g, u = R.random_weights(rng, rows, cols), R.random_weights(rng, rows, cols)
    x = R.acts(rng, n, cols) * F32(0.5 / np.sqrt(cols))
    want, tol = R.gated(R.values(*R.quantize(x, act), act), R.values(*g, 4), R.values(*u, 4))
    out, wide = strided(torch, np.full((n, rows), np.nan, F32), 3, 7.0)
    kq4.mx_gated_dev(out, strided(torch, x, 8)[0], packed(kq4, torch, *g), packed(kq4, torch, *u), act=act)
    got = wide.cpu().numpy()
    assert (np.abs(got[:, :rows] - want) <= tol).all(), (np.abs(got[:, :rows] - want) / tol).max()
    assert (got[:, rows:] == 7.0).all()


@pytest.mark.parametrize("act", [4, 6])
@pytest.mark.parametrize("n,rows,cols", [(1, 16, 32), (1, 333, 1024), (3, 100, 544), (16, 64, 512), (29, 260, 2048), (66, 129, 96),
                                         (130, 520, 640), (300, 288, 1056)])
def test_gated(kq4, torch_dev, n, rows, cols, act):
    check_gated(kq4, torch_dev, np.random.default_rng(rows), n, rows, cols, act)


def test_gate_far_from_zero(kq4, torch_dev):
    """Gates of -1e4 .. 1e4: exp overflows, the quotient does not."""
    torch, rng = torch_dev, np.random.default_rng(3)
    g, u = R.random_weights(rng, 64, 512), R.random_weights(rng, 64, 512)
    x = R.acts(rng, 9, 512) * F32(100)
    with np.errstate(over="ignore"):
        want, tol = R.gated(R.values(*R.quantize(x, 6), 6), R.values(*g, 4), R.values(*u, 4))
    out = torch.empty(9, 64, device="cuda")
    kq4.mx_gated_dev(out, up(torch, x), packed(kq4, torch, *g), packed(kq4, torch, *u))
    got = out.cpu().numpy()
    assert np.isfinite(got).all() and (np.abs(got - want) <= tol).all()


def hull(h, tol, bits):
    """Least and largest value that each element of h +- tol may be quantized to: the block's scale lies between those of its
    largest magnitude less and plus its bound."""
    lo, hi = h - tol, h + tol
    a = np.abs(h)
    n = h.shape[0]
    b = [R.quantize(np.nextafter(v.astype(F32), F32(s)), bits)[1] for v, s in ((np.maximum(a - tol, 0), 0), (a + tol, np.inf))]
    el = R.elements(bits)
    grid = np.concatenate([-el[::-1], el])
    out = []
    for sc in b:
        s = np.repeat(R.scale_values(sc), 32, 1)
        for v, side in ((lo, -1), (hi, 1)):
            y = np.clip(v / s, -el[-1], el[-1])
            i = np.abs(y[..., None] - grid).argmin(-1)
            q = grid[i] * s
            near = np.abs(np.abs(y[..., None] - grid) - np.abs(y - grid[i])[..., None]) <= 1e-6 * np.abs(y)[..., None]
            pick = np.where(near, grid, -np.inf if side > 0 else np.inf)
            q = (pick.max(-1) if side > 0 else pick.min(-1)) * s
            out.append(q)
    return np.minimum.reduce(out).reshape(n, -1), np.maximum.reduce(out).reshape(n, -1)


@pytest.mark.parametrize("act", [4, 6])
@pytest.mark.parametrize("n,dim,ffn", [(1, 96, 160), (1, 512, 1056), (5, 128, 544), (40, 256, 640), (140, 192, 288)])
@pytest.mark.parametrize("form,split", [(0, 0), (1, 0), (2, 1), (2, 2)])
def test_ffn(kq4, torch_dev, n, dim, ffn, act, form, split):
    """The block as one call: within the product's bound of some h that the fp32 sums of gate and up allow. The GEMM in one
    slice hands h over quantized."""
    with kq4.options(mx_form=form, mx_split=split):
        check_ffn(kq4, torch_dev, n, dim, ffn, act)


def check_ffn(kq4, torch_dev, n, dim, ffn, act):
    torch, rng = torch_dev, np.random.default_rng(n + ffn)
    g, u, d = R.random_weights(rng, ffn, dim), R.random_weights(rng, ffn, dim), R.random_weights(rng, dim, ffn)
    x = R.acts(rng, n, dim) * F32(0.5 / np.sqrt(dim))
    res = rng.standard_normal((n, dim)).astype(F32)
    h, tol = R.gated(R.values(*R.quantize(x, act), act), R.values(*g, 4), R.values(*u, 4))
    lo, hi = hull(h, tol, act)
    dv = R.values(*d, 4)
    mid, half = (lo + hi) / 2, (hi - lo) / 2
    want, tol = R.product(mid, dv, res)
    tol = tol * 1.01 + half @ np.abs(dv).T
    out = torch.empty(n, dim, device="cuda")
    kq4.mx_ffn_dev(out, up(torch, x), packed(kq4, torch, *g), packed(kq4, torch, *u), packed(kq4, torch, *d), act=act,
                   residual=up(torch, res))
    got = out.cpu().numpy()
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()
    assert half.max() <= 0 or (half > 0).mean() < 0.02       # the hull is a point nearly everywhere


# ---- how the calls are made ------------------------------------------------------------------------------

def step(kq4, torch, n, act, seed=0):
    """A step's calls over fresh tensors: (run(stream), outputs)."""
    rng = np.random.default_rng(seed + n)
    dim, ffn = 544, 1056
    w = {k: packed(kq4, torch, *R.random_weights(rng, r, c)) for k, (r, c) in
         dict(q=(300, dim), kv=(77, dim), o=(dim, 320), g=(ffn, dim), u=(ffn, dim), d=(dim, ffn)).items()}
    x, att = up(torch, R.acts(rng, n, dim)), up(torch, R.acts(rng, n, 320))
    new = lambda c: torch.empty(n, c, device="cuda")  # noqa: E731
    o = dict(q=new(300), kv=new(77), h=new(dim), gu=new(ffn), y=new(dim), xq=kq4.MX(n, dim, act))

    def run(stream=None):
        kq4.mx_quantize_dev(o["xq"], x, stream=stream)
        kq4.mx_matmul_q_dev(o["q"], o["xq"], w["q"], stream=stream)
        kq4.mx_matmul_q_dev(o["kv"], o["xq"], w["kv"], stream=stream)
        kq4.mx_matmul_dev(o["h"], att, w["o"], act=act, residual=x, stream=stream)
        kq4.mx_gated_dev(o["gu"], o["h"], w["g"], w["u"], act=act, stream=stream)
        kq4.mx_ffn_dev(o["y"], o["h"], w["g"], w["u"], w["d"], act=act, residual=o["h"], stream=stream)
    return run, [o[k] for k in ("q", "kv", "h", "gu", "y")], o["xq"].data


@pytest.mark.parametrize("n", [1, 12, 40, 300])
@pytest.mark.parametrize("act", [4, 6])
def test_graph_and_stream_and_repeats(kq4, torch_dev, n, act):
    """Captured and replayed between eager calls, on another stream, and again: the same bits."""
    torch = torch_dev
    run, outs, xq = step(kq4, torch, n, act)
    other, _, _ = step(kq4, torch, 2 * n, act, 1)
    run()
    torch.cuda.synchronize()
    want = [t.clone() for t in outs + [xq]]
    assert all(torch.isfinite(t).all() for t in want[:-1])

    def fresh(f):
        for t in outs:
            t.fill_(float("nan"))
        xq.fill_(1)
        torch.cuda.synchronize()
        f()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs + [xq], want))

    fresh(run)
    s = torch.cuda.Stream()
    fresh(lambda: run(s))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(torch.cuda.current_stream())
    for _ in range(4):
        fresh(graph.replay)
        other()


def test_two_graphs_share_the_workspace(kq4, torch_dev):
    """Steps of two sizes captured one after the other and replayed in turn, outputs cleared between."""
    torch = torch_dev
    steps = [step(kq4, torch, n, 6, seed) for seed, n in enumerate((300, 21))]
    for run, _, _ in steps:
        run()
    torch.cuda.synchronize()
    want = [[t.clone() for t in outs + [xq]] for _, outs, xq in steps]
    graphs = []
    for run, _, _ in steps:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            run(torch.cuda.current_stream())
    for _ in range(3):
        for t in [t for _, outs, _ in steps for t in outs]:
            t.fill_(float("nan"))
        for g in graphs + graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        for (_, outs, xq), w in zip(steps, want):
            assert all(torch.equal(a, b) for a, b in zip(outs + [xq], w))


@pytest.mark.parametrize("n", [1, 9, 40, 300])
@pytest.mark.parametrize("form", [1, 2])
def test_rows_behind_the_batch_stay(kq4, torch_dev, n, form):
    """Outputs and residuals of more rows than x: those behind are not written; x of more rows than
    a matrix."""
    torch, rng = torch_dev, np.random.default_rng(n)
    rows, cols = 260, 544
    w = [packed(kq4, torch, *R.random_weights(rng, r, c)) for r, c in ((rows, cols), (rows, cols), (cols, 288), (288, cols), (288, cols))]
    x = up(torch, R.acts(rng, n + 2, cols))
    small = [torch.empty(n, c, device="cuda") for c in (rows, rows, rows, cols)]
    large = [torch.full((n + 5, c), 7.0, device="cuda") for c in (rows, rows, rows, cols)]
    res = up(torch, rng.standard_normal((n + 1, rows)).astype(F32))
    with kq4.options(mx_form=form):
        for o in (small, large):
            xq = kq4.MX(n, cols, 6)
            kq4.mx_quantize_dev(xq, x)
            kq4.mx_matmul_dev(o[0], x[:n], w[0], residual=res)
            kq4.mx_matmul_q_dev(o[1], xq, w[0])
            kq4.mx_gated_dev(o[2], x[:n], w[0], w[1])
            kq4.mx_ffn_dev(o[3], x[:n], w[3], w[4], w[2])
    for a, b in zip(small, large):
        assert torch.equal(a, b[:n]) and (b[n:] == 7.0).all()


@pytest.mark.slow
def test_matrix_past_32_bits(kq4, torch_dev):
    """A matrix of more than 4 GiB: rows at both ends and across the borders of 2^31 and 2^32 bytes."""
    torch, rng = torch_dev, np.random.default_rng(9)
    rows, cols = 540000, 16384
    codes = torch.randint(0, 256, (rows, cols // 2), dtype=torch.uint8, device="cuda")
    scales = torch.randint(118, 123, (rows, cols // 32), dtype=torch.uint8, device="cuda")
    w = kq4.MX(rows, cols, 4)
    kq4.mx_pack_dev(w, codes, scales)
    pick = np.unique(np.concatenate([[0, 1, rows - 1, rows - 17], [(1 << s) // (cols // 2) + d for s in (31, 32) for d in (-129, -1, 0, 1, 130)],
                                     rng.integers(0, rows, 40)]))
    at = torch.from_numpy(pick).cuda()
    c = codes[at].cpu().numpy()
    full = np.stack([c & 15, c >> 4], 2).reshape(len(pick), cols)
    wv = R.values(full, scales[at].cpu().numpy(), 4)
    for n, act in ((1, 6), (20, 4), (150, 6)):
        x = R.acts(rng, n, cols)
        want, tol = R.product(R.values(*R.quantize(x, act), act), wv)
        out = torch.empty(n, rows, device="cuda")
        kq4.mx_matmul_dev(out, up(torch, x), w, act=act)
        assert (np.abs(out[:, at].cpu().numpy() - want) <= tol).all()
