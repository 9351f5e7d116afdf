"""GPU: NaN, infinities and the ends of the scales through every form of the microscaled products (rows kernel, GEMM, K slices and
their join), the gated block and the whole block; the whole block at sizes of every kernel that hands h over quantized."""
import numpy as np
import pytest

import mx_ref as R
from test_gpu_mx import check_ffn, hull, packed, up

pytestmark = pytest.mark.gpu
F32 = np.float32
FORMS = [(1, 0), (2, 1), (2, 2), (2, 3)]


def within(got, want, tol, nan):
    np.testing.assert_array_equal(np.isnan(got), nan)
    off = (np.abs(got - want) / tol)[~nan]
    assert (off <= 1).all(), off.max()


def bad_tokens(rng, n, cols):
    """(x, the tokens that hold a NaN or an infinity): in the first block, the last one, beside a border of 512 columns."""
    x = R.acts(rng, n, cols) * F32(0.5 / np.sqrt(cols))
    bad = np.zeros(n, bool)
    for t, c, v in ((n // 2, 5, np.nan), (n - 1, cols - 1, -np.inf), (n // 3, 512, np.inf)):
        if n > 2 or t == n // 2:
            x[t, c], bad[t] = v, True
    return x, bad


@pytest.mark.parametrize("act", [4, 6])
@pytest.mark.parametrize("form,split", FORMS)
@pytest.mark.parametrize("n", [1, 20, 129, 300])
def test_nan_in_tokens_and_rows(kq4, torch_dev, n, form, split, act):
    """Products and the gated block: NaN in its token and its weight's row, nowhere else."""
    torch, rng = torch_dev, np.random.default_rng(n)
    rows, cols = 150, 1120
    w, g, u = (R.random_weights(rng, rows, cols) for _ in range(3))
    w[1][77, 20] = g[1][3, 0] = u[1][149, 34] = 255
    x, bad = bad_tokens(rng, n, cols)
    xv = R.values(*R.quantize(x, act), act)
    out, h = torch.empty(n, rows, device="cuda"), torch.empty(n, rows, device="cuda")
    with kq4.options(mx_form=form, mx_split=split):
        kq4.mx_matmul_dev(out, up(torch, x), packed(kq4, torch, *w), act=act)
        kq4.mx_gated_dev(h, up(torch, x), packed(kq4, torch, *g), packed(kq4, torch, *u), act=act)
    at = lambda *rows_: bad[:, None] | np.isin(np.arange(rows), rows_)[None]  # noqa: E731
    within(out.cpu().numpy(), *R.product(xv, R.values(*w, 4)), at(77))
    within(h.cpu().numpy(), *R.gated(xv, R.values(*g, 4), R.values(*u, 4)), at(3, 149))


@pytest.mark.parametrize("act", [4, 6])
@pytest.mark.parametrize("form,split", FORMS)
@pytest.mark.parametrize("n", [1, 40, 200])
def test_scales_at_their_ends(kq4, torch_dev, n, form, split, act):
    """Weights with scales of 2^-127 and 2^93, zero and tiny tokens. Of the gated pair one matrix at a time, so that its
    product stays in range."""
    torch, rng = torch_dev, np.random.default_rng(n)
    rows, cols = 70, 1056
    w, plain = R.random_weights(rng, rows, cols), R.random_weights(rng, rows, cols)
    w[1][::4], w[1][1::4], w[1][2::4, ::2] = 0, 220, 0
    x = R.acts(rng, n, cols)
    x[0, :544] = 0
    if n > 1:
        x[1], x[2] = 0, x[2] * F32(1e-41)
    xv = R.values(*R.quantize(x, act), act)
    wv, pv = R.values(*w, 4), R.values(*plain, 4)
    m, p, xd = packed(kq4, torch, *w), packed(kq4, torch, *plain), up(torch, x)
    new = lambda: torch.empty(n, rows, device="cuda")  # noqa: E731
    out, up_ends, gate_ends = new(), new(), new()
    with kq4.options(mx_form=form, mx_split=split):
        kq4.mx_matmul_dev(out, xd, m, act=act)
        kq4.mx_gated_dev(up_ends, xd, p, m, act=act)
        kq4.mx_gated_dev(gate_ends, xd, m, p, act=act)
    none = np.zeros((n, rows), bool)
    with np.errstate(over="ignore"):
        within(out.cpu().numpy(), *R.product(xv, wv), none)
        within(up_ends.cpu().numpy(), *R.gated(xv, pv, wv), none)
        within(gate_ends.cpu().numpy(), *R.gated(xv, wv, pv), none)


def block(rng, dim, ffn):
    return R.random_weights(rng, ffn, dim), R.random_weights(rng, ffn, dim), R.random_weights(rng, dim, ffn)


def block_of(x, g, u, d, act, res=None):
    """(the block's outputs of x, their bound): the product's of some h that gate's and up's sums allow."""
    h, tol = R.gated(R.values(*R.quantize(x, act), act), R.values(*g, 4), R.values(*u, 4))
    lo, hi = hull(h, tol, act)
    dv = R.values(*d, 4)
    want, tol = R.product((lo + hi) / 2, dv, res)
    return want, tol * 1.01 + (hi - lo) / 2 @ np.abs(dv).T


@pytest.mark.parametrize("act", [4, 6])
@pytest.mark.parametrize("form,split", FORMS)
@pytest.mark.parametrize("n", [5, 40, 150])
def test_block_with_nan(kq4, torch_dev, n, form, split, act):
    """A token's NaN or infinity makes its outputs NaN, a scale of down that output of every token. Before it the workspace
    is left full of NaN blocks by a larger call."""
    torch, rng = torch_dev, np.random.default_rng(n)
    dim, ffn = 544, 1312
    g, u, d = block(rng, dim, ffn)
    d[1][100, 40] = 255
    m = [packed(kq4, torch, *v) for v in (g, u, d)]
    x, bad = bad_tokens(rng, n, dim)
    out = torch.empty(n, dim, device="cuda")
    with kq4.options(mx_form=form, mx_split=split):
        kq4.mx_ffn_dev(torch.empty(n + 300, dim, device="cuda"), torch.full((n + 300, dim), float("nan"), device="cuda"), *m, act=act)
        kq4.mx_ffn_dev(out, up(torch, x), *m, act=act)
    nan = bad[:, None] | (np.arange(dim) == 100)[None]
    within(out.cpu().numpy(), *block_of(x, g, u, d, act), nan)


@pytest.mark.parametrize("act", [4, 6])
@pytest.mark.parametrize("n,dim,ffn,form,split", [
    (2100, 96, 2080, 2, 1),        # gated GEMM of more than a tile a CU (17 x 17), ragged in tokens, columns and scales
    (4000, 160, 1120, 2, 1), (2048, 96, 2176, 2, 1), (300, 288, 2080, 2, 1),
    (2048, 1024, 4096, 0, 0),      # the planner takes the GEMM twice
    (1500, 2048, 6144, 0, 0), (700, 4096, 12288, 0, 0)])
def test_block_is_its_parts(kq4, torch_dev, n, dim, ffn, form, split, act):
    """h leaves the gated GEMM quantized: the same bits as the gated call, the quantizer and the product one after the other;
    and tokens at the tiles' borders against 64 bits."""
    torch, rng = torch_dev, np.random.default_rng(n)
    g, u, d = block(rng, dim, ffn)
    for _, scales in (g, u, d):
        scales -= 4
    m = [packed(kq4, torch, *v) for v in (g, u, d)]
    x = R.acts(rng, n, dim) * F32(8 / np.sqrt(dim))
    xd = up(torch, x)
    res = up(torch, rng.standard_normal((n, dim)).astype(F32))
    out, h, parts = torch.empty(n, dim, device="cuda"), torch.empty(n, ffn, device="cuda"), torch.empty(n, dim, device="cuda")
    hq = kq4.MX(n, ffn, act)
    with kq4.options(mx_form=form, mx_split=split):
        kq4.mx_ffn_dev(out, xd, *m, act=act, residual=res)
        kq4.mx_gated_dev(h, xd, *m[:2], act=act)
        kq4.mx_quantize_dev(hq, h)
        kq4.mx_matmul_q_dev(parts, hq, m[2], residual=res)
    assert torch.isfinite(out).all() and torch.equal(out, parts)
    tokens = np.unique(np.clip([0, 1, 31, 32, 63, 64, 127, 128, 129, n // 2, n - 129, n - 33, n - 2, n - 1], 0, n - 1))[:8 if dim > 1000 else None]
    at = torch.from_numpy(tokens).cuda()
    want, tol = block_of(x[tokens], g, u, d, act, res[at].cpu().numpy())
    off = np.abs(out[at].cpu().numpy() - want) / tol
    assert (off <= 1).all(), off.max()


@pytest.mark.parametrize("act", [4, 6])
def test_block_in_every_form(kq4, torch_dev, act):
    """Sizes past one group of rows and one scale tile each way, in every form."""
    for form, split in FORMS:
        with kq4.options(mx_form=form, mx_split=split):
            check_ffn(kq4, torch_dev, 150, 1184, 1312, act)
