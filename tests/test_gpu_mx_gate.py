"""GPU: silu(g) * u of the gated block by itself. The weights are such that g and u are exact sums: ones in the
activations, and 24 bits of g in twelve blocks of its row, two bits each; so what is off is the gate's own rounding."""
import numpy as np
import pytest

import mx_ref as R
from test_gpu_mx import packed, up

pytestmark = pytest.mark.gpu
F32 = np.float32
COLS, BLOCKS = 1056, [0, 1, 2, 9, 10, 13, 16, 17, 20, 25, 30, 32]     # three pieces of 512 columns
DIGIT = np.array([0, 2, 4, 5], np.uint8)                              # the codes of 0, 1, 2, 3


def rows_of(g):
    """(codes, scales) whose rows add up to fp32 g over ones at the blocks' first columns."""
    m, e = np.frexp(np.abs(g).astype(np.float64))
    m, e = (m * 2.0 ** 24).astype(np.int64), e - 24
    codes, scales = np.zeros((len(g), COLS), np.uint8), np.full((len(g), COLS // 32), 127, np.uint8)
    for i, b in enumerate(BLOCKS):
        codes[:, 32 * b] = DIGIT[(m >> (2 * i)) & 3] + 8 * (g < 0)
        scales[:, b] = np.where(g == 0, 127, e + 2 * i + 127)
    return codes, scales


def ones(n):
    x = np.zeros((n, COLS), F32)
    x[:, [32 * b for b in BLOCKS]] = 1
    return x


def unit(rows, power):
    """(codes, scales) of rows that add up to 2^power."""
    codes, scales = np.zeros((rows, COLS), np.uint8), np.full((rows, COLS // 32), 127, np.uint8)
    codes[:, 0], scales[:, 0] = 2, 127 + power
    return codes, scales


def gates(kq4, torch, g, power, n, act):
    """(the rows' sums, the gated outputs) of g and u = 2^power, one token's: every token of n has the same."""
    w, x = rows_of(g), up(torch, ones(n))
    gate, u = packed(kq4, torch, *w), packed(kq4, torch, *unit(len(g), power))
    sums, out = torch.empty(n, len(g), device="cuda"), torch.empty(n, len(g), device="cuda")
    kq4.mx_matmul_dev(sums, x, gate, act=act)
    kq4.mx_gated_dev(out, x, gate, u, act=act)
    assert torch.equal(sums, sums[:1].expand(n, -1)) and torch.equal(out.view(torch.int32), out[:1].view(torch.int32).expand(n, -1))
    return sums[0].cpu().numpy(), out[0].cpu().numpy()


FORMS = [(0, 0, 1), (1, 0, 20), (2, 1, 3), (2, 2, 130), (2, 1, 2300)]     # mx_form, mx_split, tokens


# Every rounding is 2^-24 of its result. e^-g: 2 for the hardware's exp2 (1 ulp), 1 for the factor that corrects its argument, 1
# for the product with it; they count by e^-g / (1 + e^-g) of the result, which is below 1. Then the sum 1 + e^-g and
# the quotient; the product with u = 2^power is exact. Below -64, where 1 + e^-g is e^-g, the two factors g e^(g/2) e^(g/2)
# count 4 each, and two products. 0.02 for what is of second order. 2^-149: a result that is subnormal before it is
# multiplied by u.
def bound(g, want, power):
    w = 1 / (1 + np.exp(np.minimum(g, 700)))
    k = np.where(g < -64, 8 + 2, 4 * w + 2) + 0.02
    return k * 2.0 ** -24 * np.abs(want) + 2.0 ** (power - 149)


@pytest.mark.parametrize("act", [4, 6])
@pytest.mark.parametrize("form,split,n", FORMS)
@pytest.mark.parametrize("lo,hi,power", [(4, 17, 0), (0, 4, 0), (-17, 0, 0), (17, 88, 0), (-64, -17, 20), (-87, -64, 60), (-104, -87, 120)])
def test_gate_is_off_by_its_roundings(kq4, torch_dev, lo, hi, power, form, split, n, act):
    rng = np.random.default_rng(hi - lo)
    g = rng.uniform(lo, hi, 2000 if n > 1000 else 6000).astype(F32)
    with kq4.options(mx_form=form, mx_split=split):
        sums, got = gates(kq4, torch_dev, g, power, n, act)
    np.testing.assert_array_equal(sums, g)
    g = g.astype(np.float64)
    want = g / (1 + np.exp(-g)) * 2.0 ** power
    off = np.abs(got - want) / bound(g, want, power)
    assert (off <= 1).all(), (off.max(), g[off.argmax()], got[off.argmax()], want[off.argmax()])


@pytest.mark.parametrize("form,split,n", FORMS)
def test_gate_at_the_ends(kq4, torch_dev, form, split, n):
    """Zeros, the least and the largest gates."""
    g = np.array([0, 1e-30, -1e-30, 88.72284, -88.72284, -88.73, -87.3365, -87.34, -64, -64.00001, -63.99999, 110, -110,
                  1e4, -1e4, 1e30, -1e30, 3e38, -3e38], F32)
    with kq4.options(mx_form=form, mx_split=split):
        sums, got = gates(kq4, torch_dev, g, 0, n, 6)
    np.testing.assert_array_equal(sums, g)
    g = g.astype(np.float64)
    with np.errstate(over="ignore"):
        want = g / (1 + np.exp(-g))
    assert (np.abs(got - want) <= bound(g, want, 0)).all(), (got, want)


@pytest.mark.parametrize("form,split,n", FORMS)
def test_gate_of_infinite_sums(kq4, torch_dev, form, split, n):
    """Sums past fp32's range: silu(inf) is inf, silu(-inf) the quotient's NaN, and u = 1 leaves them."""
    codes, scales = np.zeros((2, COLS), np.uint8), np.full((2, COLS // 32), 127, np.uint8)
    codes[:, 32], scales[:, 1] = [7, 15], 254                 # +-6 * 2^127
    x = up(torch_dev, ones(n))
    gate, u = packed(kq4, torch_dev, codes, scales), packed(kq4, torch_dev, *unit(2, 0))
    out = torch_dev.empty(n, 2, device="cuda")
    with kq4.options(mx_form=form, mx_split=split):
        kq4.mx_gated_dev(out, x, gate, u)
    got = out.cpu().numpy()
    assert (got[:, 0] == np.inf).all() and np.isnan(got[:, 1]).all()


@pytest.mark.parametrize("form,split,n", FORMS)
def test_gate_is_the_same_beside_far_ones(kq4, torch_dev, form, split, n):
    """A gate's bits do not go with its neighbours': the same gates with every seventh or none of them past 64."""
    g = np.random.default_rng(n).uniform(-64, 64, 2100).astype(F32)
    mixed = g.copy()
    mixed[::7] = np.where(np.arange(300) % 2, 3e5, -70)
    with kq4.options(mx_form=form, mx_split=split):
        alone, beside = gates(kq4, torch_dev, g, 0, n, 6)[1], gates(kq4, torch_dev, mixed, 0, n, 6)[1]
    kept = np.arange(2100) % 7 != 0
    np.testing.assert_array_equal(alone.view(np.int32)[kept], beside.view(np.int32)[kept])
