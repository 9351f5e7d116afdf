"""The attention's accuracy against 64 bits, tightly enough that each half of the split operands (queries and weights as
hi + lo of f16) shows.

The measure: a row's error, root mean square over its dimensions, relative to the row's own root mean square, and the root
mean square of that over rows. An output is a sum of weights times values of random signs, about as large as the root
of the sum of their squares, and so is what independent relative errors of the weights make of it: the measure is the
weights' relative error plus that of the two sums. In units of 2^-24, at most, for up to 2000 keys of 128 dimensions and
scores up to 6:
  scores      2 D products added, each addition off by one unit of a partial sum of up to 6: sqrt(256) * 6 = 96
              q as hi + lo: 2^-22 of the score, 24 at most and of random sign over dimensions: 24 / sqrt(128) = 2
  weights     exponent rounded at up to 16 (in powers of 2): 11; exp2, the scales' logarithm and reciprocal: 8; as hi + lo: 4
  sums        2 n additions for the output, n for the row's sum, each off by half a unit of it: sqrt(6000) / 2 = 39
in quadrature 106, below the bound of 128 = 2^-17. A factor rounded to f16 alone is off by 2^-11 / sqrt(3) of its power
of two, 2^-12.3 of itself: 3300 units for the weights, and as many times the scores' spread (1.2) for the queries."""
import numpy as np
import pytest

from kv_ref import F32, Batch

BOUND = 2.0 ** -17


def measure(got, want):
    err = np.sqrt(((got - want) ** 2).mean(-1)) / np.sqrt((want ** 2).mean(-1))
    return float(np.sqrt((err ** 2).mean()))


def batch(lens, kv_heads, dim, seed):
    rng = np.random.default_rng(seed)
    b = Batch(rng, lens, kv_heads, dim, 64, dim)
    b.fill(rng, upto="all", spread=1.0)
    return b, rng.standard_normal((b.n, 4 * kv_heads, dim)).astype(F32)


SHAPES = [([(1, 1500)], 2), ([(1, 300), (1, 77), (1, 640)], 1), ([(40, 700)], 1), ([(130, 200)], 1),
          ([(50, 400), (1, 900), (3, 250)], 1)]


def in_f16_halves(b, q, lo_q, lo_p):
    """The formulas with fp32 sums and f16 operands, with or without the lower halves of queries and weights."""
    f16 = lambda a: a.astype(np.float16).astype(F32)  # noqa: E731
    heads, out = q.shape[1], np.zeros(q.shape)
    for i, (nq, kv) in enumerate(b.lens):
        for h in range(b.hkv):
            codes, scale = np.zeros((2, kv, b.dim), F32), np.zeros((2, kv), F32)
            for g0 in range(0, kv, 16):
                p, g, _ = b.place(i, g0)
                m = min(16, kv - g0)
                codes[:, g0:g0 + m] = b.group(p, h, g)[:, :, :m].transpose(0, 2, 1)
                scale[:, g0:g0 + m] = b.scales[p, h, g][:, None]
            for t in range(nq):
                tok, n = int(b.q_start[i]) + t, kv - nq + t + 1
                y = b.rotated(q[tok, 4 * h:4 * h + 4], tok, n - 1).astype(F32)
                sh = (13 - np.floor(np.log2(np.abs(y).max(1, keepdims=True)))).astype(int)
                y = np.ldexp(y, sh)
                hi = f16(y)
                s = hi @ codes[0, :n].T
                if lo_q:
                    s = s + f16(y - hi) @ codes[0, :n].T
                lv = np.log2(scale[1, :n])
                c = scale[0, :n] * np.ldexp(F32(b.dim ** -0.5 * np.log2(np.e)), -sh)
                M = (s * c + lv).max(1, keepdims=True)
                p = np.exp2((s * c + (lv - M + F32(6))).astype(F32))
                hi = f16(p)
                o = hi @ codes[1, :n]
                if lo_p:
                    o = o + f16(p - hi) @ codes[1, :n]
                out[tok, 4 * h:4 * h + 4] = o / (p / scale[1, :n]).sum(1, keepdims=True, dtype=F32)
    return out


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,kv_heads", SHAPES)
def test_the_bound_tells_the_halves(lens, kv_heads, dim):
    b, q = batch(lens, kv_heads, dim, 41)
    want = b.attention(q, q.shape[1], float(F32(dim ** -0.5)))[0]
    assert measure(in_f16_halves(b, q, True, True), want) <= BOUND
    assert measure(in_f16_halves(b, q, True, False), want) > 8 * BOUND
    assert measure(in_f16_halves(b, q, False, True), want) > 8 * BOUND


@pytest.mark.gpu
@pytest.mark.parametrize("tile,split", [(0, 0), (16, 1), (16, 3), (128, 1), (128, 3), (256, 1), (256, 2)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,kv_heads", SHAPES)
def test_attention_accuracy(kq4, torch_dev, lens, kv_heads, dim, tile, split):
    torch = torch_dev
    b, q = batch(lens, kv_heads, dim, 41)
    want = b.attention(q, q.shape[1], float(F32(dim ** -0.5)))[0]
    out = torch.empty((b.n, q.shape[1] * dim), device="cuda")
    with kq4.options(attn_tile=tile, attn_split=split):
        kq4.attn_dev(out, torch.from_numpy(q.reshape(b.n, -1)).cuda(), b.device(torch, kq4), q.shape[1], dim ** -0.5,
                     max_q=max(n for n, _ in lens), max_kv=max(n for _, n in lens))
    assert measure(out.cpu().numpy().astype(np.float64).reshape(want.shape), want) <= BOUND
