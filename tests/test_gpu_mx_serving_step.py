"""GPU: a decoder layer over microscaled weights as an engine runs it - norm, its rows quantized once for Q, K and V, append,
attention, O projection with its residual, norm, the feed-forward block with its residual, lm_head, log probabilities - over
a prompt of two sequences and then single tokens of both. Every stage is checked against its plain form on the outputs
that the stage before it left on the GPU."""
import numpy as np
import pytest

import mx_ref as R
from conftest import rel_err
from kv_ref import F32, Batch, logprobs
from test_gpu_mx import hull, packed, up

pytestmark = pytest.mark.gpu

HID, HEADS, KV, DIM, FFN, VOCAB, EPS = 256, 4, 2, 64, 544, 1000, 1e-6


def within(got, want_tol):
    want, tol = want_tol
    assert got.shape == want.shape and (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()


@pytest.mark.parametrize("act", [4, 6])
@pytest.mark.parametrize("lens", [(37, 20), (290, 41)])
def test_prompt_and_decode_steps(kq4, torch_dev, orc, act, lens):
    torch, rng = torch_dev, np.random.default_rng(act + lens[0])
    mats = dict(q=(HEADS * DIM, HID), k=(KV * DIM, HID), v=(KV * DIM, HID), o=(HID, HEADS * DIM), gate=(FFN, HID),
                up=(FFN, HID), down=(HID, FFN), lm=(VOCAB, HID))
    raw = {n: R.random_weights(rng, *s) for n, s in mats.items()}
    for c, s in raw.values():
        s -= 3                                                   # sums near one
    w = {n: packed(kq4, torch, *raw[n]) for n in mats}
    wv = {n: R.values(*raw[n], 4) for n in mats}
    norm = (1 + 0.1 * rng.standard_normal(HID)).astype(F32)
    quantized = lambda a: R.values(*R.quantize(a, act), act)  # noqa: E731

    b = Batch(rng, [(n, n) for n in lens], KV, DIM, 16, DIM, extra_pages=1)
    b.table[:] = rng.permutation(b.table.size).reshape(b.table.shape)      # room to grow
    b.codes = rng.integers(0, 256, (b.table.size,) + b.codes.shape[1:], np.uint8)
    b.scales = np.full((b.table.size,) + b.scales.shape[1:], np.nan, F32)
    b.rope = kq4.rope_table(320, DIM, 1e4, device="cpu").numpy()
    codes, scales, table = up(torch, b.codes), up(torch, b.scales), up(torch, b.table)
    for step in range(3):
        if step:
            b.lens = [(1, kv + 1) for _, kv in b.lens]
        n = b.n = sum(q for q, _ in b.lens)
        b.q_start = np.concatenate([[0], np.cumsum([q for q, _ in b.lens])]).astype(np.int32)
        b.kv_len = np.array([kv for _, kv in b.lens], np.int32)
        kv = kq4.KVBatch(codes, scales, 16, table, up(torch, b.q_start), up(torch, b.kv_len), n, rope=up(torch, b.rope))
        x = rng.standard_normal((n, HID)).astype(F32)
        new = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
        # Q, K and V side by side in one tensor: rows of its stride
        qkv = new(n, (HEADS + 2 * KV) * DIM)
        q, k, v = (qkv[:, a * DIM:b_ * DIM] for a, b_ in ((0, HEADS), (HEADS, HEADS + KV), (HEADS + KV, HEADS + 2 * KV)))
        xd, nx, nh, att, h, y, lg = up(torch, x), new(n, HID), new(n, HID), new(n, HEADS * DIM), new(n, HID), new(n, HID), new(n, VOCAB)
        token = rng.integers(0, VOCAB, n)
        lp, ent, tlp, tid = new(n), new(n), new(n, 5), torch.empty((n, 5), dtype=torch.int32, device="cuda")
        xq = kq4.MX(n, HID, act)
        kq4.rms_norm_dev(nx, xd, up(torch, norm), EPS)
        kq4.mx_quantize_dev(xq, nx)
        for o, name in ((q, "q"), (k, "k"), (v, "v")):
            kq4.mx_matmul_q_dev(o, xq, w[name])
        kq4.kv_append_dev(kv, k, v)
        kq4.attn_dev(att, q, kv, HEADS, DIM ** -0.5, max_q=int(max(q_ for q_, _ in b.lens)), max_kv=int(b.kv_len.max()))
        kq4.mx_matmul_dev(h, att, w["o"], act=act, residual=xd)
        kq4.rms_norm_dev(nh, h, up(torch, norm), EPS)
        kq4.mx_ffn_dev(y, nh, w["gate"], w["up"], w["down"], act=act, residual=h)
        kq4.mx_matmul_dev(lg, y, w["lm"], act=act)
        kq4.logprobs_dev(lg, up(torch, token.astype(np.int32)), lp, ent, tlp, tid)
        torch.cuda.synchronize()
        nx, q, k, v, att, h, nh, y, lg = (t.cpu().numpy() for t in (nx, q, k, v, att, h, nh, y, lg))

        assert rel_err(nx, orc.rms_norm(x, norm, HID, EPS, chunked=True))[0] <= 1e-5
        for got, name in ((q, "q"), (k, "k"), (v, "v")):
            within(got, R.product(quantized(nx), wv[name]))
        b.append(k.reshape(n, KV, DIM), v.reshape(n, KV, DIM))
        np.testing.assert_array_equal(codes.cpu().numpy(), b.codes)
        np.testing.assert_array_equal(scales.cpu().numpy(), b.scales)
        want, tol, _ = b.attention(q.reshape(n, HEADS, DIM), HEADS, float(F32(DIM ** -0.5)))
        assert (np.abs(att.reshape(want.shape) - want) <= tol).all()
        within(h, R.product(quantized(att), wv["o"], x))
        lo, hi = hull(*R.gated(quantized(nh), wv["gate"], wv["up"]), act)
        want, tol = R.product((lo + hi) / 2, wv["down"], h)
        within(y, (want, tol * 1.01 + (hi - lo) / 2 @ np.abs(wv["down"]).T))
        within(lg, R.product(quantized(y), wv["lm"]))
        want = logprobs(lg, token, 5)
        np.testing.assert_array_equal(tid.cpu().numpy(), want[3])
        assert (np.abs(lp.cpu().numpy() - want[0]) <= want[4]).all()
        assert (np.abs(ent.cpu().numpy() - want[1]) <= want[4] * (want[1] + 1)).all()
        assert (np.abs(tlp.cpu().numpy() - want[2]) <= want[4][:, None]).all()
