"""GPU: a decoder layer and the reading of its logits as an engine runs them - fused norm + QKV, append, attention,
O projection with its residual, norm + gate/up, SiLU + down, lm_head, log probabilities - over a prompt of two
sequences and then single tokens of both. Every stage is checked against its plain form on the outputs that the stage
before it left on the GPU."""
import numpy as np
import pytest

import synth
from conftest import rel_err
from kv_ref import F32, Batch, logprobs

pytestmark = pytest.mark.gpu

HID, HEADS, KV, DIM, FFN, VOCAB, EPS = 256, 4, 2, 64, 512, 1000, 1e-6


def test_prompt_and_decode_steps(kq4, torch_dev, orc):
    torch, rng = torch_dev, np.random.default_rng(1)
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    mats = dict(q=(HEADS * DIM, HID), k=(KV * DIM, HID), v=(KV * DIM, HID), o=(HID, HEADS * DIM), gate=(FFN, HID),
                up=(FFN, HID), down=(HID, FFN), lm=(VOCAB, HID))
    raw = {n: synth.make_q4_weights(r, c, 10 + i) for i, (n, (r, c)) in enumerate(mats.items())}
    w = {n: kq4.prepare_dev(up(raw[n]), *mats[n]) for n in mats}
    norm = (1 + 0.1 * rng.standard_normal(HID)).astype(F32)

    b = Batch(rng, [(37, 37), (20, 20)], KV, DIM, 16, DIM, extra_pages=1)
    b.table[:] = rng.permutation(b.table.size).reshape(b.table.shape)      # room to grow
    b.codes = rng.integers(0, 256, (b.table.size,) + b.codes.shape[1:], np.uint8)
    b.scales = np.full((b.table.size,) + b.scales.shape[1:], np.nan, F32)
    b.rope = kq4.rope_table(64, DIM, 1e4, device="cpu").numpy()
    codes, scales, table = up(b.codes), up(b.scales), up(b.table)
    for step in range(4):
        if step:
            b.lens = [(1, kv + 1) for _, kv in b.lens]
        n = b.n = sum(q for q, _ in b.lens)
        b.q_start = np.concatenate([[0], np.cumsum([q for q, _ in b.lens])]).astype(np.int32)
        b.kv_len = np.array([kv for _, kv in b.lens], np.int32)
        kv = kq4.KVBatch(codes, scales, 16, table, up(b.q_start), up(b.kv_len), n, rope=up(b.rope))
        x = rng.standard_normal((n, HID)).astype(F32)
        new = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
        xd, q, k, v = up(x), new(n, HEADS * DIM), new(n, KV * DIM), new(n, KV * DIM)
        att, h, g, u, y, lg = new(n, HEADS * DIM), new(n, HID), new(n, FFN), new(n, FFN), new(n, HID), new(n, VOCAB)
        token = rng.integers(0, VOCAB, n)
        lp, ent, tlp, tid = new(n), new(n), new(n, 5), torch.empty((n, 5), dtype=torch.int32, device="cuda")
        kq4.rmsnorm_matmul_multi_dev([q, k, v], xd, up(norm), EPS, [w["q"], w["k"], w["v"]],
                                     [mats["q"][0], mats["k"][0], mats["v"][0]], HID)
        kq4.kv_append_dev(kv, k, v)
        kq4.attn_dev(att, q, kv, HEADS, DIM ** -0.5, max_q=int(max(q_ for q_, _ in b.lens)), max_kv=int(b.kv_len.max()))
        kq4.matmul_dev(h, att, w["o"], HID, HEADS * DIM, residual=xd)
        kq4.rmsnorm_matmul_multi_dev([g, u], h, up(norm), EPS, [w["gate"], w["up"]], [FFN, FFN], HID)
        kq4.matmul_silu_dev(y, g, u, w["down"], HID, FFN, residual=h)
        kq4.matmul_dev(lg, y, w["lm"], VOCAB, HID)
        kq4.logprobs_dev(lg, up(token.astype(np.int32)), lp, ent, tlp, tid)
        torch.cuda.synchronize()
        q, k, v, att, h, lg = (t.cpu().numpy() for t in (q, k, v, att, h, lg))

        normed = orc.rms_norm(x, norm, HID, EPS, chunked=True)
        for got, name in ((q, "q"), (k, "k"), (v, "v")):
            assert rel_err(got, orc.matmul(raw[name], normed, *mats[name]))[0] <= 1e-5
        b.append(k.reshape(n, KV, DIM), v.reshape(n, KV, DIM))
        np.testing.assert_array_equal(codes.cpu().numpy(), b.codes)
        np.testing.assert_array_equal(scales.cpu().numpy(), b.scales)
        want, tol, _ = b.attention(q.reshape(n, HEADS, DIM), HEADS, float(F32(DIM ** -0.5)))
        assert (np.abs(att.reshape(want.shape) - want) <= tol).all()
        assert rel_err(h, orc.matmul(raw["o"], att, *mats["o"], residual=x))[0] <= 1e-5
        want = logprobs(lg, token, 5)
        np.testing.assert_array_equal(tid.cpu().numpy(), want[3])
        assert (np.abs(lp.cpu().numpy() - want[0]) <= want[4]).all()
        assert (np.abs(ent.cpu().numpy() - want[1]) <= want[4] * (want[1] + 1)).all()
        assert (np.abs(tlp.cpu().numpy() - want[2]) <= want[4][:, None]).all()
