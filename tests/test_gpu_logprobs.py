"""GPU: log probabilities of given tokens, entropy and top alternatives against the plain form in 64 bits
(kv_ref.logprobs). The ids have to be equal, the values within the bound derived there."""
import numpy as np
import pytest

from kv_ref import F32, logprobs

pytestmark = pytest.mark.gpu


def run(kq4, torch, x, token, n_top, view=None):
    n = x.shape[0]
    d = torch.from_numpy(np.ascontiguousarray(x)).cuda() if view is None else view
    lp, ent = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    tlp = torch.empty((n, n_top), device="cuda") if n_top else None
    tid = torch.empty((n, n_top), dtype=torch.int32, device="cuda") if n_top else None
    kq4.logprobs_dev(d, token=torch.from_numpy(token.astype(np.int32)).cuda(), logprob=lp, entropy=ent, top_logprob=tlp,
                     top_id=tid)
    torch.cuda.synchronize()
    return [t.cpu().numpy() if t is not None else np.zeros((n, 0)) for t in (lp, ent, tlp, tid)]


def check(kq4, torch, x, token, n_top, view=None):
    got = run(kq4, torch, x, token, n_top, view)
    want = logprobs(x, token, n_top)
    np.testing.assert_array_equal(got[3], want[3])
    tol = want[4]
    for g, w, t in ((got[0], want[0], tol), (got[1], want[1], tol * (want[1] + 1)), (got[2], want[2], tol[:, None])):
        g = g.astype(np.float64)
        np.testing.assert_array_equal(np.isnan(g), np.isnan(w))
        np.testing.assert_array_equal(np.isneginf(g), np.isneginf(w))
        with np.errstate(invalid="ignore"):
            bad = ~(np.abs(g - w) <= t) & np.isfinite(w)
        assert not bad.any(), (g[bad][:4], w[bad][:4])


@pytest.mark.parametrize("n,vocab", [(1, 1), (3, 2), (2, 31), (5, 1000), (1, 8191), (2, 8192), (3, 8193), (4, 50257),
                                     (2, 151936), (130, 4096), (1, 1 << 20)])
@pytest.mark.parametrize("n_top", [0, 1, 5, 20, 32])
def test_rows(kq4, torch_dev, n, vocab, n_top):
    n_top = min(n_top, vocab)
    rng = np.random.default_rng(vocab + n_top)
    x = (3 * rng.standard_normal((n, vocab))).astype(F32)
    x[np.arange(n), rng.integers(0, vocab, n)] += F32(8) * rng.random(n).astype(F32)
    check(kq4, torch_dev, x, rng.integers(0, vocab, n), n_top)


def test_sure_rows_keep_their_digits(kq4, torch_dev):
    """One logit far above the rest: log p and the entropy are far below 1 and right relative to themselves."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((6, 30000)).astype(F32)
    x[np.arange(6), np.arange(6) * 4999] = [14, 20, 26, 32, 40, 60]
    token = np.arange(6) * 4999
    lp, ent, _, _ = run(kq4, torch_dev, x, token, 0)
    want = logprobs(x, token, 0)
    rel = 2.0 ** -24 * (64 + 2 * 105 + 70)                    # the bound of z, and of t, relative
    assert (np.abs(lp - want[0]) <= rel * np.abs(want[0])).all()
    assert (np.abs(ent - want[1]) <= 2 * rel * np.abs(want[1])).all()


@pytest.mark.parametrize("vocab", [100, 8192, 20001])
@pytest.mark.parametrize("what", ["equal", "two_values", "masked", "one_left", "none_left", "half", "ascending", "late",
                                  "zeros", "nan", "inf", "low"])
def test_ties_masks_and_ends(kq4, torch_dev, what, vocab):
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((3, vocab)).astype(F32)
    token = rng.integers(0, vocab, 3)
    if what == "equal":
        x[:] = 1.25
    elif what == "two_values":
        x = (rng.random((3, vocab)) < 0.5).astype(F32)
    elif what == "masked":
        x[rng.random((3, vocab)) < 0.97] = -np.inf
    elif what == "one_left":
        x[:] = -np.inf
        x[:, vocab // 2] = [-1e30, 0, 1e30]
    elif what == "none_left":
        x[1:] = -np.inf
    elif what == "half":
        x = np.round(x * 2) / 2
    elif what == "ascending":
        x = np.sort(x, 1)
    elif what == "late":                                      # the best all in one thread's elements
        x[:, 4::1024] += 50
    elif what == "zeros":
        x[:] = 0.0
        x[:, ::2] = -0.0
    elif what == "nan":
        x[0, 7] = np.nan
        x[2, [3, vocab - 1]] = np.nan
    elif what == "inf":
        x[1, 50] = np.inf
        x[2, [1, 2]] = np.inf
    elif what == "low":
        x[:, 1:] = np.finfo(F32).min
    check(kq4, torch_dev, x.astype(F32), token, min(20, vocab))


def test_tokens_outside_the_vocabulary(kq4, torch_dev):
    x = np.random.default_rng(2).standard_normal((4, 500)).astype(F32)
    check(kq4, torch_dev, x, np.array([-1, 499, 500, 1 << 30]), 3)


@pytest.mark.parametrize("offset,ld", [(0, 1003), (1, 1000), (4, 1004), (3, 1007)])
def test_strides_and_alignment(kq4, torch_dev, offset, ld):
    torch = torch_dev
    flat = torch.full((offset + 5 * ld + 8,), float("nan"), device="cuda")
    view = flat[offset:offset + 5 * ld].view(5, ld)[:, :999]
    x = np.random.default_rng(3).standard_normal((5, 999)).astype(F32)
    view.copy_(torch.from_numpy(x).cuda())
    check(kq4, torch, x, np.arange(5) * 200, 7, view=view)


def test_each_output_alone(kq4, torch_dev):
    torch = torch_dev
    x = torch.randn(9, 33000, device="cuda")
    token = torch.arange(9, dtype=torch.int32, device="cuda") * 3000
    full = [torch.empty(9, device="cuda"), torch.empty(9, device="cuda"), torch.empty((9, 4), device="cuda"),
            torch.empty((9, 4), dtype=torch.int32, device="cuda")]
    kq4.logprobs_dev(x, token, *full)
    one = [torch.empty_like(t) for t in full]
    kq4.logprobs_dev(x, token=token, logprob=one[0])
    kq4.logprobs_dev(x, entropy=one[1])
    kq4.logprobs_dev(x, top_logprob=one[2], top_id=one[3])
    for a, b in zip(full, one):
        assert torch.equal(a, b)


def test_graph_replays(kq4, torch_dev):
    torch = torch_dev
    x = torch.empty(3, 40000, device="cuda")
    token = torch.zeros(3, dtype=torch.int32, device="cuda")
    outs = [[torch.empty(3, device="cuda"), torch.empty(3, device="cuda"), torch.empty((3, 6), device="cuda"),
             torch.empty((3, 6), dtype=torch.int32, device="cuda")] for _ in range(2)]
    kq4.workspace_reserve(kq4.logprobs_workspace_bytes(3, 40000, 6))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kq4.logprobs_dev(x, token, *outs[0], stream=torch.cuda.current_stream())
    for i in range(4):
        x.copy_(torch.randn(3, 40000, generator=torch.Generator().manual_seed(i)).cuda())
        token.fill_(i * 11)
        graph.replay()
        torch.cuda.synchronize()
        kq4.logprobs_dev(x, token, *outs[1])
        torch.cuda.synchronize()
        for a, b in zip(*outs):
            assert torch.equal(a, b), i


@pytest.mark.parametrize("n,vocab,n_top", [(3, 40000, 6), (64, 151936, 20), (5, 1000, 32)])
def test_same_bits_whatever_the_order(kq4, torch_dev, n, vocab, n_top):
    """Which thread takes a candidate is not fixed, what it makes of it is: calls repeat to the bit, and an alternative
    has the log probability that its token has when it is asked for."""
    torch = torch_dev
    x = torch.randn((n, vocab), generator=torch.Generator().manual_seed(1)).cuda()
    first = None
    for k in range(n_top):
        lp, top, ids = (torch.empty(s, device="cuda", dtype=t) for s, t in
                        (((n,), torch.float32), ((n, n_top), torch.float32), ((n, n_top), torch.int32)))
        token = torch.zeros(n, dtype=torch.int32, device="cuda") if first is None else first[1][:, k].contiguous()
        kq4.logprobs_dev(x, token, logprob=lp, top_logprob=top, top_id=ids)
        torch.cuda.synchronize()
        if first is None:
            first = top, ids
        else:
            assert torch.equal(lp, first[0][:, k]), k
        assert torch.equal(top, first[0]) and torch.equal(ids, first[1]), k


def test_many_rows_of_few_logits(kq4, torch_dev):
    rng = np.random.default_rng(5)
    check(kq4, torch_dev, (3 * rng.standard_normal((5000, 7))).astype(F32), rng.integers(0, 7, 5000), 7)
