"""Performance cases of kq4's serving operators next to the linear layers: the paged int8 key/value cache,
the attention that reads it, and the reading of the logits.

A case is one of three kinds of call:

  append    keys and values of the call's tokens into the cache, the keys rotated on the way
  attn      attention of the call's queries (rotated as they are read) over the cache
  logprobs  log probabilities of given tokens, entropy and top alternatives of rows of logits

The cache of a layer is `codes`, uint8 [n_pages][kv_heads][page / 16][2][16 * dim], and `scales`, fp32
[n_pages][kv_heads][page / 16][2]: 16 consecutive tokens of a sequence are a group, with one scale for its
keys and one for its values per head; a byte is its code + 128, |code| <= 127, and stands for code * scale.
In a group the keys lie as [dim / 16][16 tokens][16], the values as [dim][16 tokens].

Appending rounds at these places, so codes and scales are whole numbers and values of their own, returned
as the cache holds them: rotated key = (x1 c - x2 s, x2 c + x1 s), exact, rounded to fp32 once;
s_new = max(fl(amax / 127), 2^-100) over the group's new tokens, the group's scale s = max(s_old, s_new) if
it holds earlier tokens, else s_new; code = rint(fl(x * fl(1 / s))); where s > s_old the earlier codes c
become rint(fl(c * fl(s_old / s))).

Head counts and sizes are those of Qwen3-VL-2B (16 query / 8 key heads), Qwen3-8B (32 / 8), a 32 / 4 layout
for long contexts, or generic.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda"
THETA = 1.0e6
TINY = 2.0 ** -100


def listed():
    return [
        # one decode token of one sequence in one layer of Qwen3-8B: the smallest call, all latency
        dict(name="append_1", kind="append", n_seq=1, q=1, kv=777, ragged=False, kv_heads=8, dim=128,
             page=64, rope=128),
        # a decode step of a continuous batch: one token of each of 64 sequences, at any place of its group
        dict(name="append_64", kind="append", n_seq=64, q=1, kv=4000, ragged=True, kv_heads=8, dim=128,
             page=64, rope=128),
        # several prompts' chunks of odd lengths at odd places, half-rotated heads of 64, small pages
        dict(name="append_ragged", kind="append", n_seq=9, q=301, kv=1999, ragged=True, kv_heads=4,
             dim=64, page=16, rope=32),
        # a whole prompt
        dict(name="append_prompt", kind="append", n_seq=1, q=4096, kv=4096, ragged=False, kv_heads=8,
             dim=128, page=64, rope=128),
        # one decode token over a short context (Qwen3-VL-2B heads): the latency of a chat turn's step
        dict(name="attn_1x1k", kind="attn", n_seq=1, q=1, kv=1001, ragged=False, heads=16, kv_heads=8,
             dim=128, page=64, rope=128, window=0),
        # a continuous batch's decode step: 32 sequences of up to 8192 tokens (Qwen3-8B heads)
        dict(name="attn_32x8k", kind="attn", n_seq=32, q=1, kv=8192, ragged=True, heads=32, kv_heads=8,
             dim=128, page=64, rope=128, window=0),
        # one decode token far into a long context
        dict(name="attn_1x128k", kind="attn", n_seq=1, q=1, kv=131072, ragged=False, heads=32,
             kv_heads=4, dim=128, page=128, rope=128, window=0),
        # odd chunks of several sequences with a sliding window, small heads and pages
        dict(name="attn_ragged", kind="attn", n_seq=7, q=190, kv=2901, ragged=True, heads=12,
             kv_heads=4, dim=64, page=16, rope=64, window=1024),
        # a whole prompt's causal attention (Qwen3-8B heads), the largest call
        dict(name="attn_prompt", kind="attn", n_seq=1, q=4096, kv=4096, ragged=False, heads=32,
             kv_heads=8, dim=128, page=64, rope=128, window=0),
        # the token that one decode step sampled, with five alternatives
        dict(name="logprobs_1", kind="logprobs", rows=1, vocab=151936, top=5, masked=False),
        # a batch of decode steps under grammars that forbid most tokens, twenty alternatives
        dict(name="logprobs_64", kind="logprobs", rows=64, vocab=151936, top=20, masked=True),
        # a prompt's token log probabilities, odd vocabulary, one alternative
        dict(name="logprobs_prompt", kind="logprobs", rows=1000, vocab=128003, top=1, masked=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: sizes log-uniform over the listed range, odd ones among them."""
    kind = rng.choice(["append", "attn", "attn", "attn", "logprobs"])
    if kind == "logprobs":
        vocab = _log_int(rng, 1000, 151936)
        rows = min(_log_int(rng, 1, 1000), 128003 * 1000 // vocab)
        return dict(kind=kind, rows=rows, vocab=vocab, top=rng.randint(0, 20), masked=rng.random() < 0.3)
    kv_heads, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128])
    c = dict(kind=kind, n_seq=_log_int(rng, 1, 64), ragged=rng.random() < 0.7, kv_heads=kv_heads, dim=dim,
             page=rng.choice([16, 32, 64, 128]), rope=rng.choice([0, 32, dim, dim]))
    if kind == "append":
        c["q"] = 1 if rng.random() < 0.4 else _log_int(rng, 2, 4096)
        c["n_seq"] = min(c["n_seq"], max(1, 4096 // c["q"]))
        c["kv"] = max(c["q"], _log_int(rng, 16, 8192))
        return c
    c["heads"] = kv_heads * rng.choice([1, 2, 3, 4, 6, 8])
    c["q"] = 1 if rng.random() < 0.5 else _log_int(rng, 2, 4096)
    c["kv"] = max(c["q"], _log_int(rng, 16, 131072 if c["q"] == 1 else 16384))
    while c["n_seq"] * (c["kv"] * kv_heads * dim) > 32 * 8192 * 8 * 128 // 2 or \
            c["n_seq"] * c["heads"] * c["q"] * c["kv"] > 32 * 4096 * 2048:
        if c["n_seq"] > 1:
            c["n_seq"] = c["n_seq"] // 2
        elif c["q"] > 1:
            c["q"] = c["q"] // 2
        else:
            c["kv"] = c["kv"] // 2
    c["window"] = _log_int(rng, 8, c["kv"] + 8) if rng.random() < 0.25 else 0
    return c


def _lens(c):
    """(tokens of the call, tokens in the cache with them) of each sequence."""
    n, q, kv = c["n_seq"], c["q"], c["kv"]
    if not c["ragged"]:
        return [(q, kv)] * n
    got = []
    for i in range(n):
        f, h = (i * 0.6180339887498949) % 1.0, (i * 0.7548776662466927) % 1.0
        qi = q - int((q - 1) * f)
        got.append((qi, max(qi, kv - int((kv - 1) * 0.9 * h))))
    return got


# ---- inputs --------------------------------------------------------------------------------------

def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed((seed * 1000003 + salt * 7919 + 17) & 0x7FFFFFFF)
    return g


def _acts(n, heads, dim, seed, salt):
    """[n][heads * dim] N(0, 1), each head with a few channels several times as large, as keys have."""
    g = _gen(seed, salt)
    gain = 1.0 + 4.0 * (torch.rand(heads * dim, device=DEV, generator=g) < 0.03).float()
    return torch.randn(n, heads * dim, device=DEV, generator=g) * gain


def _rope_table(rows, rope):
    """fp32 [rows][rope / 2][cos, sin], the angles in 64 bits; None without a rotation."""
    if not rope:
        return None
    inv = THETA ** (-torch.arange(0, rope, 2, dtype=torch.float64, device=DEV) / rope)
    a = torch.arange(rows, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], 2).float().contiguous()


def _cache(n_pages, c, seed, salt):
    """A filled cache: normal keys (with their large channels) and values, a scale per group and head."""
    hkv, dim, ng = c["kv_heads"], c["dim"], c["page"] // 16
    codes = torch.empty(n_pages, hkv, ng, 2, 16 * dim, dtype=torch.uint8, device=DEV)
    scales = torch.empty(n_pages, hkv, ng, 2, device=DEV)
    g = _gen(seed, salt)
    for part in range(2):
        gain = 1.0 + 4.0 * (torch.rand(hkv, 1, 1, dim, device=DEV, generator=g) < 0.03).float() * (1 - part)
        x = torch.randn(n_pages, hkv, ng, 16, dim, device=DEV, generator=g) * gain
        s = x.abs().amax((3, 4)) / 127
        q = (x / s[..., None, None]).round().clamp(-127, 127) + 128
        q = q.to(torch.uint8)
        q = q.view(n_pages, hkv, ng, 16, dim // 16, 16).transpose(3, 4) if part == 0 else q.transpose(3, 4)
        codes[:, :, :, part] = q.reshape(n_pages, hkv, ng, 16 * dim)
        scales[..., part] = s
    return codes, scales


def _prepare_logprobs(c, seed):
    rows, vocab, top = c["rows"], c["vocab"], c["top"]
    g = _gen(seed, 1)
    x = 2.5 * torch.randn(rows, vocab, device=DEV, generator=g)
    best = torch.randint(0, vocab, (rows, 1), device=DEV, generator=g)
    x.scatter_add_(1, best, 12.0 * torch.rand(rows, 1, device=DEV, generator=g))
    if c["masked"]:
        x.masked_fill_(torch.rand(rows, vocab, device=DEV, generator=g) < 0.97, -math.inf)
        x.scatter_(1, best, 1.0)
    token = torch.where(torch.rand(rows, 1, device=DEV, generator=g) < 0.5, best,
                        torch.randint(0, vocab, (rows, 1), device=DEV, generator=g))
    s = dict(x=x, token=token[:, 0].to(torch.int32), logprob=torch.empty(rows, device=DEV),
             entropy=torch.empty(rows, device=DEV), top_logprob=None, top_id=None)
    if top:
        s["top_logprob"] = torch.empty(rows, top, device=DEV)
        s["top_id"] = torch.empty(rows, top, dtype=torch.int32, device=DEV)
    return s


def prepare(case, seed):
    c = case
    if c["kind"] == "logprobs":
        return dict(case=c, **_prepare_logprobs(c, seed))
    lens, page = _lens(c), c["page"]
    n = sum(q for q, _ in lens)
    width = -(-max(kv for _, kv in lens) // page)
    need = [-(-kv // page) for _, kv in lens]
    pool = sum(need) + 3
    order = torch.randperm(pool, device=DEV, generator=_gen(seed, 3)).to(torch.int32)
    table = torch.zeros(c["n_seq"], width, dtype=torch.int32, device=DEV)
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = order[at:at + m]
        at += m
    starts = [0]
    for q, _ in lens:
        starts.append(starts[-1] + q)
    s = dict(case=c, n=n, table=table, max_q=max(q for q, _ in lens), max_kv=max(kv for _, kv in lens),
             q_start=torch.tensor(starts, dtype=torch.int32, device=DEV),
             kv_len=torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=DEV),
             rope=_rope_table(max(kv for _, kv in lens), c["rope"]))
    s["codes"], s["scales"] = _cache(pool, c, seed, 4)
    if c["kind"] == "append":
        s["k"], s["v"] = (_acts(n, c["kv_heads"], c["dim"], seed, salt) for salt in (5, 6))
    else:
        s["q"] = _acts(n, c["heads"], c["dim"], seed, 7)
        s["out"] = torch.empty(n, c["heads"] * c["dim"], device=DEV)
    if own:   # the handle that a program keeps for a layer's cache and its batch: addresses and sizes
        s["kv"] = _kq4().KVBatch(s["codes"], s["scales"], page, s["table"], s["q_start"], s["kv_len"], n,
                                 rope=s["rope"])
    return s


# ---- the framework's calls -------------------------------------------------------------------------

def _kq4():
    """The binding, initialised once: a program keeps the module."""
    global _binding
    if _binding is None:
        sys.path.insert(0, os.path.abspath("kestrel-llm_amd"))
        import kq4
        kq4.init(0)
        _binding = kq4
    return _binding


_binding = None


def _run_own(s):
    c, kq4 = s["case"], _kq4()
    if c["kind"] == "append":
        kq4.kv_append_dev(s["kv"], s["k"], s["v"])
        return s["codes"], s["scales"]
    if c["kind"] == "attn":
        kq4.attn_dev(s["out"], s["q"], s["kv"], c["heads"], 1 / math.sqrt(c["dim"]), window=c["window"],
                     max_q=s["max_q"], max_kv=s["max_kv"])
        return s["out"]
    kq4.logprobs_dev(s["x"], token=s["token"], logprob=s["logprob"], entropy=s["entropy"],
                     top_logprob=s["top_logprob"], top_id=s["top_id"])
    return [t for t in (s["logprob"], s["entropy"], s["top_logprob"], s["top_id"]) if t is not None]


# ---- the plain forms ---------------------------------------------------------------------------------

def _tokens(s):
    """(sequence, position in it) of each token of the call."""
    t = torch.arange(s["n"], device=DEV)
    start, length = s["q_start"].long(), s["kv_len"].long()
    seq = torch.searchsorted(start[1:], t, right=True)
    return seq, length[seq] - (start[seq + 1] - t)


def _rotate(x, rope, pos):
    """x [n, heads, dim] with its first rope.shape[1] * 2 dimensions rotated by the table's row `pos`."""
    if rope is None:
        return x
    h = rope.shape[1]
    c, s = rope[pos, None, :, 0].double(), rope[pos, None, :, 1].double()
    a, b = x[..., :h].double(), x[..., h:2 * h].double()
    return torch.cat([(a * c - b * s).float(), (b * c + a * s).float(), x[..., 2 * h:]], 2)


def _views(s):
    """The cache's keys [page, head, group, dim / 16, token, 16] and values [page, head, group, dim, token]."""
    p, h, g, _, b = s["codes"].shape
    return (s["codes"][:, :, :, 0].view(p, h, g, b // 256, 16, 16), s["codes"][:, :, :, 1].view(p, h, g, b // 16, 16))


def _divide(a, b):
    """fl(a / b) of fp32 tensors, rounded once."""
    return (a.double() / b.double()).float()


def _plain_append(s):
    c = s["case"]
    n, page, hkv, dim = s["n"], c["page"], c["kv_heads"], c["dim"]
    seq, pos = _tokens(s)
    where, group, slot = s["table"][seq, pos // page].long(), pos % page // 16, pos % 16
    t = torch.arange(n, device=DEV)
    lead = t - torch.minimum(slot, t - s["q_start"][seq])         # the call's first token of the same group
    K, V = _views(s)
    earlier = (slot[lead] > 0)[:, None]
    first = s["q_start"][:-1].long()                              # only a sequence's first group has earlier tokens
    page0, group0 = where[first], group[first]
    before = torch.arange(16, device=DEV)[None, :] < slot[first][:, None]
    k = _rotate(s["k"].view(n, hkv, dim), s["rope"], pos)
    for part, x in enumerate((k, s["v"].view(n, hkv, dim))):
        amax = torch.zeros(n, hkv, device=DEV).scatter_reduce_(0, lead[:, None].expand(n, hkv), x.abs().amax(2), "amax")
        new = _divide(amax[lead], torch.full_like(amax, 127.0)).clamp(min=TINY)
        old = torch.where(earlier, s["scales"][where, :, group, part], torch.zeros_like(new))
        scale = torch.maximum(old, new)
        ratio = torch.where(scale > old, _divide(old, scale), torch.ones_like(old))[first]
        if part == 0:
            held = K[page0, :, group0]                            # [sequence, head, dim / 16, token, 16]
            kept = (held.float() - 128) * ratio[:, :, None, None, None]
            K[page0, :, group0] = torch.where(before[:, None, None, :, None], (kept.round() + 128).to(torch.uint8), held)
        else:
            held = V[page0, :, group0]
            kept = (held.float() - 128) * ratio[:, :, None, None]
            V[page0, :, group0] = torch.where(before[:, None, None], (kept.round() + 128).to(torch.uint8), held)
        code = ((x * _divide(torch.ones_like(scale), scale)[:, :, None]).round() + 128).to(torch.uint8)
        if part == 0:
            K[where, :, group, :, slot] = code.view(n, hkv, dim // 16, 16)
        else:
            V[where, :, group, :, slot] = code
        s["scales"][where, :, group, part] = scale
    return s["codes"], s["scales"]


def _plain_attn(s):
    c = s["case"]
    n, heads, hkv, dim, page = s["n"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    seq, pos = _tokens(s)
    lq, lk, b = s["max_q"], s["max_kv"], c["n_seq"]
    at = torch.arange(s["n"], device=DEV) - s["q_start"].long()[seq]
    q = torch.zeros(b, lq, heads, dim, device=DEV)
    q[seq, at] = _rotate(s["q"].view(n, heads, dim), s["rope"], pos)
    q = q.view(b, lq, hkv, heads // hkv, dim).permute(0, 2, 3, 1, 4).reshape(b, hkv, heads // hkv * lq, dim)
    j = torch.arange(lk, device=DEV)
    where, group, slot = s["table"].long()[:, j // page], (j % page // 16)[None], (j % 16)[None]
    K, V = _views(s)
    sc = s["scales"][where, :, group]                                                # [b, lk, hkv, 2]
    k = (K[where, :, group, :, slot].reshape(b, lk, hkv, dim).float() - 128) * sc[..., :1]
    x = torch.matmul(q, k.permute(0, 2, 3, 1)) * (1 / math.sqrt(dim))
    x = x.view(b, hkv, heads // hkv, lq, lk)
    own_pos = (s["kv_len"] - (s["q_start"][1:] - s["q_start"][:-1])).long()[:, None] + torch.arange(lq, device=DEV)
    sees = (j <= own_pos[..., None]) & (j < s["kv_len"][:, None, None])
    if c["window"]:
        sees &= j > own_pos[..., None] - c["window"]
    x = x.masked_fill(~sees[:, None, None], -math.inf)
    m = x.amax(4, keepdim=True).clamp(min=-1e30)
    p = torch.exp(x - m)
    total = p.sum(4, keepdim=True)
    v = (V[where, :, group, :, slot].float() - 128) * sc[..., 1:]
    o = torch.matmul(p.view(b, hkv, heads // hkv * lq, lk), v.permute(0, 2, 1, 3)).view(b, hkv, heads // hkv, lq, dim)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    s["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(b, lq, heads * dim)[seq, at])
    return s["out"]


def _plain_logprobs(s):
    x, top = s["x"], s["case"]["top"]
    m = x.amax(1, keepdim=True)
    d = x - m
    e = torch.exp(d).masked_fill_(torch.arange(x.shape[1], device=DEV) == x.argmax(1)[:, None], 0.0)
    logz = torch.log1p(e.sum(1, dtype=torch.float64))             # the others' share of a sure row is small
    p = torch.exp(d.double() - logz[:, None])
    s["entropy"].copy_(logz - (p * d).nan_to_num_(0.0).sum(1))
    s["logprob"].copy_(d.gather(1, s["token"][:, None].long())[:, 0].double() - logz)
    got = [s["logprob"], s["entropy"]]
    if top:
        value, index = torch.sort(x, dim=1, descending=True, stable=True)
        s["top_logprob"].copy_((value[:, :top] - m).double() - logz[:, None])
        s["top_id"].copy_(index[:, :top])
        got += [s["top_logprob"], s["top_id"]]
    return got


def run(state):
    if own:
        return _run_own(state)
    return {"append": _plain_append, "attn": _plain_attn, "logprobs": _plain_logprobs}[state["case"]["kind"]](state)


# ---- 64 bits, from the definitions ---------------------------------------------------------------------

def _exact_rotation(x, c, pos, table):
    """One sequence's x [tokens, heads, dim] in 64 bits, rotated at positions pos and rounded to fp32."""
    if table is None:
        return x.double()
    h = c["rope"] // 2
    y = x.double().clone()
    t = table[pos].double()
    for i in range(h):
        co, si = t[:, i, 0:1], t[:, i, 1:2]
        y[..., i] = x[..., i].double() * co - x[..., h + i].double() * si
        y[..., h + i] = x[..., h + i].double() * co + x[..., i].double() * si
    return y.float().double()


def _exact_append(s):
    c = s["case"]
    page, hkv, dim = c["page"], c["kv_heads"], c["dim"]
    codes, scales, t0 = s["codes"], s["scales"].double(), 0
    one = lambda a: a.float().double()  # noqa: E731   a rounding to fp32
    for i, (q, kv) in enumerate(_lens(c)):
        pos = torch.arange(kv - q, kv, device=DEV)
        both = (_exact_rotation(s["k"][t0:t0 + q].view(q, hkv, dim), c, pos, s["rope"]), s["v"][t0:t0 + q].view(q, hkv, dim).double())
        t0 += q
        for g in range((kv - q) // 16, (kv - 1) // 16 + 1):
            lo, hi = max(kv - q, 16 * g), min(kv, 16 * g + 16)
            p, u = int(s["table"][i, 16 * g // page]), 16 * g % page // 16
            for part in range(2):
                x = both[part][lo - (kv - q):hi - (kv - q)]                    # [tokens, head, dim]
                new = one(x.abs().amax((0, 2)) / 127).clamp(min=TINY)
                held = codes[p, :, u, part]
                held = held.view(hkv, dim // 16, 16, 16).transpose(2, 3).reshape(hkv, dim, 16) if part == 0 else held.view(hkv, dim, 16)
                full = held.double() - 128                                     # [head, dim, token]
                if lo > 16 * g:
                    old = scales[p, :, u, part]
                    grown = torch.maximum(old, new)
                    full[:, :, :lo - 16 * g] = one(full[:, :, :lo - 16 * g] * one(old / grown)[:, None, None]).round()
                    new = grown
                full[:, :, lo - 16 * g:hi - 16 * g] = one(x.permute(1, 2, 0) * one(1 / new)[:, None, None]).round()
                full = (full + 128).to(torch.uint8)
                if part == 0:
                    full = full.view(hkv, dim // 16, 16, 16).transpose(2, 3)
                codes[p, :, u, part] = full.reshape(hkv, 16 * dim)
                scales[p, :, u, part] = new
    return codes, scales


def _exact_attn(s):
    c = s["case"]
    heads, hkv, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    out, t0 = torch.zeros(s["n"], heads, dim, dtype=torch.float64, device=DEV), 0
    for i, (q, kv) in enumerate(_lens(c)):
        pages = s["table"][i, :-(-kv // page)].long()
        x = s["codes"][pages].double() - 128                                   # [pages, head, group, 2, 16 * dim]
        x = x * s["scales"][pages].double()[..., None]
        np_, ng = x.shape[0], page // 16
        k = x[:, :, :, 0].view(np_, hkv, ng, dim // 16, 16, 16).permute(1, 0, 2, 4, 3, 5).reshape(hkv, np_ * page, dim)[:, :kv]
        v = x[:, :, :, 1].view(np_, hkv, ng, dim, 16).permute(1, 0, 2, 4, 3).reshape(hkv, np_ * page, dim)[:, :kv]
        pos = torch.arange(kv - q, kv, device=DEV)
        y = _exact_rotation(s["q"][t0:t0 + q].view(q, heads, dim), c, pos, s["rope"])
        for h in range(heads):
            kh, vh = k[h // (heads // hkv)], v[h // (heads // hkv)]
            w = y[:, h] @ kh.T / math.sqrt(dim)
            far = pos[:, None] - torch.arange(kv, device=DEV)[None, :]
            w[(far < 0) | (far >= (c["window"] or kv + 1))] = -math.inf
            out[t0:t0 + q, h] = torch.softmax(w, 1) @ vh
        t0 += q
    return out.reshape(s["n"], heads * dim)


def _exact_logprobs(s):
    out = [[], [], [], []]
    for row, token in zip(s["x"], s["token"].tolist()):
        x = row.double()
        at = int(x.argmax())
        rest = torch.exp(x - x[at])
        rest[at] = 0
        lz = torch.log1p(rest.sum())
        lp = (x - x[at]) - lz
        here = torch.isfinite(lp)
        out[0].append(lp[token])
        out[1].append(-(lp[here].exp() * lp[here]).sum())
        if s["case"]["top"]:
            index = torch.argsort(-x, stable=True)[:s["case"]["top"]]
            out[2].append(lp[index])
            out[3].append(index.to(torch.int32))
    return [torch.stack(o) for o in out if o]


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attn": _exact_attn, "logprobs": _exact_logprobs}[case["kind"]](s)


# ---- what a pass cannot do without ---------------------------------------------------------------------

def work(case):
    c = case
    if c["kind"] == "logprobs":
        return {"bytes": 4.0 * c["rows"] * (c["vocab"] + 3 + 2 * c["top"]), "flops": 4.0 * c["rows"] * c["vocab"]}
    lens = _lens(c)
    n, hkv, dim = sum(q for q, _ in lens), c["kv_heads"], c["dim"]
    table = 4.0 * c["rope"] * n
    if c["kind"] == "append":
        groups = sum((kv - 1) // 16 - (kv - q) // 16 + 1 for q, kv in lens)
        return {"bytes": n * hkv * dim * 2 * (4 + 1) + groups * hkv * 8 + table, "flops": n * hkv * (3.0 * c["rope"] + 3.0 * 2 * dim)}
    read, pairs = 0, 0
    for q, kv in lens:
        w = c["window"] or kv
        read += min(kv, q + w - 1)
        # the query at position p sees min(p + 1, w) keys
        pairs += sum(min(p + 1, w) for p in range(kv - q, kv))
    return {"bytes": read * hkv * 2 * (dim + 0.25) + n * c["heads"] * dim * 8 + table, "flops": 4.0 * dim * c["heads"] * pairs}
