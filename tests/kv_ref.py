"""Plain forms of the paged int8 key/value cache, its attention and the logits' log probabilities, in 64 bits
on the CPU, one element of the definition at a time (include/kq4.h kq4_kv)."""
import numpy as np

F32 = np.float32
TINY = 2.0 ** -100


def f32(x):
    """Rounded to binary32 once, kept in 64 bits."""
    with np.errstate(over="ignore", invalid="ignore"):
        return np.asarray(x, np.float64).astype(F32).astype(np.float64)


class Batch:
    """Host copies of a cache and a call's batch; `pages` are drawn without repetition from the pool."""

    def __init__(self, rng, lens, kv_heads, dim, page, rope_dim=0, pool=None, pad=0, extra_pages=0, theta=1e4):
        self.lens, self.hkv, self.dim, self.page = lens, kv_heads, dim, page
        need = [max(0, -(-kv // page)) for _, kv in lens]
        self.width = max([1] + need) + extra_pages
        pool = pool or sum(need) + 2
        order = rng.permutation(pool)
        self.table = np.full((len(lens), self.width), -1, np.int32)
        at = 0
        for i, m in enumerate(need):
            self.table[i, :m] = order[at:at + m]
            at += m
        self.q_start = np.concatenate([[0], np.cumsum([q for q, _ in lens])]).astype(np.int32)
        self.kv_len = np.array([kv for _, kv in lens], np.int32).reshape(len(lens))
        self.n = int(self.q_start[-1]) + pad
        self.rope_dim, self.rope, self.rope_pos = rope_dim, None, None
        if rope_dim:
            rows = max([1] + [kv for _, kv in lens])
            a = np.arange(rows)[:, None] * theta ** (-np.arange(0, rope_dim, 2) / rope_dim)
            self.rope = np.stack([np.cos(a), np.sin(a)], 2).astype(F32)
        # what no token holds is as bad as memory can be: any byte, NaN scales
        self.codes = rng.integers(0, 256, (pool, kv_heads, page // 16, 2, 16 * dim), np.uint8)
        self.scales = np.full((pool, kv_heads, page // 16, 2), np.nan, F32)

    def place(self, i, pos):
        """(page, group, slot) of a position, or None without a page of the cache."""
        if pos < 0 or pos // self.page >= self.table.shape[1]:
            return None
        p = int(self.table[i, pos // self.page])
        return None if p < 0 or p >= self.codes.shape[0] else (p, pos % self.page // 16, pos % 16)

    def group(self, p, h, g):
        """[2][dim][16 tokens] view-free codes of a group, as whole numbers around 0."""
        c = self.codes[p, h, g].astype(np.int64) - 128
        k = c[0].reshape(self.dim // 16, 16, 16).transpose(0, 2, 1).reshape(self.dim, 16)
        return np.stack([k, c[1].reshape(self.dim, 16)])

    def put_group(self, p, h, g, c):
        c = (c + 128).astype(np.uint8)
        self.codes[p, h, g, 0] = c[0].reshape(self.dim // 16, 16, 16).transpose(0, 2, 1).reshape(-1)
        self.codes[p, h, g, 1] = c[1].reshape(-1)

    def fill(self, rng, upto=None, spread=4.0):
        """Random codes and scales (log-uniform over 2^-spread .. 2^spread) of the positions held before the
        call (all of them with upto="all")."""
        for i, (q, kv) in enumerate(self.lens):
            end = kv if upto == "all" else kv - q
            for g0 in range(0, max(0, end), 16):
                at = self.place(i, g0)
                if at is None:
                    continue
                for h in range(self.hkv):
                    self.put_group(at[0], h, at[1], rng.integers(-127, 128, (2, self.dim, 16)))
                    self.scales[at[0], h, at[1]] = 2.0 ** rng.uniform(-spread, spread, 2) / 64

    def rotated(self, x, tok, pos):
        """x [heads][dim] of token `tok` at position pos: rotated, rounded to fp32 once; NaN off the table."""
        x = x.astype(np.float64)
        if not self.rope_dim:
            return x
        row = int(self.rope_pos[tok]) if self.rope_pos is not None else pos
        h, y = self.rope_dim // 2, x.copy()
        if not 0 <= row < self.rope.shape[0]:
            y[:, :2 * h] = np.nan
            return y
        c, s = self.rope[row, :, 0].astype(np.float64), self.rope[row, :, 1].astype(np.float64)
        y[:, :h] = f32(x[:, :h] * c - x[:, h:2 * h] * s)
        y[:, h:2 * h] = f32(x[:, h:2 * h] * c + x[:, :h] * s)
        return y

    def append(self, k, v):
        """k, v [n][heads][dim] fp32 into codes and scales."""
        for i, (q, kv) in enumerate(self.lens):
            groups = {}
            for t in range(q):
                pos = kv - q + t
                at = self.place(i, pos)
                if at is not None:
                    groups.setdefault((at[0], at[1]), []).append((at[2], int(self.q_start[i]) + t, pos))
            for (p, g), toks in groups.items():
                lo = toks[0][0]
                x = np.stack([np.stack([self.rotated(k[t], t, pos) for _, t, pos in toks], 2),
                              np.stack([v[t].astype(np.float64) for _, t, _ in toks], 2)])   # [2][h][d][tok]
                for h in range(self.hkv):
                    c = self.group(p, h, g)
                    for part in range(2):
                        s = f32(np.maximum(f32(np.abs(x[part, h]).max() / 127), TINY))
                        if lo > 0:
                            old = float(self.scales[p, h, g, part])
                            new = np.maximum(old, s)       # (a NaN of either is NaN)
                            if new > old:
                                c[part, :, :lo] = np.rint(f32(c[part, :, :lo] * f32(old / new)))
                            s = new
                        with np.errstate(invalid="ignore", over="ignore"):
                            code = np.rint(f32(x[part, h] * f32(1 / s)))
                        code = np.where(np.isnan(code), 0, np.clip(code, -127, 127))
                        c[part][:, [t[0] for t in toks]] = code
                        self.scales[p, h, g, part] = s
                    self.put_group(p, h, g, c)

    def keys_values(self, i, h):
        """(keys, values [len][dim], which positions there are) of one sequence and kv head."""
        n = min(int(self.kv_len[i]), self.table.shape[1] * self.page)
        kv = np.zeros((2, max(n, 0), self.dim))
        there = np.zeros(max(n, 0), bool)
        for g0 in range(0, n, 16):
            at = self.place(i, g0)
            if at is None:
                continue
            c = self.group(at[0], h, at[1]) * self.scales[at[0], h, at[1]].astype(np.float64)[:, None, None]
            m = min(16, n - g0)
            kv[:, g0:g0 + m] = c[:, :, :m].transpose(0, 2, 1)
            there[g0:g0 + m] = True
        return kv[0], kv[1], there

    def attention(self, q, heads, scale, window=0):
        """(out [n][heads][dim], bound on an fp32 result's error, rows of a sequence) of q [n][heads][dim].

        The bound: a score is a sum of 2 D products of f16 halves (|q.k| <= A in absolute values), each addition
        off by 2^-24 of at most A, and q = hi + lo is off by 2^-21 of q; with the exponent's own rounding (a few
        2^-24 of the score and of the scales' logarithms, at most 100) that is the relative error g of each
        weight, which holds for numerator and denominator; P = hi + lo is off by 2^-20; the sums over n keys and
        their joining are off by n 2^-24 at most. Each of these moves the output by at most twice itself times the
        largest |v|."""
        out = np.zeros((self.n, heads, self.dim))
        tol = np.zeros((self.n, heads, self.dim))
        rows = np.zeros(self.n, bool)
        G = heads // self.hkv
        for i, (nq, kv) in enumerate(self.lens):
            for h in range(self.hkv):
                K, V, there = self.keys_values(i, h)
                for t in range(nq):
                    tok, pos = int(self.q_start[i]) + t, kv - nq + t
                    rows[tok] = True
                    j = np.arange(len(K))
                    see = there & (j <= pos) & ((j > pos - window) if window else True)
                    if not see.any():
                        continue
                    y = self.rotated(q[tok, h * G:(h + 1) * G], tok, pos)
                    with np.errstate(invalid="ignore", over="ignore"):
                        s = y @ K[see].T * scale
                        A = np.abs(y) @ np.abs(K[see]).T * scale
                        w = np.exp(s - s.max(1, keepdims=True))
                        out[tok, h * G:(h + 1) * G] = w @ V[see] / w.sum(1, keepdims=True)
                        g = 2.0 ** -24 * (2 * self.dim + 16) * A.max(1) + 2.0 ** -21 * A.max(1)
                        g += 2.0 ** -24 * (4 * np.abs(s).max(1) + 400 + see.sum()) + 2.0 ** -20
                        tol[tok, h * G:(h + 1) * G] = 2 * g[:, None] * np.abs(V[see]).max()
        return out, tol, rows

    def device(self, torch, kq4):
        """A kq4.KVBatch of device copies."""
        up = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        return kq4.KVBatch(up(self.codes), up(self.scales), self.page, up(self.table), up(self.q_start), up(self.kv_len),
                           self.n, rope=up(self.rope), rope_pos=up(self.rope_pos))


def logprobs(x, token, n_top):
    """(logprob, entropy, top logprob, top id, bound) of logits x [n][vocab] (fp32), in 64 bits.

    The bound, absolute, for logprob and top_logprob, and times entropy + 1 for the entropy: z is a sum in a tree
    of at most 32 + 6 + 2 additions a piece and 6 + vocab / 2^19 over pieces, each off by 2^-24; each term's exponent is
    rounded at 2^-24 of at most 105 in nats (beyond, e^-d is 0 in fp32); x - m and the last subtractions are off by
    2^-24 of their results."""
    n, vocab = x.shape
    lp, ent = np.full(n, np.nan), np.zeros(n)
    tlp, tid, tol = np.zeros((n, n_top)), np.zeros((n, n_top), np.int64), np.zeros(n)
    for i in range(n):
        r = x[i].astype(np.float64)
        order = np.lexsort((np.arange(vocab), -np.where(np.isnan(r), np.inf, r), ~np.isnan(r)))[:n_top]
        tid[i] = order
        ok = 0 <= token[i] < vocab
        if np.isnan(r).any() or np.isposinf(r).any():
            ent[i], tlp[i] = np.nan, np.nan
            continue
        if np.isneginf(r).all():
            tlp[i] = -np.inf
            if ok:
                lp[i] = -np.inf
            continue
        at = int(r.argmax())
        d = r - r[at]
        e = np.exp(d)
        e[at] = 0
        lz = np.log1p(e.sum())
        p = np.exp(d - lz)
        ent[i] = lz - (p * np.where(np.isneginf(d), 0, d)).sum()
        if ok:
            lp[i] = d[token[i]] - lz
        tlp[i] = d[order] - lz
        far = np.abs(d[np.isfinite(d)]).max()
        tol[i] = 2.0 ** -24 * (64 + 2 * 105 + 2 * min(far, 1e6) + 4 * lz)
    return lp, ent, tlp, tid, tol
