"""The paged cache's index arithmetic (csrc/kq4_kv.h), compiled for the host: whatever a batch's device arrays hold,
no index leaves the call's arrays or the cache, and the key ranges of splits cover what the queries see."""
import ctypes
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("kv") / "kv_layout.so")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-fPIC", "-shared",
                        os.path.join(ROOT, "tests", "c", "kv_layout.cpp"), "-o", so], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    h = ctypes.CDLL(so)
    h.t_group_at.restype = ctypes.c_long
    return h


def ints(n):
    return (ctypes.c_int * n)()


def test_spans_stay_in_the_call(lib):
    rng = random.Random(1)
    odd = [-(1 << 31), -5, 0, 1, 7, 63, 64, 65, 100, (1 << 31) - 1]
    for _ in range(20000):
        start, end, kv = (rng.choice(odd) for _ in range(3))
        n_tok, room = rng.choice([0, 1, 64, 100]), 16 * rng.choice([1, 4, 100])
        o = ints(6)
        lib.t_span(start, end, kv, n_tok, room, o)
        q0, nq, p0, length, first, groups = o
        assert 0 <= q0 <= n_tok and 0 <= nq <= n_tok - q0 and 0 <= length <= room
        assert p0 + nq == max(kv, 0) and length <= max(kv, 0)
        # every position of the touched groups that is new is a token of the call and a place of the table
        touched = sorted({p // 16 for p in range(max(p0, 0), length)}) if nq else []
        assert groups == len(touched) and (not touched or first == touched[0])
        assert groups <= min(nq, nq // 16 + 2)


def test_groups_of_bad_pages(lib):
    """Only pages of the cache are followed; the index stays below its groups."""
    rng = random.Random(2)
    for _ in range(5000):
        log_pg, pages, heads, width = rng.randint(0, 8), rng.choice([1, 3, 1000]), rng.choice([1, 3, 8]), rng.choice([1, 5])
        row = (ctypes.c_int * width)(*[rng.choice([-1, 0, pages - 1, pages, 1 << 30, -(1 << 31)]) for _ in range(width)])
        group, head = rng.randint(-2, (width + 1) << log_pg), rng.randrange(heads)
        got = lib.t_group_at(row, width, group, head, pages, heads, log_pg)
        slot = group >> log_pg
        if group < 0 or slot >= width or not 0 <= row[slot] < pages:
            assert got == -1
        else:
            assert got == ((row[slot] * heads + head) << log_pg) + group % (1 << log_pg)
            assert 0 <= got < pages * heads << log_pg
    row = (ctypes.c_int * 1)(1 << 29)                          # groups past 32 bits
    assert lib.t_group_at(row, 1, 3, 7, 1 << 30, 8, 2) == (((1 << 29) * 8 + 7) << 2) + 3


def test_what_a_query_sees(lib):
    for length in (0, 1, 16, 100):
        for p in list(range(-3, 20)) + [99, 100, 5000]:
            for window in (0, 1, 5, 16, 200, (1 << 31) - 1):
                o = ints(2)
                lib.t_sees(p, length, window, o)
                keys = [j for j in range(length) if j <= p and (window == 0 or j > p - window)]
                assert list(range(o[0], o[1])) == keys


def test_split_ranges_cover_the_keys(lib):
    rng = random.Random(3)
    for _ in range(4000):
        nq, kv = rng.randint(1, 90), rng.randint(0, 700)
        length, p0 = min(kv, 600), kv - nq
        t0 = rng.randrange(nq)
        t1 = rng.randrange(t0, nq)
        window, chunk, ns = rng.choice([0, 1, 40, 500]), 64 * rng.randint(1, 5), rng.randint(1, 9)
        o = ints(2)
        used = lib.t_ranges(nq, p0, length, t0, t1, window, chunk, ns, o)
        base, end = o
        assert 1 <= used <= ns and base % 64 == 0 and base >= 0 and end <= max(length, 0)
        seen = {j for t in range(t0, t1 + 1) for j in range(length)
                if j <= p0 + t and (window == 0 or j > p0 + t - window)}
        got = set()
        for s in range(used):
            b = base + s * chunk
            got |= set(range(b, end if s + 1 == used else b + chunk))
            assert s == 0 or b < end                           # no split without a key beside the first
        assert seen <= got


def test_parts_cover_a_range_and_fit_the_shares(lib):
    """Ranges by shares: of any number of turns they cover it without an empty one, a shorter range of the sequence has
    no more of them, and those of a batch fit the items that its launch has."""
    used = ints(1)
    for share in (1, 2, 3, 5, 7, 40):
        for most in (1, 2, 4, 9, 64):
            before = 1
            for turns in range(200):
                n = lib.t_parts(turns, share, most)
                assert before <= n <= max(1, min(most, -(-turns // share)))
                before = n
                part = lib.t_part(turns, n, used)
                assert 1 <= used[0] <= n and part >= 1
                assert part * used[0] >= turns and (used[0] == 1 or part * (used[0] - 1) < turns)
    rng = random.Random(3)
    for _ in range(3000):
        n_seq, shares = rng.randint(1, 64), rng.randint(1, 256)
        turns = [rng.choice([0, 1, 2, rng.randint(0, 500)]) for _ in range(n_seq)]
        share = max(1, -(-sum(turns) // shares))
        assert sum(lib.t_parts(t, share, 1000) for t in turns) <= shares + n_seq
