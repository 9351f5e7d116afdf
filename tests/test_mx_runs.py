"""What the microscaled GEMM loads of a matrix (csrc/kq4_mx.h kq4_mx_run, compiled for the host). The hardware's range
check compares a load's offset with the bytes left behind the scalar offset, so that must never pass the bytes."""
import ctypes
import os
import subprocess

import pytest

import mx_ref as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("mx") / "mx_run.so")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-fPIC", "-shared",
                        os.path.join(ROOT, "tests", "c", "mx_run.cpp"), "-o", so], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    h = ctypes.CDLL(so)

    def f(*args):
        o = (ctypes.c_long * 3)()
        h.t_run(*args, o)
        return tuple(o)
    return f


@pytest.mark.parametrize("bits", [4, 6])
@pytest.mark.parametrize("nt", list(range(1, 26)))
@pytest.mark.parametrize("cols", [32, 128, 160, 512, 544, 1024, 1536, 4096, 12288])
def test_runs_stay_in_the_matrix(run, nt, cols, bits):
    """Every run of a workgroup's two groups of row tiles, past the last group too, in every stage: the scalar offset
    is within the bytes; a run that starts in a tile of the matrix starts at that tile's byte; others have no bytes."""
    rows, (_, kt, kq) = 16 * nt - 3, R.dims(16 * nt, cols)
    size = nt * kt * 256 * bits + nt * kq * 256
    for scales, tile, stages, base in ((0, 256 * bits, kt, 0), (1, 256, kq, nt * kt * 256 * bits)):
        for t0 in range(0, nt + 8, 8):
            for off in range(0, 16 * tile, 1024):
                at, left, step = run(rows, cols, bits, scales, t0, off)
                assert 0 <= at <= size and left == size - at
                assert (stages - 1) * step <= left
                t = t0 + off // tile
                if t >= nt:
                    assert left == step == 0
                    continue
                group = t // 8 * 8
                held = min(8, nt - group)
                assert step == held * tile and at == base + group * stages * tile + (t - group) * tile + off % tile
                assert (stages - 1) * step < left


def test_matrix_past_31_bits(run):
    rows, cols = 1 << 20, 16384
    for t0 in (0, (1 << 16) - 8):
        at, left, step = run(rows, cols, 4, 0, t0, 1024)
        assert at == t0 * 128 * 1024 + 1024 and step == 8192
        assert left == min(rows * cols // 32 * 17 - at, (1 << 31) - 1)
