"""Microscaled matrices without a GPU: the layout's index arithmetic and the choice of a block's scale (csrc/kq4_mx.h,
compiled for the host) against the plain form (mx_ref.py), and the plain form against the formats."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import mx_ref as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("mx") / "mx_layout.so")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-fPIC", "-shared",
                        os.path.join(ROOT, "tests", "c", "mx_layout.cpp"), "-o", so], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    h = ctypes.CDLL(so)
    h.t_size.restype = h.t_codes.restype = ctypes.c_size_t
    h.t_code_at.restype = h.t_scale_at.restype = ctypes.c_long
    return h


SHAPES = [(1, 32), (16, 128), (17, 160), (128, 512), (130, 544), (257, 1056), (40, 640)]


@pytest.mark.parametrize("bits", [4, 6])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_every_element_and_scale(lib, rows, cols, bits):
    rng = np.random.default_rng(rows + cols)
    codes = rng.integers(0, 1 << bits, (rows, cols), np.uint8)
    scales = rng.integers(0, 256, (rows, cols // 32)).astype(np.uint8)
    m = R.matrix(codes, scales, bits)
    assert m.size == lib.t_size(rows, cols, bits)
    for r in range(rows):
        for c in range(0, cols, 32):
            at = [lib.t_code_at(rows, cols, bits, r, c, y) for y in range(4 * bits)]
            assert at[0] % 16 == 0 and (bits == 4 or at[16] % 8 == 0)
            np.testing.assert_array_equal(m[at], R.row_major(codes[r:r + 1, c:c + 32], bits)[0])
            assert m[lib.t_scale_at(rows, cols, bits, r, c)] == scales[r, c // 32]


def test_sizes_past_32_bits(lib):
    rows, cols = 1 << 20, 16384
    assert lib.t_size(rows, cols, 4) == rows * cols // 2 + rows * cols // 32
    assert lib.t_code_at(rows, cols, 4, rows - 1, cols - 1, 15) == rows * cols // 2 - 1
    assert lib.t_scale_at(rows, cols, 4, rows - 1, cols - 1) == rows * cols // 2 + rows * cols // 32 - 1


@pytest.mark.parametrize("bits", [4, 6])
def test_scale_of_a_block(lib, bits):
    rng = np.random.default_rng(bits)
    edge = [(m * 2.0 ** e) for e in (-149, -140, -127, -126, -125, -119, -118, -117, -1, 0, 1, 100, 127)
            for m in (1, 1.25, 1.5, 1.74, 1.7499999, 1.75, 1.7500001, 1.875, 1.93, 1.9374999, 1.9375, 1.9375001, 1.9999999)]
    a = np.array([0.0] + [v for v in edge if v < 3.4028235e38], np.float32)
    a = np.concatenate([a, np.exp2(rng.uniform(-149, 127.9, 500)).astype(np.float32), np.float32([3.4028235e38])])
    x = np.zeros((a.size, 32), np.float32)
    x[:, 3] = a
    _, b = R.quantize(x, bits)
    for v, want in zip(a, b[:, 0]):
        got = lib.t_scale_byte(int(v.view(np.uint32)), bits)
        assert got == want, (v, got, want)
        assert np.uint32(lib.t_scale_bits(got)).view(np.float32) == np.exp2(float(got) - 127)
    assert lib.t_scale_byte(0x7f800000, bits) == lib.t_scale_byte(0x7fc00001, bits) == 255


@pytest.mark.parametrize("bits", [4, 6])
def test_no_element_is_off_by_more_than_half_a_step(bits):
    """What the scale's rule is for: relative to the element half of eps, or half of the least step."""
    rng = np.random.default_rng(7)
    x = (rng.standard_normal((400, 64)) * np.exp2(rng.integers(-130, 100, (400, 1)))).astype(np.float32)
    code, b = R.quantize(x, bits)
    v, s = R.values(code, b, bits), np.repeat(R.scale_values(b), 32, 1)
    half, least = (2.0 ** -2, 0.25) if bits == 4 else (2.0 ** -4, 2.0 ** -4)
    assert (np.abs(v - x) <= np.maximum(np.abs(x.astype(np.float64)) * half, least * s)).all()


def test_kq4_mx_bytes(kq4_cpu):
    f = kq4_cpu.lib().kq4_mx_bytes
    for rows, cols in SHAPES:
        nt, kt, kq = R.dims(rows, cols)
        for bits in (4, 6):
            assert f(rows, cols, bits) == nt * kt * 256 * bits + nt * kq * 256
    for bad in ((0, 32, 4), (-1, 32, 4), (1, 0, 4), (1, 31, 4), (1, 48, 6), (1, 32, 8), (1, -32, 4), (1 << 25, 32, 4),
                (1 << 24, 16384, 4), (16, (1 << 20) + 32, 4), ((1 << 31) - 1, 1 << 30, 6)):
        assert f(*bad) == 0
        with pytest.raises(kq4_cpu.KQ4Error):
            kq4_cpu.MX(*bad, device="cpu")
    assert kq4_cpu.mx_workspace_bytes(0, 64) == kq4_cpu.mx_workspace_bytes(1, 33) == 0
    assert kq4_cpu.mx_ffn_workspace_bytes(1, 64, 33) == kq4_cpu.mx_ffn_workspace_bytes(1, 0, 32) == 0
