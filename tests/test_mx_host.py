"""The host side of the microscaled calls without a GPU, on the stand-in for the HIP runtime (tests/c/hip_standin.c):
what they refuse, launch and ask of the workspace; and the binding's refusals."""
import os
import subprocess
import sys

import pytest

import kq4
from test_workspace_routes import standin  # noqa: F401

SETUP = """
def quantize(m=at(1), x=at(2), ldx=512, rows=5, cols=512, type=4):
    return k.kq4_mx_quantize_dev(m, x, ldx, rows, cols, type, None)

def pack(m=at(1), codes=at(2), scales=at(3), rows=5, cols=512, type=4):
    return k.kq4_mx_pack_dev(m, codes, scales, rows, cols, type, None)

def unpack(codes=at(2), scales=at(3), m=at(1), rows=5, cols=512, type=4):
    return k.kq4_mx_unpack_dev(codes, scales, m, rows, cols, type, None)

def matmul(out=at(1), ldo=300, x=at(2), ldx=512, res=at(3), w=at(4), rows=300, cols=512, n=5, act=6):
    return k.kq4_mx_matmul_dev(out, ldo, x, ldx, res, w, rows, cols, n, act, None)

def matmul_q(out=at(1), ldo=300, xq=at(2), res=at(3), w=at(4), rows=300, cols=512, n=5, act=6):
    return k.kq4_mx_matmul_q_dev(out, ldo, xq, res, w, rows, cols, n, act, None)

def gated(out=at(1), ldo=300, x=at(2), ldx=512, gate=at(3), up=at(4), rows=300, cols=512, n=5, act=6):
    return k.kq4_mx_gated_dev(out, ldo, x, ldx, gate, up, rows, cols, n, act, None)

def ffn(out=at(1), ldo=512, x=at(2), ldx=512, res=at(3), gate=at(4), up=at(5), down=at(6), dim=512, ffn=320, n=5, act=6):
    return k.kq4_mx_ffn_dev(out, ldo, x, ldx, res, gate, up, down, dim, ffn, n, act, None)

def launched(f):
    hip.standin_clear()
    rc = f()
    return rc, len(hip.standin_log().decode().split("\\n")) - 1
"""


@pytest.mark.parametrize("call", [
    "quantize(m=None)", "quantize(m=at(1) + 8)", "quantize(x=None)", "quantize(x=at(2) + 4)", "quantize(ldx=508)",
    "quantize(ldx=514)", "quantize(ldx=-512)", "quantize(rows=-1)", "quantize(cols=0)", "quantize(cols=500)", "quantize(type=8)",
    "quantize(rows=1 << 24, cols=16384, ldx=16384)", "quantize(rows=(1 << 31) - 1)",
    "pack(m=None)", "pack(m=at(1) + 4)", "pack(codes=None)", "pack(scales=None)", "pack(codes=at(2) + 8)", "pack(rows=0)",
    "pack(cols=48)", "pack(type=0)", "unpack(m=None)", "unpack(codes=None)", "unpack(scales=None)", "unpack(type=-4)",
    "unpack(codes=at(2) + 1)",
    "matmul(out=None)", "matmul(out=at(1) + 2)", "matmul(ldo=299)", "matmul(ldo=-300)", "matmul(x=None)",
    "matmul(x=at(2) + 8)", "matmul(ldx=511)", "matmul(ldx=510)", "matmul(ldx=513)", "matmul(res=at(3) + 1)", "matmul(w=None)",
    "matmul(w=at(4) + 8)", "matmul(rows=0, ldo=0)", "matmul(rows=-4)", "matmul(cols=33, ldx=36)", "matmul(n=-1)",
    "matmul(n=(1 << 24) + 1)", "matmul(act=5)", "matmul(act=0)", "matmul(act=16)", "matmul(out=at(2))", "matmul(out=at(2) + 16)",
    "matmul(out=at(2) + 4 * 300, ldo=512)", "matmul(res=at(1) + 4)", "matmul(res=at(1) + 4 * 300)",
    "matmul(n=1 << 20, rows=1 << 24, ldo=1 << 24, cols=32, ldx=32, res=None)", "matmul_q(xq=None)", "matmul_q(xq=at(2) + 8)", "matmul_q(out=None)", "matmul_q(act=3)", "matmul_q(w=None)", "matmul_q(n=-5)",
    "matmul_q(ldo=10)", "matmul_q(res=at(1) + 4)",
    "gated(gate=None)", "gated(up=None)", "gated(gate=at(3) + 4)", "gated(up=at(4) + 4)", "gated(out=None)", "gated(x=None)",
    "gated(ldo=200)", "gated(out=at(2) + 64)", "gated(n=-1)", "gated(act=9)", "gated(rows=0)", "gated(cols=0)",
    "ffn(gate=None)", "ffn(up=None)", "ffn(down=None)", "ffn(down=at(6) + 8)", "ffn(ffn=300)", "ffn(ffn=0)", "ffn(dim=0)",
    "ffn(dim=500)", "ffn(ldo=500)", "ffn(out=at(2))", "ffn(act=1)", "ffn(x=None)", "ffn(out=None)", "ffn(n=-1)",
    "ffn(res=at(1) + 4)", "ffn(n=1 << 24, ffn=16384)",
    "quantize(m=at(2))", "quantize(m=at(2) + 16 * 512)", "quantize(x=at(1) + 16 * 256)", "pack(m=at(2))", "pack(scales=at(2) + 1279)",
    "pack(m=at(3))", "unpack(m=at(2) + 1264)", "unpack(scales=at(1) + 16 * 256 + 255)", "unpack(scales=at(2))",
    "matmul_q(out=at(2))", "matmul_q(out=at(2) + 16 * 384 + 252, res=None)", "matmul_q(xq=at(1) + 4 * 5 * 300 - 8 - 8)",
    "matmul_q(out=at(4))", "matmul(out=at(4) + 19 * 16 * 256, res=None)", "matmul(w=at(1) + 16, res=None)", "gated(out=at(3) + 64)",
    "gated(out=at(4))", "ffn(out=at(4), res=None)", "ffn(out=at(5) + 256, res=None)", "ffn(out=at(6), res=None)",
])
def test_refusals(standin, call):  # noqa: F811
    assert standin(SETUP + f"result = launched(lambda: {call})") == [-1, 0]


def test_nothing_to_do_launches_nothing(standin):  # noqa: F811
    calls = ["quantize(rows=0)", "matmul(n=0)", "matmul_q(n=0)", "gated(n=0)", "ffn(n=0)"]
    body = "result = [" + ", ".join(f"launched(lambda: {c})" for c in calls) + "]"
    assert standin(SETUP + body) == [[0, 0]] * len(calls)


def test_calls_that_are_taken(standin):  # noqa: F811
    """No residual, the residual in place, one row of any stride, columns of one wider tensor for x and out."""
    calls = ["matmul(res=None)", "matmul(res=at(1))", "matmul(out=at(2) + 4 * 512, ldo=1024, ldx=1024, res=None)",
             "matmul(x=at(1) + 4 * 304, ldx=816, ldo=816, res=None)", "gated(out=at(2) + 4 * 512, ldo=812, ldx=812)",
             "matmul(res=at(1) + 4 * 5 * 300)", "matmul_q(res=at(1))", "ffn(res=None)", "ffn(res=at(1))", "quantize(type=6)", "pack(type=6)",
             "unpack()", "quantize(m=at(2) + 5 * 512 * 4)", "quantize(x=at(1) + 17 * 256)", "pack(scales=at(2) + 1280)",
             "matmul_q(out=at(2) + 16 * 384 + 256)"]
    body = "result = [launched(f)[0] for f in (" + ", ".join(f"lambda: {c}" for c in calls) + ",)]"
    assert standin(SETUP + body) == [0] * len(calls)


@pytest.mark.parametrize("n", [1, 5, 40, 300, 2000])
@pytest.mark.parametrize("act", [4, 6])
def test_workspace_of_captured_calls(standin, n, act):  # noqa: F811
    """Calls that need the workspace: refused on a capturing stream that cannot grow it, done after a reservation of the
    bytes they name, also for smaller sizes than those reserved for."""
    res = standin(SETUP + """
calls = [lambda: matmul(n=n, act=act, rows=4096, ldo=4096, cols=12288, ldx=12288), lambda: gated(n=n, act=act), lambda: ffn(n=n, act=act),
         lambda: matmul_q(n=n, act=act, rows=70, ldo=70, cols=12288)]
hip.standin_capture(1)
before = [launched(f) for f in calls]
hip.standin_capture(0)
assert k.kq4_workspace_reserve(max(k.kq4_mx_workspace_bytes(n, 12288), k.kq4_mx_ffn_workspace_bytes(n, 512, 320))) == 0
hip.standin_capture(1)
after = [launched(f) for f in calls]
calls = [lambda m=m, r=r, c=c: matmul(n=m, act=act, rows=r, ldo=r, cols=c, ldx=c) for m in (n, (n + 1) // 2, 1) for r in (16, 1024, 151936)
         for c in (32, 4096, 12288)]
smaller = [launched(f)[0] for f in calls]
result = [before, after, smaller]
""", n=n, act=act)
    before, after, smaller = res
    for b, a in zip(before, after):
        assert b in ([-1, 0], a)          # refused whole or done whole
        assert a[0] == 0 and a[1] >= 1
    assert before[2] == [-1, 0]           # the block always has h between its launches
    assert smaller == [0] * len(smaller)


@pytest.mark.parametrize("shape,want", [
    ((1, 4096, 4096, "matmul"), ["rows"]), ((4, 4096, 4096, "matmul"), ["rows"]), ((9, 4096, 4096, "matmul"), ["quantize", "rows"]), ((1, 151936, 2048, "matmul"), ["rows"]),
    ((6, 151936, 2048, "matmul"), ["rows"]), ((8, 151936, 2048, "matmul"), ["quantize", "rows"]),
    ((16, 151936, 2048, "matmul"), ["quantize", "rows"]), ((64, 4096, 12288, "matmul"), ["quantize", "rows"]),
    ((256, 4096, 4096, "matmul"), ["quantize", "rows"]), ((768, 4096, 4096, "matmul"), ["quantize", "gemm"]),
    ((512, 4096, 12288, "matmul"), ["quantize", "gemm", "join"]), ((4096, 4096, 12288, "matmul"), ["quantize", "gemm"]),
    ((1, 12288, 4096, "gated"), ["rows"]), ((29, 6144, 2048, "gated"), ["quantize", "rows"]),
    ((2048, 12288, 4096, "gated"), ["quantize", "gemm"]), ((300, 1024, 512, "gated"), ["rows"]), ((40, 1024, 512, "gated"), ["rows"]), ((40, 6144, 2048, "gated"), ["quantize", "rows"]),
    ((1, 4096, 12288, "ffn"), ["rows", "rows"]), ((12, 4096, 12288, "ffn"), ["quantize", "rows", "quantize", "rows"]),
    ((2048, 4096, 12288, "ffn"), ["quantize", "gemm", "gemm"]),
])
def test_launches(standin, shape, want):  # noqa: F811
    """Which kernels a call takes on 256 CUs (6-bit activations): one launch for few tokens, h quantized in the GEMM."""
    res = standin(SETUP + """
n, rows, cols, kind = shape
hip.standin_clear()
far = dict(out=at(200), x=at(300))
rc = matmul(n=n, rows=rows, ldo=rows, cols=cols, ldx=cols, res=None, w=at(4), **far) if kind == "matmul" else \\
    gated(n=n, rows=rows, ldo=rows, cols=cols, ldx=cols, **far) if kind == "gated" else \\
    ffn(n=n, dim=rows, ffn=cols, ldo=rows, ldx=rows, res=None, **far)
result = [rc] + [s.split(" ")[0] for s in hip.standin_log().decode().split("\\n")[:-1]]
""", shape=shape)
    assert res[0] == 0
    assert [next(k for k in ("quantize", "rows", "gemm", "join") if "kq4_mx_" + k in s) for s in res[1:]] == want


def test_planner_options(standin):  # noqa: F811
    """mx_form and mx_split choose the form and the slices; a split that K does not have is the most that it has."""
    res = standin(SETUP + """
def names(**o):
    for k_, v in o.items():
        assert k.kq4_set_option(k_.encode(), v) == 0
    hip.standin_clear()
    rc = matmul(n=300, rows=600, ldo=600, cols=1536, ldx=1536, res=None, out=at(20))
    return [rc] + [s.split(" ")[0].split("kq4_mx_")[1][:4] + " " + s.split(" ")[1] for s in hip.standin_log().decode().split("\\n")[1:-1]]
result = [names(mx_form=1), names(mx_form=2, mx_split=1), names(mx_split=2), names(mx_split=99), names(mx_form=-1, mx_split=-1)]
""")
    assert [r[0] for r in res] == [0] * 5
    assert res[1][1:] == ["gemm 15"] and res[2][1:] == ["gemm 30", "join 300"] and res[3][1:] == ["gemm 45", "join 300"]
    assert len(res[0]) == 2 and res[0][1].startswith("rows") and res[4] == res[0]


def test_binding_refuses_host_tensors_and_shapes(kq4_cpu):
    import torch
    with pytest.raises(kq4_cpu.KQ4Error, match="device tensor"):
        kq4_cpu.MX(4, 64, 4, data=torch.zeros(4096, dtype=torch.uint8))
    with pytest.raises(kq4_cpu.KQ4Error, match="expected a 4-bit MX"):
        kq4_cpu.mx_matmul_dev(None, torch.zeros(1, 64), torch.zeros(4, 64))
    with pytest.raises(kq4_cpu.KQ4Error, match="expected an MX"):
        kq4_cpu.mx_matmul_q_dev(None, torch.zeros(1, 64), None)
    with pytest.raises(kq4_cpu.KQ4Error, match="expected a 4-bit MX"):
        kq4_cpu.mx_gated_dev(None, torch.zeros(1, 64), None, None)
    for call in (lambda: kq4_cpu.mx_quantize_dev(None, torch.zeros(1, 64)),
                 lambda: kq4_cpu.mx_pack_dev(None, torch.zeros(1, 32, dtype=torch.uint8), torch.zeros(1, 2, dtype=torch.uint8))):
        with pytest.raises(kq4_cpu.KQ4Error, match="expected an MX"):
            call()


def test_the_bindings_first_call_may_be_any():
    """Without a call before it that loads the library: the binding's own error."""
    code = ("import sys, torch; sys.path.insert(0, %r)\nimport kq4\n"
            "try: kq4.logprobs_dev(torch.zeros(2, 8))\nexcept kq4.KQ4Error as e: assert 'device' in str(e), e\nelse: assert 0\n"
            % os.path.dirname(kq4.__file__))
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300)
