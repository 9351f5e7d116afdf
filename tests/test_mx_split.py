"""The microscaled GEMM's K slices as the option mx_split asks for them, on the stand-in for the HIP runtime."""
import pytest

from test_mx_host import SETUP
from test_workspace_routes import standin  # noqa: F401


@pytest.mark.parametrize("want,slices", [(1, 1), (2, 2), (3, 3), (99, 3), (100000, 3), (1 << 24, 3), ((1 << 31) - 1, 3)])
def test_a_split_that_k_does_not_have_is_the_most_that_it_has(standin, want, slices):  # noqa: F811
    res = standin(SETUP + """
assert k.kq4_set_option(b"mx_form", 2) == 0 and k.kq4_set_option(b"mx_split", want) == 0
hip.standin_clear()
rc = matmul(n=300, rows=600, ldo=600, cols=1536, ldx=1536, res=None, out=at(20))
result = [rc] + [s.split(" ")[1] for s in hip.standin_log().decode().split("\\n") if "kq4_mx_gemm" in s]
""", want=want)
    assert res == [0, str(15 * slices)]
