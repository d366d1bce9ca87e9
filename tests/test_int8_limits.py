"""How large an int8 product may be: as large as its declaration says. B is NULL, which is refused after the sizes, so that nothing is
launched."""
import pytest

import gonngpu as G
from tests.test_int8_refusals import GEMM, LINEAR


@pytest.mark.parametrize("name,good", [("gn_int8_gemm", GEMM), ("gn_int8_linear", LINEAR)])
@pytest.mark.parametrize("across", [1, 3, 100, 8192, 1 << 21])
def test_blocks(name, good, across):
    most = min(16 * ((1 << 26) // across), 1 << 25)
    for n in {16 * across - 15, 16 * across}:
        for m, word in ((most, "NULL B"), (most + 1, "too large")):
            for M, N in ((m, n), (n, m)):
                rc, msg = G.call_rc(name, *{**good, "M": M, "N": N, "ldc": N, "A": 1 << 20, "B": None}.values() if name == "gn_int8_gemm"
                                    else {**good, "M": M, "N": N, "ldc": N, "B": None}.values())
                assert rc == -1 and word in msg, (M, N, msg)
