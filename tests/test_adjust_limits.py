"""How many pieces of rows the logits-adjusting entry points take: as many as their declarations say. The matrices are NULL, which
is refused after the sizes, so that nothing is launched."""
import pytest

import gonngpu as G
from tests.test_int8_refusals import ADJUST, ADJUST_GRAD

# Columns to a piece, pieces below which a call has to stay; by the tokens of history.
SPLITS = [(0, 2048, 1 << 24), (1023, 2048, 1 << 24), (1024, 8192, 1 << 22), (5000, 8192, 1 << 22)]


@pytest.mark.parametrize("name,good", [("gn_adjust_logits", ADJUST), ("gn_adjust_logits_backward", ADJUST_GRAD)])
@pytest.mark.parametrize("h,piece,limit", SPLITS)
@pytest.mark.parametrize("pieces", [1, 2, 3, 5, 7, 16, 1000])
def test_pieces(name, good, h, piece, limit, pieces):
    most = (limit - 1) // pieces
    for cols in {(pieces - 1) * piece + 1, pieces * piece}:
        sizes = {k: cols for k in ("ld", "ldo", "ldg") if k in good}
        for rows, word in ((most, "NULL logits"), (most + 1, "too large")):
            rc, msg = G.call_rc(name, *{**good, **sizes, "cols": cols, "ldmask": -(-cols // 32), "h": h, "rows": rows, "x": None,
                                        "out": None, **({"g": None} if "g" in good else {})}.values())
            assert rc == -1 and (word in msg or (word == "NULL logits" and h == 0 and "NULL grad_out" in msg)), (rows, cols, msg)
