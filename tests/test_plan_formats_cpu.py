"""The plans of products with 4-bit operands, without a GPU: K-blocks of 256 elements where both operands are E2M1, the even-rows form from
48 or 64 weight rows per CTA where one is; every element of C covered once, and scratch that serves whatever formats a call has."""
import pytest

from hipkittensp_b200 import _lib
from hipkittensp_b200._lib import E2M1, E2M3, E4M3, debug_plan
from tests.test_plan_cpu import SHAPES, SM, _cover_pair, _cover_single

PAIRS = [(E2M1, E2M1), (E4M3, E2M1), (E2M1, E4M3), (E2M3, E2M3)]
MORE = [(16, 20480, 8192), (16, 14336, 4096), (3, 14400, 512), (16, 19500, 4224), (32, 15001, 1024), (1, 28672, 256), (16, 512, 8192), (64, 38400, 1024), (16, 640, 128)]


@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("shape", SHAPES + MORE)
def test_plan_covers_c_exactly_once(shape, pair):
    M, N, K = shape
    pl = debug_plan(M, N, K, SM, fmt_a=pair[0], fmt_b=pair[1])
    assert 1 <= pl["grid"] <= SM * pl["ctas"]
    if pl["ctas"] == 2:
        least = 80 if E2M1 not in pair else 48 if K <= 4096 else 64
        assert pl["swap"] and not pl["streamk"] and pl["bn"] <= 32 and least <= pl["p_tile"] <= 128
    cover = _cover_pair(pl, M, N)[0] if pl["pair"] else _cover_single(pl, M, N)
    assert (cover == 1).all()
    assert (pl["scratch"] > 0) == bool(pl["streamk"])


def test_even_rows_form_of_4_bit_operands():
    for shape in ((16, 20480, 8192), (16, 14336, 4096)):
        for pair in PAIRS[:3]:
            pl = debug_plan(*shape, SM, fmt_a=pair[0], fmt_b=pair[1])
            assert pl["ctas"] == 2 and not pl["streamk"] and pl["p_tile"] == -(-shape[1] // (2 * SM))
        assert debug_plan(*shape, SM)["streamk"]                                 # the wider formats keep their rule
    assert debug_plan(16, 14336, 8192, SM, fmt_a=E2M1)["streamk"]                 # 49 rows, long K


def test_split_work_follows_the_longer_k_blocks():
    """K = 8192: 64 K-blocks of 128 elements or 32 of 256, four a CTA at least."""
    assert debug_plan(16, 512, 8192, SM)["grid"] == 64 and debug_plan(16, 512, 8192, SM, fmt_a=E2M1)["grid"] == 32
    assert debug_plan(16, 512, 8192, SM, fmt_a=E4M3, fmt_b=E2M1)["grid"] == 64
    assert debug_plan(16, 512, 384, SM, fmt_a=E2M1)["grid"] == 2                  # 1.5 blocks of 256 count as two


@pytest.mark.parametrize("sm", [148, 132, 16])
def test_reported_workspace_serves_every_format_and_result(sm):
    for shape in SHAPES + MORE:
        needs = [debug_plan(*shape, sm, requant=r, fmt_a=a, fmt_b=b) for a, b in PAIRS for r in (False, True)]
        assert max(p["scratch"] for p in needs) == needs[0]["workspace"]


def test_bad_formats_are_refused():
    for pair in ((5, 0), (0, -1)):
        with pytest.raises(_lib.Mxfp6Error):
            debug_plan(16, 512, 512, SM, fmt_a=pair[0], fmt_b=pair[1])
