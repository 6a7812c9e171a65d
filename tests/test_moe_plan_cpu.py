"""Which kernel a grouped product takes (148 SMs where there is no GPU): the shapes of
moe_shapes.py reach every variant, so that a change of the rule cannot leave one untested."""
import pytest

from moe_shapes import NARROW, WIDE, plan
from mxfp4_b200 import capi


def even(N, name):
    return N - N % 16 if name == "swiglu" else N


@pytest.mark.parametrize("name", ["none", "swiglu"])
def test_shapes_reach_every_variant(name):
    """Wide: tiles of 128 and 256 weight rows, scale rows by TMA and by lines, several tiles a
    pair.  Narrow: 16 and 64 rows; K whole with one and several tiles a CTA, halved with several
    tiles, split four and eight ways."""
    wide, narrow = set(), set()
    for E, M, N, K in WIDE:
        rows, n, ranks, tiles, clusters = plan(E, M, even(N, name), K, name)
        assert rows == 256 and ranks == 1
        if M // rows * -(-even(N, name) // n) > clusters:  # tiles of an even split, at least
            wide.add((n, K % 512 == 0))
    assert wide == {(n, tma) for n in (128, 256) for tma in (True, False)}
    for E, M, N, K in NARROW:
        rows, n, ranks, tiles, clusters = plan(E, M, even(N, name), K, name)
        assert n == (256 if name == "swiglu" else 128)
        narrow.add((rows, ranks, tiles > clusters))
    assert narrow >= {(rows, *v) for rows in (16, 64) for v in ((1, False), (1, True), (2, True), (4, False), (8, False))}


def test_a_quantized_result_splits_k_less():
    """A quantized block of 32 columns has one owner: at most four CTAs split K."""
    assert plan(1, 60, 336, 7200)[2] == 8
    assert plan(1, 60, 352, 7200, quantized=True)[2] == 4


@pytest.mark.parametrize("E,M,N,K,act", [(0, 1, 64, 32, 0), (513, 1, 64, 32, 0), (1, 0, 64, 32, 0), (1, 1, 60, 32, 0),
                                         (1, 1, 72, 32, 6), (1, 1, 64, 48, 0), (1, 1, 64, 32, 7), (4, 1, 1 << 30, 32, 0)])
def test_refusals(E, M, N, K, act):
    import ctypes
    out = (ctypes.c_int64 * 5)()
    assert capi.status_of("mxb_grouped_gemm_plan", M, E, N, K, act, 0, 1, out) == 1
    assert "grouped_gemm_plan" in capi.last_error()
    assert capi.status_of("mxb_grouped_gemm_plan", 1, 1, 64, 32, 0, 0, 1, None) == 1
