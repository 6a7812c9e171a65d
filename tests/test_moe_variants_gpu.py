"""The MXFP4 expert operators at the ends of their ranges and through every variant of their
kernels, against plain 64-bit forms."""
import pytest
import torch

import helpers as H
import moe_ref as R
from moe_shapes import NARROW, WIDE, plan
from mxfp4_b200 import capi
from omo_python_api import mxfp4_moe as moe
from test_moe_gpu import act_grad_ref, check_wgrad, dev, randn, splits_of, weights

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.fixture(autouse=True)
def _no_wait_gave_up(cuda):
    yield
    torch.cuda.synchronize()
    assert capi.reset_wait_timeouts() == 0


@pytest.mark.parametrize("name", R.ACTS)
def test_slopes_of_large_values(cuda, name):
    """|z| from 16 to 2^126, where the slopes are 0, 1, 2 z or (swiglu) one half times the other.
    One rounding to BF16 (2^-9 of the value, 2^-8 allowed); a logistic below 2^-126 is 0, which
    leaves at most 88 * 2^-126 times the other half (here at most 3) of a tail: 4e-36."""
    big = torch.exp2(torch.arange(4, 127).double())
    big = torch.cat((big, -big, 1.37 * big[:-1], -1.37 * big[:-1]))
    big = torch.cat((big, big[:-big.numel() % 64])).reshape(-1, 64).to(BF).cuda()
    pre = big
    if name == "swiglu":
        other = torch.tensor([1.25, -3.0], device=cuda).repeat(32).to(BF).expand_as(big)
        pre = torch.cat((torch.cat((big, other), 1), torch.cat((other, big), 1)))
    dy = torch.ones(pre.shape[0], 64, dtype=BF, device=cuda)
    got = moe.omo_bias_act_grad(dy, pre, None, name, bias_grad=False)
    want = act_grad_ref(dy, pre, name)
    R.check(got, want, 2.0 ** -8 * want.abs() + 4e-36)


# ---------------------------------------------------------------- the grouped product's kernels
def grouped_case(E, M, N, K, name, seed=0):
    gated = name == "swiglu"
    N -= N % 16 if gated else 0
    seed += E + M + N + K
    splits = splits_of(E, M, seed, empty=(1,) if E > 2 else ())
    ac, asc = R.mxfp4(M, K, seed)
    bc, bs, bt = weights(E, N, K, seed + 1, gated)
    return N, N // 2 if gated else N, splits, ac, asc, bc, bs, bt


def check_grouped(cuda, E, M, N, K, name):
    N, W, splits, ac, asc, bc, bs, bt = grouped_case(E, M, N, K, name)
    m, quantize = dev(splits), W % 32 == 0
    bias = randn(E, N, seed=2, dtype=torch.float32 if N % 32 else BF)
    res = randn(M, W, seed=3)
    out = moe.omo_grouped_gemm_mxfp4(ac, asc, bc, bt, m, bias=bias, activation=name, residual=res, save_pre=True,
                                     quantize=quantize)
    z, y, bz, by = R.grouped(ac, asc, bc, bs, splits, bias, name, res)
    R.check(out[1], z, bz, "pre")
    R.check(out[0], y, by, "c")
    if quantize:
        q, s = H.quant_rows(out[0])
        assert torch.equal(out[2], q) and torch.equal(out[3], s)
    alone = moe.omo_grouped_gemm_mxfp4(ac, asc, bc, bt, m, activation=name)
    _, y, _, by = R.grouped(ac, asc, bc, bs, splits, None, name, None)
    R.check(alone, y, by, "c alone")
    again = moe.omo_grouped_gemm_mxfp4(ac, asc, bc, bt, m, activation=name)
    assert torch.equal(again.view(torch.int16), alone.view(torch.int16)), "a second call differs"


@pytest.mark.parametrize("name", R.ACTS)
@pytest.mark.parametrize("E,M,N,K", WIDE)
def test_wide(cuda, E, M, N, K, name):
    check_grouped(cuda, E, M, N, K, name)


@pytest.mark.parametrize("name", ["none", "gelu", "swiglu"])
@pytest.mark.parametrize("E,M,N,K", NARROW)
def test_narrow(cuda, E, M, N, K, name):
    check_grouped(cuda, E, M, N, K, name)


@pytest.mark.parametrize("E,M,N,K", [WIDE[1], WIDE[3], NARROW[0], NARROW[1], NARROW[6]])
def test_nan_scales_stay_in_their_row_in_later_tiles(cuda, E, M, N, K):
    """E8M0 bytes 255 in the last step of rows and weight rows all over the tiles."""
    N, _, splits, ac, asc, bc, bs, _ = grouped_case(E, M, N, K, "none")
    asc[::37, K // 32 - 1] = 255
    bs[:, 5::211, K // 32 - 1] = 255
    c = moe.omo_grouped_gemm_mxfp4(ac, asc, bc, moe.omo_swizzle_scales_grouped(bs), dev(splits))
    _, y, _, by = R.grouped(ac, asc, bc, bs, splits, None, "none", None)
    R.check(c, y, by)


@pytest.mark.parametrize("E,M,N,K", [WIDE[0], WIDE[2], NARROW[2], NARROW[5]])
def test_scale_rows_by_lines_are_those_of_tma(cuda, E, M, N, K):
    """The same sizes with scale rows at any address, 256 weight rows a tile among them, give the
    bytes of aligned ones."""
    N, _, splits, ac, asc, bc, _, bt = grouped_case(E, M, N, K, "none")
    if (E, M, N, K) == WIDE[2]:
        assert plan(E, M, N, K, aligned=False)[:2] == plan(E, M, N, K, aligned=True)[:2] == (256, 256)
    want = moe.omo_grouped_gemm_mxfp4(ac, asc, bc, bt, dev(splits))
    n = sum(splits)
    for pad, off in ((3, 1), (4, 4), (16, 16), (0, 15)):
        big = torch.full((M, K // 32 + pad + off), 255, dtype=torch.uint8, device=cuda)
        big[:, off:off + K // 32] = asc
        got = moe.omo_grouped_gemm_mxfp4(ac, big[:, off:off + K // 32], bc, bt, dev(splits))
        assert torch.equal(got[:n].view(torch.int16), want[:n].view(torch.int16))


# ---------------------------------------------------------------- weight gradient: many tiles a pair
@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("E,M,N,K,empty", [(5, 1500, 1032, 1056, (2,)), (8, 3000, 2056, 1056, (0, 4, 7)),
                                           (2, 700, 4104, 2080, ())])
def test_wgrad_many_tiles(cuda, E, M, N, K, empty, dtype):
    """More 256 x 256 tiles than pairs of SMs, several 64-row steps each, experts without rows
    between them."""
    assert E * -(-N // 256) * -(-K // 256) > 74
    splits = splits_of(E, M, M + N, empty=empty)
    xc, xs = R.mxfp4(M, K, 1)
    dy = randn(M, N, seed=2, scale=0.1)
    dw = moe.omo_grouped_wgrad_mxfp4(dy, xc, xs, dev(splits), out_dtype=dtype)
    check_wgrad(dw, dy, xc, xs, splits)
    assert torch.equal(moe.omo_grouped_wgrad_mxfp4(dy, xc, xs, dev(splits), out_dtype=dtype), dw)
    if dtype == torch.float32:
        base = randn(E, N, K, seed=3, dtype=torch.float32)
        acc = base.clone()
        moe.omo_grouped_wgrad_mxfp4(dy, xc, xs, dev(splits), accumulate_into=acc)
        check_wgrad(acc, dy, xc, xs, splits, base)


@pytest.mark.parametrize("E,M,N,K", [(3, 90, 72, 96), (3, 700, 520, 544), (4, 900, 2056, 1536)])
def test_wgrad_strided_rows(cuda, E, M, N, K):
    """dy with a pitch above N, codes and scales side by side in wire rows: the same bytes as
    contiguous ones."""
    splits = splits_of(E, M, 5)
    xc, xs = R.mxfp4(M, K, 1)
    dy = randn(M, N, seed=2)
    wire = torch.full((M, (17 * K // 32 + 15) // 16 * 16), 255, dtype=torch.uint8, device=cuda)
    wire[:, :K // 2], wire[:, K // 2:17 * K // 32] = xc, xs
    big = torch.full((M, N + 24), float("nan"), dtype=BF, device=cuda)
    big[:, 8:8 + N] = dy
    want = moe.omo_grouped_wgrad_mxfp4(dy, xc, xs, dev(splits))
    got = moe.omo_grouped_wgrad_mxfp4(big[:, 8:8 + N], wire[:, :K // 2], wire[:, K // 2:17 * K // 32], dev(splits))
    assert torch.equal(got, want)
    check_wgrad(got, dy, xc, xs, splits)


# ---------------------------------------------------------------- epilogue gradient: 128 rows a CTA
@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("name", ["none", "gelu", "swiglu"])
def test_bias_act_grad_many_rows(cuda, name, quantize):
    """Enough rows and columns for chunks of 128 rows (fewer take 32), over uneven experts.  Bounds
    as in test_bias_act_grad; a bias gradient adds up to 4100 terms, 2^-18 of their sizes."""
    E, M = 5, 4100
    N = 5120 if name == "swiglu" else 2560
    W = N // 2 if name == "swiglu" else N
    ws = capi.load().mxb_bias_act_grad_workspace(M, E, N)
    assert ws == (M // 128 + E) * N * 4
    splits = splits_of(E, M, 11, empty=(2,))
    dy, pre = randn(M, W, seed=1), randn(M, N, seed=2, scale=2.0)
    out = moe.omo_bias_act_grad(dy, pre, dev(splits), name, quantize=quantize)
    want = act_grad_ref(dy, pre, name)
    mag = torch.cat((dy, dy), -1).double().abs() if name == "swiglu" else dy.double().abs()
    mag = mag * (R.slope_bound(pre.double(), name) + pre.double().abs() + 1)
    R.check(out[0], want, 2.0 ** -8 * want.abs() + 2.0 ** -18 * mag)
    for e, (i, j) in enumerate(R.spans(splits, M)):
        R.check(out[1][e], want[i:j].sum(0), 2.0 ** -18 * mag[i:j].sum(0) + 1e-40, f"bias of {e}")
    if quantize:
        q, s = H.quant_rows(out[0])
        assert torch.equal(out[2], q) and torch.equal(out[3], s)


# ---------------------------------------------------------------- results that the caller allocates
def test_extension_forms_with_outputs_given(cuda):
    """The operators of the extension that write into given tensors, against the wrappers."""
    import omo
    M, N, E = 700, 256, 3
    dy, pre, m = randn(M, N // 2, seed=1), randn(M, N, seed=2), dev([300, 0, 400])
    want = moe.omo_bias_act_grad(dy, pre, m, "swiglu", quantize=True)
    got = [torch.empty_like(t) for t in want]
    work = torch.empty(omo.omo_bias_act_grad_workspace(M, E, N), dtype=torch.uint8, device=cuda)
    omo.omo_bias_act_grad(dy, pre, m, E, N, capi.ACTIVATIONS["swiglu"], got[0], got[2], got[3], got[1], work)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    T, k = 50, 3
    y, dout, w = randn(T * k, N, seed=3), randn(T, N, seed=4), torch.rand(T, k, device=cuda)
    at = torch.randperm(T * k, device=cuda).to(torch.int32).reshape(T, k)
    out = torch.empty(T, N, dtype=BF, device=cuda)
    omo.omo_moe_unpermute(y, at, w, k, out)
    assert torch.equal(out, moe.omo_moe_unpermute(y, at, w))
    want = moe.omo_moe_unpermute_grad(dout, y, at, w, quantize=True)
    got = [torch.empty_like(t) for t in want]
    omo.omo_moe_unpermute_grad(dout, y, T * k, at, w, k, got[0], got[2], got[3], got[1])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
