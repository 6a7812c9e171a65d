"""CPU-only contracts of the MXFP4 expert entry points: out-of-contract calls are refused with
a status and a message before any CUDA call, and empty ones do nothing."""
import ctypes

import pytest

from mxfp4_b200 import capi

A = 4096  # an aligned stand-in for a device pointer (never read)


def gemm(a=A, ap=64, s=A, sp=4, M=8, m=A, E=2, b=A, bs=A, N=64, K=128, c=A, ep="default", **epi):
    e = None
    if ep == "default":
        e = ctypes.byref(capi.Epilogue(**{"c_ld": 64, **epi}))
    return ("mxb_grouped_gemm_mxfp4", (a, ap, s, sp, M, m, E, b, bs, N, K, e, c, None))


def wgrad(dy=A, ld=64, x=A, xp=64, s=A, sp=4, M=8, m=A, E=2, N=64, K=128, dw=A, f32=1, acc=0):
    return ("mxb_grouped_wgrad_mxfp4", (dy, ld, x, xp, s, sp, M, m, E, N, K, dw, f32, acc, None))


def grad(dy=A, pre=A, M=8, m=A, E=2, N=64, act=3, dz=A, q=None, s=None, db=A, w=None, wb=0):
    return ("mxb_bias_act_grad", (dy, pre, M, m, E, N, act, dz, q, s, db, w, wb, None))


def unp(y=A, R=16, H=64, m=A, mp=2, k=2, w=A, T=8, out=A):
    return ("mxb_moe_unpermute", (y, R, H, m, mp, k, w, T, out, None))


def unpg(d=A, y=A, R=16, H=64, m=A, mp=2, k=2, w=A, T=8, dy=A, q=None, s=None, dw=A):
    return ("mxb_moe_unpermute_grad", (d, y, R, H, m, mp, k, w, T, dy, q, s, dw, None))


@pytest.mark.parametrize("call,status,needle", [
    (gemm(ep=None), 1, "epilogue"),
    (gemm(activation=7), 1, "activation"),
    (gemm(activation=-1), 1, "activation"),
    (gemm(M=-1), 1, "M"),
    (gemm(E=0), 1, "E"),
    (gemm(E=513), 1, "E"),
    (gemm(N=60), 1, "N"),
    (gemm(N=72, activation=6), 1, "N"),
    (gemm(K=96 + 16), 1, "K"),
    (gemm(K=0), 1, "K"),
    (gemm(N=1 << 30, E=4), 1, "E * N"),
    (gemm(a=None), 1, "null"),
    (gemm(m=None), 1, "null"),
    (gemm(c=None), 1, "no output"),
    (gemm(c_codes=A), 1, "quantized"),
    (gemm(c_codes=A, c_scales=A, N=72, c_ld=72), 1, "quantized"),
    (gemm(ap=63), 1, "pitch"),
    (gemm(sp=3), 1, "pitch"),
    (gemm(c_ld=56), 1, "pitch"),
    (gemm(residual=A, residual_ld=8), 1, "pitch"),
    (gemm(pre=A, pre_ld=8), 1, "pitch"),
    (gemm(a=A + 8), 2, "aligned"),
    (gemm(ap=72), 2, "aligned"),
    (gemm(c=A + 2), 2, "aligned"),
    (gemm(c_ld=68), 2, "multiples of 8"),
    (gemm(bias=A + 1), 2, "bias"),
    (wgrad(N=60), 1, "N"),
    (wgrad(K=48), 1, "K"),
    (wgrad(E=513), 1, "E"),
    (wgrad(f32=0, acc=1), 4, "accumulates"),
    (wgrad(dw=None), 1, "null"),
    (wgrad(dy=None), 1, "null"),
    (wgrad(m=None), 1, "null"),
    (wgrad(ld=56), 1, "pitch"),
    (wgrad(xp=63), 1, "pitch"),
    (wgrad(ld=68), 2, "aligned"),
    (wgrad(x=A + 4), 2, "aligned"),
    (grad(act=9), 1, "activation"),
    (grad(N=60), 1, "N"),
    (grad(N=72, act=6), 1, "N"),
    (grad(q=A), 1, "quantized"),
    (grad(q=A, s=A, N=96, act=6), 1, "quantized"),
    (grad(dz=None, db=None), 1, "no output"),
    (grad(pre=None), 1, "null"),
    (grad(m=None), 1, "null"),
    (grad(M=513), 1, "workspace"),
    (grad(dy=A + 8), 2, "aligned"),
    (unp(H=60), 1, "H"),
    (unp(k=0), 1, "topk"),
    (unp(mp=1), 1, "map_pitch"),
    (unp(k=1025, mp=2000), 1, "topk"),
    (unp(y=None), 1, "null"),
    (unp(out=A + 8), 2, "aligned"),
    (unpg(H=40, q=A, s=A), 1, "quantized"),
    (unpg(dy=None, dw=None), 1, "no output"),
    (unpg(y=None), 1, "null"),
    (unpg(dy=A + 2), 2, "aligned"),
    (("mxb_swizzle_scales_grouped", (A, 2, 7, 4, 2, A, None)), 1, "parts"),
    (("mxb_swizzle_scales_grouped", (A, 2, 8, 4, 3, A, None)), 1, "parts"),
    (("mxb_swizzle_scales_grouped", (None, 2, 8, 4, 1, A, None)), 1, "null"),
    (("mxb_swizzle_scales_grouped", (A, 2, 8, 4, 1, A + 4, None)), 2, "aligned"),
])
def test_refused_before_any_cuda_call(call, status, needle):
    assert capi.status_of(call[0], *call[1]) == status, capi.last_error()
    assert needle in capi.last_error(), capi.last_error()
    assert "CUDA" not in capi.last_error()


@pytest.mark.parametrize("call", [gemm(M=0, a=None), gemm(N=0), wgrad(N=0), wgrad(K=0),
                                  wgrad(M=0, acc=1), grad(N=0), grad(M=0, db=None), unp(T=0),
                                  unp(H=0), unpg(T=0)])
def test_empty_calls_do_nothing(call):
    assert capi.status_of(call[0], *call[1]) == 0, capi.last_error()


def test_workspace_size():
    f = capi.load().mxb_bias_act_grad_workspace
    assert f(512, 8, 4096) == 0          # a cluster has an expert's rows: no partial sums
    assert f(513, 8, 4096) == (16 + 8) * 4096 * 4
    assert f(16384, 8, 4096) == (128 + 8) * 4096 * 4


def test_expert_order():
    """Rows sorted by expert, tokens in order within an expert; empty experts have no rows."""
    import torch
    from mxfp4_b200.moe import expert_order
    idx = torch.tensor([[2, 0], [0, 3], [2, 3], [3, 0]])
    dst, splits = expert_order(idx, 5)
    assert splits.tolist() == [3, 0, 2, 3, 0] and splits.dtype == torch.int32
    assert dst.tolist() == [[3, 0], [1, 5], [4, 6], [7, 2]] and dst.dtype == torch.int32
