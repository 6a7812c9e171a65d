"""The MXFP4 expert operators through their public wrappers, against plain 64-bit forms:
grouped and dense products with the epilogue, weight gradients, the epilogue's gradient, the
weighted unpermute and its gradient, and the expert layer that runs them together."""
import math

import pytest
import torch

import helpers as H
import moe_ref as R
from mxfp4_b200 import capi
from omo_python_api import mxfp4_moe as moe

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.fixture(autouse=True)
def _no_wait_gave_up(cuda):
    yield
    torch.cuda.synchronize()
    assert capi.reset_wait_timeouts() == 0


def splits_of(E, M, seed, empty=()):
    g = torch.Generator().manual_seed(seed)
    p = torch.rand(E, generator=g) + 0.1
    for e in empty:
        p[e] = 0
    m = torch.bincount(torch.multinomial(p, M, replacement=True, generator=g), minlength=E)
    return m.tolist()


def dev(splits):
    return torch.tensor(splits, dtype=torch.int32, device="cuda")


def randn(*shape, seed, scale=1.0, dtype=BF):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def weights(E, N, K, seed, gated):
    bc, bs = R.mxfp4((E, N), K, seed, 112, 120)
    return bc, bs, moe.omo_swizzle_scales_grouped(bs, gated)


# every kernel: few rows an expert (16- and 64-row tiles, alone and splitting K), many (wide
# tiles of 128 and, with long K or scale rows that TMA cannot take, 256 weight rows)
GROUPED = [
    # E, M, N, K
    (1, 1, 64, 32),
    (8, 9, 512, 2048),
    (5, 1, 80, 160),
    (3, 40, 272, 96),
    (40, 37, 48, 7168),
    (1, 16, 1000, 288),
    (2, 100, 176, 1056),
    (3, 259, 336, 64),
    (1, 130, 2064, 512),
    (2, 1000, 4400, 96),
    (1, 200, 19200, 256),
    (5, 3001, 1424, 544),
    (1, 30, 1032, 2048),
    (1, 60, 336, 7200),
    (3, 300, 72, 9216),
    (3, 2600, 2600, 4096),
    (4, 2000, 4400, 2080),
    (2, 1500, 4400, 3712),
]


@pytest.mark.parametrize("name", R.ACTS)
@pytest.mark.parametrize("E,M,N,K", GROUPED)
def test_grouped(cuda, E, M, N, K, name):
    gated = name == "swiglu"
    N -= N % 16 if gated else 0
    W = N // 2 if gated else N
    seed = E + M + N + K + len(name)
    splits = splits_of(E, M, seed, empty=(0,) if E > 2 else ())
    ac, asc = R.mxfp4(M, K, seed)
    bc, bs, bt = weights(E, N, K, seed + 1, gated)
    bias = randn(E, N, seed=seed + 2, dtype=torch.float32 if seed % 2 else BF)
    res = randn(M, W, seed=seed + 3) if seed % 3 else None
    c, pre = moe.omo_grouped_gemm_mxfp4(ac, asc, bc, bt, dev(splits), bias=bias, activation=name,
                                        residual=res, save_pre=True)
    z, y, bz, by = R.grouped(ac, asc, bc, bs, splits, bias, name, res)
    R.check(pre, z, bz, "pre")
    R.check(c, y, by, "c")
    # the result alone, without bias and residual
    c2 = moe.omo_grouped_gemm_mxfp4(ac, asc, bc, bt, dev(splits), activation=name)
    _, y, _, by = R.grouped(ac, asc, bc, bs, splits, None, name, None)
    R.check(c2, y, by, "c alone")
    again = moe.omo_grouped_gemm_mxfp4(ac, asc, bc, bt, dev(splits), activation=name)
    assert torch.equal(again.view(torch.int16), c2.view(torch.int16)), "a second call differs"


@pytest.mark.parametrize("name", ["none", "gelu", "swiglu"])
@pytest.mark.parametrize("E,M,W,K", [(4, 30, 96, 1024), (2, 90, 160, 288), (3, 1500, 2368, 128),
                                     (3, 2600, 1312, 4096)])
def test_quantized_result_is_the_quantizer_on_c(cuda, E, M, W, K, name):
    N = 2 * W if name == "swiglu" else W
    splits = splits_of(E, M, W + M)
    ac, asc = R.mxfp4(M, K, 5)
    bc, bs, bt = weights(E, N, K, 6, name == "swiglu")
    c, q, s = moe.omo_grouped_gemm_mxfp4(ac, asc, bc, bt, dev(splits), activation=name, quantize=True)
    rq, rs = H.quant_rows(c)
    assert torch.equal(q, rq) and torch.equal(s, rs)
    q2, s2 = moe.omo_grouped_gemm_mxfp4(ac, asc, bc, bt, dev(splits), activation=name, quantize=True,
                                        bf16_out=False)
    assert torch.equal(q2, rq) and torch.equal(s2, rs)


@pytest.mark.parametrize("M", [4, 3000])
@pytest.mark.parametrize("name", R.ACTS)
def test_activations_alone(cuda, M, name):
    """Zero operands leave the bias: act(z) over z in [-80, 80], the tails included, against the
    64-bit formula without cancellation.  One rounding to BF16 (2^-9, 2^-8 allowed) and the f32
    evaluation (2^-16: an exponent of up to 115 rounded to f32); below 1e-36 f32 may underflow."""
    W = 4096
    gated = name == "swiglu"
    z = torch.cat((torch.linspace(-80, 80, W // 2), torch.linspace(-6, 6, W // 2))).cuda()
    bias = torch.cat((z, torch.linspace(-3, 3, W).cuda())) if gated else z
    N = bias.numel()
    ac = torch.zeros(M, 16, dtype=torch.uint8, device=cuda)
    asc = torch.full((M, 1), 127, dtype=torch.uint8, device=cuda)
    bc = torch.zeros(N, 16, dtype=torch.uint8, device=cuda)
    bt = moe.omo_swizzle_scales_grouped(torch.full((1, N, 1), 127, dtype=torch.uint8, device=cuda), gated)
    c = moe.omo_gemm_mxfp4_act(ac, asc, bc, bt[0], bias=bias, activation=name)
    d = bias.double()
    want = 0.5 * d * torch.special.erfc(-d / math.sqrt(2)) if name == "gelu" else \
        d * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (d + 0.044715 * d ** 3)) if name == "gelu_tanh" else R.act(d, name)
    R.check(c, want.expand(M, -1), (2.0 ** -8 + 2.0 ** -16) * want.abs().expand(M, -1) + 1e-36)


@pytest.mark.parametrize("M,N,K", [(1, 7168, 2048), (77, 1000, 1056), (129, 264, 4096), (300, 9600, 512)])
@pytest.mark.parametrize("name", ["none", "silu", "swiglu"])
def test_dense(cuda, M, N, K, name):
    N -= N % 16
    W = N // 2 if name == "swiglu" else N
    ac, asc = R.mxfp4(M, K, 1)
    bc, bs, bt = weights(1, N, K, 2, name == "swiglu")
    bias, res = randn(N, seed=3), randn(M, W, seed=4)
    c = moe.omo_gemm_mxfp4_act(ac, asc, bc[0], bt[0], bias=bias, activation=name, residual=res)
    _, y, _, by = R.grouped(ac, asc, bc, bs, [M], bias[None], name, res)
    R.check(c, y, by)


def test_dense_equals_the_plain_gemm(cuda):
    """The same bytes as omo_gemm_mxfp4 where that one takes the sizes."""
    from omo_python_api.mxfp4 import omo_gemm_mxfp4
    ac, asc = R.mxfp4(2560, 1024, 1)
    bc, bs, bt = weights(1, 2048, 1024, 2, False)
    a = omo_gemm_mxfp4(ac, asc, bc[0], bs[0])
    b = moe.omo_gemm_mxfp4_act(ac, asc, bc[0], bt[0])
    assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("M,splits", [
    (40, [10, -5, 0, 12]),      # a negative split counts as zero, the last 18 rows are nobody's
    (40, [30, 30, 7, 1]),       # more rows than there are: cut at M
    (40, [0, 0, 0, 0]),
    (700, [300, -1, 100, 250]),
    (3000, [700, 1400, 0, 300]),
    (3000, [2000, 2000, 2 ** 31 - 1, 2 ** 31 - 1]),
])
@pytest.mark.parametrize("K", [96, 2080])
def test_rows_outside_the_splits_are_left_alone(cuda, M, splits, K):
    N = 4800 if M == 3000 else 160
    ac, asc = R.mxfp4(M, K, 1)
    bc, bs, bt = weights(4, N, K, 2, False)
    mark = torch.full((M, N), 3.0, dtype=BF, device=cuda)
    pre = mark.clone()
    ep = capi.Epilogue(c_ld=N, pre=pre.data_ptr(), pre_ld=N)
    m = dev(splits)
    capi.call("mxb_grouped_gemm_mxfp4", ac.data_ptr(), K // 2, asc.data_ptr(), K // 32, M,
              m.data_ptr(), 4, bc.data_ptr(), bt.data_ptr(), N, K, ep, mark.data_ptr(), H.stream())
    _, y, _, by = R.grouped(ac, asc, bc, bs, splits, None, "none", None)
    y = torch.where(torch.isnan(y), 3.0, y)
    for x in (mark, pre):
        R.check(x, y, torch.where(torch.isnan(by), 1e-30, by))


@pytest.mark.parametrize("E,M,N,K", [(3, 20, 96, 256), (3, 20, 96, 160), (2, 150, 96, 256), (2, 150, 96, 160),
                                     (2, 1200, 4800, 256), (2, 1200, 4800, 160), (4, 2000, 4400, 2080),
                                     (3, 2600, 2600, 4096)])
def test_strided_rows_and_pitches(cuda, E, M, N, K):
    """Wire rows (codes and scales side by side) as A, and padded c, pre and residual."""
    splits = splits_of(E, M, 7)
    ac, asc = R.mxfp4(M, K, 1)
    wire = torch.full((M, (17 * K // 32 + 15) // 16 * 16), 255, dtype=torch.uint8, device=cuda)
    wire[:, :K // 2], wire[:, K // 2:17 * K // 32] = ac, asc
    bc, bs, bt = weights(E, N, K, 2, False)
    big = torch.full((3, M, N + 24), 7.0, dtype=BF, device=cuda)
    c, pre, res = (t[:, 8:8 + N] for t in big)
    res.copy_(randn(M, N, seed=3))
    import omo
    omo.omo_grouped_gemm_mxfp4(wire[:, :K // 2], wire[:, K // 2:17 * K // 32], dev(splits), bc, bt, c,
                               None, 3, res, pre)
    z, y, bz, by = R.grouped(ac, asc, bc, bs, splits, None, "silu", res)
    R.check(c, y, by)
    R.check(pre, z, bz)
    assert (big[:2, :, :8] == 7).all() and (big[:2, :, 8 + N:] == 7).all()


@pytest.mark.parametrize("K", [512, 384, 288, 4096])
@pytest.mark.parametrize("E,M,N", [(3, 20, 96), (2, 150, 96), (2, 1200, 4800)])
def test_scale_rows_at_any_address(cuda, E, M, N, K):
    """A's scale rows at an odd base and pitch give the same bytes as aligned ones."""
    splits = splits_of(E, M, 7)
    ac, asc = R.mxfp4(M, K, 1)
    bc, bs, bt = weights(E, N, K, 2, False)
    want = moe.omo_grouped_gemm_mxfp4(ac, asc, bc, bt, dev(splits))
    for pad, off in ((3, 1), (4, 4), (16, 16)):
        big = torch.full((M, K // 32 + pad + off), 255, dtype=torch.uint8, device=cuda)
        big[:, off:off + K // 32] = asc
        got = moe.omo_grouped_gemm_mxfp4(ac, big[:, off:off + K // 32], bc, bt, dev(splits))
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("E,M,N,K", [(3, 20, 96, 320), (3, 150, 96, 320), (3, 1300, 4800, 320),
                                     (3, 2600, 2600, 4096), (4, 2000, 4400, 2080)])
def test_nan_scales_stay_in_their_row(cuda, E, M, N, K):
    """A row or weight row whose E8M0 byte is NaN (255) makes its own results NaN only."""
    splits = splits_of(E, M, 3)
    ac, asc = R.mxfp4(M, K, 1)
    bc, bs, _ = weights(E, N, K, 2, False)
    asc[M // 2, 3] = 255
    asc[M - 1, 9] = 255
    bs[1, 5, 0] = 255
    bs[2, N - 1, 9] = 255
    bt = moe.omo_swizzle_scales_grouped(bs)
    c = moe.omo_grouped_gemm_mxfp4(ac, asc, bc, bt, dev(splits))
    _, y, _, by = R.grouped(ac, asc, bc, bs, splits, None, "none", None)
    R.check(c, y, by)


def test_many_experts(cuda):
    E, M, N, K = capi_max_experts(), 300, 64, 64
    splits = splits_of(E, M, 9)
    ac, asc = R.mxfp4(M, K, 1)
    bc, bs, bt = weights(E, N, K, 2, False)
    c = moe.omo_grouped_gemm_mxfp4(ac, asc, bc, bt, dev(splits))
    _, y, _, by = R.grouped(ac, asc, bc, bs, splits, None, "none", None)
    R.check(c, y, by)
    dy = randn(M, N, seed=4)
    dw = moe.omo_grouped_wgrad_mxfp4(dy, ac, asc, dev(splits))
    check_wgrad(dw, dy, ac, asc, splits)


def capi_max_experts():
    import re
    from test_capi_cpu import ROOT
    txt = (ROOT / "include" / "mxfp4_b200.h").read_text()
    return int(re.search(r"define MXB_MAX_EXPERTS (\d+)", txt).group(1))


def test_another_stream(cuda):
    ac, asc = R.mxfp4(500, 512, 1)
    bc, bs, bt = weights(2, 320, 512, 2, False)
    m = dev([200, 300])
    want = moe.omo_grouped_gemm_mxfp4(ac, asc, bc, bt, m, activation="gelu")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = moe.omo_grouped_gemm_mxfp4(ac, asc, bc, bt, m, activation="gelu")
    s.synchronize()
    assert torch.equal(got, want)


def test_two_streams_at_once(cuda):
    """Products that split K over clusters, wide products and weight gradients issued on two
    streams without ordering between them: each stream's results are those of a run alone."""
    ac, asc = R.mxfp4(300, 4096, 1)
    bc, bs, bt = weights(4, 256, 4096, 2, False)
    dy = randn(300, 256, seed=5)
    few, many = dev([1, 2, 0, 5]), dev([100, 50, 0, 150])

    def work():
        return [moe.omo_grouped_gemm_mxfp4(ac[:8], asc[:8], bc, bt, few),
                moe.omo_grouped_gemm_mxfp4(ac, asc, bc, bt, many, activation="silu"),
                moe.omo_grouped_wgrad_mxfp4(dy, ac, asc, many)]

    want = work()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for s, g in zip(streams, got):
            with torch.cuda.stream(s):
                g.append(work())
    torch.cuda.synchronize()
    for g in got:
        for outs in g:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_in_a_graph(cuda):
    """Captured once, replayed with other splits: nothing of the routing is on the host."""
    ac, asc = R.mxfp4(64, 512, 1)
    bc, bs, bt = weights(4, 320, 512, 2, False)
    m = dev([16, 16, 16, 16])
    moe.omo_grouped_gemm_mxfp4(ac, asc, bc, bt, m)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c = moe.omo_grouped_gemm_mxfp4(ac, asc, bc, bt, m)
    for splits in ([0, 64, 0, 0], [1, 2, 3, 58]):
        m.copy_(dev(splits))
        g.replay()
        _, y, _, by = R.grouped(ac, asc, bc, bs, splits, None, "none", None)
        R.check(c, y, by)


@pytest.mark.parametrize("E,N,S,gated", [(1, 128, 4, False), (3, 72, 5, False), (2, 200, 7, True),
                                         (2, 512, 65, True)])
def test_swizzle_scales_grouped(cuda, E, N, S, gated):
    """Each part of each expert equals mxb_swizzle_scales on it."""
    s = torch.randint(0, 256, (E, N, S), dtype=torch.uint8, device=cuda)
    got = moe.omo_swizzle_scales_grouped(s, gated)
    parts = 2 if gated else 1
    n = N // parts
    for e in range(E):
        for h in range(parts):
            one = s[e, h * n:(h + 1) * n].contiguous()
            want = torch.empty((n + 127) // 128 * 128, (S + 3) // 4 * 4, dtype=torch.uint8, device=cuda)
            capi.call("mxb_swizzle_scales", one.data_ptr(), n, S, want.data_ptr(), H.stream())
            assert torch.equal(got[e].reshape(parts, *want.shape)[h], want)


# ---------------------------------------------------------------- weight gradient
def check_wgrad(dw, dy, xc, xs, splits, base=None):
    """f32 accumulation: 2^-16 of the sum of |dy x| (rows / 16 partial sums at 2^-24 each,
    with margin), and 2^-8 of a BF16 result for its rounding."""
    M = dy.shape[0]
    x = R.values(xc, xs)
    for e, (i, j) in enumerate(R.spans(splits, M)):
        d = dy[i:j].double()
        want = d.T @ x[i:j]
        bound = 2.0 ** -16 * (d.abs().T @ x[i:j].abs())
        if base is not None:
            want = want + base[e].double()
            bound = bound + 2.0 ** -23 * base[e].double().abs()
        if dw.dtype == BF:
            bound = bound + 2.0 ** -8 * want.abs()
        R.check(dw[e], want, bound + 1e-40, f"expert {e}")


@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("E,M,N,K", [(1, 1, 8, 32), (1, 64, 256, 128), (2, 65, 264, 160), (3, 300, 128, 384),
                                     (8, 301, 520, 768), (4, 7, 1000, 96), (5, 3001, 328, 288)])
def test_wgrad(cuda, E, M, N, K, dtype):
    splits = splits_of(E, M, M + N, empty=(1,) if E > 2 else ())
    xc, xs = R.mxfp4(M, K, 1)
    dy = randn(M, N, seed=2, scale=0.1)
    dw = moe.omo_grouped_wgrad_mxfp4(dy, xc, xs, dev(splits), out_dtype=dtype)
    check_wgrad(dw, dy, xc, xs, splits)
    again = moe.omo_grouped_wgrad_mxfp4(dy, xc, xs, dev(splits), out_dtype=dtype)
    assert torch.equal(dw, again)
    if E == 1:
        assert torch.equal(moe.omo_grouped_wgrad_mxfp4(dy, xc, xs, None, out_dtype=dtype), dw)


def test_wgrad_accumulates(cuda):
    E, M, N, K = 4, 500, 264, 192
    splits = splits_of(E, M, 3, empty=(2,))
    xc, xs = R.mxfp4(M, K, 1)
    dy = randn(M, N, seed=2)
    base = randn(E, N, K, seed=3, dtype=torch.float32)
    dw = base.clone()
    out = moe.omo_grouped_wgrad_mxfp4(dy, xc, xs, dev(splits), accumulate_into=dw)
    assert out is dw and torch.equal(dw[2], base[2])
    check_wgrad(dw, dy, xc, xs, splits, base)


def test_wgrad_neighbours_infinities_stay_out(cuda):
    """Rows of the next expert, and rows of nobody, hold infinities and NaN."""
    E, M, N, K = 3, 200, 128, 128
    splits = [37, 90, 20]
    xc, xs = R.mxfp4(M, K, 1)
    dy = randn(M, N, seed=2)
    dy[37:127] = math.inf
    dy[50] = math.nan
    dy[147:] = math.nan
    xs[147:] = 255
    dw = moe.omo_grouped_wgrad_mxfp4(dy, xc, xs, dev(splits))
    for e, (i, j) in ((0, (0, 37)), (2, (127, 147))):
        d, x = dy[i:j].double(), R.values(xc[i:j], xs[i:j])
        R.check(dw[e], d.T @ x, 2.0 ** -16 * (d.abs().T @ x.abs()) + 1e-40)
    assert not torch.isfinite(dw[1]).any()


@pytest.mark.parametrize("lo,hi", [(0, 3), (1, 2), (60, 64), (200, 204), (252, 253)])
def test_wgrad_scale_range(cuda, lo, hi):
    M, N, K = 40, 64, 64
    xc, xs = R.mxfp4(M, K, 1, lo, hi)
    dy = randn(M, N, seed=2, scale=2.0 ** (127 - hi if hi > 127 else 0))
    dw = moe.omo_grouped_wgrad_mxfp4(dy, xc, xs, None)
    d, x = dy.double(), R.values(xc, xs)
    # a product below f32's normal range may be flushed: 2^-126 each
    R.check(dw[0], d.T @ x, 2.0 ** -16 * (d.abs().T @ x.abs()) + M * 2.0 ** -126)


def test_wgrad_without_rows_is_zero(cuda):
    xc, xs = R.mxfp4(0, 64, 1)
    dy = torch.empty(0, 64, dtype=BF, device=cuda)
    assert (moe.omo_grouped_wgrad_mxfp4(dy, xc, xs, dev([0, 0])) == 0).all()
    xc, xs = R.mxfp4(10, 64, 1)
    dy = randn(10, 64, seed=1)
    assert (moe.omo_grouped_wgrad_mxfp4(dy, xc, xs, dev([0, 0])) == 0).all()


# ---------------------------------------------------------------- epilogue gradient
def act_grad_ref(dy, pre, name):
    z = pre.double().requires_grad_(True)
    R.act(z, name).backward(dy.double())
    return z.grad


@pytest.mark.parametrize("name", R.ACTS)
@pytest.mark.parametrize("E,M,N", [(1, 1, 64), (1, 64, 64), (1, 65, 576), (1, 100, 1088), (3, 129, 512), (8, 333, 1024),
                                   (1, 512, 128), (2, 513, 128), (8, 1000, 320), (2, 5000, 64)])
def test_bias_act_grad(cuda, E, M, N, name):
    W = N // 2 if name == "swiglu" else N
    splits = splits_of(E, M, M, empty=(1,) if E > 2 else ())
    dy, pre = randn(M, W, seed=1), randn(M, N, seed=2, scale=2.0)
    dz, db, q, s = moe.omo_bias_act_grad(dy, pre, dev(splits), name, quantize=True)
    want = act_grad_ref(dy, pre, name)
    # evaluated in f32 to about 2^-18 of the terms it is made of, rounded once to BF16
    mag = torch.cat((dy, dy), -1).double().abs() if name == "swiglu" else dy.double().abs()
    mag = mag * (R.slope_bound(pre.double(), name) + pre.double().abs() + 1)
    R.check(dz, want, 2.0 ** -8 * want.abs() + 2.0 ** -18 * mag)
    rq, rs = H.quant_rows(dz)
    assert torch.equal(q, rq) and torch.equal(s, rs)
    for e, (i, j) in enumerate(R.spans(splits, M)):
        R.check(db[e], want[i:j].sum(0), 2.0 ** -18 * mag[i:j].sum(0) + 1e-40, f"bias of {e}")
    dz2, db2 = moe.omo_bias_act_grad(dy, pre, dev(splits), name)
    assert torch.equal(dz2, dz) and torch.equal(db2, db)
    assert torch.equal(moe.omo_bias_act_grad(dy, pre, dev(splits), name, bias_grad=False), dz)


@pytest.mark.parametrize("name", R.ACTS)
def test_act_grad_against_differences(cuda, name):
    """The slope that the kernel returns for dy = 1 against central differences of the
    activation in 64 bits; a step of 1e-4 leaves at most 1e-7, the BF16 result 2^-8."""
    z = torch.linspace(-9, 9, 64 * 64, device=cuda).to(BF).reshape(64, 64)
    dy = torch.ones(64, 32 if name == "swiglu" else 64, dtype=BF, device=cuda)
    got = moe.omo_bias_act_grad(dy, z, None, name, bias_grad=False).double()
    h = 1e-4
    d = z.double()
    parts = [slice(0, 32), slice(32, 64)] if name == "swiglu" else [slice(0, 64)]
    for cols in parts:
        up, dn = d.clone(), d.clone()
        up[:, cols] += h
        dn[:, cols] -= h
        diff = (R.act(up, name) - R.act(dn, name)) / (2 * h)
        kink = (d[:, cols].abs() < 2 * h) & torch.tensor(name in ("relu", "relu2"), device=cuda)
        err = (got[:, cols] - diff).abs() - (2.0 ** -8 * diff.abs() + 1e-5)
        assert (err[~kink] <= 0).all(), err.max()


def test_act_grad_rows_of_nobody(cuda):
    dy, pre = randn(50, 64, seed=1), randn(50, 64, seed=2)
    dz = torch.full_like(pre, 5.0)
    db = torch.empty(2, 64, dtype=torch.float32, device=cuda)
    m = dev([10, -3])
    assert capi.load().mxb_bias_act_grad_workspace(50, 2, 64) == 0
    capi.call("mxb_bias_act_grad", dy.data_ptr(), pre.data_ptr(), 50, m.data_ptr(), 2, 64, 3,
              dz.data_ptr(), None, None, db.data_ptr(), None, 0, H.stream())
    assert (dz[10:] == 5).all() and (db[1] == 0).all()


# ---------------------------------------------------------------- unpermute
def unpermute_ref(y, m, w):
    ok = (m >= 0) & (m < y.shape[0])
    rows = y.double()[torch.where(ok, m, 0).long()] * ok[..., None]
    w = (ok if w is None else torch.where(ok, w, 0)).double()
    return rows, w, ok


@pytest.mark.parametrize("T,k,H_", [(1, 1, 8), (16, 8, 7168), (7, 3, 264), (100, 9, 64), (33, 20, 136),
                                    (5, 1, 10000)])
@pytest.mark.parametrize("weighted", [True, False])
def test_unpermute(cuda, T, k, H_, weighted):
    g = torch.Generator().manual_seed(T + k)
    rows = T * k + 5
    y = randn(rows, H_, seed=1)
    m = torch.randperm(rows, generator=g)[:T * k].reshape(T, k).to(torch.int32)
    m[torch.rand(T, k, generator=g) < 0.2] = -1
    m[0] = -1                        # a token without rows
    if k > 2:
        m[T - 1, 1] = rows           # out of range: no row
    m = m.cuda()
    w = torch.rand(T, k, generator=g).cuda() if weighted else None
    out = moe.omo_moe_unpermute(y, m, w)
    x, wd, ok = unpermute_ref(y, m, w)
    want = (x * wd[..., None]).sum(1)
    mag = (x.abs() * wd[..., None]).sum(1)
    R.check(out, want, 2.0 ** -8 * want.abs() + k * 2.0 ** -23 * mag + 1e-40)
    assert (out[0] == 0).all()
    dout = randn(T, H_, seed=3)
    r = moe.omo_moe_unpermute_grad(dout, y, m, w, quantize=H_ % 32 == 0, zero_unnamed=True)
    dy, dw = r[0], r[1]
    want = torch.zeros(rows, H_, dtype=torch.float64, device=cuda)
    want[m[ok].long()] = (wd[..., None] * dout.double()[:, None])[ok]
    R.check(dy, want, 2.0 ** -8 * want.abs())
    dots, mags = (x * dout.double()[:, None]).sum(-1), (x * dout.double()[:, None]).abs().sum(-1)
    R.check(dw, dots, 2.0 ** -18 * mags + 1e-40)
    assert (dw[~ok] == 0).all()
    if H_ % 32 == 0:
        rq, rs = H.quant_rows(dy)
        named = torch.zeros(rows, dtype=torch.bool, device=cuda)
        named[m[ok].long()] = True
        assert torch.equal(r[2][named], rq[named]) and torch.equal(r[3][named], rs[named])
        assert (r[2][~named] == 0).all() and (r[3][~named] == 0).all()


def test_unpermute_takes_a_row_id_map(cuda):
    """Transformer Engine's map [T, 2E + 1]: destinations in the first columns, then -1."""
    T, E, H_ = 40, 12, 128
    routing = torch.rand(T, E, device=cuda) < 0.3
    rid = torch.empty(T, 2 * E + 1, dtype=torch.int32, device=cuda)
    work = torch.empty(E, dtype=torch.int32, device=cuda)
    capi.call("mxb_moe_make_row_id_map", routing.data_ptr(), T, E, rid.data_ptr(), work.data_ptr(), H.stream())
    n = int(routing.sum())
    y = randn(n, H_, seed=1)
    out = moe.omo_moe_unpermute(y, rid, None, topk=E)
    x, w, _ = unpermute_ref(y, rid[:, :E], None)
    want = (x * w[..., None]).sum(1)
    R.check(out, want, 2.0 ** -8 * want.abs() + E * 2.0 ** -23 * x.abs().sum(1) + 1e-40)


# ---------------------------------------------------------------- refusals through the wrappers
@pytest.mark.parametrize("what,bad", [
    ("dtype", lambda a: a.update(ac=a["ac"].to(torch.int8))),
    ("rows", lambda a: a.update(asc=a["asc"][:-1])),
    ("device", lambda a: a.update(m=a["m"].cpu())),
    ("splits", lambda a: a.update(m=a["m"].long())),
    ("experts", lambda a: a.update(m=a["m"][:1])),
    ("scales", lambda a: a.update(bt=a["bt"][:, :64])),
    ("bias", lambda a: a.update(bias=torch.zeros(2, 95, device="cuda"))),
    ("residual", lambda a: a.update(res=torch.zeros(9, 96, device="cuda", dtype=BF))),
    ("name", lambda a: a.update(name="swish")),
    ("alignment", lambda a: a.update(ac=torch.zeros(10, 72, dtype=torch.uint8, device="cuda")[:, 8:])),
])
def test_refusals(cuda, what, bad):
    ac, asc = R.mxfp4(10, 128, 1)
    bc, bs, bt = weights(2, 96, 128, 2, False)
    a = dict(ac=ac, asc=asc, bt=bt, m=dev([4, 6]), bias=None, res=None, name="none")
    bad(a)
    with pytest.raises(RuntimeError):
        moe.omo_grouped_gemm_mxfp4(a["ac"], a["asc"], bc, a["bt"], a["m"], bias=a["bias"],
                                   activation=a["name"], residual=a["res"])


# ---------------------------------------------------------------- the layer that runs them together
def plain_experts(x, idx, w, w1, w2):
    """The same layer in FP32 without quantization."""
    out = torch.zeros(x.shape[0], x.shape[1], device=x.device)
    for e in range(w1.shape[0]):
        t, k = (idx == e).nonzero(as_tuple=True)
        out = out.index_add(0, t, w[t, k, None] * (R.act(x[t] @ w1[e].T, "swiglu") @ w2[e].T))
    return out


def cos(a, b):
    return torch.nn.functional.cosine_similarity(a.float().reshape(1, -1), b.float().reshape(1, -1)).item()


@pytest.mark.parametrize("T,E,k,Hd,F", [(5, 4, 2, 256, 96), (700, 6, 3, 512, 256)])
def test_expert_layer(cuda, T, E, k, Hd, F):
    """Against the unquantized layer: an E2M1 value is off by about 0.11 of itself (rms), a
    product of two such operands by 0.16, two products in a row by 0.22, a gradient passes
    three or four: cosines of 0.97 and 0.94 are expected, 0.9 and 0.85 asked for (a wrong expert,
    half, weight or transposition leaves less than 0.7).  An expert nobody is routed to gets zeros."""
    from mxfp4_b200.moe import MXFP4Experts, expert_order
    torch.manual_seed(3)
    layer = MXFP4Experts(E, Hd, F, device=cuda)
    layer.quantize_weights()
    x = torch.randn(T, Hd, device=cuda).to(BF).requires_grad_(True)
    idx = torch.stack([torch.randperm(E - 1, device=cuda)[:k] for _ in range(T)])  # expert E - 1: nobody
    w = torch.rand(T, k, device=cuda).requires_grad_(True)
    out = layer(x, idx, w)
    dout = torch.randn(T, Hd, device=cuda).to(BF)
    out.backward(dout)
    xr, wr = x.detach().float().requires_grad_(True), w.detach().clone().requires_grad_(True)
    w1, w2 = (p.detach().float().requires_grad_(True) for p in (layer.w1, layer.w2))
    want = plain_experts(xr, idx, wr, w1, w2)
    want.backward(dout.float())
    assert cos(out, want) > 0.9
    for got, ref in ((x.grad, xr.grad), (w.grad, wr.grad), (layer.w1.grad, w1.grad), (layer.w2.grad, w2.grad)):
        assert got.shape == ref.shape and cos(got, ref) > 0.85
    assert (layer.w1.grad[E - 1] == 0).all() and (layer.w2.grad[E - 1] == 0).all()
    # the same gradient added to an FP32 buffer
    layer.w1.main_grad = torch.ones_like(layer.w1, dtype=torch.float32)
    layer.w1.grad = None
    g2 = layer.w2.grad.clone()
    layer.w2.grad = None
    layer(x, idx, w).backward(dout)
    assert layer.w1.grad is None and torch.equal(layer.w2.grad, g2)
    dst, splits = expert_order(idx, E)
    assert splits.sum() == T * k and torch.equal(dst.flatten().sort().values.cpu(), torch.arange(T * k, dtype=torch.int32))
    assert cos(layer.w1.main_grad - 1, w1.grad) > 0.85


def test_expert_layer_needs_quantized_weights(cuda):
    from mxfp4_b200.moe import MXFP4Experts
    layer = MXFP4Experts(2, 64, 32, device=cuda)
    with pytest.raises(RuntimeError, match="quantize_weights"):
        layer(torch.zeros(1, 64, dtype=BF, device=cuda), torch.zeros(1, 1, dtype=torch.long, device=cuda),
              torch.ones(1, 1, device=cuda))
