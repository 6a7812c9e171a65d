"""The MXFP4 expert layer step by step against 64-bit forms: each step's result per element,
from the operands that the step before really handed on."""
import pytest
import torch

import helpers as H
import moe_ref as R
from mxfp4_b200 import capi
from mxfp4_b200.moe import MXFP4Experts, expert_order
from omo_python_api import mxfp4_moe as moe
from test_moe_gpu import act_grad_ref, check_wgrad

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def stacked(w):
    """Rowwise MXFP4 of every expert's weights, scales row-major."""
    q = [H.quant_rows(w[e].contiguous()) for e in range(w.shape[0])]
    return torch.stack([c for c, _ in q]), torch.stack([s for _, s in q])


def weighted(rows, dst, w):
    """The sum over k of w * rows[dst] where there is a row, and the sum of its terms' sizes."""
    ok = dst >= 0
    x = rows.double()[torch.where(ok, dst, 0).long()] * ok[..., None]
    x = torch.where(ok[..., None], x, 0.0)
    w = torch.where(ok, w.double(), 0.0)[..., None]
    return (x * w).sum(1), (x * w).abs().sum(1), x


@pytest.mark.parametrize("lost", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("T,E,k,Hd,F,dtype", [(5, 4, 2, 256, 96, BF), (300, 6, 3, 512, 256, BF),
                                              (1000, 3, 2, 320, 160, torch.float32)])
def test_layer_step_by_step(cuda, T, E, k, Hd, F, dtype, lost):
    """`lost`: the share of ids that are -1, experts of another rank.  Bounds as in the operators'
    own tests; a sum over k terms is off by k * 2^-23 of their sizes and one rounding to BF16."""
    g = torch.Generator().manual_seed(T)
    torch.manual_seed(T)
    layer = MXFP4Experts(E, Hd, F, dtype=dtype, device=cuda)
    layer.quantize_weights()
    x = torch.randn(T, Hd, generator=g).to(BF).cuda().requires_grad_(True)
    idx = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)])
    idx[torch.rand(T, k, generator=g) < lost] = -1
    idx = idx.to(torch.int32).cuda()
    w = torch.rand(T, k, generator=g).cuda().requires_grad_(True)
    dout = torch.randn(T, Hd, generator=g).to(BF).cuda()
    out = layer(x, idx, w)
    out.backward(dout)
    dst, splits = expert_order(idx, E)
    ms, rows, ok, n = splits.tolist(), T * k, dst >= 0, int(splits.sum())
    assert n == int((idx >= 0).sum())

    def there(*ts):  # rows past the last expert's are nobody's
        return [t[:n] for t in ts]

    # the rows of every expert, and its weights
    codes, scales = H.quant_rows(x.detach())
    xc = torch.zeros(rows, Hd // 2, dtype=torch.uint8, device=cuda)
    xs = torch.full((rows, Hd // 32), 127, dtype=torch.uint8, device=cuda)
    token = torch.arange(T, device=cuda)[:, None].expand(T, k)
    xc[dst[ok].long()], xs[dst[ok].long()] = codes[token[ok]], scales[token[ok]]
    w1, w2 = (p.detach().to(BF) for p in (layer.w1, layer.w2))
    c1, s1 = stacked(w1)
    c2, s2 = stacked(w2)
    c1t, s1t = stacked(w1.transpose(1, 2))
    c2t, s2t = stacked(w2.transpose(1, 2))
    q1, q2 = layer._q
    for mine, theirs in ((c1, q1.codes), (c2, q2.codes), (c1t, q1.codes_t), (c2t, q2.codes_t)):
        assert torch.equal(mine, theirs)

    # forward
    pre, hc, hs = moe.omo_grouped_gemm_mxfp4(xc, xs, q1.codes, q1.scales, splits, activation="swiglu",
                                             save_pre=True, quantize=True, bf16_out=False)
    z, h, bz, bh = there(*R.grouped(xc, xs, c1, s1, ms, None, "swiglu", None))
    R.check(pre[:n], z, bz, "pre")
    # E2M1 is off by at most a quarter of the value, and by a quarter of the smallest step's scale
    step = torch.exp2(hs[:n].double() - 127).repeat_interleave(32, -1)
    R.check(R.values(hc, hs)[:n], h, bh + 0.25 * h.abs() + 0.25 * step, "h")
    y = moe.omo_grouped_gemm_mxfp4(hc, hs, q2.codes, q2.scales, splits)
    _, yw, _, by = there(*R.grouped(hc, hs, c2, s2, ms, None, "none", None))
    R.check(y[:n], yw, by, "y")
    want, mag, yk = weighted(y, dst, w.detach())
    R.check(out.detach(), want, 2.0 ** -8 * want.abs() + k * 2.0 ** -23 * mag + 1e-40, "out")

    # backward
    dots, mags = (yk * dout.double()[:, None]).sum(-1), (yk * dout.double()[:, None]).abs().sum(-1)
    R.check(w.grad, dots, 2.0 ** -18 * mags + 1e-40, "weights' gradient")
    assert (w.grad[~ok] == 0).all()
    dy, dyc, dys = moe.omo_moe_unpermute_grad(dout, y, dst, w.detach(), weight_grad=False, quantize=True,
                                              zero_unnamed=True)
    dyw = torch.zeros(rows, Hd, dtype=torch.float64, device=cuda)
    dyw[dst[ok].long()] = (w.detach().double()[..., None] * dout.double()[:, None])[ok]
    R.check(dy, dyw, 2.0 ** -8 * dyw.abs(), "dy")
    check_wgrad(layer.w2.grad, dy, hc, hs, ms)
    dh = moe.omo_grouped_gemm_mxfp4(dyc, dys, q2.codes_t, q2.scales_t, splits)
    _, dhw, _, bdh = there(*R.grouped(dyc, dys, c2t, s2t, ms, None, "none", None))
    R.check(dh[:n], dhw, bdh, "dh")
    dz, dzc, dzs = moe.omo_bias_act_grad(dh, pre, splits, "swiglu", bias_grad=False, quantize=True)
    dzw = act_grad_ref(dh[:n], pre[:n], "swiglu")
    size = torch.cat((dh, dh), -1)[:n].double().abs() * (R.slope_bound(pre[:n].double(), "swiglu") +
                                                         pre[:n].double().abs() + 1)
    R.check(dz[:n], dzw, 2.0 ** -8 * dzw.abs() + 2.0 ** -18 * size, "dz")
    check_wgrad(layer.w1.grad, dz, xc, xs, ms)
    dxp = moe.omo_grouped_gemm_mxfp4(dzc, dzs, q1.codes_t, q1.scales_t, splits)
    _, dxw, _, bdx = there(*R.grouped(dzc, dzs, c1t, s1t, ms, None, "none", None))
    R.check(dxp[:n], dxw, bdx, "rows' gradient")
    want, mag, _ = weighted(dxp, dst, torch.ones_like(w.detach()))
    R.check(x.grad, want, 2.0 ** -8 * want.abs() + k * 2.0 ** -23 * mag + 1e-40, "x's gradient")
    torch.cuda.synchronize()
    assert capi.reset_wait_timeouts() == 0


def test_second_derivative_is_refused(cuda):
    """With a graph of gradients the first ones are the same bytes, and a penalty on them raises."""
    layer = MXFP4Experts(3, 128, 64, device=cuda)
    layer.quantize_weights()
    x = torch.randn(9, 128, device=cuda).to(BF).requires_grad_(True)
    idx = torch.stack([torch.randperm(3, device=cuda)[:2] for _ in range(9)])
    w = torch.rand(9, 2, device=cuda).requires_grad_(True)
    inputs = (x, w, layer.w1, layer.w2)
    want = torch.autograd.grad(layer(x, idx, w).sum(), inputs)
    got = torch.autograd.grad(layer(x, idx, w).sum(), inputs, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for g in got:
        with pytest.raises(RuntimeError, match="second derivative"):
            g.float().square().sum().backward(retain_graph=True)
