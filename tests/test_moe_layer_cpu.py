"""The MXFP4 expert layer on the CPU: its routing, and its autograd function over plain operators."""
import pytest
import torch

from mxfp4_b200 import moe
from mxfp4_b200.ep import build_route
from mxfp4_b200.moe import expert_order


def order_ref(idx, E):
    """Row by row from the definition: expert by expert, token by token."""
    dst, splits, at = [[-1] * idx.shape[1] for _ in range(idx.shape[0])], [0] * E, 0
    for e in range(E):
        for t, ids in enumerate(idx.tolist()):
            for k, i in enumerate(ids):
                if i == e:
                    dst[t][k] = at
                    splits[e] += 1
                    at += 1
    return dst, splits


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("T,k,E,lo,hi", [(4, 2, 5, 0, 5), (33, 4, 7, -1, 7), (5, 3, 2, -1, 0), (1, 1, 1, -1, 0),
                                         (40, 2, 6, -3, 9), (0, 2, 3, 0, 3)])
def test_ids_without_an_expert_here_have_no_row(T, k, E, lo, hi, dtype):
    g = torch.Generator().manual_seed(T + k)
    idx = torch.randint(lo, hi, (T, k), generator=g).to(dtype)
    dst, splits = expert_order(idx, E)
    want_dst, want_splits = order_ref(idx, E)
    assert dst.dtype == splits.dtype == torch.int32 and splits.is_contiguous()
    assert splits.tolist() == want_splits and dst.shape == (T, k)
    assert dst.tolist() == want_dst


def test_takes_a_dispatchers_ids():
    """What build_route hands a rank: ids local to it and -1 elsewhere."""
    g = torch.Generator().manual_seed(1)
    idx = torch.stack([torch.randperm(8, generator=g)[:3] for _ in range(20)])
    route = build_route(idx, torch.rand(20, 3, generator=g), 2, 8)
    assert (route.local_topk == -1).any()
    dst, splits = expert_order(route.local_topk, 4)
    assert int(splits.sum()) == int((route.local_topk >= 0).sum())
    assert torch.equal(dst >= 0, route.local_topk >= 0)


class Plain:
    """The layer's operators in float64 without quantization: codes are the values."""

    @staticmethod
    def omo_per_token_group_quant_mxfp4(x):
        return x, x[:, :0]

    @staticmethod
    def omo_moe_permute_mxfp4(codes, scales, dst, rows):
        out = codes.new_zeros(rows, codes.shape[1])
        t, k = (dst >= 0).nonzero(as_tuple=True)
        out[dst[t, k].long()] = codes[t]
        return out, out[:, :0]

    @staticmethod
    def omo_grouped_gemm_mxfp4(a, sa, b, sb, splits, activation="none", save_pre=False, quantize=False, bf16_out=True):
        z = a.new_zeros(a.shape[0], b.shape[1])
        n = int(splits.sum())
        z[:n] = torch.cat([x @ w.T for x, w in zip(a[:n].split(splits.tolist()), b)])
        if activation == "none":
            return z
        g, u = z.chunk(2, -1)
        return z, g * torch.sigmoid(g) * u, z[:, :0]

    @staticmethod
    def omo_moe_unpermute(y, dst, w=None):
        rows = y[dst.clamp(min=0).long()] * (dst >= 0)[..., None]
        return (rows if w is None else rows * w[..., None]).sum(1)

    @staticmethod
    def omo_moe_unpermute_grad(dout, y, dst, w, quantize):
        dy = torch.zeros_like(y)
        t, k = (dst >= 0).nonzero(as_tuple=True)
        dy[dst[t, k].long()] = w[t, k, None] * dout[t]
        dw = (y[dst.clamp(min=0).long()] * dout[:, None]).sum(-1) * (dst >= 0)
        return dy, dw, dy, dy[:, :0]

    @staticmethod
    def omo_bias_act_grad(dh, pre, splits, activation, bias_grad, quantize):
        g, u = pre.chunk(2, -1)
        s = torch.sigmoid(g)
        dz = torch.cat((dh * u * s * (1 + g * (1 - s)), dh * g * s), -1)
        return dz, dz, dz[:, :0]

    @staticmethod
    def omo_grouped_wgrad_mxfp4(dy, xc, xs, splits, out_dtype=None, accumulate_into=None):
        n, m = int(splits.sum()), splits.tolist()
        dw = torch.stack([d.T @ x for d, x in zip(dy[:n].split(m), xc[:n].split(m))])
        return dw if accumulate_into is None else accumulate_into.add_(dw)


@pytest.fixture
def plain_layer(monkeypatch):
    """A float64 layer whose operators are the plain ones."""
    monkeypatch.setattr(moe, "Q", Plain)
    monkeypatch.setattr(moe, "M", Plain)
    torch.manual_seed(0)
    layer = moe.MXFP4Experts(3, 64, 32, dtype=torch.float64)
    weights = []
    for w in (layer.w1, layer.w2):
        q = moe.QuantizedWeights.__new__(moe.QuantizedWeights)
        q.codes, q.codes_t, q.scales, q.scales_t = w.detach(), w.detach().transpose(1, 2), None, None
        weights.append(q)
    layer._q = tuple(weights)
    x = torch.randn(6, 64, dtype=torch.float64, requires_grad=True)
    return layer, x, torch.tensor([[0, 2], [2, -1], [1, 0], [-1, -1], [2, 1], [0, 1]]), torch.rand(6, 2, requires_grad=True)


def test_first_derivatives(plain_layer):
    """The layer's own backward pass against differences (steps of 1e-6: 1e-7 of the values) and,
    with a graph, the same gradients."""
    layer, x, idx, w = plain_layer
    d = torch.randn(6, 64, dtype=torch.float64)
    inputs = [x, w, layer.w1, layer.w2]
    grads = torch.autograd.grad((layer(x, idx, w) * d).sum(), inputs)
    again = torch.autograd.grad((layer(x, idx, w) * d).sum(), inputs, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    g = torch.Generator().manual_seed(1)
    for _ in range(20):
        t, c = int(torch.randint(6, (1,), generator=g)), int(torch.randint(64, (1,), generator=g))
        with torch.no_grad():
            sides = []
            for h in (1e-6, -1e-6):
                y = x.clone()
                y[t, c] += h
                sides.append((layer(y, idx, w) * d).sum())
        want = (sides[0] - sides[1]) / 2e-6
        assert abs(want - grads[0][t, c]) <= 1e-6 * (1 + abs(want))


def test_second_derivatives_are_refused(plain_layer):
    """A penalty on any gradient of the layer beside another loss raises instead of counting for
    nothing, whether or not the incoming gradient needs one itself."""
    layer, x, idx, w = plain_layer
    for scale in (torch.ones(()), torch.ones((), requires_grad=True)):
        for at in (x, w, layer.w1, layer.w2):
            out = layer(x, idx, w)
            g, = torch.autograd.grad(out.sum() * scale, at, create_graph=True)
            with pytest.raises(RuntimeError, match="second derivative"):
                (out.sum() + g.square().sum()).backward()


def test_a_graph_of_gradients_beside_the_layer_still_works(plain_layer):
    """A penalty on a gradient behind the layer needs the layer's first derivative only."""
    layer, x, idx, w = plain_layer
    head = torch.randn(64, dtype=torch.float64, requires_grad=True)
    g, = torch.autograd.grad((layer(x, idx, w) @ head).square().sum(), head, create_graph=True)
    g.square().sum().backward()
    assert x.grad is not None and torch.isfinite(x.grad).all() and (x.grad != 0).any()
