"""The expert layer of a mixture-of-experts model with MXFP4 operands, forward and backward.

    experts = MXFP4Experts(num_experts, hidden, ffn).cuda()
    experts.quantize_weights()                    # once per weight update
    out = experts(x, topk_idx, topk_w)            # x BF16 [T, H], ids [T, k], weights [T, k]

Under expert parallelism the layer holds a rank's own experts and takes what the dispatch
delivers: ids local to the rank, -1 where a token's expert is on another rank.  Such an entry
adds nothing to its token and its weight's gradient is 0.

Forward: the tokens are quantized once and permuted as MXFP4 rows; the gate and up product
applies SwiGLU in its epilogue and hands its result on as MXFP4; the down product's rows
are weighted and summed back per token.  Backward: the rows that wait for it are the
MXFP4 ones of both products (4.25 bits a value) and, in BF16, the rows before the activation
[T * k, 2F] and the down product's [T * k, H], which the routing weights' gradient needs; they
are made and kept whether or not a gradient is asked for.  The input gradients
are the same products with the transposed weights, the weight gradients come from BF16
output gradients and the saved MXFP4 rows.  Nothing synchronises with the host: the rows per
expert stay on the device and the buffers hold T * k rows.  A second derivative through the
layer (a penalty on its gradients) raises.

A weight with an FP32 `main_grad` attribute of its shape (Megatron's gradient buffer) gets
its gradient added there; any other gets `.grad` in its own dtype.
"""
from __future__ import annotations

import torch

import mxfp4_b200  # noqa: F401
from omo_python_api import mxfp4 as Q
from omo_python_api import mxfp4_moe as M


def expert_order(topk_idx: torch.Tensor, num_experts: int):
    """Where the rows of tokens routed to topk_idx [T, k] go when sorted by expert, tokens in
    order within an expert: (dst int32 [T, k], m_splits int32 [E]).  An id outside
    [0, num_experts), as the dispatchers' -1 for an expert of another rank, has no row: its dst
    is -1 and no expert counts it."""
    flat = topk_idx.reshape(-1).long()
    here = (flat >= 0) & (flat < num_experts)
    key = torch.where(here, flat, num_experts)  # rows of nobody sort last
    order = torch.sort(key, stable=True).indices
    dst = torch.empty_like(order, dtype=torch.int32)
    dst[order] = torch.arange(flat.numel(), dtype=torch.int32, device=flat.device)
    splits = torch.zeros(num_experts + 1, dtype=torch.int32, device=flat.device)
    splits.scatter_add_(0, key, torch.ones_like(key, dtype=torch.int32))
    return torch.where(here, dst, -1).reshape(topk_idx.shape), splits[:num_experts]


class QuantizedWeights:
    """Stacked weights [E, N, K] as MXFP4 for the product (blocks along K) and, transposed,
    for the input gradient (blocks along N)."""

    def __init__(self, w: torch.Tensor, gated: bool):
        E, N, K = w.shape
        dev = w.device
        new = lambda *s: torch.empty(s, dtype=torch.uint8, device=dev)  # noqa: E731
        self.codes, scales = new(E, N, K // 2), new(E, N, K // 32)
        self.codes_t, scales_t = new(E, K, N // 2), new(E, K, N // 32)
        for e in range(E):
            (self.codes[e], scales[e], self.codes_t[e], scales_t[e]) = \
                Q.omo_per_token_group_quant_mxfp4_rowcol(w[e].contiguous())
        self.scales = M.omo_swizzle_scales_grouped(scales, gated)
        self.scales_t = M.omo_swizzle_scales_grouped(scales_t)


class _FirstOrder(torch.autograd.Function):
    """Gradients as they are, with a graph that refuses to be differentiated.  `anchor` is what
    makes the graph: the gradients may not need one themselves and yet depend on saved tensors
    that do (a loss that is the plain sum of the outputs)."""

    @staticmethod
    def forward(ctx, anchor, *grads):
        return grads

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("MXFP4Experts has no second derivative: the operators of its backward "
                           "pass are not differentiable")


class _Experts(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, topk_w, w1, w2, q1, q2, dst, splits):
        codes, scales = Q.omo_per_token_group_quant_mxfp4(x)
        xc, xs = Q.omo_moe_permute_mxfp4(codes, scales, dst, dst.numel())
        pre, hc, hs = M.omo_grouped_gemm_mxfp4(xc, xs, q1.codes, q1.scales, splits,
                                               activation="swiglu", save_pre=True, quantize=True,
                                               bf16_out=False)
        y = M.omo_grouped_gemm_mxfp4(hc, hs, q2.codes, q2.scales, splits)
        ctx.save_for_backward(xc, xs, pre, hc, hs, y, dst, topk_w, splits, w1, w2)
        ctx.q1, ctx.q2 = q1, q2
        return M.omo_moe_unpermute(y, dst, topk_w)

    @staticmethod
    def backward(ctx, dout):
        with torch.no_grad():
            grads = _Experts._grads(ctx, dout)
        if torch.is_grad_enabled():  # create_graph: autograd does not see through the operators
            there = [i for i, g in enumerate(grads) if g is not None]
            anchor = torch.zeros((), device=dout.device, requires_grad=True)
            for i, g in zip(there, _FirstOrder.apply(anchor, *(grads[i] for i in there))):
                grads[i] = g
        return (*grads, None, None, None, None)

    @staticmethod
    def _grads(ctx, dout):
        xc, xs, pre, hc, hs, y, dst, topk_w, splits, w1, w2 = ctx.saved_tensors
        dy, dtopk, dyc, dys = M.omo_moe_unpermute_grad(dout.contiguous(), y, dst, topk_w,
                                                       quantize=True)
        dh = M.omo_grouped_gemm_mxfp4(dyc, dys, ctx.q2.codes_t, ctx.q2.scales_t, splits)
        dw2 = _weight_grad(w2, dy, hc, hs, splits)
        dz, dzc, dzs = M.omo_bias_act_grad(dh, pre, splits, "swiglu", bias_grad=False, quantize=True)
        dx = None
        if ctx.needs_input_grad[0]:
            dxp = M.omo_grouped_gemm_mxfp4(dzc, dzs, ctx.q1.codes_t, ctx.q1.scales_t, splits)
            dx = M.omo_moe_unpermute(dxp, dst)
        dw1 = _weight_grad(w1, dz, xc, xs, splits)
        return [dx, dtopk, dw1, dw2]


def _weight_grad(w, dy, xc, xs, splits):
    if not w.requires_grad:
        return None
    main = getattr(w, "main_grad", None)
    if main is not None:
        M.omo_grouped_wgrad_mxfp4(dy, xc, xs, splits, accumulate_into=main)
        return None
    return M.omo_grouped_wgrad_mxfp4(dy, xc, xs, splits, out_dtype=w.dtype)


class MXFP4Experts(torch.nn.Module):
    """SwiGLU experts: w1 [E, 2F, H] (gate rows above up rows) and w2 [E, H, F], BF16 (or FP32
    masters, quantized through BF16).  H and F are multiples of 32."""

    def __init__(self, num_experts: int, hidden: int, ffn: int, dtype=torch.bfloat16, device=None):
        super().__init__()
        if hidden % 32 or ffn % 32:
            raise ValueError("hidden and ffn must be multiples of 32")
        self.num_experts = num_experts
        kw = dict(dtype=dtype, device=device)
        self.w1 = torch.nn.Parameter(torch.randn(num_experts, 2 * ffn, hidden, **kw) * hidden ** -0.5)
        self.w2 = torch.nn.Parameter(torch.randn(num_experts, hidden, ffn, **kw) * ffn ** -0.5)
        self._q = None

    def quantize_weights(self) -> None:
        """Lay the weights out as MXFP4; call it after every weight update."""
        with torch.no_grad():
            self._q = (QuantizedWeights(self.w1.to(torch.bfloat16), gated=True),
                       QuantizedWeights(self.w2.to(torch.bfloat16), gated=False))

    def forward(self, x: torch.Tensor, topk_idx: torch.Tensor, topk_w: torch.Tensor) -> torch.Tensor:
        if self._q is None:
            raise RuntimeError("quantize_weights() has to be called before the first forward")
        dst, splits = expert_order(topk_idx, self.num_experts)
        return _Experts.apply(x.contiguous(), topk_w.float().contiguous(), self.w1, self.w2,
                              self._q[0], self._q[1], dst, splits)


def main() -> None:
    """A few training steps of one small layer towards a fixed target (needs a B200)."""
    torch.manual_seed(0)
    E, H, F, T, k = 8, 1024, 512, 2048, 2
    experts = MXFP4Experts(E, H, F, dtype=torch.float32, device="cuda")
    opt = torch.optim.AdamW(experts.parameters(), lr=2e-3)
    x = torch.randn(T, H, device="cuda", dtype=torch.bfloat16)
    target = torch.randn(T, H, device="cuda") * 0.5
    probs = torch.softmax(torch.randn(T, E, device="cuda"), -1)
    topk_w, topk_idx = probs.topk(k, -1)
    for step in range(20):
        experts.quantize_weights()
        loss = (experts(x, topk_idx, topk_w).float() - target).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        if step % 5 == 0 or step == 19:
            print(f"step {step:2d}  loss {loss.item():.4f}")


if __name__ == "__main__":
    main()
