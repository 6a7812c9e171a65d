"""Cases of the MXFP4 mixture-of-experts operators, with their plain forms.

Five operators, each reached through `omo_python_api.mxfp4_moe`:

  grouped    rows sorted by expert times each expert's own MXFP4 weights (ragged groups), with the
             bias / activation epilogue; the same call with transposed weights is the input gradient
  dense      one MXFP4 product with bias, activation and residual in its epilogue
  wgrad      the experts' weight gradients from BF16 output gradients and the saved MXFP4 rows
  act_grad   the gradient of the epilogue: activation and per-expert bias
  unpermute  the weighted sum of expert rows back into token order, and its gradient

MXFP4 operands are code bytes [rows, K/2] (element 2i in the low nibble) and E8M0 bytes
[rows, K/32]; a weight's E8M0 bytes are held as the framework wants them, in the 128x4-tile
layout, laid out once when the weights are made (the two halves of a gate and up projection each in
tiles of their own).
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---------------------------------------------------------------------------- cases
def listed():
    return [
        # one decoding step of a small expert layer: nine rows over eight experts, launch latency counts
        dict(name="experts decode small", op="grouped", E=8, M=9, N=1024, K=2048, act="swiglu", bias=False, pre=False),
        # one decoding step of 16 sequences, top-8 of the 32 experts that a rank hosts: every
        # weight is read for a handful of rows
        dict(name="experts decode", op="grouped", E=32, M=128, N=4096, K=7168, act="swiglu", bias=False, pre=False),
        # a prefill chunk through experts of odd widths, with biases
        dict(name="experts ragged", op="grouped", E=16, M=3001, N=1416, K=2080, act="gelu_tanh", bias=True, pre=False),
        # a training step's gate and up projections of 4096 tokens x top-8: the rows before the
        # activation are kept for the backward pass
        dict(name="experts training", op="grouped", E=32, M=32768, N=4096, K=7168, act="swiglu", bias=False, pre=True),
        # one token through an output projection with its residual
        dict(name="dense one token", op="dense", M=1, N=7168, K=2048, act="none", bias=True, residual=True, pre=False),
        # a training step's dense layer
        dict(name="dense training", op="dense", M=8192, N=8192, K=7168, act="gelu", bias=True, residual=True, pre=True),
        # weight gradients of small experts that saw few rows, some of them none
        dict(name="wgrad small", op="wgrad", E=8, M=301, N=1024, K=768, out="float32"),
        # a training step's weight gradients
        dict(name="wgrad training", op="wgrad", E=8, M=16384, N=4096, K=7168, out="float32"),
        # the epilogue's gradient of a small dense layer
        dict(name="act grad small", op="act_grad", E=1, M=333, N=1024, act="gelu"),
        # the epilogue's gradient of a training step's gate and up projections
        dict(name="act grad training", op="act_grad", E=8, M=16384, N=8192, act="swiglu"),
        # the way back of one decoding step
        dict(name="unpermute decode", op="unpermute", T=16, topk=8, H=7168, grad=False),
        # the way back of a training step and its gradient
        dict(name="unpermute training", op="unpermute", T=4096, topk=8, H=7168, grad=True),
    ]


def _log(rng, lo, hi, mult=1):
    """A size between lo and hi, spread over its logarithm, rounded to a multiple."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(mult, int(round(v / mult)) * mult)


def draw(rng):
    op = rng.choice(["grouped", "grouped", "dense", "wgrad", "act_grad", "unpermute"])
    act = rng.choice(["none", "relu", "relu2", "silu", "gelu", "gelu_tanh", "swiglu"])
    if op == "grouped":
        c = dict(op=op, E=_log(rng, 1, 64), M=_log(rng, 1, 20000), N=_log(rng, 128, 4096, 16),
                 K=_log(rng, 128, 7168, 32), act=act, bias=rng.random() < 0.5, pre=rng.random() < 0.5)
    elif op == "dense":
        c = dict(op=op, M=_log(rng, 1, 8192), N=_log(rng, 128, 8192, 16), K=_log(rng, 128, 7168, 32), act=act,
                 bias=rng.random() < 0.7, residual=rng.random() < 0.7, pre=rng.random() < 0.5)
    elif op == "wgrad":
        c = dict(op=op, E=_log(rng, 1, 32), M=_log(rng, 1, 16384), N=_log(rng, 64, 4096, 8), K=_log(rng, 64, 4096, 32),
                 out=rng.choice(["float32", "bfloat16"]))
    elif op == "act_grad":
        c = dict(op=op, E=_log(rng, 1, 32), M=_log(rng, 1, 16384), N=_log(rng, 128, 8192, 16), act=act)
    else:
        c = dict(op=op, T=_log(rng, 1, 4096), topk=rng.randint(1, 8), H=_log(rng, 64, 7168, 8), grad=rng.random() < 0.5)
    return c


def _width(case):
    """Columns of the activation's result."""
    return case["N"] // 2 if case.get("act") == "swiglu" else case["N"]


def _shares(E):
    """The experts' shares of the rows: uneven, the busiest about seven times the least busy."""
    return [math.exp(2.0 * ((e * 7) % E) / max(1, E - 1)) for e in range(E)]


def work(case):
    op = case["op"]
    if op == "unpermute":
        T, k, H = case["T"], case["topk"], case["H"]
        one = 2.0 * T * k * H + 2.0 * T * H + 8.0 * T * k  # expert rows, token rows, map and weights
        if not case["grad"]:
            return {"bytes": one, "flops": 2.0 * T * k * H}
        return {"bytes": one + 2.0 * T * H + 2.0 * T * k * H + 4.0 * T * k, "flops": 5.0 * T * k * H}
    E, M, N = case.get("E", 1), case["M"], case["N"]
    if op == "act_grad":
        return {"bytes": 2.0 * M * (_width(case) + 2 * N) + 4.0 * E * N, "flops": 10.0 * M * N}
    K = case["K"]
    if op == "wgrad":
        size = 4.0 if case["out"] == "float32" else 2.0
        return {"bytes": 2.0 * M * N + M * K * 17 / 32 + size * E * N * K, "flops": 2.0 * M * N * K}
    p = _shares(E)
    active = sum(1 - (1 - x / sum(p)) ** M for x in p)  # experts that get a row
    outs = _width(case) * (2 if case.get("residual") else 1) + (N if case["pre"] else 0)
    return {"bytes": (M + active * N) * K * 17 / 32 + 2.0 * M * outs + (2.0 * active * N if case["bias"] else 0),
            "flops": 2.0 * M * N * K}


# ---------------------------------------------------------------------------- inputs
def _quantize(x):
    """Rowwise MXFP4 of a float tensor: blocks of 32 along the last dimension, the shared scale
    2^ceil(log2(amax / 6)), codes to the nearest (ties to even)."""
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    e = torch.ceil(torch.log2(torch.clamp(b.abs().amax(-1) / 6, min=1e-10)))
    v = b * torch.exp2(-e)[..., None]
    a = v.abs().clamp(max=6)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = torch.round(a / step) * step
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = (code | ((v < 0).to(torch.uint8) << 3)).reshape(*x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _tiles(s, parts):
    """E8M0 bytes [E, N, S] -> the bytes of each of an expert's parts in the 128x4-tile layout,
    [E, parts * round_up(N / parts, 128), round_up(S, 4)]: byte (r, c) of a part at
    ((r / 128) * S4 + c / 4) * 512 + (r % 32) * 16 + (r % 128) / 32 * 4 + c % 4."""
    E, N, S = s.shape
    p = torch.nn.functional.pad(s.reshape(E * parts, N // parts, S), (0, -S % 4, 0, -(N // parts) % 128))
    t = p.reshape(E * parts, p.shape[1] // 128, 4, 32, p.shape[2] // 4, 4).permute(0, 1, 4, 3, 2, 5)
    return t.reshape(E, parts * p.shape[1], p.shape[2]).contiguous()


def _untiles(t, N, S, parts):
    E, Np, Sp = t.shape
    r = t.reshape(E * parts, Np // parts // 128, Sp // 4, 32, 4, 4).permute(0, 1, 4, 3, 2, 5)
    return r.reshape(E * parts, Np // parts, Sp)[:, :N // parts, :S].reshape(E, N, S)


def _splits(case, gen):
    """Rows per expert of an uneven routing, as int32 on the GPU and as a list."""
    p = torch.tensor(_shares(case["E"]))
    picks = torch.multinomial(p, case["M"], replacement=True, generator=gen)
    m = torch.bincount(picks, minlength=case["E"])
    return m.to(torch.int32).to(DEV), m.tolist()


def _rows(M, K, g):
    """Activations: normal, with a few channels of larger magnitude."""
    x = torch.randn(M, K, device=DEV, generator=g)
    return x * (1 + 7 * (torch.rand(K, device=DEV, generator=g) < 0.01))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case)
    op = case["op"]
    if op == "unpermute":
        T, k, H = case["T"], case["topk"], case["H"]
        R = T * k
        s["y"] = torch.randn(R, H, device=DEV, generator=g).to(torch.bfloat16)
        s["map"] = torch.randperm(R, device=DEV, generator=g).to(torch.int32).reshape(T, k)
        s["w"] = torch.softmax(torch.randn(T, k, device=DEV, generator=g), -1)
        s["dout"] = torch.randn(T, H, device=DEV, generator=g).to(torch.bfloat16)
        return s
    s["E"] = E = case.get("E", 1)
    M, N = case["M"], case["N"]
    s["splits"], s["counts"] = _splits(s, torch.Generator().manual_seed(seed))
    if op == "act_grad":
        s["dy"] = (torch.randn(M, _width(case), device=DEV, generator=g) * 1e-2).to(torch.bfloat16)
        s["pre_rows"] = (torch.randn(M, N, device=DEV, generator=g) * 1.5).to(torch.bfloat16)
        return s
    K = case["K"]
    s["a"], s["sa"] = _quantize(_rows(M, K, g))
    if op == "wgrad":
        s["dy"] = (torch.randn(M, N, device=DEV, generator=g) * 1e-2).to(torch.bfloat16)
        return s
    s["b"] = torch.empty(E, N, K // 2, dtype=torch.uint8, device=DEV)
    sb = torch.empty(E, N, K // 32, dtype=torch.uint8, device=DEV)
    for e in range(E):
        s["b"][e], sb[e] = _quantize(torch.randn(N, K, device=DEV, generator=g) * K ** -0.5)
    s["parts"] = 2 if case["act"] == "swiglu" else 1
    s["sb"] = _tiles(sb, s["parts"])
    s["bias_rows"] = (torch.randn(E, N, device=DEV, generator=g) * 0.3).to(torch.bfloat16) if case["bias"] else None
    s["res"] = torch.randn(M, _width(case), device=DEV, generator=g).to(torch.bfloat16) if case.get("residual") else None
    return s


# ---------------------------------------------------------------------------- plain forms
def _values(codes, scales):
    """MXFP4 -> float32."""
    t = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    v = torch.stack((t[(codes & 15).long()], t[(codes >> 4).long()]), -1).reshape(*codes.shape[:-1], -1, 32)
    return (v * torch.exp2(scales.float() - 127)[..., None]).reshape(*codes.shape[:-1], -1)


def _padded(s):
    """Index of each expert's rows in a [E, most] grid (row 0 where there is none), and which are rows."""
    most = max(1, max(s["counts"]))
    ends = torch.cumsum(s["splits"], 0)
    at = torch.arange(most, device=DEV)
    there = at < s["splits"][:, None]
    return torch.where(there, (ends - s["splits"])[:, None] + at, 0).long(), there


def _expert(s):
    return torch.repeat_interleave(torch.arange(s["E"], device=DEV), s["splits"].long(), output_size=s["M"])


def _act(z, act):
    if act == "swiglu":
        a, b = z.chunk(2, -1)
        return a / (1 + torch.exp(-a)) * b
    if act == "relu":
        return torch.clamp(z, min=0)
    if act == "relu2":
        return torch.clamp(z, min=0) ** 2
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3)))
    return z


def _act_grad(z, dy, act):
    if act == "swiglu":
        a, b = z.chunk(2, -1)
        sg = 1 / (1 + torch.exp(-a))
        return torch.cat((dy * b * sg * (1 + a * (1 - sg)), dy * a * sg), -1)
    if act == "relu":
        return dy * (z > 0)
    if act == "relu2":
        return dy * 2 * torch.clamp(z, min=0)
    if act == "silu":
        sg = 1 / (1 + torch.exp(-z))
        return dy * sg * (1 + z * (1 - sg))
    if act == "gelu":
        return dy * (0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) / (2 * math.pi) ** 0.5)
    if act == "gelu_tanh":
        c = (2 / math.pi) ** 0.5
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return dy * (0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z))
    return dy * 1.0


def _plain(s):
    op = s["op"]
    bf = torch.bfloat16
    if op == "unpermute":
        rows = s["y"].float()[s["map"].long()]
        out = (s["w"][..., None] * rows).sum(1).to(bf)
        if not s["grad"]:
            return out
        d = s["dout"].float()
        dy = torch.empty_like(s["y"])
        dy[s["map"].long().reshape(-1)] = (s["w"][..., None] * d[:, None]).to(bf).reshape(-1, s["H"])
        return {"out": out, "dy": dy, "dw": (rows * d[:, None]).sum(-1)}
    if op == "act_grad":
        dz = _act_grad(s["pre_rows"].float(), s["dy"].float(), s["act"])
        at, there = _padded(s)
        return {"dz": dz.to(bf), "dbias": (dz[at] * there[..., None]).sum(1)}
    a = _values(s["a"], s["sa"])
    at, there = _padded(s)
    if op == "wgrad":
        dy = s["dy"].float()[at] * there[..., None]
        return torch.matmul(dy.transpose(1, 2), a[at]).to(getattr(torch, s["out"]))
    z = torch.matmul(a[at], _values(s["b"], _untiles(s["sb"], s["N"], s["K"] // 32, s["parts"])).transpose(1, 2))[there]
    if s["bias_rows"] is not None:
        z = z + s["bias_rows"].float()[_expert(s)]
    y = _act(z, s["act"])
    if s["res"] is not None:
        y = y + s["res"].float()
    return {"c": y.to(bf), "pre": z.to(bf)} if s["pre"] else y.to(bf)


# ---------------------------------------------------------------------------- the framework's calls
_ops = None


def _own():
    global _ops
    if _ops is None:
        pkg = os.path.join(os.getcwd(), "mxfp4-hopper_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from omo_python_api import mxfp4_moe
        _ops = mxfp4_moe
    return _ops


def run(state):
    s = state
    if not own:
        return _plain(s)
    ops, op = _own(), s["op"]
    if op == "unpermute":
        out = ops.omo_moe_unpermute(s["y"], s["map"], s["w"])
        if not s["grad"]:
            return out
        dy, dw = ops.omo_moe_unpermute_grad(s["dout"], s["y"], s["map"], s["w"])
        return {"out": out, "dy": dy, "dw": dw}
    if op == "act_grad":
        dz, dbias = ops.omo_bias_act_grad(s["dy"], s["pre_rows"], s["splits"], s["act"])
        return {"dz": dz, "dbias": dbias}
    if op == "wgrad":
        return ops.omo_grouped_wgrad_mxfp4(s["dy"], s["a"], s["sa"], s["splits"], out_dtype=getattr(torch, s["out"]))
    if op == "dense":
        r = ops.omo_gemm_mxfp4_act(s["a"], s["sa"], s["b"][0], s["sb"][0],
                                   bias=None if s["bias_rows"] is None else s["bias_rows"][0],
                                   activation=s["act"], residual=s["res"], save_pre=s["pre"])
    else:
        r = ops.omo_grouped_gemm_mxfp4(s["a"], s["sa"], s["b"], s["sb"], s["splits"], bias=s["bias_rows"],
                                       activation=s["act"], save_pre=s["pre"])
    return {"c": r[0], "pre": r[1]} if s["pre"] else r


# ---------------------------------------------------------------------------- 64 bits
def _decode64(codes, scales):
    """Code by code from the format: sign, two exponent bits, one mantissa bit, times 2^(scale - 127)."""
    q = torch.stack((codes % 16, codes // 16), -1).flatten(-2)
    sign = 1.0 - 2.0 * (q // 8).double()
    ex, man = ((q % 8) // 2).int(), (q % 2).double()
    mag = torch.where(ex == 0, man / 2, torch.ldexp(1 + man / 2, ex - 1))
    return torch.ldexp(sign * mag, torch.repeat_interleave(scales.int(), 32, -1) - 127)


def _act64(z, act):
    if act == "swiglu":
        h = z.shape[1] // 2
        return z[:, :h] * torch.sigmoid(z[:, :h]) * z[:, h:]
    if act in ("relu", "relu2"):
        return torch.where(z > 0, z, 0.0) ** (2 if act == "relu2" else 1)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    if act == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
    return z


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "unpermute":
        T, k, H = case["T"], case["topk"], case["H"]
        y, w, d, m = s["y"].double(), s["w"].double(), s["dout"].double(), s["map"].long()
        out = torch.zeros(T, H, dtype=torch.float64, device=DEV)
        dy, dw = torch.zeros_like(y), torch.zeros(T, k, dtype=torch.float64, device=DEV)
        for j in range(k):
            out += w[:, j:j + 1] * y[m[:, j]]
            dy[m[:, j]] = w[:, j:j + 1] * d
            dw[:, j] = torch.einsum("th,th->t", d, y[m[:, j]])
        return {"out": out, "dy": dy, "dw": dw} if case["grad"] else out
    starts = [0]
    for m in s["counts"]:
        starts.append(starts[-1] + m)
    parts = [(e, slice(starts[e], starts[e + 1])) for e in range(s["E"])]
    N = case["N"]
    if op == "act_grad":
        z = s["pre_rows"].double().requires_grad_(True)
        with torch.enable_grad():
            y = _act64(z, case["act"])
            dz, = torch.autograd.grad(y, z, s["dy"].double())
        return {"dz": dz, "dbias": torch.stack([dz[r].sum(0) for _, r in parts])}
    if op == "wgrad":
        dw = torch.empty(s["E"], N, case["K"], dtype=torch.float64, device=DEV)
        for e, r in parts:
            dw[e] = s["dy"][r].double().t() @ _decode64(s["a"][r], s["sa"][r])
        return dw
    z = torch.empty(case["M"], N, dtype=torch.float64, device=DEV)
    sb = _untiles(s["sb"], N, case["K"] // 32, s["parts"])
    for e, r in parts:
        z[r] = _decode64(s["a"][r], s["sa"][r]) @ _decode64(s["b"][e], sb[e]).t()
        if s["bias_rows"] is not None:
            z[r] += s["bias_rows"][e].double()
    y = _act64(z, case["act"])
    if s["res"] is not None:
        y = y + s["res"].double()
    return {"c": y, "pre": z} if case["pre"] else y
