"""Plain 64-bit forms of the MXFP4 expert operators, and their inputs."""
import math

import torch

ACTS = ["none", "relu", "relu2", "silu", "gelu", "gelu_tanh", "swiglu"]
MAG = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def values(codes, scales):
    """MXFP4 codes [.., K/2] and E8M0 bytes [.., K/32] -> float64 [.., K]; byte 255 is NaN."""
    t = torch.tensor(MAG + tuple(-v for v in MAG), dtype=torch.float64, device=codes.device)
    v = torch.stack((t[(codes & 15).long()], t[(codes >> 4).long()]), -1).flatten(-2)
    f = torch.where(scales == 255, math.nan, torch.exp2(scales.double() - 127))
    return v * f.repeat_interleave(32, -1)


def mxfp4(rows, K, seed, lo=118, hi=130, device="cuda"):
    """Random codes and scale bytes in [lo, hi): rows [*rows, K/2] and [*rows, K/32]."""
    g = torch.Generator().manual_seed(seed)
    rows = rows if isinstance(rows, tuple) else (rows,)
    c = torch.randint(0, 256, (*rows, K // 2), generator=g, dtype=torch.uint8)
    s = torch.randint(lo, hi, (*rows, K // 32), generator=g).to(torch.uint8)
    return c.to(device), s.to(device)


def spans(splits, M):
    """Row ranges of the experts: negative splits count as 0, rows end at M."""
    out, at = [], 0
    for m in splits:
        end = min(at + max(m, 0), M)
        out.append((min(at, M), end))
        at += max(m, 0)
    return out


def act(z, name):
    if name == "swiglu":
        a, b = z.chunk(2, -1)
        return a * torch.sigmoid(a) * b
    if name == "relu":
        return torch.where(z > 0, z, 0.0)
    if name == "relu2":
        return torch.where(z > 0, z * z, 0.0)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z / math.sqrt(2)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def slope_bound(z, name):
    """A bound on the activation's change per unit change of z, elementwise [.., N]."""
    if name == "relu2":
        return 2 * z.abs() + 1
    if name == "swiglu":
        a, b = z.chunk(2, -1)
        return torch.cat((1.2 * b.abs(), a.abs()), -1) + 1
    return torch.full_like(z, 1.2)


def grouped(ac, asc, bc, bsc, splits, bias, name, residual):
    """z, c and the bound on c's and z's error, per element, all float64; rows without an
    expert are NaN.  The bound: one rounding to BF16 (2^-9 of the result, 2^-8 allowed),
    plus the f32 accumulation at 2^-18 of the sum of |a b| (K / 64 partial sums at 2^-24
    each, with margin) times the activation's slope, plus 2^-20 of the activation's own
    value for its f32 evaluation."""
    M, N = ac.shape[0], bc.shape[1]
    z = torch.full((M, N), math.nan, dtype=torch.float64, device=ac.device)
    ab = torch.zeros_like(z)
    for e, (i, j) in enumerate(spans(splits, M)):
        a, b = values(ac[i:j], asc[i:j]), values(bc[e], bsc[e])
        z[i:j] = a @ b.T
        ab[i:j] = a.abs() @ b.abs().T
        if bias is not None:
            z[i:j] += bias[e].double()
            ab[i:j] += bias[e].double().abs()
    acc = 2.0 ** -18 * ab
    y = act(z, name)
    prop = acc * slope_bound(z, name)
    if name == "swiglu":
        prop = prop[:, :N // 2] + prop[:, N // 2:]
    prop = prop + 2.0 ** -20 * y.abs()
    if residual is not None:
        y = y + residual.double()
    return z, y, 2.0 ** -8 * z.abs() + acc, 2.0 ** -8 * y.abs() + prop + 1e-38


def check(got, want, bound, what=""):
    """|got - want| <= bound wherever want is finite; NaN where it is NaN."""
    got = got.double()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN in other places"
    err = torch.where(nan, 0.0, (got - want).abs())
    bound = torch.where(nan, 1.0, bound)
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst error / bound = {(err / bound)[bad].max():.3f}"
