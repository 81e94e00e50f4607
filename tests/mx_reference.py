"""MXFP4 in plain 64-bit torch, from the format's definition, for tests."""
import torch

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def block_exponents(x):
    """e of the scale 2**e of every block of 32 along the last dimension (x finite)."""
    top = x.double().unflatten(-1, (-1, 32)).abs().amax(-1)
    _, e = torch.frexp(top)
    return torch.where(top > 0, (e - 3).clamp(min=-127), torch.full_like(e, -127))


def codes_at(x, e):
    """The code of every value of x under the scales 2**e: the nearest, ties to the even code."""
    q = x.double().unflatten(-1, (-1, 32)) * torch.pow(2.0, -e.double()).unsqueeze(-1)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    d = (q.abs().unsqueeze(-1) - grid).abs()
    # the distances of a tie are equal; an even code wins over an odd one
    odd = torch.arange(8, device=x.device) % 2
    near = d == d.amin(-1, keepdim=True)
    code = torch.where(near & (odd == 0), 0, torch.where(near, 1, 2)).argmin(-1)
    return (code + 8 * torch.signbit(q).long()).flatten(-2)


def quantize(x):
    """(codes uint8 [..., K/2], scales uint8 [..., K/32]), NaN and infinities included."""
    bad = (~torch.isfinite(x)).unflatten(-1, (-1, 32)).any(-1)
    e = block_exponents(torch.nan_to_num(x.double(), 0, 0, 0))
    c = codes_at(torch.nan_to_num(x.double(), 0, 0, 0), e)
    c = torch.where(bad.repeat_interleave(32, -1), 0, c)
    byte = torch.where(bad, 255, e + 127)
    return (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8), byte.to(torch.uint8)


def values(codes, scales):
    """The 64-bit values that codes and scales stand for."""
    grid = torch.tensor(GRID, dtype=torch.float64, device=codes.device)
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    v = torch.where(n >= 8, -grid[n & 7], grid[n & 7])
    s = torch.where(scales == 255, float("nan"), torch.pow(2.0, scales.double() - 127))
    return v * s.repeat_interleave(32, -1)


def rounded(x):
    return values(*quantize(x))


def sum_error(k):
    """Bound on the error of an fp32 sum of k exact products over the sum of their magnitudes: a tree of 7
    levels inside a step of 128, the steps one after another, and up to 8 parts joined, each addition off by
    at most 2^-23 (a truncated one) of what it adds up."""
    return (7 + -(-k // 128) + 8) * 2.0 ** -23


def gemm(a, w, bias=None):
    """(a @ w^T + bias, bound on an fp32 evaluation's error) of 64-bit values."""
    y, size = a @ w.t(), a.abs() @ w.abs().t()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y, size * (sum_error(a.shape[1]) + 2.0 ** -23)


def act(g, kind):
    if kind == "silu":
        return g * torch.sigmoid(g)
    return torch.nn.functional.gelu(g, approximate="tanh")


def moe(x, weights, ids, w1, w2, kind):
    """(out, bound on the kernels' error before the last rounding): x [T, H] any type, w1 [E, 2I, H] and w2
    [E, H, I] 64-bit values.  The intermediate is rounded to MXFP4, so an fp32 error can move it over a
    rounding border: the bound takes the codes at both ends of its error."""
    xq = rounded(x)
    out, off = torch.zeros_like(xq), torch.zeros_like(xq)
    inter, experts, slots = w2.shape[2], w1.shape[0], ids.shape[1]
    weights = weights.to(xq.device).double()
    for e in range(experts):
        rows, slot = (ids.to(xq.device) == e).nonzero(as_tuple=True)
        if not rows.numel():
            continue
        gu, dgu = gemm(xq[rows], w1[e])
        g, u, dg, du = gu[:, :inter], gu[:, inter:], dgu[:, :inter], dgu[:, inter:]
        h = act(g, kind) * u
        # |act'| < 1.13; exp2 and reciprocal in hardware: a few 2^-23 of |act|, as |t| 2^-23 grows with g
        dh = 1.13 * dg * (u.abs() + du) + act(g, kind).abs() * du + h.abs() * (16 + 4 * g.abs()) * 2.0 ** -23
        size = h.abs()
        ends = [(size - dh).clamp(min=0), size + dh]
        hq = rounded(h)
        near = [rounded(v) for v in ends] + [v for end in ends for v in values_at(size, dh, block_exponents(end))]
        slack = torch.stack(near).sub(hq.abs()).abs().amax(0)
        y, dy = gemm(hq, w2[e])
        dy = dy + slack @ w2[e].abs().t()
        w = weights[rows, slot].unsqueeze(1)
        out.index_add_(0, rows, w * y)
        off.index_add_(0, rows, w.abs() * (dy + y.abs() * (slots + 1) * 2.0 ** -23))
    return out, off


def values_at(size, d, e):
    """The values of size - d and size + d under given scales."""
    grid = torch.tensor(GRID, dtype=torch.float64, device=size.device)
    s = torch.pow(2.0, e.double()).repeat_interleave(32, -1)
    return [grid[codes_at(v, e)] * s for v in ((size - d).clamp(min=0), size + d)]


def half_step(y, dtype):
    """What one rounding to dtype can be off: half a step, or half the smallest subnormal."""
    f = torch.finfo(dtype)
    return y.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2
