"""The 8-bit projections and adapters from their definitions, in 64 bits, with
the error bounds their kernels have to stay within (shared by the GPU tests).

Bounds count roundings: one to bf16 is off by at most 2^-8 of the value, one
to fp32 by 2^-24; a sum of K products that the tensor cores accumulate in
fp32 (they may truncate: 2^-23 per addition) is off by at most the number
of additions times 2^-23 of the sum of the magnitudes.  An 8-bit MMA adds 32
products at a time, a 16-bit one 16."""
import torch

TOP, TINY = 448.0, 2.0 ** -100
BF16, F32, SUM = 2.0 ** -8, 2.0 ** -24, 2.0 ** -23


def e4m3_step(v):
    """Distance between e4m3 neighbours around v (3 mantissa bits, exponents from -6)."""
    _, e = torch.frexp(v)
    return torch.ldexp(torch.ones_like(v), torch.clamp_min(e - 1, -6) - 3)


def quant(y):
    """(values the 8 bits are rounded from, scale) of the rows of y (fp64)."""
    s = torch.clamp_min(y.abs().amax(dim=1), TINY) / TOP
    return y / s[:, None], s


def check_quant(q, s, y, s_tol):
    """q / s against the rows of y: the scale within s_tol, every value one of
    the (at most two) e4m3 numbers nearest to y / s, fp32 rounding apart."""
    v, s_ref = quant(y)
    assert ((s.double() - s_ref).abs() <= s_ref * s_tol).all(), ((s.double() - s_ref).abs() / s_ref).max()
    off = (q.double() - v).abs()
    lim = e4m3_step(v) / 2 + v.abs() * 2.0 ** -21
    assert (off <= lim).all(), (off - lim).max()


def linear(xq, xs, wq, ws):
    """(x w^T with scales, bound of its fp32 error) in fp64."""
    x, w = xq.double() * xs.double()[:, None], wq.double() * ws.double()[:, None]
    K = x.shape[1]
    return x @ w.t(), (K / 32 + 16) * SUM * (x.abs() @ w.abs().t())


def silu_mul(g, eg, u, eu):
    s = g * torch.sigmoid(g)
    # |silu'| <= 1.1; expf and the division: a few fp32 roundings
    return s * u, 1.1 * eg * u.abs() + (s.abs() + 1.1 * eg) * eu + 2.0 ** -20 * (s * u).abs()


def lora(y, x, a, b, adapter, scale, ranks, slices):
    """(y + adapters, bound) in fp64."""
    out, err = y.double(), torch.zeros_like(y, dtype=torch.float64)
    slices = [y.shape[1]] if slices is None else slices
    R, K = b.shape[2], x.shape[1]
    for ad in sorted(set(adapter.tolist())):
        if ad < 0 or ad >= a.shape[0]:
            continue
        rows = (adapter == ad).nonzero()[:, 0]
        r = R if ranks is None else int(ranks[ad])
        sc = 1.0 if scale is None else scale[ad].double()
        at = 0
        for i, w in enumerate(slices):
            A, Bm, xr = a[ad, i * R:i * R + r].double(), b[ad, at:at + w, :r].double(), x[rows].double()
            t = xr @ A.t() * sc
            # the first sum, the scale's rounding and the two bf16 words of t
            et = (K / 16 + 80) * SUM * (xr.abs() @ A.abs().t()) * abs(sc) + (2.0 ** -16 + 2 * F32) * t.abs()
            out[rows, at:at + w] += t @ Bm.t()
            err[rows, at:at + w] += et @ Bm.abs().t() + (R / 4 + 4) * SUM * (t.abs() @ Bm.abs().t())
            at += w
    return out, err


def check_bf16(got, ref, err):
    """A bf16 result: one rounding (2^-8) on top of the fp32 error `err`."""
    off, lim = (got.double() - ref).abs(), ref.abs() * BF16 + err * (1 + BF16) + 1e-37
    assert torch.isfinite(got.float()).all()
    assert (off <= lim).all(), f"{(off / lim).max().item()} of the bound"
