"""Weights of 4 bits in 64 bits: their quantiser from its definition, products with them, and how far a kernel may be off."""
import torch

LEAST = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}


def quantize(w, group, scale_dtype):
    """(values int8 (..., N, K), scale (..., N, K / group)); groups that are not finite: NaN and zeros."""
    parts = w.unflatten(-1, (-1, group))
    peak = parts.float().abs().amax(-1)
    scale = torch.maximum(peak * torch.tensor(1 / 7, device=w.device), torch.tensor(LEAST[scale_dtype], device=w.device)).to(scale_dtype)
    bad = ~(torch.isfinite(peak) & torch.isfinite(scale))
    scale = torch.where(bad, torch.tensor(float("nan"), dtype=scale_dtype, device=w.device), scale)
    values = torch.round(parts.double() / scale.double()[..., None]).clamp(-8, 7)
    values = torch.where(bad[..., None], torch.zeros_like(values), values).to(torch.int8)
    return values.flatten(-2), scale


def weights(values, scale):
    return (values.double().unflatten(-1, (scale.shape[-1], -1)) * scale.double()[..., None]).flatten(-2)


def unpack(q, scale, columns):
    """(values, scale) of tiles, element by element from the description of the layout."""
    lead, (strips, tiles) = q.shape[:-3], q.shape[-3:-1]
    n, k = torch.arange(strips * 16), torch.arange(columns)
    r, within = n % 16, k % 128
    j, c, e = within // 32, within % 32 // 8, within % 8
    # columns (0,2), (4,6), (1,3), (5,7) in bytes 0 .. 3, the first in the low four bits
    byte = 16 * (r[:, None] + 16 * c) + 4 * j + 2 * (e % 2) + e // 4
    high = e // 2 % 2
    raw = q.cpu().reshape(-1, strips, tiles, 1024)[:, (n // 16)[:, None], (k // 128)[None, :], byte]
    values = torch.where(high.bool(), raw >> 4, raw & 15).to(torch.int8) - 8
    per = scale.shape[-1]
    g = torch.arange(columns // (128 // per))
    s = scale.cpu().reshape(-1, strips, tiles, 16, per)[:, (n // 16)[:, None], (g // per)[None, :], r[:, None], (g % per)[None, :]]
    return values.reshape(*lead, strips * 16, columns), s.reshape(*lead, strips * 16, -1)


def mm(x, values, scale, ends):
    """(product, sum of |x| scale), both in float64; `values` (E, N, K)."""
    y = torch.zeros((x.shape[0], values.shape[1]), dtype=torch.float64, device=x.device)
    m = torch.zeros_like(y)
    start = 0
    for g, end in enumerate(ends):
        if end > start:
            xd = x[start:end].double()
            y[start:end] = xd @ weights(values[g], scale[g]).t()
            m[start:end] = xd.abs() @ weights(torch.ones_like(values[g]), scale[g]).abs().t()
            start = end
    return y, m


def sums_bound(m, k, group):
    """The kernels sum (24 + q) x and -24 x over a group, 2 group terms of 55 |x| together at most, then K / group scaled sums over
    up to 8 waves: every fp32 addition is off by at most one unit in the last place (2^-23) of a partial sum, which no sum of
    magnitudes is below."""
    return (2 * group + k / group + 10) * 2.0 ** -23 * 55 * m


def check(got, ref, m, k, group):
    """... then one rounding to the output's type."""
    half, info = torch.finfo(got.dtype).eps / 2, torch.finfo(got.dtype)
    sums = sums_bound(m, k, group)
    bad = (got.double() - ref).abs() > sums + half * (ref.abs() + sums) + info.smallest_normal * half
    assert torch.isfinite(got).all()
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())
