"""The ragged expert products in 64 bits, and how far a kernel that sums in fp32 may be from them."""
import torch


def spans(ends):
    start = 0
    for g, end in enumerate(ends):
        if end > start:
            yield g, start, end
        start = max(start, end)


def mm(x, w, ends):
    """(product, product of the magnitudes), both in float64."""
    y = torch.zeros((x.shape[0], w.shape[1]), dtype=torch.float64, device=x.device)
    s = torch.zeros_like(y)
    for g, a, b in spans(ends):
        xd, wd = x[a:b].double(), w[g].double()
        y[a:b] = xd @ wd.t()
        s[a:b] = xd.abs() @ wd.abs().t()
    return y, s


def mm_int8(x, w, x_scale, w_scale, ends):
    """The integer sums, which float64 holds exactly (so that a sum of zero is one here too), then the scales."""
    y = torch.zeros((x.shape[0], w.shape[1]), dtype=torch.float64, device=x.device)
    for g, a, b in spans(ends):
        y[a:b] = (x[a:b].double() @ w[g].double().t()) * x_scale[a:b].double()[:, None] * w_scale[g].double()
    return y


def wgrad(dy, x, ends):
    w = torch.zeros((len(ends), dy.shape[1], x.shape[1]), dtype=torch.float64, device=x.device)
    s = torch.zeros_like(w)
    for g, a, b in spans(ends):
        w[g] = dy[a:b].double().t() @ x[a:b].double()
        s[g] = dy[a:b].double().abs().t() @ x[a:b].double().abs()
    return w, s


def check(got, ref, mags, depth):
    """|got - ref| against what the arithmetic allows: `depth` fp32 additions, each off by at most one unit in the last place
    (2^-23) of a partial sum, which no sum of magnitudes is below, then one rounding to the output's type (half a step, or half
    of the smallest step)."""
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * half
    sums = depth * 2.0 ** -23 * mags
    bound = sums + half * (ref.abs() + sums) + tiny
    off = (got.double() - ref).abs()
    assert torch.isfinite(got).all()
    bad = off > bound
    assert not bad.any(), (int(bad.sum()), float((off - bound).max()), bad.nonzero()[:4].tolist())


def sized(total, groups, gen, empty=0.3):
    """Ends of `groups` ragged groups over `total` rows, some of them empty."""
    p = torch.rand((groups,), generator=gen) * (torch.rand((groups,), generator=gen) >= empty)
    if float(p.sum()) == 0:
        p[-1] = 1.0
    counts = torch.bincount(torch.multinomial(p, total, replacement=True, generator=gen), minlength=groups) if total else torch.zeros(groups)
    return torch.cumsum(counts, 0).to(torch.int64).tolist()
