"""A layer of experts from its definition in 64 bits, and how far a kernel with sums in fp32 may be from it."""
import torch

ULP = 2.0 ** -23


def select(scores, top_k):
    """The top_k largest of every row, largest first, ties to the lower index, NaN above every number."""
    key = torch.where(torch.isnan(scores), torch.full_like(scores, float("inf")), scores)
    # (a NaN before an infinity, whichever comes first)
    order = torch.argsort(torch.isnan(scores).to(torch.int8), dim=-1, descending=True, stable=True)
    order = order.gather(-1, torch.argsort(key.gather(-1, order), dim=-1, descending=True, stable=True))
    return order[:, :top_k]


class Layer:
    """`w1` (E, 2H, K), `w2` (E, K, H): the weights that stand there, in any type; `mag1`, `mag2`: what bounds the magnitudes that
    the kernel sums for a unit of |x| (the weights' own; for 4 bits see int4_ref.sums_bound); `depth1`, `depth2`: the longest chain of
    additions.  A chain of a lane has K / 16 products, of which two make an addition or two; 30 additions join lanes, waves
    and tokens."""

    def __init__(self, x, gate, w1, w2, top_k, bias, mag1=None, mag2=None, depth1=None, depth2=None):
        self.x, self.top_k = x.double(), top_k
        K, H = x.shape[1], w2.shape[2]
        self.scores = self.x @ gate.double().t() + (0 if bias is None else bias.double())
        self.scores_off = (K / 16 + 30) * ULP * (self.x.abs() @ gate.double().abs().t() + (0 if bias is None else bias.double().abs()))
        self.w1, self.w2 = w1, w2
        self.mag1, self.mag2 = w1.abs() if mag1 is None else mag1, w2.abs() if mag2 is None else mag2
        self.depth1, self.depth2 = depth1 or K / 16 + 30, depth2 or H / 8 + 30
        self.dtype = x.dtype

    def check(self, out, ids, weights):
        T = self.x.shape[0]
        want = select(self.scores, self.top_k)
        # the selection is the exact one wherever no two candidates are closer than the kernel's error
        ranked = self.scores.sort(dim=-1, descending=True).values
        off = 2 * self.scores_off.amax(-1, keepdim=True)
        near = ranked[:, :-1] - ranked[:, 1:] <= off
        for t in range(T):
            if not near[t, :self.top_k].any():
                assert ids[t].tolist() == want[t].tolist(), t
            else:
                assert len(set(ids[t].tolist())) == self.top_k
                assert (self.scores[t, ids[t].long()] >= ranked[t, :self.top_k] - off[t]).all(), t
        chosen = self.scores.gather(-1, ids.long())
        share = torch.softmax(chosen, -1)
        share_off = share * (2 * off + 2.0 ** -18)
        assert ((weights.double() - share).abs() <= share_off + 1e-30).all()
        ref, bound = torch.zeros_like(self.x), torch.zeros_like(self.x)
        half = torch.finfo(self.dtype).eps / 2
        for e in torch.unique(ids).tolist():
            t, r = torch.nonzero(ids == e, as_tuple=True)
            x = self.x[t]
            h, d = x @ self.w1[e].double().t(), self.depth1 * ULP * (x.abs() @ self.mag1[e].double().t())
            g, u = h.chunk(2, -1)
            dg, du = d.chunk(2, -1)
            act = g * torch.sigmoid(g) * u
            # |silu'| <= 1.1, |silu(g)| <= |g|; exponential, reciprocal and two products: 2^-18 (1 + |g|) of the value; the activation as
            # two numbers of the type: the rest of a rest, or half of the type's smallest step
            bent = 1.1 * u.abs() * dg + g.abs() * du + 1.1 * dg * du
            bent = bent + (2.0 ** -18 * (1 + g.abs()) + half * half) * (act.abs() + bent) + torch.finfo(self.dtype).smallest_normal * half
            y = act @ self.w2[e].double().t()
            dy = bent @ self.w2[e].double().abs().t() + self.depth2 * ULP * ((act.abs() + bent) @ self.mag2[e].double().t())
            a, da = share[t, r][:, None], share_off[t, r][:, None]
            ref[t] += a * y
            bound[t] += a * dy + da * (y.abs() + dy) + 40 * ULP * a * y.abs()
        assert torch.isfinite(out).all()
        bound = bound + half * (ref.abs() + bound) + torch.finfo(self.dtype).smallest_normal * half
        bad = (out.double() - ref).abs() > bound
        assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float(((out.double() - ref).abs() - bound).max()))
        return ref
