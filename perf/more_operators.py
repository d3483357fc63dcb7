"""Performance cases of decoding: a whole layer of experts for a few tokens, and products with weights of 4 bits.

The operators:

    moe_layer(x, gate, w1, w2, top_k, bias)           router (products with the gate, top-k, softmax over the selected logits), experts
                                                      (gate and up projection, SwiGLU, down projection), weighted sum; up to 16 tokens
    moe_layer_int4(..., w1, w1_scale, w2, w2_scale)   the same with the experts in 4 bits
    grouped_mm_int4(x, w, w_scale, offsets)           rows by their expert's matrix in 4 bits; without offsets a single matrix
    quantize_int4(w, group), dequantize_int4(q, s)    to 4 bits and back: scale = amax / 7 of every `group` values of a row

A weight of 4 bits stands for value * scale: an integer from -8 to 7 and a 16-bit scale per 32, 64 or 128 consecutive values of
its row.  The layers are those of the repository's other cases: the README's, the Mixtral-, Qwen3- and DeepSeek-V3-like ones
and the grid of the reference's benchmark.  x ~ N(0, 1), weights of variance 1/K.
"""
import math
import os
import sys

import torch

own = False

# layer -> (hidden size, experts, gate and up rows, top_k, routing).  routing: "normal" (gate logits N(0, 1)), "biased" (a
# popularity of 0.5 N(0, 1) per expert on top), "zipf" (popularity rank^-1.2).
LAYERS = {
    "readme": (4096, 8, 512, 4, "normal"),
    "mixtral": (4096, 8, 28672, 2, "normal"),
    "qwen3": (2048, 128, 1536, 8, "biased"),
    "bench_grid": (2048, 32, 2048, 4, "normal"),
    "test_grid_37": (4096, 37, 256, 9, "normal"),
    "dsv3": (7168, 256, 4096, 8, "normal"),
    "dsv3_zipf": (7168, 256, 4096, 8, "zipf"),
}

# (operator, layer, fewest and most tokens): the ranges that the listed cases stand for and draw() draws from.
RANGES = [
    ("layer", "readme", 1, 16),
    ("layer", "mixtral", 1, 7),
    ("layer", "qwen3", 1, 16),
    ("layer", "bench_grid", 1, 16),
    ("layer", "test_grid_37", 1, 16),
    ("layer", "dsv3", 1, 3),
    ("layer_int4", "readme", 1, 16),
    ("layer_int4", "mixtral", 1, 16),
    ("layer_int4", "qwen3", 1, 16),
    ("layer_int4", "dsv3", 1, 16),
    ("mm", "mixtral", 1, 64),
    ("mm", "qwen3", 1, 64),
    ("mm", "dsv3_zipf", 1, 64),
    ("mm", "test_grid_37", 1, 64),
    ("mm_dense", "mixtral", 1, 64),
    ("mm_dense", "dsv3", 1, 64),
    ("mm_dense", "readme", 1, 64),
    ("quantize", "readme", 1, 8),
    ("quantize", "qwen3", 1, 128),
    ("quantize", "mixtral", 1, 3),
]


def _case(op, layer, tokens, side="up", dtype="bf16", group=128, behind=0):
    """`side`: "up" takes rows of the hidden size to the gate and up rows, "down" rows of half of those back.  `behind`: rows
    of the batch behind the last expert's (pairs that were dropped).  `tokens` of "quantize": matrices."""
    return {"op": op, "layer": layer, "tokens": tokens, "side": side, "dtype": dtype, "group": group, "behind": behind}


def listed():
    def case(name, *a, **k):
        return {"name": name, **_case(*a, **k)}

    return [
        # one sequence decoding through many small experts, all latency
        case("layer_1", "layer", "qwen3", 1),
        # a few sequences and few small experts, in fp16: less work still
        case("layer_readme_5", "layer", "readme", 5, dtype="fp16"),
        # a small batch: half of the experts are touched, by a row or two each
        case("layer_16", "layer", "qwen3", 16),
        # a few sequences through large experts, bound by the stream of weights
        case("layer_mixtral_3", "layer", "mixtral", 3),
        # one sequence, weights of 4 bits: all latency
        case("layer_int4_1", "layer_int4", "qwen3", 1),
        # a small batch on the largest layer, in 4 bits, groups of 32
        case("layer_int4_16", "layer_int4", "dsv3", 16, group=32),
        # a token through a shared expert in 4 bits, all latency
        case("mm_dense_1", "mm_dense", "dsv3", 1),
        # an odd batch through a large dense layer
        case("mm_dense_27", "mm_dense", "mixtral", 27, dtype="fp16", group=64),
        # batched decode with skewed routing, some pairs dropped
        case("mm_64", "mm", "dsv3_zipf", 64, behind=7),
        # the down projections of a token
        case("mm_down_1", "mm", "qwen3", 1, side="down", group=32),
        # one matrix to 4 bits
        case("quantize_1", "quantize", "readme", 1, dtype="fp16", group=64),
        # a whole layer's matrices to 4 bits, memory bound
        case("quantize_128", "quantize", "qwen3", 128),
    ]


def draw(rng):
    op, layer, lo, hi = rng.choice(RANGES)
    tokens = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return _case(op, layer, tokens, side=rng.choice(("up", "down")) if op in ("mm", "mm_dense", "quantize") else "up",
                 dtype=rng.choice(("bf16", "fp16")), group=rng.choice((32, 64, 128)),
                 behind=rng.randrange(0, 20) if op == "mm" and rng.random() < 0.3 else 0)


DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _matrix(case):
    """(rows, columns) of an expert's matrix on the case's side"""
    hidden, _, gate_up, _, _ = LAYERS[case["layer"]]
    return (gate_up, hidden) if case["side"] == "up" else (hidden, gate_up // 2)


def _counts(case, seed):
    """Rows of each expert: every token's top_k of the gate's values."""
    _, experts, _, top_k, routing = LAYERS[case["layer"]]
    gen = torch.Generator().manual_seed(seed)
    logits = torch.randn((case["tokens"], experts), generator=gen)
    if routing == "biased":
        logits += 0.5 * torch.randn((experts,), generator=gen)
    elif routing == "zipf":  # the top_k of log popularity + Gumbel noise are draws without replacement
        noise = -torch.log(torch.empty((case["tokens"], experts)).exponential_(generator=gen))
        logits = noise - 1.2 * torch.log(torch.arange(1, experts + 1, dtype=torch.float32))
    return torch.bincount(torch.topk(logits, top_k, dim=-1).indices.flatten(), minlength=experts)


def _normal(shape, std, dtype, gen):
    return torch.empty(shape, dtype=dtype, device=gen.device).normal_(0.0, std, generator=gen)


def _weights(shape, group, dtype, gen):
    """Values of 4 bits and their scales; the products have the variance 1/K."""
    values = torch.randint(-8, 8, shape, dtype=torch.int8, device=gen.device, generator=gen)
    scale = torch.rand(shape[:-1] + (shape[-1] // group,), dtype=torch.float32, device=gen.device, generator=gen)
    return values, ((scale + 0.5) * (0.21 * shape[-1] ** -0.5)).to(dtype)


def _inputs(case, seed):
    device = torch.device("cuda:0")
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    op, dtype, group, tokens = case["op"], DTYPES[case["dtype"]], case["group"], case["tokens"]
    hidden, experts, gate_up, top_k, routing = LAYERS[case["layer"]]
    state = {"op": op, "dtype": dtype, "group": group, "top_k": top_k}
    n, k = _matrix(case)
    if op == "quantize":
        state["w"] = _normal((tokens, n, k), k ** -0.5, dtype, gen)
    elif op in ("layer", "layer_int4"):
        state["x"] = _normal((tokens, hidden), 1.0, dtype, gen)
        state["gate"] = _normal((experts, hidden), hidden ** -0.5, dtype, gen)
        state["bias"] = _normal((experts,), 0.5, torch.float32, gen) if routing == "biased" else None
        for name, shape in (("w1", (experts, gate_up, hidden)), ("w2", (experts, hidden, gate_up // 2))):
            if op == "layer":
                state[name] = _normal(shape, shape[-1] ** -0.5, dtype, gen)
            else:
                state[name], state[name + "_scale"] = _weights(shape, group, dtype, gen)
    else:
        rows, lead = tokens, ()
        if op == "mm":
            ends = torch.cumsum(_counts(case, seed), 0)
            state["ends"] = ends.tolist()
            state["offsets"] = ends.to(torch.int32).to(device)
            rows, lead = tokens * top_k + case["behind"], (experts,)
        else:
            state["ends"] = [tokens]
        state["x"] = _normal((rows, k), 1.0, dtype, gen)
        state["w"], state["w_scale"] = _weights(lead + (n, k), group, dtype, gen)
    return state


def _package():
    folder = os.path.join(os.getcwd(), "prime-flash-moe_amd")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import prime_moe
    return prime_moe


def prepare(case, seed):
    state = _inputs(case, seed)
    if own:  # weights of 4 bits are laid out once, when they are loaded
        for name in ("w", "w1", "w2"):
            if name + "_scale" in state:
                state[name], state[name + "_scale"] = _package().pack_int4(state[name], state[name + "_scale"])
    return state


# ---- the plain forms: elementary operations in 32 bits, an expert at a time, rounded once at the end


def _plain_weight(values, scale, group):
    return values.float() * scale.float().repeat_interleave(group, dim=-1)


def _plain_layer(s):
    """The gate's products are taken in 64 bits: logits next to each other."""
    x, top_k = s["x"].float(), s["top_k"]
    logits = s["x"].double() @ s["gate"].double().t()
    if s["bias"] is not None:
        logits = logits + s["bias"].double()
    values, ids = torch.sort(logits, dim=-1, descending=True, stable=True)
    values, ids = values[:, :top_k], ids[:, :top_k]
    weights = torch.exp(values - values[:, :1])
    weights = (weights / weights.sum(-1, keepdim=True)).float()
    out = torch.zeros_like(x)
    half = s["w1"].shape[1] // 2
    for e in torch.unique(ids).tolist():
        token, slot = torch.nonzero(ids == e, as_tuple=True)
        if s["op"] == "layer":
            w1, w2 = s["w1"][e].float(), s["w2"][e].float()
        else:
            w1 = _plain_weight(s["w1"][e], s["w1_scale"][e], s["group"])
            w2 = _plain_weight(s["w2"][e], s["w2_scale"][e], s["group"])
        h = x[token] @ w1.t()
        gate, up = h[:, :half], h[:, half:]
        y = (gate / (1 + torch.exp(-gate)) * up) @ w2.t()
        out[token] += y * weights[token, slot][:, None]
    return {"out": out.to(s["dtype"]), "ids": ids.to(torch.int32), "weights": weights}


def _plain_mm(s):
    y = torch.zeros((s["x"].shape[0], s["w"].shape[-2]), dtype=s["dtype"], device=s["x"].device)
    start = 0
    for g, end in enumerate(s["ends"]):
        if end > start:
            w, scale = (s["w"], s["w_scale"]) if s["w"].dim() == 2 else (s["w"][g], s["w_scale"][g])
            y[start:end] = (s["x"][start:end].float() @ _plain_weight(w, scale, s["group"]).t()).to(s["dtype"])
        start = end
    return y


def _plain_quantize(w, group):
    """The quotient is taken in 64 bits: values next to a border between two integers."""
    pieces = w.reshape(*w.shape[:-1], -1, group)
    least = 2.0 ** -24 if w.dtype == torch.float16 else 2.0 ** -126
    scale = (pieces.float().abs().amax(-1) * (1.0 / 7.0)).clamp_min(least).to(w.dtype)
    q = torch.empty_like(pieces, dtype=torch.int8)
    for i in range(w.shape[0]):
        q[i] = torch.round(pieces[i].double() / scale[i].double()[..., None]).clamp(-8, 7)
    return (q.float() * scale.float()[..., None]).to(w.dtype).reshape(w.shape)


def run(s):
    op = s["op"]
    if own:
        prime_moe = _package()
        if op == "layer":
            out, ids, weights = prime_moe.moe_layer(s["x"], s["gate"], s["w1"], s["w2"], s["top_k"], s["bias"])
            return {"out": out, "ids": ids, "weights": weights}
        if op == "layer_int4":
            out, ids, weights = prime_moe.moe_layer_int4(s["x"], s["gate"], s["w1"], s["w1_scale"], s["w2"], s["w2_scale"],
                                                         s["top_k"], s["bias"])
            return {"out": out, "ids": ids, "weights": weights}
        if op == "mm":
            return {"y": prime_moe.grouped_mm_int4(s["x"], s["w"], s["w_scale"], s["offsets"])}
        if op == "mm_dense":
            return {"y": prime_moe.grouped_mm_int4(s["x"], s["w"], s["w_scale"])}
        return {"w": prime_moe.dequantize_int4(*prime_moe.quantize_int4(s["w"], s["group"]))}
    if op in ("layer", "layer_int4"):
        return _plain_layer(s)
    if op in ("mm", "mm_dense"):
        return {"y": _plain_mm(s)}
    return {"w": _plain_quantize(s["w"], s["group"])}


# ---- from the definitions, in 64 bits


def _exact_weight(values, scale):
    n, k = values.shape
    return (values.double().view(n, scale.shape[-1], -1) * scale.double().unsqueeze(-1)).view(n, k)


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "quantize":
        out = torch.empty(s["w"].shape, dtype=torch.float64, device=s["w"].device)
        for i, w in enumerate(s["w"]):
            parts = w.unflatten(-1, (-1, case["group"]))
            peak = parts.abs().max(dim=-1, keepdim=True).values.to(torch.float32)
            least = torch.tensor(2.0 ** (-24 if case["dtype"] == "fp16" else -126), device=w.device)
            scale = torch.maximum(peak * torch.tensor(1.0 / 7.0, device=w.device), least).to(w.dtype).double()
            out[i] = (torch.clamp((parts.double() / scale).round(), -8, 7) * scale).flatten(-2)
        return {"w": out}
    x = s["x"].double()
    if op in ("mm", "mm_dense"):
        dense = op == "mm_dense"
        y = torch.zeros((x.shape[0], s["w"].shape[-2]), dtype=torch.float64, device=x.device)
        begin = [0] + s["ends"][:-1]
        for g, end in enumerate(s["ends"]):
            if end > begin[g]:
                w = _exact_weight(s["w"] if dense else s["w"][g], s["w_scale"] if dense else s["w_scale"][g])
                y[begin[g]:end] = torch.mm(x[begin[g]:end], w.t())
        return {"y": y}
    score = torch.mm(x, s["gate"].double().t())
    if s["bias"] is not None:
        score += s["bias"].double()
    tokens, top_k = x.shape[0], LAYERS[case["layer"]][3]
    left = score.clone()
    ids = torch.empty((tokens, top_k), dtype=torch.int64, device=x.device)
    for r in range(top_k):  # the largest that is left, the lowest index of equal ones
        best = left.max(dim=1, keepdim=True).values
        ids[:, r] = (left == best).to(torch.int8).argmax(dim=1)
        left.scatter_(1, ids[:, r:r + 1], -math.inf)
    weights = torch.softmax(torch.gather(score, 1, ids), dim=1)
    share = torch.zeros_like(score).scatter_(1, ids, weights)
    out = torch.zeros_like(x)
    for e in range(score.shape[1]):
        rows = (share[:, e] > 0).nonzero().flatten()
        if rows.numel() == 0:
            continue
        if op == "layer":
            w1, w2 = s["w1"][e].double(), s["w2"][e].double()
        else:
            w1, w2 = _exact_weight(s["w1"][e], s["w1_scale"][e]), _exact_weight(s["w2"][e], s["w2_scale"][e])
        gate, up = torch.mm(x[rows], w1.t()).chunk(2, dim=1)
        out[rows] += torch.mm(gate * torch.sigmoid(gate) * up, w2.t()) * share[rows, e:e + 1]
    return {"out": out, "ids": ids.to(torch.int32), "weights": weights}


def work(case):
    """Rows, the gate, the touched experts' weights and their scales read once, the outputs written once; the operations of
    every row.  A layer's touched experts: as many as evenly routed tokens reach on average."""
    hidden, experts, gate_up, top_k, _ = LAYERS[case["layer"]]
    op, tokens, group = case["op"], case["tokens"], case["group"]
    n, k = _matrix(case)
    if op == "quantize":  # to 4 bits and back
        return {"bytes": int(tokens * n * k * (2 + 2 + 2 * (0.5 + 2 / group))), "flops": 4 * tokens * n * k}
    if op in ("layer", "layer_int4"):
        touched = experts * (1 - (1 - top_k / experts) ** tokens)
        per_weight = 2 if op == "layer" else 0.5 + 2 / group
        expert = 3 * hidden * gate_up // 2
        return {"bytes": int(touched * expert * per_weight) + 2 * experts * hidden + 4 * tokens * hidden + 8 * tokens * top_k,
                "flops": 2 * tokens * (top_k * expert + experts * hidden)}
    rows = tokens * (top_k if op == "mm" else 1)
    touched = int((_counts(case, 0) > 0).sum()) if op == "mm" else 1
    return {"bytes": int(touched * n * k * (0.5 + 2 / group)) + 2 * rows * (n + k) + 2 * case["behind"] * n, "flops": 2 * rows * n * k}
