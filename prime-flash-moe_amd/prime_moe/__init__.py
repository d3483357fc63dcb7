"""prime_moe for MI355X (gfx950): the fused-MoE forward behind the reference's op surface.

Drop-in for the reference package (prime_moe/__init__.py:1-122 and the op schemas of
prime_moe/csrc/torch_interface.cpp:271-324): the same three ``prime_moe::`` torch-library
ops with the same schemas, the same Python wrappers returning ``out``, ``BLOCK`` and
``pack_scales_blocked``.  The schemas and fake impls are defined here, the implementations in
``_torch_ops.so`` (csrc/torch_ops.cpp), which calls hand-written HIP kernels through the C ABI
of ``libprime_moe_hip.so`` (``include/prime_moe_hip.h``); the PyTorch-ROCm device is dispatch
key ``CUDA``.  Argument checks raise ``RuntimeError`` for the conditions the reference's
``TORCH_CHECK``s reject (torch_interface.cpp:85-87, :132-155, :208-241).

Extras that the reference leaves to its callers: a fake impl for ``moe_align`` (so all
three ops trace), :func:`quantize_mx`, the OCP-MX quantiser in front of the mxfp8 op, and
:func:`route`, the router front-end (top-k + softmax + ``moe_align``) in front of both.

Next to the fused forward pass, the experts' products on their own, for training, other activations and 8-bit integers:
:func:`grouped_mm` (differentiable), :func:`grouped_mm_wgrad`, :func:`grouped_mm_int8`, :func:`quantize_int8` and
:func:`expert_offsets`, which makes their ``offsets`` from a schedule.

For decoding: :func:`moe_layer`, a whole layer for up to 16 tokens, and experts of 4 bits in it (:func:`moe_layer_int4`) and on
their own (:func:`grouped_mm_int4`; :func:`quantize_int4`, :func:`pack_int4`, :func:`dequantize_int4`).
"""
from __future__ import annotations

import torch

BLOCK = 32  # MX scale block size

_LIB = torch.library.Library("prime_moe", "FRAGMENT")
_LIB.define(
    "fused_moe_bf16(Tensor x, Tensor w, Tensor w2, Tensor sorted_token_ids, Tensor expert_ids, "
    "Tensor num_tokens_post_padded, Tensor topk_weights, Tensor(a!) out, int top_k, int block_m, "
    "int block_n, int warp_n, int stages, int bpc, int cpc, bool split=True) -> ()"
)
_LIB.define(
    "fused_moe_mxfp8(Tensor x, Tensor x_scales, Tensor w, Tensor w_scales, Tensor w2, "
    "Tensor w2_scales, Tensor sorted_token_ids, Tensor expert_ids, Tensor num_tokens_post_padded, "
    "Tensor topk_weights, Tensor(a!) out, int top_k, int block_m, int block_n, int warp_n, "
    "int stages, int bpc, bool split=True) -> ()"
)
_LIB.define("moe_align(Tensor topk_ids, int num_experts, int block_m, int bpc) -> (Tensor, Tensor, Tensor)")
_LIB.define("expert_offsets(Tensor expert_ids, Tensor num_tokens_post_padded, int num_experts) -> Tensor")
_LIB.define("grouped_mm(Tensor x, Tensor w, Tensor offsets) -> Tensor")
_LIB.define("grouped_mm_wgrad(Tensor dy, Tensor x, Tensor offsets) -> Tensor")
_LIB.define("grouped_mm_int8(Tensor x, Tensor w, Tensor x_scale, Tensor w_scale, Tensor? offsets, ScalarType out_dtype) -> Tensor")
_LIB.define("quantize_int8(Tensor x) -> (Tensor, Tensor)")
_LIB.define("grouped_mm_int4(Tensor x, Tensor w, Tensor w_scale, Tensor? offsets) -> Tensor")
_LIB.define("quantize_int4(Tensor w, int group, ScalarType scale_dtype) -> (Tensor, Tensor)")
_LIB.define("dequantize_int4(Tensor q, Tensor scale, int columns) -> Tensor")
_LIB.define("moe_layer(Tensor x, Tensor gate, Tensor w1, Tensor w2, int top_k, Tensor? bias) -> (Tensor, Tensor, Tensor)")
_LIB.define("moe_layer_int4(Tensor x, Tensor gate, Tensor w1, Tensor w1_scale, Tensor w2, Tensor w2_scale, int top_k, Tensor? bias) "
            "-> (Tensor, Tensor, Tensor)")


try:
    # host side of the ops (csrc/torch_ops.cpp): registers their CUDA-key implementations, does the argument checks
    from . import _torch_ops
except ImportError as _err:
    # Not built, or built against another torch or library: the package still imports (its build module has to), and
    # everything that needs the native code raises.
    class _Unavailable:
        def __init__(self, reason):
            self._reason = reason

        def _raise(self, *args, **kwargs):
            raise RuntimeError(f"prime_moe: _torch_ops.so cannot be loaded ({self._reason}). Build the native code "
                               "first: python prime-flash-moe_amd/prime_moe/build.py (there is no fallback path).")

        def __getattr__(self, name):
            return self._raise

    _torch_ops = _Unavailable(str(_err))
    for _op in ("moe_align", "fused_moe_bf16", "fused_moe_mxfp8", "expert_offsets", "grouped_mm", "grouped_mm_wgrad",
                "grouped_mm_int8", "quantize_int8", "grouped_mm_int4", "quantize_int4", "dequantize_int4", "moe_layer",
                "moe_layer_int4"):
        _LIB.impl(_op, _torch_ops._raise, "CUDA")


# ------------------------------------------------------------------------------- moe_align

def align_sizes(n: int, num_experts: int, block_m: int, bpc: int):
    """(pad_to, max_padded, max_blocks) as torch_interface.cpp:88-91 computes them."""
    pad_to = block_m * bpc
    max_padded = (n + num_experts * (pad_to - 1) + pad_to - 1) // pad_to * pad_to
    return pad_to, max_padded, max_padded // block_m


def _validate_align(topk_ids, num_experts, block_m, bpc, placement: bool = True) -> None:
    """Argument checks of the op.  `placement=False` skips the device check (what is left can then be
    exercised with CPU tensors)."""
    _torch_ops.validate_align(topk_ids, num_experts, block_m, bpc, placement)


def _moe_align_fake(topk_ids, num_experts, block_m, bpc):
    _, max_padded, max_blocks = align_sizes(topk_ids.numel(), num_experts, block_m, bpc)
    mk = lambda n: torch.empty((n,), dtype=torch.int32, device=topk_ids.device)
    return mk(max_padded), mk(max_blocks), mk(1)


# ------------------------------------------------------------------------------- fused_moe_bf16

def _validate_bf16(x, w, w2, sorted_token_ids, expert_ids, num_tokens_post_padded, topk_weights, out,
                   top_k, block_m, block_n, warp_n, stages, bpc, cpc, split, placement: bool = True) -> None:
    """Argument checks of the op.  `placement=False` skips the device and alignment checks."""
    _torch_ops.validate_bf16(x, w, w2, sorted_token_ids, expert_ids, num_tokens_post_padded, topk_weights, out,
                             top_k, block_m, block_n, warp_n, stages, bpc, cpc, split, placement)


def _fused_moe_bf16_fake(x, w, w2, sorted_token_ids, expert_ids, num_tokens_post_padded, topk_weights,
                         out, top_k, block_m, block_n, warp_n, stages, bpc, cpc, split=True):
    return None


# ------------------------------------------------------------------------------- fused_moe_mxfp8

def _validate_mxfp8(x, x_scales, w, w_scales, w2, w2_scales, sorted_token_ids, expert_ids,
                    num_tokens_post_padded, topk_weights, out, top_k, block_m, block_n, warp_n, stages,
                    bpc, split, placement: bool = True) -> None:
    """Argument checks of the op.  `placement=False` skips the device and alignment checks."""
    _torch_ops.validate_mxfp8(x, x_scales, w, w_scales, w2, w2_scales, sorted_token_ids, expert_ids,
                              num_tokens_post_padded, topk_weights, out, top_k, block_m, block_n, warp_n, stages,
                              bpc, split, placement)


def _fused_moe_mxfp8_fake(x, x_scales, w, w_scales, w2, w2_scales, sorted_token_ids, expert_ids,
                          num_tokens_post_padded, topk_weights, out, top_k, block_m, block_n, warp_n,
                          stages, bpc, split=True):
    return None


# ------------------------------------------------------------------------------- ragged expert products

def _expert_offsets_fake(expert_ids, num_tokens_post_padded, num_experts):
    return expert_ids.new_empty((num_experts,))


def _grouped_mm_fake(x, w, offsets):
    return x.new_empty((x.shape[0], w.shape[1]))


def _grouped_mm_wgrad_fake(dy, x, offsets):
    return x.new_empty((offsets.shape[0], dy.shape[1], x.shape[1]))


def _grouped_mm_int8_fake(x, w, x_scale, w_scale, offsets, out_dtype):
    return x.new_empty((x.shape[0], w.shape[-2]), dtype=out_dtype)


def _quantize_int8_fake(x):
    return x.new_empty(x.shape, dtype=torch.int8), x.new_empty(x.shape[:-1], dtype=torch.float32)


def _grouped_mm_int4_fake(x, w, w_scale, offsets):
    return x.new_empty((x.shape[0], w.shape[-3] * 16))


def _quantize_int4_fake(w, group, scale_dtype):
    lead, (n, k) = w.shape[:-2], w.shape[-2:]
    tiles = (k + 127) // 128
    return (w.new_empty((*lead, n // 16, tiles, 1024), dtype=torch.uint8),
            w.new_empty((*lead, n // 16, tiles, 16, 128 // group), dtype=scale_dtype))


def _dequantize_int4_fake(q, scale, columns):
    return scale.new_empty((*q.shape[:-3], q.shape[-3] * 16, columns))


def _moe_layer_fake(x, gate, w1, w2, top_k, bias):
    pairs = (x.shape[0], top_k)
    return torch.empty_like(x), x.new_empty(pairs, dtype=torch.int32), x.new_empty(pairs, dtype=torch.float32)


def _moe_layer_int4_fake(x, gate, w1, w1_scale, w2, w2_scale, top_k, bias):
    return _moe_layer_fake(x, gate, w1, w2, top_k, bias)


torch.library.register_fake("prime_moe::moe_align", _moe_align_fake, lib=_LIB)
torch.library.register_fake("prime_moe::fused_moe_bf16", _fused_moe_bf16_fake, lib=_LIB)
torch.library.register_fake("prime_moe::fused_moe_mxfp8", _fused_moe_mxfp8_fake, lib=_LIB)
torch.library.register_fake("prime_moe::expert_offsets", _expert_offsets_fake, lib=_LIB)
torch.library.register_fake("prime_moe::grouped_mm", _grouped_mm_fake, lib=_LIB)
torch.library.register_fake("prime_moe::grouped_mm_wgrad", _grouped_mm_wgrad_fake, lib=_LIB)
torch.library.register_fake("prime_moe::grouped_mm_int8", _grouped_mm_int8_fake, lib=_LIB)
torch.library.register_fake("prime_moe::quantize_int8", _quantize_int8_fake, lib=_LIB)
torch.library.register_fake("prime_moe::grouped_mm_int4", _grouped_mm_int4_fake, lib=_LIB)
torch.library.register_fake("prime_moe::quantize_int4", _quantize_int4_fake, lib=_LIB)
torch.library.register_fake("prime_moe::dequantize_int4", _dequantize_int4_fake, lib=_LIB)
torch.library.register_fake("prime_moe::moe_layer", _moe_layer_fake, lib=_LIB)
torch.library.register_fake("prime_moe::moe_layer_int4", _moe_layer_int4_fake, lib=_LIB)


# ------------------------------------------------------------------------------- public wrappers

def fused_moe_bf16(x, w, w2, sorted_token_ids, expert_ids, num_tokens_post_padded, topk_weights, out,
                   top_k: int, block_m: int, block_n: int, warp_n: int, stages: int, bpc: int = 1,
                   cpc: int = 1, split: bool = True) -> torch.Tensor:
    """Runs ``prime_moe::fused_moe_bf16`` and returns ``out`` (reference __init__.py:27-49)."""
    torch.ops.prime_moe.fused_moe_bf16(
        x, w, w2, sorted_token_ids, expert_ids, num_tokens_post_padded, topk_weights, out,
        top_k, block_m, block_n, warp_n, stages, bpc, cpc, split)
    return out


def fused_moe_mxfp8(x, x_scales, w, w_scales, w2, w2_scales, sorted_token_ids, expert_ids,
                    num_tokens_post_padded, topk_weights, out, top_k: int, block_m: int, block_n: int,
                    warp_n: int, stages: int, bpc: int = 1, split: bool = True) -> torch.Tensor:
    """Runs ``prime_moe::fused_moe_mxfp8`` and returns ``out`` (reference __init__.py:75-100)."""
    torch.ops.prime_moe.fused_moe_mxfp8(
        x, x_scales, w, w_scales, w2, w2_scales, sorted_token_ids, expert_ids,
        num_tokens_post_padded, topk_weights, out, top_k, block_m, block_n, warp_n, stages, bpc, split)
    return out


def pack_scales_blocked(scales: torch.Tensor) -> torch.Tensor:
    """Row-major ``(..., MN, K/32)`` e8m0 scales -> the 128x4 blocked tiles the kernels read.

    Layout contract of the reference (__init__.py:106-115): tiles of 128 rows x 4 K-blocks, 512
    bytes each, ordered [row tile][K tile]; inside a tile the scale of (row r, block b) is byte
    ``(r % 32) * 16 + (r % 128 // 32) * 4 + b % 4``, so the four scales of one row over 128
    consecutive K form one aligned 32-bit word.  Load-time work, plain torch.
    """
    u = scales.view(torch.uint8)
    mn, kb = u.shape[-2], u.shape[-1]
    assert mn % 128 == 0, f"MN ({mn}) must be a multiple of 128"
    assert kb % 4 == 0, f"K ({kb * 32}) must be a multiple of 128"
    lead = u.shape[:-2]
    # axes: [lead, row tile, quarter (r%128//32), r%32, K tile, b%4] -> [lead, row tile, K tile, r%32, quarter, b%4]
    tiles = u.reshape(-1, mn // 128, 4, 32, kb // 4, 4).permute(0, 1, 4, 3, 2, 5)
    return tiles.contiguous().reshape(*lead, -1).view(torch.float8_e8m0fnu)


def quantize_mx(t: torch.Tensor):
    """OCP-MX quantisation of the last dimension of a bf16 tensor on the GPU.

    Returns ``(float8_e4m3fn values, float8_e8m0fnu scales)`` with scales of shape
    ``t.shape[:-1] + (K // 32,)`` row major -- the format ``fused_moe_mxfp8`` takes for ``x``
    and, after :func:`pack_scales_blocked`, for the weights (specification: the reference's
    test/test_mxfp8.py:21-38).
    """
    return _torch_ops.quantize_mx(t)


def route(logits: torch.Tensor, top_k: int, block_m: int = 128, bpc: int = 1, bias: torch.Tensor = None):
    """Router front-end: gate logits ``(T, E)`` -> top-k, softmax weights and the ``moe_align`` schedule.

    The step the reference leaves to its callers (README.md:147-149): returns
    ``(topk_ids (T, top_k) int32, topk_weights (T, top_k) fp32, sorted_token_ids, expert_ids,
    num_tokens_post_padded)``; the last three are what ``torch.ops.prime_moe.moe_align(topk_ids, E,
    block_m, bpc)`` returns.  Selection: the ``top_k`` largest of ``logits[t] (+ bias)``, largest first,
    ties to the lower expert index; weights: softmax over the selected values in fp32.  One top-k kernel
    plus the align kernels on the current stream, no host synchronisation.
    """
    return _torch_ops.route(logits, top_k, block_m, bpc, bias)


def expert_offsets(expert_ids: torch.Tensor, num_tokens_post_padded: torch.Tensor, num_experts: int) -> torch.Tensor:
    """``offsets`` of the ragged products below, from a schedule of ``moe_align`` / :func:`route` with ``block_m=1``.

    Such a schedule is the permutation that sorts the pairs by expert without padding: ``sorted_token_ids`` holds the pair of
    every row, ``expert_ids`` its expert.  Returns the end of every expert's rows, ``(num_experts,)`` int32.  Pairs that the
    schedule drops (ids outside the experts) are in none of its rows: behind the last end ``sorted_token_ids`` is -1, which a
    program that drops pairs has to leave out (or clamp, with the weight zero) before it gathers and scatters by it.
    """
    return torch.ops.prime_moe.expert_offsets(expert_ids, num_tokens_post_padded, num_experts)


def grouped_mm(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """Rows by their expert's matrix: ``out[r] = w[g] @ x[r]`` for the rows ``offsets[g-1] <= r < offsets[g]`` of expert ``g``.

    ``x`` (M, K), ``w`` (E, N, K), both bfloat16 or float16; ``offsets`` (E,) int32 on the same GPU, non-decreasing, at most
    1024 experts.  Rows from ``offsets[-1]`` on come out as zeros.  Sums in fp32, rounded once.  ``x`` needs a contiguous last
    dimension; ``w`` may be stored either way (``w.transpose(1, 2)`` of an (E, K, N) tensor; for few rows per expert, as in
    decoding, (E, N, K) is 1.4 to 5.6 times faster, as only that layout has a streaming kernel).  K, N and the strides are
    multiples of 8, tensors start 16-byte aligned.  Differentiable in ``x`` and ``w`` (backward, any number of times; a tensor
    with a forward-mode tangent is refused).  Offsets are read on the device and not checked: with other values the output is
    unspecified, but nothing outside the arguments is read or written.
    """
    return torch.ops.prime_moe.grouped_mm(x, w, offsets)


def grouped_mm_wgrad(dy: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """Gradient of :func:`grouped_mm` with respect to ``w``: ``dw[g]`` is the sum of ``dy[r] x[r]^T`` over expert g's rows.

    ``dy`` (M, N), ``x`` (M, K); returns (E, N, K), zeros for an expert without rows.  What the backward pass of
    ``grouped_mm`` calls; for programs that accumulate weight gradients themselves.
    """
    return torch.ops.prime_moe.grouped_mm_wgrad(dy, x, offsets)


def grouped_mm_int8(x: torch.Tensor, w: torch.Tensor, x_scale: torch.Tensor, w_scale: torch.Tensor,
                    offsets: torch.Tensor = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """:func:`grouped_mm` of 8-bit integers: ``out[r, n] = (x[r] . w[g, n]) * x_scale[r] * w_scale[g, n]``.

    ``x`` (M, K) and ``w`` (E, N, K) int8, ``x_scale`` (M,) and ``w_scale`` (E, N) float32.  Without ``offsets`` it is a dense
    product with ``w`` (N, K) and ``w_scale`` (N,), such as a shared expert's.  Sums are exact (K < 131072); ``out_dtype``
    bfloat16, float16 or float32.  N is a multiple of 8, K and the strides are multiples of 16.  No gradients.
    """
    return torch.ops.prime_moe.grouped_mm_int8(x, w, x_scale, w_scale, offsets, out_dtype)


def quantize_int8(x: torch.Tensor):
    """``(q, scale)`` of every row of the last dimension: ``scale = max(amax * (1 / 127), 2**-126)`` in float32, ``q`` the
    integer nearest to ``x / scale`` (exactly, ties to even).

    ``x`` (..., K) bfloat16, float16 or float32, K a multiple of 8; ``q`` int8 of the same shape, ``scale`` float32 of
    ``x.shape[:-1]``: what :func:`grouped_mm_int8` takes for rows and, applied to (E, N, K) weights, for ``w``.  A row that
    holds an infinity or a NaN gets the scale NaN and zeros.
    """
    return torch.ops.prime_moe.quantize_int8(x)


def quantize_int4(w: torch.Tensor, group: int = 128, scale_dtype: torch.dtype = None):
    """``(q, scale)``: a matrix (N, K), or a stack (..., N, K), to 4 bits with a scale per ``group`` (32, 64 or 128) values of a row.

    A weight stands for ``value * scale``: ``scale`` is the number of ``scale_dtype`` (bfloat16 or float16; ``w``'s own type, and
    bfloat16 for float32) nearest to ``max(amax * (1 / 7), least)`` in float32, ``least`` being 2**-126 (bfloat16) or 2**-24
    (float16), ``value`` the integer nearest to ``w / scale`` (exactly, ties to even) from -8 to 7.  A group that holds an infinity or
    a NaN, or whose scale is beyond the type, gets the scale NaN and zeros.

    ``w`` is contiguous, bfloat16, float16 or float32; N is a multiple of 16, K of ``group``.  ``q`` (..., N / 16, ceil(K / 128),
    1024) uint8 and ``scale`` (..., N / 16, ceil(K / 128), 16, 128 / group) hold tiles of 16 x 128 in the order the kernels read;
    :func:`pack_int4` makes them from integers of another quantiser, :func:`dequantize_int4` gives the weights back.
    """
    if scale_dtype is None:
        scale_dtype = torch.bfloat16 if w.dtype == torch.float32 else w.dtype
    return torch.ops.prime_moe.quantize_int4(w, group, scale_dtype)


def pack_int4(values: torch.Tensor, scale: torch.Tensor):
    """``(q, scale)`` as :func:`quantize_int4` lays them out, from integers ``values`` (..., N, K) int8, -8 to 7, and their scales
    (..., N, K / group), bfloat16 or float16.  Load-time work, plain torch, on the device of ``values``, with about 2.5 bytes a
    weight beside its arguments at the peak and two waits for the device (a large stack may be packed matrix by matrix)."""
    if values.dtype != torch.int8 or values.dim() < 2:
        raise RuntimeError("pack_int4: values must be int8 (..., N, K)")
    if scale.dtype not in (torch.bfloat16, torch.float16):
        raise RuntimeError("pack_int4: scale must be bfloat16 or float16")
    lead, (n, k) = values.shape[:-2], values.shape[-2:]
    group = k // scale.shape[-1] if scale.dim() == values.dim() and scale.shape[-1] > 0 else 0
    if group not in (32, 64, 128) or scale.shape != (*lead, n, k // group) or k % group != 0:
        raise RuntimeError(f"pack_int4: scale must be (..., N, K / group) with a group of 32, 64 or 128, got {tuple(scale.shape)} "
                           f"for values {tuple(values.shape)}")
    if n == 0 or n % 16 != 0:
        raise RuntimeError(f"pack_int4: N must be a positive multiple of 16, got {n}")
    if values.numel() > 0 and not (int(values.amin()) >= -8 and int(values.amax()) <= 7):
        raise RuntimeError("pack_int4: values must lie in -8 .. 7")
    tiles, per = (k + 127) // 128, 128 // group
    v = torch.nn.functional.pad(values, (0, tiles * 128 - k)) + 8
    # axes: [lead, strip, row, tile, 32 columns, 8 columns, column] -> two columns a byte -> [lead, strip, tile, 8 columns, row, 32 columns, byte]
    v = v.view(torch.uint8).reshape(-1, n // 16, 16, tiles, 4, 4, 8)
    v = v[..., [0, 4, 1, 5]] | (v[..., [2, 6, 3, 7]] << 4)
    q = v.permute(0, 1, 3, 5, 2, 4, 6).reshape(*lead, n // 16, tiles, 1024)
    s = torch.nn.functional.pad(scale, (0, tiles * per - scale.shape[-1])).reshape(-1, n // 16, 16, tiles, per)
    return q.contiguous(), s.transpose(2, 3).reshape(*lead, n // 16, tiles, 16, per).contiguous()


def dequantize_int4(q: torch.Tensor, scale: torch.Tensor, columns: int = None) -> torch.Tensor:
    """The weights (..., N, K) that ``(q, scale)`` stand for, in the type of ``scale``; for products of many rows, with
    :func:`grouped_mm` for example.  ``columns``: K, where it is not a multiple of 128."""
    return torch.ops.prime_moe.dequantize_int4(q, scale, q.shape[-2] * 128 if columns is None else columns)


def grouped_mm_int4(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, offsets: torch.Tensor = None) -> torch.Tensor:
    """:func:`grouped_mm` with weights of 4 bits: ``w``, ``w_scale`` from :func:`quantize_int4` or :func:`pack_int4`, of (E, N, K)
    weights, or of an (N, K) matrix without ``offsets`` (a dense product).

    Made for few rows per expert, as in decoding: every 16 rows of an expert read its weights again, or, where the experts have more
    than 14 on average (a single matrix more than 16), every 32 (for many rows: :func:`dequantize_int4`).  ``x`` (M, K) bfloat16 or float16 with a contiguous last dimension, rows a multiple of 8 elements
    apart, 16-byte aligned; ``w_scale`` of the same type.  Sums in fp32, rounded once; a row of ``x`` that holds an infinity or a
    NaN comes out as NaN.  No gradients.
    """
    return torch.ops.prime_moe.grouped_mm_int4(x, w, w_scale, offsets)


def moe_layer(x: torch.Tensor, gate: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, top_k: int, bias: torch.Tensor = None):
    """A whole layer of experts for up to 16 tokens: router, experts and weighted sum.  Returns ``(out, topk_ids, topk_weights)``.

    What ``route(x @ gate.T, top_k, bias=bias)`` and a fused forward pass compute, with fp32 logits: ``topk_ids`` (T, top_k) int32,
    the ``top_k`` largest of ``x @ gate.T + bias``, largest first, ties to the lower index; ``topk_weights`` (T, top_k) float32,
    softmax over the selected logits; ``out`` (T, K) the sum of ``weight * (w2[e] @ (silu(g) * u))`` with ``g`` and ``u`` the two
    halves of ``w1[e] @ x``.  ``x`` (T, K), ``gate`` (E, K), ``w1`` (E, 2H, K) with the gate rows first, ``w2`` (E, K, H): contiguous,
    all bfloat16 or all float16, K and H multiples of 8, at most 512 experts; ``bias`` (E,) float32.  Sums in fp32, the activation
    in its range and with 16 bits of mantissa or more in both types, one rounding to 16 bits at the end; the same bits every time.
    Made for few tokens per expert: every four of them read its weights again.  No gradients.  More than 16 tokens: :func:`route` and :func:`fused_moe_bf16`, in
    float16 :func:`route`, :func:`expert_offsets` and :func:`grouped_mm`.
    """
    return torch.ops.prime_moe.moe_layer(x, gate, w1, w2, top_k, bias)


def moe_layer_int4(x: torch.Tensor, gate: torch.Tensor, w1: torch.Tensor, w1_scale: torch.Tensor, w2: torch.Tensor,
                   w2_scale: torch.Tensor, top_k: int, bias: torch.Tensor = None):
    """:func:`moe_layer` with experts of 4 bits: ``w1``, ``w1_scale`` and ``w2``, ``w2_scale`` from :func:`quantize_int4` or
    :func:`pack_int4`, of (E, 2H, K) and (E, K, H) weights with one group size and scales of the type of ``x``.  K and H are
    multiples of the group (and with it of 16).  A token whose ``x`` or activation holds an infinity or a NaN comes out as NaN.  More than 16 tokens: :func:`route`, :func:`expert_offsets` and
    :func:`grouped_mm_int4`, or :func:`grouped_mm` on what :func:`dequantize_int4` returns."""
    return torch.ops.prime_moe.moe_layer_int4(x, gate, w1, w1_scale, w2, w2_scale, top_k, bias)


__all__ = [
    "dequantize_int4",
    "grouped_mm_int4",
    "moe_layer",
    "moe_layer_int4",
    "pack_int4",
    "quantize_int4",
    "expert_offsets",
    "grouped_mm",
    "grouped_mm_int8",
    "grouped_mm_wgrad",
    "quantize_int8",
    "route",
    "fused_moe_bf16",
    "fused_moe_mxfp8",
    "pack_scales_blocked",
    "quantize_mx",
    "BLOCK",
]
