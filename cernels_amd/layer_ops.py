"""The decoder layer around the experts, over the C ABI: layer norm, rotary positions, a paged cache's writes and attention.

Conventions are those of ``cernels_amd.ops``, which offers these entries too: CUDA (HIP) tensors, ``RuntimeError`` for a call that
breaks the contract, new output tensors, kernels on the current HIP stream of the tensors' device, no host synchronisation,
scratch memory from torch's caching allocator.

``layer_norm`` and ``rotary`` are differentiable (once). The paged entries serve: a call that would have to carry a gradient is
refused.

Paged cache: ``k_pages`` and ``v_pages`` [pages, page_size, kv_heads, dim] hold the keys and values of one layer, in any order of
strides whose last dimension is contiguous. ``block_table`` [sequences, blocks] int32 names the page of each block of page_size
positions of a sequence; entries outside [0, pages) have no page: nothing is written there and their keys add nothing.
``lengths`` [sequences] int32 counts each sequence's tokens with the step's new ones, which are its last; ``q_offsets``
[sequences + 1] int32 says which rows of q, k and v are whose (None: the same number for all). Rows behind the last sequence are not
written.
"""

from __future__ import annotations

import ctypes
import math

import torch

from cernels_amd import _native
from cernels_amd._call import launch as _launch, require as _require

_DTYPES = {torch.bfloat16: _native.DTYPE_BF16, torch.float16: _native.DTYPE_F16, torch.float32: _native.DTYPE_F32}
_CACHE_DTYPES = {torch.bfloat16: _native.DTYPE_BF16, torch.float16: _native.DTYPE_F16}
_FREQ_DTYPES = {torch.float32: _native.DTYPE_F32, torch.float64: _native.DTYPE_F64}
_POSITION_DTYPES = {torch.int32: _native.INDEX_I32, torch.int64: _native.INDEX_I64}
_Strides = ctypes.c_int64 * 6
_ATTENTION_DIMS = (64, 128, 256)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _dense_like(t):
    """A new contiguous tensor of t's shape, type and device, whatever t's strides."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _refuse_gradient(what, *tensors) -> None:
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no backward pass: call it under torch.no_grad()")


def _once(backward):
    """A backward pass whose gradients have none of their own: differentiating them raises. Only a graph of the gradients needs the
    wrapper that says so; without one (gradients are computed with grad mode off) its 4 us on autograd's thread are left out."""
    guarded = torch.autograd.function.once_differentiable(backward)

    def entry(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return entry


# ---- layer norm ---------------------------------------------------------------------------------------------------------


def _check_norm(x, weight, bias):
    _require(all(isinstance(t, torch.Tensor) for t in (x, weight)) and (bias is None or isinstance(bias, torch.Tensor)),
             "x, weight and bias must be tensors")
    _require(x.is_cuda and weight.device == x.device and (bias is None or bias.device == x.device),
             "x, weight and bias must be CUDA (HIP) tensors on one device")
    _require(x.dtype in _DTYPES, "x must be bfloat16, float16 or float32")
    _require(weight.dtype in (x.dtype, torch.float32) and (bias is None or bias.dtype == weight.dtype),
             "weight must have x's type or float32, bias the weight's type")
    _require(x.dim() >= 1 and x.size(-1) >= 1 and weight.shape == x.shape[-1:] and (bias is None or bias.shape == weight.shape),
             "weight and bias must be [N] for x [..., N]")
    _require(x.is_contiguous() and weight.is_contiguous() and (bias is None or bias.is_contiguous()),
             "x, weight and bias must be contiguous")


def _norm_ok(x, weight, bias) -> bool:
    """Whether a call holds to _check_norm's contract, in one expression on every short call's path; what it refuses goes to
    _check_norm, which says what is wrong. A condition added there belongs here too."""
    try:
        dev, dt, wt, n = x.get_device(), x.dtype, weight.dtype, weight.shape
        return (dev >= 0 and dt in _DTYPES and (wt is dt or wt is torch.float32) and len(n) == 1 and n[0] > 0 and x.shape[-1:] == n
                and weight.get_device() == dev and x.is_contiguous() and weight.is_contiguous()
                and (bias is None or (bias.dtype is wt and bias.shape == n and bias.get_device() == dev and bias.is_contiguous())))
    except (AttributeError, TypeError):
        return False


def _norm_forward(x, weight, bias, eps, keep_stats):
    cols = x.size(-1)
    rows = x.numel() // cols
    y = torch.empty_like(x)
    stats = x.new_empty((rows, 2), dtype=torch.float32) if keep_stats else None
    if rows:
        _launch("cernels_layer_norm", x.get_device(), _native.lib().cernels_layer_norm, x.data_ptr(), weight.data_ptr(), _ptr(bias),
                rows, cols, _DTYPES[x.dtype], _DTYPES[weight.dtype], eps, y.data_ptr(), _ptr(stats))
    return y, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _norm_forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        rows, cols = stats.size(0), x.size(-1)
        dy = dy.contiguous()
        dx = torch.empty_like(x) if want_x else None
        dw = torch.empty_like(weight) if want_w else None
        db = torch.empty_like(weight) if want_b else None
        L, dtype = _native.lib(), _DTYPES[x.dtype]
        nbytes = L.cernels_layer_norm_backward_workspace_bytes(rows, cols, dtype) if want_w or want_b else 0
        ws = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        _launch("cernels_layer_norm_backward", x.get_device(), L.cernels_layer_norm_backward, dy.data_ptr(), x.data_ptr(),
                weight.data_ptr(), stats.data_ptr(), rows, cols, dtype, _DTYPES[weight.dtype], _ptr(dx), _ptr(dw), _ptr(db),
                _ptr(ws), nbytes)
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight (+ bias) over x's last dimension, x [..., N] bf16, fp16 or fp32; weight and bias [N] in
    x's type or fp32. Sums are fp32 and the result is rounded once. Differentiable in x, weight and bias; the gradients are the
    same bits every run."""
    if not _norm_ok(x, weight, bias):
        _check_norm(x, weight, bias)
    if _wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _norm_forward(x, weight, bias, float(eps), False)[0]


# ---- rotary positions ---------------------------------------------------------------------------------------------------


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: dict | None = None, device=None):
    """(inverse frequencies [rotary_dim / 2] float64, scale) of a head's turned part, for ``rotary`` and ``paged_append``.

    ``scaling`` stretches a model to longer contexts; its keys are those of a checkpoint's ``rope_scaling``, by ``rope_type``:
      - ``linear``: every frequency divided by ``factor``;
      - ``llama3``: low frequencies (wavelength over original / low_freq_factor) divided by ``factor``, high ones kept (under
        original / high_freq_factor), in between a linear blend, original = ``original_max_position_embeddings``;
      - ``yarn`` (Peng et al., 2023): a blend by the number of turns in the original context, from ``beta_fast`` (32) turns, kept,
        to ``beta_slow`` (1), divided by ``factor``; the scale is ``attention_factor`` or 0.1 ln(factor) + 1. ``truncate``
        (default true) takes the blend's ends as whole indices.
    """
    _require(rotary_dim >= 0 and rotary_dim % 2 == 0, "rotary_dim must be even")
    index = torch.arange(rotary_dim // 2, dtype=torch.float64)
    inv = float(base) ** (-2 * index / max(rotary_dim, 1))
    kind = "default" if scaling is None else scaling.get("rope_type", scaling.get("type", "default"))
    scale = 1.0
    if kind != "default":
        factor = float(scaling["factor"])
    if kind == "linear":
        inv = inv / factor
    elif kind == "llama3":
        original = float(scaling["original_max_position_embeddings"])
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        turns = original * inv / (2 * math.pi)  # in the original context
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        inv = inv * keep + inv / factor * (1 - keep)
    elif kind == "yarn":
        original = float(scaling["original_max_position_embeddings"])

        def index_of(turns):
            return rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

        first, last = index_of(float(scaling.get("beta_fast") or 32.0)), index_of(float(scaling.get("beta_slow") or 1.0))
        if scaling.get("truncate", True):
            first, last = math.floor(first), math.ceil(last)
        first, last = max(first, 0), min(last, rotary_dim - 1)
        stretch = ((index - first) / max(last - first, 1e-3)).clamp(0, 1)
        inv = inv / factor * stretch + inv * (1 - stretch)
        given = scaling.get("attention_factor")
        scale = float(given) if given is not None else (0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0)
    else:
        _require(kind == "default", f"unknown rope_type {kind!r}")
    return inv.to(device), scale


def _check_heads(t, name, tokens, dim, like):
    _require(isinstance(t, torch.Tensor) and t.device == like.device and t.dtype == like.dtype,
             f"{name} must be a tensor of the same type on the same device")
    _require(t.dim() == 3 and (tokens is None or t.size(0) == tokens) and (dim is None or t.size(2) == dim),
             f"{name} must be [tokens, heads, dim], tokens and dim as the others")
    _require(t.stride(2) == 1 or t.size(2) <= 1, f"{name}'s last dimension must be contiguous")


def _check_frequencies(inv_freq, dim, device):
    _require(isinstance(inv_freq, torch.Tensor) and inv_freq.device == device and inv_freq.dtype in _FREQ_DTYPES
             and inv_freq.dim() == 1 and inv_freq.is_contiguous(),
             "inv_freq must be a contiguous float32 or float64 [pairs] tensor on the same device")
    _require(2 * inv_freq.numel() <= dim, "inv_freq must hold at most dim / 2 frequencies")


def _check_rotary(q, k, positions, inv_freq):
    _require(isinstance(q, torch.Tensor) and q.is_cuda and q.dtype in _DTYPES, "q must be a bfloat16, float16 or float32 CUDA (HIP) tensor")
    _check_heads(q, "q", None, None, q)
    if k is not None:
        _check_heads(k, "k", q.size(0), q.size(2), q)
    _check_frequencies(inv_freq, q.size(2), q.device)
    _require(isinstance(positions, torch.Tensor) and positions.device == q.device and positions.dtype in _POSITION_DTYPES
             and positions.shape == q.shape[:1] and positions.is_contiguous(),
             "positions must be a contiguous int32 or int64 [tokens] tensor on the same device")


def _frequencies_ok(inv_freq, dim, dev) -> bool:
    return (inv_freq.get_device() == dev and inv_freq.dtype in _FREQ_DTYPES and inv_freq.dim() == 1 and inv_freq.is_contiguous()
            and 2 * inv_freq.numel() <= dim)


def _rotary_ok(q, k, positions, inv_freq) -> bool:
    """_check_rotary's contract in one expression (as _norm_ok)."""
    try:
        tokens, _, dim = q.shape
        dev, dt = q.get_device(), q.dtype
        return (dev >= 0 and dt in _DTYPES and q.stride(2) == 1
                and (k is None or (k.dim() == 3 and k.size(0) == tokens and k.size(2) == dim and k.stride(2) == 1 and k.dtype is dt
                                   and k.get_device() == dev))
                and _frequencies_ok(inv_freq, dim, dev) and positions.get_device() == dev and positions.dtype in _POSITION_DTYPES
                and positions.shape == (tokens,) and positions.is_contiguous())
    except (AttributeError, TypeError, ValueError):
        return False


def _rotary_launch(q, k, positions, inv_freq, interleaved, scale, backward):
    first = q if q is not None else k
    tokens, _, dim = first.shape
    outs = [None if t is None else _dense_like(t) for t in (q, k)]
    if tokens:
        heads = [(None, 0, 0, 0) if t is None else (t.data_ptr(), t.stride(0), t.stride(1), t.size(1)) for t in (q, k)]
        _launch("cernels_rotary", first.get_device(), _native.lib().cernels_rotary, *heads[0], *heads[1], positions.data_ptr(),
                _POSITION_DTYPES[positions.dtype], inv_freq.data_ptr(), _FREQ_DTYPES[inv_freq.dtype], tokens, dim, inv_freq.numel(),
                interleaved, scale, backward, _DTYPES[first.dtype], _ptr(outs[0]), _ptr(outs[1]))
    return outs


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, interleaved, scale):
        ctx.save_for_backward(positions, inv_freq)
        ctx.set_materialize_grads(False)
        ctx.layout = (interleaved, scale)
        return tuple(_rotary_launch(q, k, positions, inv_freq, interleaved, scale, 0))

    @staticmethod
    @_once
    def backward(ctx, dq, dk):
        positions, inv_freq = ctx.saved_tensors
        grads = [t if want else None for t, want in zip((dq, dk), ctx.needs_input_grad)]
        grads = [t if t is None or t.stride(2) == 1 else t.contiguous() for t in grads]
        if grads[0] is not None or grads[1] is not None:
            grads = _rotary_launch(*grads, positions, inv_freq, *ctx.layout, 1)
        return *grads, None, None, None, None


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor, *,
           interleaved: bool = False, scale: float = 1.0):
    """(q, k) turned to their positions: new tensors [tokens, heads, dim] for q and k (or None) of that shape, any token and head
    strides. The first 2 * len(inv_freq) elements of a head are pairs, elements (2i, 2i + 1) if ``interleaved``, (i, i + pairs) if
    not; pair i turns by positions[t] * inv_freq[i] and is multiplied by ``scale``; the rest of the head is copied. Angles are
    formed in 64 bits, so positions of a million lose nothing. Differentiable in q and k."""
    if not _rotary_ok(q, k, positions, inv_freq):
        _check_rotary(q, k, positions, inv_freq)
    if _wants_grad(q, k):
        return _Rotary.apply(q, k, positions, inv_freq, int(bool(interleaved)), float(scale))
    return tuple(_rotary_launch(q, k, positions, inv_freq, int(bool(interleaved)), float(scale), 0))


# ---- paged cache --------------------------------------------------------------------------------------------------------


def _check_step(like, k_pages, v_pages, block_table, lengths, q_offsets, tokens, dim, kv_heads):
    dev = like.device
    _require(like.is_cuda and like.dtype in _CACHE_DTYPES, "the step's tensors must be bfloat16 or float16 CUDA (HIP) tensors")
    for t, name in ((k_pages, "k_pages"), (v_pages, "v_pages")):
        _require(isinstance(t, torch.Tensor) and t.device == dev and t.dtype == like.dtype and t.dim() == 4,
                 f"{name} must be [pages, page_size, kv_heads, dim] of the step's type and device")
        _require(t.size(3) == dim and (kv_heads is None or t.size(2) == kv_heads), f"{name}'s heads and dim must be those of the step")
        _require(t.stride(3) == 1, f"{name}'s last dimension must be contiguous")
    _require(k_pages.shape == v_pages.shape, "k_pages and v_pages must have one shape")
    _require(k_pages.size(0) >= 1 and k_pages.size(1) >= 16 and k_pages.size(1) % 16 == 0, "page_size must be a multiple of 16")
    _require(isinstance(block_table, torch.Tensor) and block_table.device == dev and block_table.dtype == torch.int32
             and block_table.dim() == 2 and (block_table.stride(1) == 1 or block_table.size(1) <= 1),
             "block_table must be int32 [sequences, blocks] with contiguous rows on the step's device")
    seqs, blocks = block_table.shape
    _require(seqs <= 1 or block_table.stride(0) >= blocks, "block_table's rows must not overlap")
    _require(isinstance(lengths, torch.Tensor) and lengths.device == dev and lengths.dtype == torch.int32
             and lengths.shape == (seqs,) and lengths.is_contiguous(), "lengths must be contiguous int32 [sequences] on the step's device")
    if q_offsets is None:
        _require(tokens % max(seqs, 1) == 0, "without q_offsets every sequence has the same number of tokens")
    else:
        _require(isinstance(q_offsets, torch.Tensor) and q_offsets.device == dev and q_offsets.dtype == torch.int32
                 and q_offsets.shape == (seqs + 1,) and q_offsets.is_contiguous(),
                 "q_offsets must be contiguous int32 [sequences + 1] on the step's device")


def _step_ok(like, k_pages, v_pages, block_table, lengths, q_offsets, tokens, dim, kv_heads) -> bool:
    """_check_step's contract in one expression (as _norm_ok); the caller catches what a wrong type raises."""
    dev, dt = like.get_device(), like.dtype
    pages, page_size, heads, d = shape = k_pages.shape
    seqs, blocks = block_table.shape
    return (dev >= 0 and dt in _CACHE_DTYPES and d == dim and (kv_heads is None or heads == kv_heads) and v_pages.shape == shape
            and k_pages.dtype is dt and v_pages.dtype is dt and k_pages.get_device() == dev and v_pages.get_device() == dev
            and k_pages.stride(3) == 1 and v_pages.stride(3) == 1 and pages >= 1 and page_size >= 16 and page_size % 16 == 0
            and block_table.dtype is torch.int32 and block_table.get_device() == dev and (block_table.stride(1) == 1 or blocks <= 1)
            and (block_table.stride(0) >= blocks or seqs <= 1) and lengths.dtype is torch.int32 and lengths.get_device() == dev and lengths.shape == (seqs,) and lengths.is_contiguous()
            and (tokens % max(seqs, 1) == 0 if q_offsets is None else
                 (q_offsets.dtype is torch.int32 and q_offsets.get_device() == dev and q_offsets.shape == (seqs + 1,)
                  and q_offsets.is_contiguous())))


def _heads_ok(t, tokens, dim, like) -> bool:
    return (t.dim() == 3 and t.size(0) == tokens and t.size(2) == dim and t.stride(2) == 1 and t.dtype is like.dtype
            and t.get_device() == like.get_device())


def _append_ok(k, v, k_pages, v_pages, block_table, lengths, q_offsets, q, inv_freq) -> bool:
    try:
        tokens, kv_heads, dim = k.shape
        return (k.stride(2) == 1 and _heads_ok(v, tokens, dim, k) and v.size(1) == kv_heads
                and (q is None or _heads_ok(q, tokens, dim, k))
                and _step_ok(k, k_pages, v_pages, block_table, lengths, q_offsets, tokens, dim, kv_heads)
                and (inv_freq is None or _frequencies_ok(inv_freq, dim, k.get_device())))
    except (AttributeError, TypeError, ValueError):
        return False


def _check_append(k, v, k_pages, v_pages, block_table, lengths, q_offsets, q, inv_freq):
    _require(all(isinstance(t, torch.Tensor) for t in (k, v)) and (q is None or isinstance(q, torch.Tensor)),
             "q, k and v must be tensors")
    _check_heads(k, "k", None, None, k)
    tokens, kv_heads, dim = k.shape
    _check_heads(v, "v", tokens, dim, k)
    _require(v.size(1) == kv_heads, "k and v must have the same heads")
    if q is not None:
        _check_heads(q, "q", tokens, dim, k)
    _check_step(k, k_pages, v_pages, block_table, lengths, q_offsets, tokens, dim, kv_heads)
    if inv_freq is not None:
        _check_frequencies(inv_freq, dim, k.device)


def _attention_ok(q, k_pages, v_pages, block_table, lengths, q_offsets, sinks, out) -> bool:
    try:
        tokens, heads, dim = q.shape
        kv_heads = k_pages.size(2)
        return (q.stride(2) == 1 and dim in _ATTENTION_DIMS and kv_heads >= 1 and heads >= 1 and heads % kv_heads == 0
                and _step_ok(q, k_pages, v_pages, block_table, lengths, q_offsets, tokens, dim, None)
                and (sinks is None or (sinks.dtype is torch.float32 and sinks.shape == (heads,) and sinks.is_contiguous()
                                       and sinks.get_device() == q.get_device()))
                and (out is None or (_heads_ok(out, tokens, dim, q) and out.size(1) == heads and out.is_contiguous())))
    except (AttributeError, TypeError, ValueError):
        return False


def _check_attention(q, k_pages, v_pages, block_table, lengths, q_offsets, sinks, out):
    _require(isinstance(q, torch.Tensor), "q must be a tensor")
    _check_heads(q, "q", None, None, q)
    tokens, heads, dim = q.shape
    _check_step(q, k_pages, v_pages, block_table, lengths, q_offsets, tokens, dim, None)
    kv_heads = k_pages.size(2)
    _require(kv_heads >= 1 and heads >= 1 and heads % kv_heads == 0, "q's heads must be a multiple of the pages' heads")
    _require(dim in _ATTENTION_DIMS, "paged_attention takes head sizes 64, 128 and 256")
    _require(sinks is None or (isinstance(sinks, torch.Tensor) and sinks.device == q.device and sinks.dtype == torch.float32
                               and sinks.shape == (heads,) and sinks.is_contiguous()),
             "sinks must be contiguous float32 [heads] on q's device")
    _require(out is None or (isinstance(out, torch.Tensor) and out.device == q.device and out.dtype == q.dtype and out.is_contiguous()
                             and out.shape == q.shape), "out must be a contiguous tensor of q's shape, type and device")


def _pages_args(k_pages, v_pages):
    pages, page_size, heads, _ = k_pages.shape
    strides = _Strides(*k_pages.stride()[:3], *v_pages.stride()[:3])
    if heads == 1:  # a stride that is never taken may be anything
        strides[2] = strides[5] = 0
    if pages == 1:
        strides[0] = strides[3] = 0
    return strides, pages, page_size


def _table_args(block_table, lengths):
    blocks = block_table.size(1)
    stride = block_table.stride(0) if block_table.size(0) > 1 else blocks
    return block_table.data_ptr(), stride, blocks, lengths.data_ptr()


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                 lengths: torch.Tensor, q_offsets: torch.Tensor | None = None, *, q: torch.Tensor | None = None,
                 inv_freq: torch.Tensor | None = None, interleaved: bool = False, scale: float = 1.0) -> torch.Tensor | None:
    """Writes the step's keys and values [tokens, kv_heads, dim] to their slots of the pages, the keys turned to their positions as
    ``rotary`` does where ``inv_freq`` is given. ``q`` [tokens, heads, dim] is turned in the same launch and returned as a new
    tensor (None without q). A position past the table's end is not written."""
    if not _append_ok(k, v, k_pages, v_pages, block_table, lengths, q_offsets, q, inv_freq):
        _refuse_gradient("paged_append", q, k, v, k_pages, v_pages)
        _check_append(k, v, k_pages, v_pages, block_table, lengths, q_offsets, q, inv_freq)
    _refuse_gradient("paged_append", q, k, v, k_pages, v_pages)
    tokens, kv_heads, dim = k.shape
    pairs = freq = 0
    if inv_freq is not None:
        pairs, freq = inv_freq.numel(), _FREQ_DTYPES[inv_freq.dtype]
    out = None if q is None else _dense_like(q)
    seqs = block_table.size(0)
    if tokens and seqs:
        head = (None, 0, 0, 0) if q is None else (q.data_ptr(), q.stride(0), q.stride(1), q.size(1))
        _launch("cernels_paged_append", k.get_device(), _native.lib().cernels_paged_append, *head, _ptr(out), k.data_ptr(),
                k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), kv_heads, dim, _CACHE_DTYPES[k.dtype],
                _ptr(inv_freq), freq, pairs, int(bool(interleaved)), float(scale), k_pages.data_ptr(), v_pages.data_ptr(),
                *_pages_args(k_pages, v_pages), *_table_args(block_table, lengths), _ptr(q_offsets), seqs, tokens)
    return out


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    lengths: torch.Tensor, q_offsets: torch.Tensor | None = None, *, scale: float | None = None, window: int = 0,
                    sinks: torch.Tensor | None = None, max_new: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the step's queries [tokens, heads, dim] over their sequences' pages, the step's own keys among them (append them
    first); one token per sequence, chunks behind a cache and whole prompts alike.

    The query at position p sees keys up to p, with ``window`` > 0 the last ``window`` of them. Query heads share key heads in
    consecutive groups. ``scale`` (default 1 / sqrt(dim)) multiplies the scores. ``sinks`` [heads] fp32 is one more score per head that
    takes weight and has no value. A row that sees nothing is 0. ``max_new`` is the largest number of new tokens of a sequence, where
    the caller knows it: it picks the kernels, and the result holds for any value. Head sizes 64, 128 and 256."""
    if not _attention_ok(q, k_pages, v_pages, block_table, lengths, q_offsets, sinks, out):
        _refuse_gradient("paged_attention", q, k_pages, v_pages, sinks)
        _check_attention(q, k_pages, v_pages, block_table, lengths, q_offsets, sinks, out)
    _refuse_gradient("paged_attention", q, k_pages, v_pages, sinks)
    tokens, heads, dim = q.shape
    kv_heads = k_pages.size(2)
    _require(0 <= window < 2 ** 31, "window must be 0 (none) or a number of keys under 2^31")
    scale = dim ** -0.5 if scale is None else float(scale)
    _require(0.0 < scale < math.inf, "scale must be positive")
    if out is None:
        out = _dense_like(q)
    seqs, blocks, page_size = block_table.size(0), block_table.size(1), k_pages.size(1)
    if tokens and seqs:
        L = _native.lib()
        # of a sequence's new tokens; 0: not known
        most = tokens // seqs if q_offsets is None else int(max_new) if max_new is not None else 0
        nbytes = L.cernels_paged_attention_workspace_bytes(tokens, seqs, heads, kv_heads, dim, page_size, blocks, most)
        if nbytes == 0:
            raise RuntimeError(f"cernels_paged_attention: invalid dimensions tokens={tokens} heads={heads}/{kv_heads} dim={dim} "
                               f"sequences={seqs} blocks={blocks} x {page_size}, max_new={max_new}")
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        _launch("cernels_paged_attention", q.get_device(), L.cernels_paged_attention, q.data_ptr(), q.stride(0), q.stride(1), heads,
                kv_heads, dim, _CACHE_DTYPES[q.dtype], k_pages.data_ptr(), v_pages.data_ptr(), *_pages_args(k_pages, v_pages),
                *_table_args(block_table, lengths), _ptr(q_offsets), seqs, tokens, most, scale, int(window), _ptr(sinks),
                out.data_ptr(), ws.data_ptr(), nbytes)
    return out


__all__ = ["layer_norm", "rotary_frequencies", "rotary", "paged_append", "paged_attention"]
