"""``scaled_dot_product_attention`` for device tensors, mirroring DenseCore's Python API.

Follows ``python/densecore/functional.py:276-388`` of the reference: the same argument checks
and messages, the same scale rule (``None`` means the double ``1/sqrt(E)``), the same
"flash eligibility" predicate and the same mask conversion (a bool mask is True where
attention is allowed and becomes 0 / -inf; a float mask is added), feeding the native
``_flash_attention`` / ``_flash_attention_backward`` pair through an autograd Function that
saves (q, k, v, out, lse) for the backward.

Inputs the flash path does not take (dropout, rank 3, Ev != E, masks the flash path rejects,
float masks that require a gradient) go through the reference's math path
(``functional.py:318-340``), composed on the device from this library's kernels
(``include/dc_math.h``): the two batched products are ``dc_bmm`` (the device entry of the
reference's bmm registry, ``src/batched_matmul.rs:28-49``, with its gradient as two more bmm
calls on transposed views), the mask add, safe softmax and its gradient are the softmax
kernels.  ``multi_head_attention_forward`` (``functional.py:400-461``) composes the same pieces
around its input and output projections.

Differences, all on the device side of the boundary:
  * tensors are ``torch`` tensors on the GPU, float32 or bfloat16 (bf16 is new: the reference
    flash path is float32 only, ``functional.py:314``); the math path is float32 only, as the
    reference's is;
  * masks are passed as broadcast views, not materialised to (B, H, L, S) on the host;
  * ``enable_gqa`` passes the kv heads straight to the flash kernels (they index kv head
    h // repeat, as ``src/torch_attention.rs:159-167`` does) instead of widening K and V first;
    the math path widens them as the reference does;
  * nothing falls back to the CPU: an input no device path takes raises ``NotImplementedError``.
"""
import math
import numbers

import numpy as np
import torch

from . import _native


def scaled_dot_product_attention(query, key, value, attn_mask=None, dropout_p=0.0, is_causal=False,
                                 scale=None, enable_gqa=False):
    """softmax(query @ key^T * scale + mask) @ value for rank-4 (N, H, L, E) device tensors."""
    for name, t in (("query", query), ("key", key), ("value", value)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"attention {name} must be a Tensor")
    rank = query.dim()
    gqa = enable_gqa and rank == 4 and key.dim() == 4 and key.shape[1] != query.shape[1]
    if rank not in (3, 4) or key.dim() != rank or value.dim() != rank:
        raise ValueError("attention query, key and value must all be rank 3 or all rank 4")
    lead, (length, embed) = tuple(query.shape[:-2]), tuple(query.shape[-2:])
    source = key.shape[-2]
    klead, vlead = tuple(key.shape[:-2]), tuple(value.shape[:-2])
    if gqa:
        if query.shape[1] % key.shape[1]:
            raise ValueError("attention shapes must be (..., L, E), (..., S, E), (..., S, Ev)")
        klead = vlead = lead  # each kv head serves H // Hkv query heads
        if tuple(key.shape[:2]) != tuple(value.shape[:2]) or key.shape[0] != query.shape[0]:
            raise ValueError("attention shapes must be (..., L, E), (..., S, E), (..., S, Ev)")
    if klead != lead or vlead != lead or key.shape[-1] != embed or value.shape[-2] != source:
        raise ValueError("attention shapes must be (..., L, E), (..., S, E), (..., S, Ev)")
    if type(is_causal) is not bool:
        raise TypeError("is_causal must be a bool")
    if is_causal and attn_mask is not None:
        raise ValueError("attn_mask and is_causal cannot both be set")
    if scale is None:
        scale = 1.0 / math.sqrt(embed) if embed else 1.0
    elif isinstance(scale, (bool, np.bool_)) or not isinstance(scale, numbers.Real):
        raise TypeError("scale must be real")
    flash_dtypes = (torch.float32, torch.bfloat16)
    if (rank == 4 and not dropout_p and value.shape[-1] == embed and length and source and embed
            and query.dtype in flash_dtypes and key.dtype == query.dtype and value.dtype == query.dtype):
        flash_mask = _flash_mask(attn_mask, tuple(query.shape), source, query.device)
        if attn_mask is None or flash_mask is not None:
            return _flash_attention(query, key, value, is_causal, float(scale), flash_mask)
    if gqa:
        # Each kv head serves H // Hkv query heads (functional.py:287-293).
        groups = query.shape[1] // key.shape[1]
        key = key.repeat_interleave(groups, dim=1)
        value = value.repeat_interleave(groups, dim=1)
    return _math_attention(query, key, value, attn_mask, dropout_p, is_causal, float(scale))


def _math_attention(query, key, value, attn_mask, dropout_p, is_causal, scale):
    """PyTorch's math path as the reference composes it (``functional.py:318-340``): q and k^T
    each scaled by sqrt(|scale|), one batched product, the additive mask, the safe softmax
    (rows that are all -inf give 0), dropout, and the product with v."""
    if any(t.dtype != torch.float32 for t in (query, key, value)):
        raise NotImplementedError("the math attention path on the GPU takes float32 tensors "
                                  "(the reference's math path is float32)")
    if query.device.type != "cuda" or key.device != query.device or value.device != query.device:
        raise ValueError("attention tensors must be on one GPU")
    factor = math.sqrt(abs(scale))
    q = query * float(-factor if scale < 0 else factor)
    attn = _matmul(q, (key * float(factor)).transpose(-2, -1))
    length, source = attn.shape[-2], attn.shape[-1]
    if is_causal:
        attn_mask = torch.ones((length, source), dtype=torch.bool, device=attn.device).tril()
    additive = None
    if attn_mask is not None:
        if isinstance(attn_mask, torch.Tensor):
            m = attn_mask.to(attn.device)
        else:
            m = torch.from_numpy(np.ascontiguousarray(np.asarray(attn_mask))).to(attn.device)
        if m.dtype == torch.bool:
            additive = torch.zeros(m.shape, dtype=torch.float32, device=attn.device).masked_fill_(
                ~m, float("-inf"))
        else:
            additive = m if m.dtype == torch.float32 else m.float()
    weights = softmax_masked(attn, additive, safe=additive is not None)
    if dropout_p:
        weights = dropout(weights, dropout_p, True)
    return _matmul(weights, value)


class _Bmm(torch.autograd.Function):
    """``bmm`` with its gradient: dA = dC B^T and dB = A^T dC, both ``dc_bmm`` on transposed
    views (no copies)."""

    @staticmethod
    def forward(ctx, a, b):
        ctx.save_for_backward(a, b)
        return _native._bmm(a, b)

    @staticmethod
    def backward(ctx, grad):
        a, b = ctx.saved_tensors
        da = _native._bmm(grad, b.transpose(1, 2)) if ctx.needs_input_grad[0] else None
        db = _native._bmm(a.transpose(1, 2), grad) if ctx.needs_input_grad[1] else None
        return da, db


def bmm(a, b):
    """The reference's ``bmm`` (``src/batched_matmul.rs:9-49``) on float32 GPU tensors:
    (batch, m, k) x (batch, k, n) -> (batch, m, n), strided operands, autograd."""
    return _Bmm.apply(a, b)


def _matmul(x, y):
    """x @ y for x (..., m, k) and y (..., k, n) with equal leading dimensions (rank 3 or 4), as
    one ``bmm`` over the flattened leading dimensions."""
    lead = tuple(x.shape[:-2])
    if tuple(y.shape[:-2]) != lead:
        raise ValueError("bmm batch or inner dimensions mismatch")
    batch = math.prod(lead)  # explicit: reshape cannot infer -1 for tensors with no elements
    out = bmm(x.reshape((batch,) + tuple(x.shape[-2:])), y.reshape((batch,) + tuple(y.shape[-2:])))
    return out.reshape(lead + tuple(out.shape[-2:]))


class _Softmax(torch.autograd.Function):
    """Softmax over the last axis with the additive mask fused in; gradient
    ``softmax_backward_lastdim`` (``src/torch_softmax.rs:90-97``).  A mask that requires a
    gradient receives the scores' gradient summed over its broadcast dimensions, as the
    reference's separate ``attn + additive`` would give it."""

    @staticmethod
    def forward(ctx, scores, mask, safe):
        y = _native._softmax(scores, mask, safe)
        ctx.save_for_backward(y)
        ctx.mask_shape = None if mask is None else tuple(mask.shape)
        return y

    @staticmethod
    def backward(ctx, grad):
        (y,) = ctx.saved_tensors
        dx = _native._softmax_backward(grad, y)
        dmask = None
        if ctx.needs_input_grad[1]:
            dmask = dx.sum_to_size(ctx.mask_shape) if ctx.mask_shape else dx.sum()
        return dx, dmask, None


def softmax_masked(scores, mask=None, safe=False):
    """``softmax(scores + mask, -1)`` on the GPU; ``safe`` makes rows that are all -inf give 0
    (the math path's ``_safe_softmax``, ``functional.py:334-337``)."""
    return _Softmax.apply(scores, mask, bool(safe))


def softmax(input, dim=-1):
    """``Tensor.softmax`` over the last axis (``src/torch_softmax.rs:57-67``) for float32 GPU
    tensors (other axes are moved last and back)."""
    if dim < 0:
        dim += input.dim()
    if dim != input.dim() - 1:
        return softmax(input.movedim(dim, -1), -1).movedim(-1, dim)
    return _Softmax.apply(input, None, False)


def _dropout_probability(p):
    """``python/densecore/functional.py:219-226``."""
    if isinstance(p, (bool, np.bool_)) or not isinstance(p, numbers.Real):
        raise TypeError("dropout probability must be real")
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError("dropout probability must be in [0, 1]")
    return p


class _Dropout(torch.autograd.Function):
    """``input * noise`` with noise = keep / float32(1 - p): the same product forward and
    backward (``dc_dropout_apply``)."""

    @staticmethod
    def forward(ctx, x, bits, scale):
        ctx.save_for_backward(bits)
        ctx.scale = scale
        return _native._dropout_apply(bits, x, scale)

    @staticmethod
    def backward(ctx, grad):
        (bits,) = ctx.saved_tensors
        return _native._dropout_apply(bits, grad, ctx.scale), None, None


def dropout(input, p=0.5, training=True, generator=None):
    """``functional.dropout`` (``python/densecore/functional.py:229-244``): zero elements with
    probability p and scale survivors by 1/(1-p) while training.  The mask is
    ``Generator::bernoulli(n, 1 - p)`` drawn on the GPU from the reference's generator stream
    (``densecore_amd.random``), so a seed gives the reference's mask bit for bit; the noise
    value is float32(1) / float32(1 - p) as ``_dropout_noise`` (:638-641) rounds it."""
    from . import random as _random
    if not isinstance(input, torch.Tensor):
        raise TypeError("dropout input must be a Tensor")
    p = _dropout_probability(p)
    if type(training) is not bool:
        raise TypeError("training must be a bool")
    if not training or p == 0.0:
        return input
    if p == 1.0:
        return input * torch.zeros((), dtype=input.dtype, device=input.device)
    if input.device.type != "cuda":
        raise ValueError("dropout on this path takes tensors on the GPU")
    if input.dtype != torch.float32:
        raise NotImplementedError("dropout on the GPU takes float32 tensors")
    gen = _random.default_generator(input.device) if generator is None else generator
    bits = gen._bernoulli_bits(input.numel(), 1 - p)
    scale = float(np.float32(1.0) / np.float32(1 - p))
    return _Dropout.apply(input, bits, scale)


def _flash_mask(attn_mask, qshape, source, device):
    """The additive float32 (B, H, L, S) mask the flash kernels read, as a broadcast view, or
    None when the reference would not take the flash path for this mask
    (``python/densecore/functional.py:343-364``)."""
    if attn_mask is None:
        return None
    if isinstance(attn_mask, torch.Tensor):
        if attn_mask.requires_grad or attn_mask.dtype not in (torch.bool, torch.float32):
            return None
        values = attn_mask.to(device)
    else:
        arr = np.asarray(attn_mask)
        if arr.dtype not in (np.bool_, np.float32):
            return None
        values = torch.from_numpy(np.ascontiguousarray(arr)).to(device)
    batch, heads, length = qshape[:3]
    if values.dim() not in (2, 4) or values.shape[-2] not in (1, length) or values.shape[-1] not in (1, source):
        return None
    if values.dim() == 4 and (values.shape[0] not in (1, batch) or values.shape[1] not in (1, heads)):
        return None
    if values.dtype == torch.bool:
        values = torch.where(values, torch.zeros((), dtype=torch.float32, device=device),
                             torch.full((), float("-inf"), dtype=torch.float32, device=device))
    return values.expand(batch, heads, length, source)


class _FlashAttention(torch.autograd.Function):
    """``FlashAttention`` (``python/densecore/functional.py:371-386``)."""

    @staticmethod
    def forward(ctx, q, k, v, causal, scale, mask):
        out, lse = _native._flash_attention(q, k, v, causal, scale, mask)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.causal, ctx.scale, ctx.mask = causal, scale, mask
        return out

    @staticmethod
    def backward(ctx, grad):
        q, k, v, out, lse = ctx.saved_tensors
        dq, dk, dv = _native._flash_attention_backward(grad, q, k, v, out, lse, ctx.causal,
                                                       ctx.scale, ctx.mask)
        return dq, dk, dv, None, None, None


def _flash_attention(query, key, value, causal, scale, mask=None):
    """The fused path (``python/densecore/functional.py:367-388``)."""
    return _FlashAttention.apply(query, key, value, causal, scale, mask)


def flash_decode(query, key, value, scale=None):
    """One decode step: query (B, H, 1, E) against the whole KV cache (B, Hkv, S, E)."""
    return _native._flash_decode(query, key, value, None if scale is None else float(scale))[0]


def _window_numbers(window, sinks, offset, scale):
    for name, n, least in (("window", window, 1), ("sinks", sinks, 0), ("offset", offset, 0)):
        if isinstance(n, (bool, np.bool_)) or not isinstance(n, numbers.Integral):
            raise TypeError(f"window attention {name} must be an int")
        if n < least:
            raise ValueError(f"window attention {name} must be at least {least}")
    if scale is not None:
        if isinstance(scale, (bool, np.bool_)) or not isinstance(scale, numbers.Real):
            raise TypeError("scale must be real")
        scale = float(scale)
        if not math.isfinite(scale):
            raise ValueError("window attention scale must be finite")
    return int(window), int(sinks), int(offset), scale


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks, offset, scale):
        out, lse, rest = _native._window_attention(q, k, v, window, sinks, offset, scale, with_rest=True)
        ctx.save_for_backward(q, k, v, out, lse, rest)
        ctx.args = (window, sinks, offset, scale)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return (*_native._window_attention_backward(grad, *ctx.saved_tensors, *ctx.args), None, None, None, None)


def window_attention(query, key, value, window, sinks=0, offset=0, scale=None):
    """Causal attention in which a query sees the last ``window`` keys, its own among them, and the first
    ``sinks`` ones: query (B, H, L, E) over key and value (B, Hkv, S, E), H a multiple of Hkv.

    The query in row l stands at position ``offset + l`` and key s at position s: key s is visible iff
    ``s <= p and (s > p - window or s < sinks)`` (``offset`` 0 is the alignment of ``is_causal``; the next
    L tokens of a sequence of S have ``offset = S - L``).  The work is that of the visible pairs, no mask
    is formed, and keys that are not visible have no influence, whatever they hold.  A query that sees no
    key gives 0 and no gradients.  Float32 or bf16, head dims up to 128, any strides; gradients are
    identical from run to run.  No counterpart in the reference."""
    _check_tensors("attention", query=query, key=key, value=value)
    args = _window_numbers(window, sinks, offset, scale)
    if torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad):
        return _WindowAttention.apply(query, key, value, *args)
    return _native._window_attention(query, key, value, *args)[0]


def window_decode(query, key, value, window, sinks=0, lengths=None, scale=None):
    """One decode step of ``window_attention``: query (B, H, 1, E) over a cache (B, Hkv, S, E) of which
    sequence b holds its first ``lengths[b]`` rows (int32 or int64 on the GPU; values are clamped to 0 .. S;
    None: all S), the query's own key the last of them.  Reads the visible rows alone; a sequence of
    length 0 gives 0.  Head dims up to 256, any strides; forward only."""
    _check_tensors("attention", query=query, key=key, value=value)
    _check_optional("attention", lengths=lengths)
    window, sinks, _, scale = _window_numbers(window, sinks, 0, scale)
    return _native._window_decode(query, key, value, window, sinks, lengths, scale)[0]


def rotary_frequencies(rotary_dim, base=10000.0, scaling=None, factor=1.0, original_length=None, beta_fast=32.0,
                       beta_slow=1.0, device=None):
    """``(inv_freq, magnitude)`` for ``rotary_embedding`` and ``qk_norm_rotary``: the angle per position
    of each of ``rotary_dim / 2`` pairs (float64) and the factor on the turned values.

    Plain: ``base ** (-2 i / rotary_dim)``.  For contexts ``factor`` times as long as the trained one,
    ``scaling`` is ``"linear"`` (positions divided by the factor), ``"ntk"`` (the base times ``factor **
    (R / (R - 2))``, so that the slowest pair is divided by the factor and the fastest kept) or ``"yarn"``
    (Peng et al., "YaRN", 2023): pairs that turn more than ``beta_fast`` times over ``original_length``
    positions are kept, those that turn less than ``beta_slow`` times divided by the factor, in between a
    ramp, and the magnitude is ``0.1 ln(factor) + 1``."""
    if isinstance(rotary_dim, bool) or not isinstance(rotary_dim, numbers.Integral) or rotary_dim < 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be an even number")
    if not base > 1.0 or not factor >= 1.0:
        raise ValueError("rotary base must be above 1 and factor at least 1")
    R = int(rotary_dim)
    i = torch.arange(R // 2, dtype=torch.float64)
    magnitude = 1.0
    if scaling == "ntk" and R > 2:
        base = base * factor ** (R / (R - 2))
    freq = torch.tensor(float(base), dtype=torch.float64) ** (-2.0 * i / max(R, 1))
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        if original_length is None or original_length <= 0:
            raise ValueError("yarn scaling takes the trained length as original_length")
        if not beta_fast > beta_slow > 0:
            raise ValueError("yarn scaling takes beta_fast above beta_slow above 0")

        def pair(turns):
            return R * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(pair(beta_fast)), 0), min(math.ceil(pair(beta_slow)), R - 1)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = freq / factor * ramp + freq * (1 - ramp)
        magnitude = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "ntk"):
        raise ValueError("rotary scaling must be None, 'linear', 'ntk' or 'yarn'")
    return freq.to(device), magnitude


class _Rotary(torch.autograd.Function):
    """The rotation, with or without the norm (``weights`` None: without); its gradient takes nothing
    but the positions without the norm, and the inputs again with it."""

    @staticmethod
    def forward(ctx, q, k, wq, wk, norm, inv_freq, positions, args, eps):
        qo, ko, fields = _native._rotary(q, k, inv_freq, positions, *args, (wq, wk) if norm else None, eps,
                                         with_fields=True)
        ctx.save_for_backward(*(q, k, wq, wk) if norm else (None,) * 4, inv_freq, positions)
        ctx.norm, ctx.args, ctx.eps, ctx.fields, ctx.has_k = norm, args, eps, fields, k is not None
        return qo, ko

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):
        q, k, wq, wk, inv_freq, positions = ctx.saved_tensors
        gk = gk if ctx.has_k else None
        if not ctx.norm:
            q, k = gq, gk
        need = ctx.needs_input_grad
        dq, dk, dwq, dwk = _native._rotary_backward(
            gq, gk, q, k, inv_freq, positions, *ctx.args, (wq, wk) if ctx.norm else None, ctx.eps,
            (need[2], need[3]), ctx.fields)
        return dq, dk, dwq, dwk, None, None, None, None, None


def _turn_args(offset, interleaved, magnitude):
    if isinstance(offset, bool) or not isinstance(offset, numbers.Integral):
        raise TypeError("rotary offset must be an int")
    if type(interleaved) is not bool:
        raise TypeError("interleaved must be a bool")
    if isinstance(magnitude, bool) or not isinstance(magnitude, numbers.Real):
        raise TypeError("rotary magnitude must be real")
    return int(offset), interleaved, float(magnitude)


def _refuse_frequency_gradient(inv_freq):
    if inv_freq.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("rotary inv_freq has no gradient")


def _check_tensors(what, **tensors):
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what} {name} must be a Tensor")


def _check_optional(what, **tensors):
    _check_tensors(what, **{name: t for name, t in tensors.items() if t is not None})


def rotary_embedding(query, key, inv_freq, positions=None, offset=0, interleaved=False, magnitude=1.0):
    """Queries (B, H, L, E) and keys (B, Hkv, L, E) turned by their positions: ``(query, key)``, contiguous.

    Token (b, l) stands at ``positions[b, l]`` (int32 or int64, (L,) or (B, L)), or at ``offset + l``.
    Pair i of a head's first ``2 len(inv_freq)`` dims is turned by the angle position x ``inv_freq[i]``
    (float64, ``rotary_frequencies``) and multiplied by ``magnitude``; pairs are (i, i + len(inv_freq)), or
    (2i, 2i + 1) when ``interleaved``; the dims behind them are passed on.  Float32 or bf16 in any strides
    (a projection's (B, L, H, E) is transposed on the way); angles are formed in float64.  ``key`` may be
    None: then the turned query alone is returned.  No counterpart in the reference."""
    _check_tensors("rotary", query=query, inv_freq=inv_freq)
    _check_optional("rotary", key=key, positions=positions)
    args = _turn_args(offset, interleaved, magnitude)
    _refuse_frequency_gradient(inv_freq)
    if torch.is_grad_enabled() and (query.requires_grad or (key is not None and key.requires_grad)):
        q, k = _Rotary.apply(query, key, None, None, False, inv_freq, positions, args, 0.0)
    else:
        q, k = _native._rotary(query, key, inv_freq, positions, *args)
    return q if key is None else (q, k)


def qk_norm_rotary(query, key, query_weight, key_weight, inv_freq, positions=None, offset=0, interleaved=False,
                   magnitude=1.0, eps=1e-6):
    """``rotary_embedding`` of each head's queries and keys divided by their root mean square:
    ``x / sqrt(mean(x^2) + eps) * weight`` over the head's E dims, then turned, in one pass.

    The weights are (E,) vectors, float32 or bf16, shared by the heads (None: no weight); with an empty
    ``inv_freq`` there is the norm alone.  Gradients: queries, keys and weights, the weights' summed in a
    fixed order.  No counterpart in the reference."""
    _check_tensors("rotary", query=query, key=key, inv_freq=inv_freq)
    _check_optional("rotary", positions=positions, query_weight=query_weight, key_weight=key_weight)
    args = _turn_args(offset, interleaved, magnitude)
    _refuse_frequency_gradient(inv_freq)
    if isinstance(eps, bool) or not isinstance(eps, numbers.Real):
        raise TypeError("norm eps must be real")
    if not eps >= 0:
        raise ValueError("norm eps must not be negative")
    leaves = (query, key, query_weight, key_weight)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in leaves):
        return _Rotary.apply(*leaves, True, inv_freq, positions, args, float(eps))
    return _native._rotary(query, key, inv_freq, positions, *args, (query_weight, key_weight), float(eps))


def _float_mask(mask):
    """MHA masks (``functional.py:391-397``): a bool mask is True where attention is NOT
    allowed (-inf); a float mask is added."""
    if mask is None:
        return None
    if mask.dtype == torch.bool:
        return torch.zeros(mask.shape, dtype=torch.float32, device=mask.device).masked_fill_(
            mask, float("-inf"))
    return mask


def _append_position(mask):
    """A mask over the keys with one more key at the end, always visible (a zero column)."""
    return None if mask is None else torch.nn.functional.pad(mask, (0, 1))


def multi_head_attention_forward(query, key, value, embed_dim_to_check, num_heads, in_proj_weight,
                                 in_proj_bias, bias_k, bias_v, add_zero_attn, dropout_p,
                                 out_proj_weight, out_proj_bias, training=True,
                                 key_padding_mask=None, need_weights=True, attn_mask=None,
                                 use_separate_proj_weight=False, q_proj_weight=None,
                                 k_proj_weight=None, v_proj_weight=None, static_k=None,
                                 static_v=None, average_attn_weights=True, is_causal=False):
    """Multi-head attention with PyTorch's ``F.multi_head_attention_forward`` signature and
    semantics (the reference composes the same steps, ``functional.py:400-461``), on the GPU.

    query is (L, N, E) or unbatched (L, E); key and value (S, N, kdim / vdim) or (S, kdim / vdim).
    The steps, in PyTorch's order: project q, k, v (the packed ``in_proj_weight`` holds the three
    projections in that order, or the three separate weights); append ``bias_k`` / ``bias_v`` as
    one more key position; split the heads; substitute ``static_k`` / ``static_v``; append a zero
    key position (``add_zero_attn``); fold ``key_padding_mask`` into the additive mask; attention
    weights softmax(q k^T / sqrt(head_dim) + mask), dropped out when training; their product with
    v, merged heads, output projection.  Masks that gain a key position gain a zero column.  Bool
    masks are True where attention is not allowed.  ``is_causal`` is only a hint: ``attn_mask``
    must still be given, and is what is applied.  The projections are device BLAS calls
    (``F.linear``); the two batched products are this library's ``bmm``, the mask add and the
    softmax its softmax kernel (rows whose keys are all masked come out NaN, as PyTorch's do), and
    the dropout its dropout."""
    F = torch.nn.functional
    if is_causal and attn_mask is None:
        raise RuntimeError("Need attn_mask if specifying the is_causal hint")
    unbatched = query.dim() != 3
    if unbatched:  # one sequence: a batch of one along dim 1
        query, key, value = (x.unsqueeze(1) for x in (query, key, value))
        key_padding_mask = None if key_padding_mask is None else key_padding_mask.unsqueeze(0)
    tgt_len, batch, embed_dim = query.shape
    if embed_dim != embed_dim_to_check:
        raise ValueError(f"was expecting embedding dimension of {embed_dim_to_check}, but got {embed_dim}")
    head_dim = embed_dim // num_heads
    rows = batch * num_heads

    # Input projections.
    if use_separate_proj_weight:
        proj_w = (q_proj_weight, k_proj_weight, v_proj_weight)
    else:
        proj_w = in_proj_weight.chunk(3)
    proj_b = in_proj_bias.chunk(3) if in_proj_bias is not None else (None, None, None)
    q = F.linear(query, proj_w[0], proj_b[0])
    k = F.linear(key, proj_w[1], proj_b[1])
    v = F.linear(value, proj_w[2], proj_b[2])

    mask = _float_mask(attn_mask)
    if mask is not None and mask.dim() == 2:
        mask = mask.unsqueeze(0)  # one (L, S) mask for every (batch, head)
    key_pad = _float_mask(key_padding_mask)
    if bias_k is not None and bias_v is not None:
        k = torch.cat([k, bias_k.expand(1, batch, embed_dim)])
        v = torch.cat([v, bias_v.expand(1, batch, embed_dim)])
        mask, key_pad = _append_position(mask), _append_position(key_pad)

    # (seq, batch, heads * head_dim) -> (batch * heads, seq, head_dim)
    def heads(x):
        return x.reshape(x.shape[0], rows, head_dim).transpose(0, 1)

    q = heads(q)
    k = heads(k) if static_k is None else static_k
    v = heads(v) if static_v is None else static_v
    if add_zero_attn:
        k = torch.cat([k, k.new_zeros(rows, 1, head_dim)], 1)
        v = torch.cat([v, v.new_zeros(rows, 1, head_dim)], 1)
        mask, key_pad = _append_position(mask), _append_position(key_pad)
    src_len = k.shape[1]
    if key_pad is not None:
        per_row = key_pad.reshape(batch, 1, 1, src_len).expand(batch, num_heads, 1, src_len)
        per_row = per_row.reshape(rows, 1, src_len)
        mask = per_row if mask is None else mask + per_row

    attn = softmax_masked(bmm(q * math.sqrt(1.0 / head_dim), k.transpose(1, 2)), mask, safe=False)
    if training and dropout_p > 0:
        attn = dropout(attn, dropout_p, True)
    merged = bmm(attn, v).transpose(0, 1).reshape(tgt_len * batch, embed_dim)
    out = F.linear(merged, out_proj_weight, out_proj_bias).reshape(tgt_len, batch, -1)
    if unbatched:
        out = out.squeeze(1)
    if not need_weights:
        return out, None
    attn = attn.reshape(batch, num_heads, tgt_len, src_len)
    if average_attn_weights:
        attn = attn.mean(1)
    return out, attn.squeeze(0) if unbatched else attn

