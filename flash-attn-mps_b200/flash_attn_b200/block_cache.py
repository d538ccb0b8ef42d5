"""Serving over a paged KV cache held in E4M3 with one scale per block of tokens.

The cache is ``k_cache``/``v_cache`` ``[pages, page, kv_heads, dim]`` in
``float8_e4m3fn`` (page a power of two, at least 16) with ``k_scale``/``v_scale``
``[pages, page // block, kv_heads]`` in float32 (block 16, 32, 64 or 128); a
cached value is ``code * scale``. Unlike the per-request descales of
``flash_attn_varlen_func`` the scales follow the data, so no calibration is
needed before the first token. One step of a (speculative) decoder calls

* ``append_kvcache_block_scaled``: rotate Q and K at their one- or
  several-axis positions and append K and V;
* ``flash_attn_with_block_scaled_kvcache``: causal attention of one token, a
  few drafted tokens or a prompt chunk per request, optionally with a sliding
  window and first tokens that stay visible;
* ``verify_draft_tokens``: keep the drafted tokens that the target accepts and
  sample the one behind them.

Arguments are checked before the launch (``ValueError``); every call is
asynchronous on the current stream and reads no tensor value on the host, so a
step can be captured in a CUDA graph. Inference only.
"""

import ctypes
import struct

import torch

from . import _capi

_FLOATS = (torch.float16, torch.bfloat16, torch.float32)
_TENSOR = struct.Struct("@Qii8q")  # fa_tensor: pointer, dtype, ndim, 4 sizes, 4 element strides


class _Arguments:
    """A packed argument struct of the C ABI: ``tensors`` fa_tensors, then scalars."""

    def __init__(self, tensors, scalars):
        self.tensors = tensors
        self.objects = struct.Struct("@%dP" % tensors)
        self.scalars = struct.Struct("@" + scalars + "0q")
        self.at = tensors * _TENSOR.size
        self.size = self.at + self.scalars.size
        self.buffer = ctypes.c_char * self.size

    def pack(self, tensors, scalars, index):
        """The struct as a ctypes buffer; None stands for an absent tensor."""
        raw = bytearray(self.size)
        view = self.buffer.from_buffer(raw)
        describe, exchange = _describe or _find_describe()
        if exchange:
            rc = describe(self.objects.pack(*[0 if t is None else id(t) for t in tensors]), self.tensors, exchange, view, 0)
            if rc:
                _capi.check(rc)
        else:
            _device(*[t for t in tensors if t is not None])
            for i, t in enumerate(tensors):
                if t is not None:
                    ctypes.memmove(ctypes.addressof(view) + i * _TENSOR.size, ctypes.byref(_capi.tensor(t)), _TENSOR.size)
        try:
            self.scalars.pack_into(raw, self.at, *scalars)
        except (struct.error, OverflowError) as e:
            raise ValueError(f"lengths, windows and counts must be 32-bit integers, the softmax scale a float: {e}") from None
        return raw, view


_describe = None


def _find_describe():
    """(fa_describe, torch's exchange function or None)."""
    global _describe
    _describe = (_capi.describe_function(), _capi.exchange_function())
    return _describe


# key value query query_out cu_seqlens seqlens cos sin positions rotary_axes, cache (k v k_scale v_scale block_table)
_APPEND = _Arguments(15, "iii")
# q out lse cu_seqlens_q seqlens s_aux workspace, cache
_ATTEND = _Arguments(12, "iiifiiii")
# logits draft_tokens cu_drafts uniform noise draft_probs temperature tokens accepted workspace
_VERIFY = _Arguments(10, "ii")


def _device(first, *others):
    """The CUDA device that all tensors are on (its index)."""
    if not first.is_cuda:
        raise ValueError("operations require CUDA tensors")
    index = first.get_device()
    for t in others:
        if t.get_device() != index:
            raise ValueError("all tensors must be on one CUDA device")
    return index


def _cuda_index(t):
    if not t.is_cuda:
        raise ValueError("operations require CUDA tensors")
    return t.get_device()


def _no_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise NotImplementedError("flash_attn_b200 is inference only; autograd is not supported")


def _call(fn, packed, index):
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            rc = fn(packed, torch.cuda.current_stream().cuda_stream)
    else:
        rc = fn(packed, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _capi.check(rc)


def _call_with_workspace(size_fn, fn, arguments, at, tensors, scalars, like, index):
    """Ask for the workspace of the arguments, put it in as tensor number ``at``, launch."""
    raw, view = arguments.pack(tensors, scalars, index)
    size = ctypes.c_size_t()
    rc = size_fn(view, ctypes.byref(size))
    if rc:
        _capi.check(rc)
    n = size.value
    if n:
        workspace = like.new_empty(n, dtype=torch.uint8)
        _TENSOR.pack_into(raw, _TENSOR.size * at, workspace.data_ptr(), 8, 1, n, 0, 0, 0, 1, 0, 0, 0)
    _call(fn, view, index)


def _like(x):
    """An uninitialised tensor of x's shape and dtype, contiguous."""
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def _packed(x, name):
    """[tokens, heads, dim] view of a packed or [batch, new, heads, dim] tensor."""
    if x.ndim == 4:
        return x.flatten(0, 1)
    if x.ndim != 3:
        raise ValueError(f"{name} must be packed [tokens, heads, dim] or [batch, new_tokens, heads, dim]")
    return x


def _offsets(x, cu_seqlens, max_seqlen, index):
    """(cu_seqlens, max_seqlen) of packed rows, or those of a [batch, new, ...] tensor."""
    if x.ndim == 4:
        if cu_seqlens is not None:
            raise ValueError("cu_seqlens goes with packed [tokens, heads, dim] tensors")
        batch, new = x.shape[:2]
        return torch.arange(0, batch * new + 1, max(new, 1), dtype=torch.int32,
                            device=x.device)[:batch + 1] if new else torch.zeros(
                                batch + 1, dtype=torch.int32, device=x.device), new
    if cu_seqlens is None or max_seqlen is None:
        raise ValueError("packed tensors need cu_seqlens and the longest sequence's length")
    return cu_seqlens, max_seqlen


def rotary_axis_map(sections, *, interleaved=False, device=None):
    """int32 ``[sum(sections)]``: the position axis of every rotary pair.

    ``sections[a]`` pairs belong to axis ``a``: the first ``sections[0]`` pairs
    to axis 0 and so on, or, ``interleaved``, dealt out in turn while an axis
    has pairs left.
    """
    sections = [int(n) for n in sections]
    if not sections or min(sections) < 0:
        raise ValueError("sections must be nonnegative pair counts, one per axis")
    if interleaved:
        left, axes = list(sections), []
        while sum(left):
            for axis, n in enumerate(left):
                if n:
                    axes.append(axis)
                    left[axis] -= 1
    else:
        axes = [axis for axis, n in enumerate(sections) for _ in range(n)]
    return torch.tensor(axes, dtype=torch.int32, device=device)


def append_kvcache_block_scaled(
    key, value, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table, *,
    cu_seqlens=None, max_seqlen=None, query=None, query_out=None, rotary_cos=None, rotary_sin=None,
    positions=None, rotary_axes=None, rotary_interleaved=False,
):
    """Append new K/V behind ``cache_seqlens`` tokens of each request; rotate K and ``query``.

    ``key``/``value`` are packed ``[tokens, kv_heads, dim]`` with ``cu_seqlens``
    (int32 ``[batch + 1]``) and ``max_seqlen`` (the most new tokens of a
    request), or ``[batch, new_tokens, kv_heads, dim]``. Token ``j`` of request
    ``b`` lands at position ``cache_seqlens[b] + j``; lengths are not modified,
    and tokens whose page is outside the table or the cache are skipped.

    With ``rotary_cos``/``rotary_sin`` (float32 ``[positions, rotary_dim / 2]``)
    pair ``i`` of a row is rotated at ``positions[rotary_axes[i], row]``:
    ``positions`` is int32 ``[tokens]`` or ``[axes, tokens]`` (default: the
    cache position), ``rotary_axes`` int32 ``[rotary_dim / 2]``
    (``rotary_axis_map``; default: axis 0). Positions past the tables are
    clamped to their last row.

    A scale is the least power of two that holds the block's values within
    +-448; it grows, and the block's older codes are re-rounded, when a larger
    value arrives in a block that already holds tokens.

    Returns the rotated ``query`` (in ``query_out`` when given, which may be
    ``query`` itself), or None.
    """
    index = _cuda_index(key)
    _no_grad(key, value, query)
    if key.dtype not in _FLOATS or value.dtype != key.dtype:
        raise TypeError("key and value must be float16, bfloat16 or float32 of one dtype")
    cu, longest = _offsets(key, cu_seqlens, max_seqlen, index)
    if query is not None:
        if query.dtype not in _FLOATS:
            raise TypeError("query must be float16, bfloat16 or float32")
        if query_out is None:
            query_out = _like(query)
        elif query_out.shape != query.shape or query_out.dtype != query.dtype:
            raise ValueError("query_out must have the query's shape and dtype")
        if query_out.ndim == 4 and not query_out.is_contiguous():
            raise ValueError("a 4-D query_out must be contiguous")
    if rotary_cos is not None and rotary_cos.dtype != torch.float32:
        rotary_cos = rotary_cos.float()
    if rotary_sin is not None and rotary_sin.dtype != torch.float32:
        rotary_sin = rotary_sin.float()
    if cache_seqlens.ndim != 1:
        raise ValueError("cache_seqlens must be int32 [batch]")
    # Held until the launch: a head-major tensor's packed form is a copy, whose memory another thread could be given.
    tensors = (_packed(key, "key"), _packed(value, "value"), None if query is None else _packed(query, "query"),
               None if query is None else _packed(query_out, "query_out"), cu, cache_seqlens, rotary_cos, rotary_sin,
               positions, rotary_axes, k_cache, v_cache, k_scale, v_scale, block_table)
    _, view = _APPEND.pack(tensors, (cache_seqlens.shape[0], longest, bool(rotary_interleaved)), index)
    _call(_capi.library().fa_append_block_scaled, view, index)
    return query_out if query is not None else None


def flash_attn_with_block_scaled_kvcache(
    q, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table, *,
    cu_seqlens_q=None, max_seqlen_q=None, max_seqlen_k=None, softmax_scale=None, causal=True,
    window_size=(-1, -1), first_tokens=0, s_aux=None, out=None, num_splits=0, return_softmax_lse=False,
):
    """Attention of ``q`` over the ``cache_seqlens[b]`` cached tokens of each request.

    ``q`` is packed ``[tokens, heads, dim]`` with ``cu_seqlens_q`` and
    ``max_seqlen_q``, or ``[batch, queries, heads, dim]``; ``cache_seqlens``
    (int32) counts the queries' own tokens, which are the last ones. A query at
    position ``i`` sees key ``j`` when ``j <= i`` (``causal``) and, with
    ``window_size=(left, -1 or 0)`` and ``left >= 0``, only while
    ``i - j <= left`` or ``j < first_tokens``. ``s_aux`` (one value per head)
    joins the softmax's denominator. Rows that see nothing are 0 with an LSE of
    -inf. ``max_seqlen_k`` bounds ``cache_seqlens`` (default: what the block
    table holds); it sizes the launch and reads no tensor.

    Scores, maxima and sums are float32. Probabilities are rounded to 2^-9 of
    their value for bfloat16 queries and 2^-12 for float16, down to 20 nats
    below the largest in reach (prompt chunks in float16: 14), each taken with
    its V block's scale; float32 queries keep them in float32.

    A NaN in a query or in a visible K makes the rows that see it NaN; one in V
    its element of these rows and of those computed in a tile with them.

    Returns ``out`` (q's shape and dtype), with ``return_softmax_lse`` also the
    natural-log LSE: ``[heads, tokens]``, or ``[batch, heads, queries]`` for a
    4-D ``q``.
    """
    index = _cuda_index(q)
    _no_grad(q)
    if q.dtype not in _FLOATS:
        raise TypeError("q must be float16, bfloat16 or float32")
    cu, longest = _offsets(q, cu_seqlens_q, max_seqlen_q, index)
    left, right = window_size
    if right > 0 or (right == 0 and not causal):
        raise NotImplementedError("only a left window is supported over a block-scaled cache")
    if out is None:
        out = _like(q)
    elif out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError("out must have q's shape and dtype")
    elif out.ndim == 4 and not out.is_contiguous():
        raise ValueError("a 4-D out must be contiguous")
    rows = _packed(q, "q")
    lse = q.new_empty((rows.shape[1], rows.shape[0]), dtype=torch.float32)
    if k_cache.ndim != 4 or block_table.ndim != 2 or cache_seqlens.ndim != 1:
        raise ValueError("caches must be [pages, page, heads, dim], block_table [batch, pages], cache_seqlens [batch]")
    if max_seqlen_k is None:
        max_seqlen_k = min(block_table.shape[1] * k_cache.shape[1], 2 ** 31 - 1)
    if softmax_scale is None:
        softmax_scale = q.shape[-1] ** -0.5
    lib = _capi.library()
    _call_with_workspace(
        lib.fa_block_attention_workspace_size, lib.fa_block_attention_fwd, _ATTEND, 6,
        (rows, _packed(out, "out"), lse, cu, cache_seqlens, s_aux, None, k_cache, v_cache, k_scale, v_scale, block_table),
        (cache_seqlens.shape[0], longest, max_seqlen_k, softmax_scale, bool(causal), left, first_tokens, num_splits), q, index)
    if not return_softmax_lse:
        return out
    if q.ndim == 4:
        lse = lse.view(q.shape[2], q.shape[0], q.shape[1]).transpose(0, 1)
    return out, lse


def verify_draft_tokens(target_logits, draft_tokens, cu_seqlens_draft, uniform, noise, *, max_draft,
                        draft_probs=None, temperature=None):
    """Accept drafted tokens against the target's probabilities and sample the next one.

    Request ``b`` has ``cu_seqlens_draft[b + 1] - cu_seqlens_draft[b]`` drafts
    (0..``max_draft``) and one more row of ``target_logits``
    ``[drafts + batch, vocabulary]`` (rows packed per request). With ``p`` the
    softmax of a row over ``temperature[b]`` (default 1; 0 puts all mass on the
    first maximum) and ``q`` the draft's ``draft_probs`` row (default: all mass
    on the drafted token), draft ``x`` is accepted while
    ``uniform * q[x] < p[x]``. Behind the accepted ones comes the first maximum
    of ``w / noise[b]``, ``w = max(p - q, 0)`` at the first rejection (``p``
    where that is zero throughout) and ``p`` after the last draft: with
    ``noise`` drawn from Exp(1), a sample of ``w``, so that the tokens follow
    the target's distribution. ``uniform`` is float32 ``[drafts]`` in [0, 1),
    ``noise`` float32 ``[batch, vocabulary]``, positive. Probabilities and
    quotients are float32: of decisions that lie within a few units of its
    rounding either may be taken.

    Returns ``tokens`` (int64 ``[batch, max_draft + 1]``, -1 behind the last)
    and ``accepted`` (int32 ``[batch]``).
    """
    index = _cuda_index(target_logits)
    _no_grad(target_logits, draft_probs)
    if target_logits.dtype not in _FLOATS or (draft_probs is not None and draft_probs.dtype not in _FLOATS):
        raise TypeError("logits and draft probabilities must be float16, bfloat16 or float32")
    batch = cu_seqlens_draft.numel() - 1
    if batch < 1 or cu_seqlens_draft.ndim != 1:
        raise ValueError("cu_seqlens_draft must be int32 [batch + 1]")
    tokens = target_logits.new_empty((batch, max_draft + 1), dtype=torch.int64)
    accepted = target_logits.new_empty(batch, dtype=torch.int32)
    lib = _capi.library()
    _call_with_workspace(
        lib.fa_verify_workspace_size, lib.fa_verify_draft_tokens, _VERIFY, 9,
        (target_logits, draft_tokens, cu_seqlens_draft, uniform, noise, draft_probs, temperature, tokens, accepted, None),
        (batch, max_draft), target_logits, index)
    return tokens, accepted
