"""A KV pool held in 8 bits: rows are quantised as they are committed, read in place by the attention, and turned back
into bf16 or fp32 on request.

Every row of ``head_dim`` elements is held as 8-bit codes and one fp32 scale; an element stands for ``code * scale``.
With ``a`` the row's largest magnitude:

* ``"int8"`` (``torch.int8``): ``scale = a / 127``, ``code = round(x * (127 / a))``, quotients and product rounded to
  fp32, halves to even.  An element is off by at most half a step, ``a / 254`` (and a few fp32 roundings).
* ``"e4m3"`` (``torch.float8_e4m3fn``): ``scale`` is the smallest power of two with ``a / scale <= 448``, ``code`` is
  ``x / scale`` rounded to e4m3, halves to even.  An element is off by at most 2^-4 of itself, or 2^-10 of the scale.

A row whose largest magnitude is below 2^-100 is held as zeros with scale 0.  A row with an infinity or NaN gets scale
NaN: it reads back as NaN throughout, and a query that sees it returns NaN.  The upstream project keeps its pool in
bf16 (models/cache.py:43-60); these operators have no counterpart there.  All of them are for inference.
"""

from __future__ import annotations

import torch

from . import _native

STORAGE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_QUANTISED = (torch.int8, torch.float8_e4m3fn)
_ROWS = (torch.bfloat16, torch.float32)


def _refuse_grad(what: str, *tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled() and True in [t.requires_grad for t in tensors]:
        raise ValueError(f"{what} has no gradients: call it under torch.no_grad()")


def _int_vector(name: str, t: torch.Tensor, batch: int, device: torch.device) -> torch.Tensor:
    if t.shape != (batch,) or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be integer (B,)")
    if t.device != device:
        raise ValueError(f"{name} must be on the pool's device")
    return t if t.is_contiguous() else t.contiguous()


def _aligned(t: torch.Tensor) -> tuple[torch.Tensor, int, tuple[int, int, int]]:
    """(tensor, address, strides) of the tensor itself where its rows have unit stride and start on 16 bytes, else of a copy."""
    address, (batch, head, token, inner) = t.data_ptr(), t.stride()
    if inner != 1 or (address | (batch | head | token) * t.element_size()) & 15:
        t = t.contiguous()
        address, (batch, head, token, inner) = t.data_ptr(), t.stride()
    return t, address, (batch, head, token)


def _check_pool(keys: torch.Tensor, values: torch.Tensor, key_scales, value_scales) -> None:
    if keys.ndim != 4 or keys.shape != values.shape:
        raise ValueError("pool keys and values must be matching (B,HKV,N,D) tensors")
    if keys.dtype != values.dtype or keys.device != values.device:
        raise ValueError("pool keys and values must share dtype and device")
    if not keys.is_cuda:
        raise ValueError("sm100 pool operators require CUDA tensors")
    if keys.stride()[3] != 1 or values.stride()[3] != 1:
        raise ValueError("pool rows must have unit stride in head_dim")
    if keys.dtype in _QUANTISED:
        for name, scales in (("key_scales", key_scales), ("value_scales", value_scales)):
            if scales is None or scales.shape != keys.shape[:3] or scales.dtype != torch.float32 or scales.device != keys.device:
                raise ValueError(f"{name} must be float32 (B,HKV,N) on the pool's device")
    elif key_scales is not None or value_scales is not None:
        raise ValueError("only pools in int8 or float8_e4m3fn have scales")


def pool_commit(
    keys: torch.Tensor, values: torch.Tensor, key_scales, value_scales, lengths: torch.Tensor, new_keys: torch.Tensor,
    new_values: torch.Tensor, lead: int, index: torch.Tensor | None, counts: torch.Tensor | None,
) -> int:
    """Checks and the launch behind every commit that quantises or picks rows; returns how many rows a sequence can get."""
    _check_pool(keys, values, key_scales, value_scales)
    batch, heads, slots, dim = keys.shape
    if new_keys.ndim != 4 or new_keys.shape != new_values.shape or new_keys.shape[:2] != (batch, heads) or new_keys.shape[3] != dim:
        raise ValueError("new rows must be (B, heads, n, D) for both K and V")
    if new_keys.dtype not in _ROWS or new_values.dtype != new_keys.dtype:
        raise ValueError("new rows must be bfloat16 or float32")
    if keys.dtype not in _QUANTISED and keys.dtype != new_keys.dtype:
        raise ValueError("new rows must have the pool's dtype")
    if any(t.device != keys.device for t in (new_keys, new_values)):
        raise ValueError("new rows must be on the pool's device")
    _refuse_grad("a pool commit", new_keys, new_values)
    lengths = _int_vector("lengths", lengths, batch, keys.device)
    rows = new_keys.shape[2]
    if index is not None:
        if index.ndim != 2 or index.shape[0] != batch or index.dtype not in (torch.int32, torch.int64) or index.device != keys.device:
            raise ValueError("index must be integer (B, n) on the pool's device")
        rows = index.shape[1]
        if index.dtype != torch.int32:  # numbers beyond the source stay beyond it
            index = index.clamp(-1, new_keys.shape[2]).to(torch.int32)
        index = index.contiguous()
    if counts is not None:
        counts = _int_vector("counts", counts, batch, keys.device)
        if counts.dtype != torch.int32:
            counts = counts.clamp(0, rows).to(torch.int32)
    if not batch or not heads or not slots or not dim or not rows or not new_keys.shape[2]:
        return rows
    a = _native.PoolCommitArgs()
    new_keys, a.new_keys, a.new_key_strides = _aligned(new_keys)
    new_values, a.new_values, a.new_value_strides = _aligned(new_values)
    a.keys, a.values = keys.data_ptr(), values.data_ptr()
    a.key_strides, a.value_strides = keys.stride()[:3], values.stride()[:3]
    if key_scales is not None:
        a.key_scales, a.value_scales = key_scales.data_ptr(), value_scales.data_ptr()
        a.key_scale_strides, a.value_scale_strides = key_scales.stride(), value_scales.stride()
    a.lengths, a.lengths_is64 = lengths.data_ptr(), lengths.dtype == torch.int64
    if index is not None:
        a.index = index.data_ptr()
    if counts is not None:
        a.counts = counts.data_ptr()
    a.storage, a.dtype = _native.storage_code(keys.dtype), _native.dtype_code(new_keys.dtype)
    a.batch, a.heads, a.slots, a.head_dim = batch, heads, slots, dim
    a.rows, a.source_rows, a.lead = rows, new_keys.shape[2], lead
    _native.call("wm_pool_commit", a, keys.device)
    return rows


def quantized_pool_append(
    keys: torch.Tensor,
    values: torch.Tensor,
    key_scales: torch.Tensor,
    value_scales: torch.Tensor,
    lengths: torch.Tensor,
    new_keys: torch.Tensor,
    new_values: torch.Tensor,
    *,
    use_dummy_token: bool = False,
    index: torch.Tensor | None = None,
    counts: torch.Tensor | None = None,
) -> None:
    """Quantise new K and V rows into an 8-bit pool behind each sequence's committed tokens, in one launch.

    The pool is (B,H,N,D) in ``torch.int8`` or ``torch.float8_e4m3fn`` with fp32 scales (B,H,N), the new rows are
    (B,H,n,D) in bf16 or fp32, D a multiple of 16 up to 128.  Row i of sequence b goes to slot ``lengths[b] + i``
    (one further with ``use_dummy_token``).  ``index`` (B,m) picks the rows instead: slot i gets row ``index[b,i]``;
    ``counts`` (B,) bounds the number of rows per sequence -- together they commit the accepted branch of a draft.
    Rows that would not fit the pool, and indices outside the new rows, are skipped: their slots keep what they held.
    The lengths stay as they are.
    """
    if type(use_dummy_token) is not bool:
        raise ValueError("use_dummy_token must be boolean")
    if keys.dtype not in _QUANTISED:
        raise ValueError("the pool must be int8 or float8_e4m3fn")
    pool_commit(keys, values, key_scales, value_scales, lengths, new_keys, new_values, int(use_dummy_token), index, counts)


def dequantize_kv_rows(
    codes: torch.Tensor,
    scales: torch.Tensor,
    *,
    lengths: torch.Tensor | None = None,
    use_dummy_token: bool = False,
    dtype: torch.dtype = torch.bfloat16,
) -> torch.Tensor:
    """The rows that a pool's codes (B,H,N,D) and scales (B,H,N) stand for, as a new (B,H,N,D) tensor in bf16 or fp32.

    With ``lengths`` (B,) only the committed rows (and the dummy slot with ``use_dummy_token``) are read; the rows
    behind them come back as zeros.
    """
    if type(use_dummy_token) is not bool:
        raise ValueError("use_dummy_token must be boolean")
    if codes.ndim != 4 or codes.dtype not in _QUANTISED:
        raise ValueError("codes must be (B,H,N,D) in int8 or float8_e4m3fn")
    if dtype not in _ROWS:
        raise ValueError("rows are read back in bfloat16 or float32")
    _check_pool(codes, codes, scales, scales)
    batch, heads, slots, dim = codes.shape
    if lengths is not None:
        lengths = _int_vector("lengths", lengths, batch, codes.device)
    out = torch.empty(codes.shape, dtype=dtype, device=codes.device)
    if not out.numel():
        return out
    a = _native.PoolDequantArgs()
    a.codes, a.scales, a.out = codes.data_ptr(), scales.data_ptr(), out.data_ptr()
    a.code_strides, a.scale_strides, a.out_strides = codes.stride()[:3], scales.stride(), out.stride()[:3]
    if lengths is not None:
        a.lengths, a.lengths_is64 = lengths.data_ptr(), lengths.dtype == torch.int64
    a.storage, a.dtype = _native.storage_code(codes.dtype), _native.dtype_code(dtype)
    a.batch, a.heads, a.slots, a.head_dim = batch, heads, slots, dim
    a.lead = int(use_dummy_token)
    _native.call("wm_pool_dequant", a, codes.device)
    return out


def pool_attention(
    query: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, key_scales, value_scales, kv_lengths, use_dummy_token: bool,
    key_mask, softmax_scale, draft=None,
) -> torch.Tensor:
    """Checks and the launch behind every read of queries that stand behind the committed tokens; ``draft`` is
    (draft keys, draft values, ancestors, depths) or None."""
    if type(use_dummy_token) is not bool:
        raise ValueError("use_dummy_token must be boolean")
    if query.ndim != 4:
        raise ValueError("query must be (B,H,T,D)")
    _check_pool(keys, values, key_scales, value_scales)
    batch, heads, length, dim = query.shape
    kv_heads, slots = keys.shape[1], keys.shape[2]
    if keys.shape[0] != batch or keys.shape[3] != dim or not kv_heads or heads % kv_heads:
        raise ValueError("Q/K/V require matching batch/head_dim and divisible heads")
    if query.device != keys.device:
        raise ValueError("Q/K/V must share a device")
    if query.dtype not in _ROWS:
        raise ValueError("query must be bfloat16 or float32")
    if keys.dtype not in _QUANTISED and keys.dtype != query.dtype:
        raise ValueError("the pool must be held in 8 bits or in the query's dtype")
    if slots < int(use_dummy_token) or (not slots and draft is not None):
        raise ValueError("the pool must have a slot")
    if kv_lengths is not None:
        kv_lengths = _int_vector("kv_lengths", kv_lengths, batch, query.device)
    if key_mask is not None and (key_mask.shape != (batch, slots) or key_mask.dtype != torch.bool or key_mask.device != query.device):
        raise ValueError("key_mask must be boolean (B,N) on the pool's device")
    _refuse_grad("pool attention", query, *(draft[:2] if draft is not None else ()))
    if dim > 128 or dim * query.element_size() % 16 or dim * keys.element_size() % 16:
        raise RuntimeError("sm100 pool attention needs rows of a multiple of 16 bytes and head_dim <= 128")
    out = torch.empty((batch, length, heads, dim), dtype=query.dtype, device=query.device)
    if not out.numel():
        return out
    if not slots:
        return out.zero_()
    a = _native.PoolAttnArgs()
    query, a.q, a.q_strides = _aligned(query)
    a.k, a.v, a.out = keys.data_ptr(), values.data_ptr(), out.data_ptr()
    a.k_strides, a.v_strides = keys.stride()[:3], values.stride()[:3]
    a.out_strides = length * heads * dim, dim, heads * dim
    if key_scales is not None:
        a.k_scales, a.v_scales = key_scales.data_ptr(), value_scales.data_ptr()
        a.k_scale_strides, a.v_scale_strides = key_scales.stride(), value_scales.stride()
    if kv_lengths is not None:
        a.lengths, a.lengths_is64 = kv_lengths.data_ptr(), kv_lengths.dtype == torch.int64
    if key_mask is not None:
        key_mask = key_mask.contiguous()
        a.key_mask = key_mask.data_ptr()
    if draft is not None:
        draft_keys, draft_values, ancestors, depths = draft
        draft_keys, a.draft_k, a.draft_k_strides = _aligned(draft_keys)
        draft_values, a.draft_v, a.draft_v_strides = _aligned(draft_values)
        ancestors, depths = ancestors.contiguous(), depths.contiguous()
        a.ancestors, a.depths = ancestors.data_ptr(), depths.data_ptr()
        a.shared_tree = depths.shape[0] == 1
    a.dtype, a.storage = _native.dtype_code(query.dtype), _native.storage_code(keys.dtype)
    a.batch, a.q_heads, a.q_len, a.head_dim = batch, heads, length, dim
    a.kv_heads, a.k_len, a.lead = kv_heads, slots, int(use_dummy_token)
    a.scale = dim**-0.5 if softmax_scale is None else float(softmax_scale)
    nbytes = _native.load_library().wm_pool_attn_workspace_bytes(_native.ctypes.byref(a))
    if nbytes:
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=query.device)
        a.workspace, a.workspace_bytes = workspace.data_ptr(), nbytes
    _native.call("wm_pool_attn", a, query.device)
    return out


def quantized_pool_attention(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    key_scales: torch.Tensor,
    value_scales: torch.Tensor,
    *,
    kv_lengths: torch.Tensor | None = None,
    use_dummy_token: bool = False,
    key_mask: torch.Tensor | None = None,
    softmax_scale: float | None = None,
) -> torch.Tensor:
    """Attention of queries that stand behind the committed tokens over an 8-bit pool, read in place.

    ``query`` is (B,H,T,D) in bf16 or fp32: one token per sequence, or T new ones that do not see one another.  The pool
    is (B,HKV,N,D) in ``torch.int8`` or ``torch.float8_e4m3fn`` with fp32 scales (B,HKV,N); any strides with unit stride
    in D and 16-byte aligned rows, so a channel view of a larger pool will do.  Every query sees the real slots
    s < ``kv_lengths[b]`` (all of them without lengths) and, with ``use_dummy_token``, slot 0, as far as ``key_mask``
    (B,N) keeps them; slots that are not seen may hold anything.  Rows without a visible slot return zero.  The
    lengths stay on the device, so the call can be captured in a CUDA graph.  Returns (B,T,H,D).
    """
    if key.dtype not in _QUANTISED:
        raise ValueError("the pool must be int8 or float8_e4m3fn")
    return pool_attention(query, key, value, key_scales, value_scales, kv_lengths, use_dummy_token, key_mask, softmax_scale)
