"""A KV pool held in 8 bits: rows are quantised as they are committed, read in place by the attention, and turned back
into bf16 or fp32 on request.

Every row of ``head_dim`` elements is held as 8-bit codes and one fp32 scale; an element stands for ``code * scale``.
With ``a`` the row's largest magnitude:

* ``"int8"`` (``torch.int8``): ``scale = a / 127``, ``code = round(x * (127 / a))``, quotients and product rounded to
  fp32, halves to even.  An element is off by at most half a step, ``a / 254`` (and a few fp32 roundings).
* ``"e4m3"`` (``torch.float8_e4m3fn``): ``scale`` is the smallest power of two with ``a / scale <= 448``, ``code`` is
  ``x / scale`` rounded to e4m3, halves to even.  An element is off by at most 2^-4 of itself, or 2^-10 of the scale; one of
  248 * 2^120 or more rounds to 2^128, which reads back as infinity.

A row whose largest magnitude is below 2^-100 is held as zeros with scale 0.  A row with an infinity or NaN gets scale
NaN: it reads back as NaN throughout, and a query that sees it returns NaN.  A pool that was quantised elsewhere may hold
e4m3's NaN codes: a query that sees one among the keys returns NaN, one among the values makes its element NaN.  The upstream project keeps its pool in
bf16 (models/cache.py:43-60); these operators have no counterpart there.  All of them are for inference, and not for tracing:
they pass addresses to the library, which ends a ``torch.compile`` graph (``fullgraph=True`` raises); CUDA graphs capture them.
"""

from __future__ import annotations

import functools

import torch
from torch.autograd import forward_ad

from . import _native

STORAGE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_QUANTISED = (torch.int8, torch.float8_e4m3fn)
_ROWS = (torch.bfloat16, torch.float32)


def _refuse_grad(what: str, *tensors: torch.Tensor | None) -> None:
    if torch.is_grad_enabled() and True in [t is not None and t.requires_grad for t in tensors]:
        raise ValueError(f"{what} has no gradients: call it under torch.no_grad()")
    if getattr(forward_ad, "_current_level", 0) >= 0:  # inside a dual level: tangents are not switched off by torch.no_grad()
        if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
            raise ValueError(f"{what} has no forward-mode derivatives: unpack the dual tensors first")


def _int_vector(name: str, t: torch.Tensor, batch: int, index: int) -> torch.Tensor:
    if t.shape != (batch,) or (t.dtype != torch.int32 and t.dtype != torch.int64):
        raise ValueError(f"{name} must be integer (B,)")
    if t.get_device() != index:
        raise ValueError(f"{name} must be on the pool's device")
    return t if t.is_contiguous() else t.contiguous()


def _aligned(t: torch.Tensor) -> tuple[torch.Tensor, int, tuple[int, int, int]]:
    """(tensor, address, strides) of the tensor itself where its rows have unit stride and start on 16 bytes, else of a copy."""
    address, (batch, head, token, inner) = t.data_ptr(), t.stride()
    if inner != 1 or (address | (batch | head | token) * t.element_size()) & 15:
        t = t.clone(memory_format=torch.contiguous_format)  # (a contiguous tensor may start off 16 bytes)
        address, (batch, head, token, inner) = t.data_ptr(), t.stride()
    return t, address, (batch, head, token)


_NO_STRIDES = (0, 0, 0)


def _check_pool(keys: torch.Tensor, values: torch.Tensor, key_scales, value_scales) -> tuple:
    """Checks of a pool's tensors; returns (shape, device index, is held in 8 bits, code of the element type, strides of keys,
    values and both scales, the scales' addresses)."""
    shape, dtype = keys.shape, keys.dtype
    if len(shape) != 4 or (values is not keys and values.shape != shape):
        raise ValueError("pool keys and values must be matching (B,HKV,N,D) tensors")
    index = keys.get_device()
    if values is not keys and (values.dtype != dtype or values.get_device() != index):
        raise ValueError("pool keys and values must share dtype and device")
    if index < 0:
        raise ValueError("sm100 pool operators require CUDA tensors")
    k0, k1, k2, k3 = keys.stride()
    v0, v1, v2, v3 = values.stride()
    if k3 != 1 or v3 != 1:
        raise ValueError("pool rows must have unit stride in head_dim")
    if dtype in _QUANTISED:
        rows = shape[:3]
        for name, scales in (("key_scales", key_scales), ("value_scales", value_scales)):
            if scales is None or scales.shape != rows or scales.dtype != torch.float32 or scales.get_device() != index:
                raise ValueError(f"{name} must be float32 (B,HKV,N) on the pool's device")
        storage = _native.WM_INT8 if dtype == torch.int8 else _native.WM_E4M3
        return shape, index, True, storage, (k0, k1, k2), (v0, v1, v2), key_scales.stride(), value_scales.stride(), key_scales.data_ptr(), value_scales.data_ptr()
    if key_scales is not None or value_scales is not None:
        raise ValueError("only pools in int8 or float8_e4m3fn have scales")
    return shape, index, False, _native.dtype_code(dtype), (k0, k1, k2), (v0, v1, v2), _NO_STRIDES, _NO_STRIDES, 0, 0


def pool_commit(
    keys: torch.Tensor, values: torch.Tensor, key_scales, value_scales, lengths: torch.Tensor, new_keys: torch.Tensor,
    new_values: torch.Tensor, lead: int, index: torch.Tensor | None, counts: torch.Tensor | None, *, advance_to: int | None = None,
) -> None:
    """Checks and the launch behind every commit that quantises or picks rows.  With ``advance_to``, a capacity, the lengths then move
    over the rows that were written: with an index, those before the first one outside the new rows."""
    (batch, heads, slots, dim), device, quantised, storage, k_strides, v_strides, ks_strides, vs_strides, ks, vs = _check_pool(
        keys, values, key_scales, value_scales
    )
    shape, dtype = new_keys.shape, new_keys.dtype
    if len(shape) != 4 or new_values.shape != shape or shape[0] != batch or shape[1] != heads or shape[3] != dim:
        raise ValueError("new rows must be (B, heads, n, D) for both K and V")
    if dtype not in _ROWS or new_values.dtype != dtype:
        raise ValueError("new rows must be bfloat16 or float32")
    if not quantised and keys.dtype != dtype:
        raise ValueError("new rows must have the pool's dtype")
    if new_keys.get_device() != device or new_values.get_device() != device:
        raise ValueError("new rows must be on the pool's device")
    _refuse_grad("a pool commit", keys, values, key_scales, value_scales, new_keys, new_values)
    held, lengths = lengths, _int_vector("lengths", lengths, batch, device)
    rows = source_rows = shape[2]
    if index is not None:
        if index.ndim != 2 or index.shape[0] != batch or index.dtype not in (torch.int32, torch.int64) or index.get_device() != device:
            raise ValueError("index must be integer (B, n) on the pool's device")
        rows = index.shape[1]
        if index.dtype != torch.int32:  # numbers beyond the source stay beyond it
            index = index.clamp(-1, source_rows).to(torch.int32)
        index = index.contiguous()
    if counts is not None:
        counts = _int_vector("counts", counts, batch, device)
        if counts.dtype != torch.int32:
            counts = counts.clamp(0, rows).to(torch.int32)
    if not (batch and heads and slots and dim and rows and source_rows):
        return
    new_keys, nk, nk_strides = _aligned(new_keys)
    new_values, nv, nv_strides = _aligned(new_values)
    at, at_index, at_counts = lengths.data_ptr(), 0 if index is None else index.data_ptr(), 0 if counts is None else counts.data_ptr()
    record = _native.pack_pool_commit(
        keys.data_ptr(), values.data_ptr(), ks, vs, nk, nv, at, at_index, at_counts,
        *k_strides, *v_strides, *ks_strides, *vs_strides, *nk_strides, *nv_strides,
        storage, _native.WM_F32 if dtype == torch.float32 else _native.WM_BF16, batch, heads, slots, rows, source_rows, dim, lead,
        lengths.dtype == torch.int64,
    )
    _native.call_record("wm_pool_commit", device, record)
    if advance_to is not None:
        _native.call_record("wm_pool_advance", device, at, lengths.dtype == torch.int64, at_index, at_counts, batch, rows, source_rows, advance_to)
        if held is not lengths:
            held.copy_(lengths)


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
    The lengths stay as they are.  The new rows must not be views of the pool that the call writes.
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
    (batch, heads, slots, dim), device, _, storage, strides, _, scale_strides, _, scale, _ = _check_pool(codes, codes, scales, scales)
    _refuse_grad("a read back", scales)
    if lengths is not None:
        lengths = _int_vector("lengths", lengths, batch, device)
    out = torch.empty_like(codes, dtype=dtype, memory_format=torch.contiguous_format)
    if not (batch and heads and slots and dim):
        return out
    record = _native.pack_pool_dequant(
        codes.data_ptr(), scale, 0 if lengths is None else lengths.data_ptr(), out.data_ptr(),
        *strides, *scale_strides, heads * slots * dim, slots * dim, dim,
        storage, _native.WM_F32 if dtype == torch.float32 else _native.WM_BF16, batch, heads, slots, dim, int(use_dummy_token),
        lengths is not None and lengths.dtype == torch.int64,
    )
    _native.call_record("wm_pool_dequant", device, record)
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
    (pool_batch, kv_heads, slots, pool_dim), device, quantised, storage, k_strides, v_strides, ks_strides, vs_strides, ks, vs = _check_pool(
        keys, values, key_scales, value_scales
    )
    batch, heads, length, dim = query.shape
    dtype = query.dtype
    if pool_batch != batch or pool_dim != dim or not kv_heads or heads % kv_heads:
        raise ValueError("Q/K/V require matching batch/head_dim and divisible heads")
    if query.get_device() != device:
        raise ValueError("Q/K/V must share a device")
    if dtype not in _ROWS:
        raise ValueError("query must be bfloat16 or float32")
    if not quantised and keys.dtype != dtype:
        raise ValueError("the pool must be held in 8 bits or in the query's dtype")
    if slots < use_dummy_token or (not slots and draft is not None):
        raise ValueError("the pool must have a slot")
    if kv_lengths is not None:
        kv_lengths = _int_vector("kv_lengths", kv_lengths, batch, device)
    if key_mask is not None:
        if key_mask.shape != (batch, slots) or key_mask.dtype != torch.bool or key_mask.get_device() != device:
            raise ValueError("key_mask must be boolean (B,N) on the pool's device")
        key_mask = key_mask.contiguous()
    wide = 4 if dtype == torch.float32 else 2
    if dim > 128 or dim * wide % 16 or (quantised and dim % 16):
        raise RuntimeError("sm100 pool attention needs rows of a multiple of 16 bytes and head_dim <= 128")
    if draft is None:
        _refuse_grad("pool attention", query, keys, values, key_scales, value_scales)
    else:
        _refuse_grad("pool attention", query, keys, values, key_scales, value_scales, draft[0], draft[1])
    out = query.new_empty((batch, length, heads, dim))
    if not (batch and length and heads and dim):
        return out
    if not slots:
        return out.zero_()
    query, q, q_strides = _aligned(query)
    dk = dv = ancestors = depths = shared = 0
    dk_strides = dv_strides = _NO_STRIDES
    if draft is not None:
        draft_keys, draft_values, ancestor_bits, depth_rows = draft
        draft_keys, dk, dk_strides = _aligned(draft_keys)
        draft_values, dv, dv_strides = _aligned(draft_values)
        ancestor_bits, depth_rows = ancestor_bits.contiguous(), depth_rows.contiguous()
        ancestors, depths, shared = ancestor_bits.data_ptr(), depth_rows.data_ptr(), depth_rows.shape[0] == 1
    lengths, lengths64 = (0, 0) if kv_lengths is None else (kv_lengths.data_ptr(), kv_lengths.dtype == torch.int64)
    mask = 0 if key_mask is None else key_mask.data_ptr()
    code, lead = _native.WM_F32 if wide == 4 else _native.WM_BF16, int(use_dummy_token)
    nbytes = _workspace_bytes(code, storage, batch, heads, kv_heads, length, slots, dim, draft is not None)
    workspace = 0
    if nbytes:
        held = torch.empty(nbytes, dtype=torch.uint8, device=query.device)
        workspace = held.data_ptr()
    record = _native.pack_pool_attn(
        q, keys.data_ptr(), values.data_ptr(), ks, vs, dk, dv, ancestors, depths, lengths, mask, out.data_ptr(), workspace, nbytes,
        *q_strides, *k_strides, *v_strides, *ks_strides, *vs_strides, *dk_strides, *dv_strides, length * heads * dim, dim, heads * dim,
        code, storage, batch, heads, kv_heads, length, slots, dim, lead, lengths64, shared,
        dim**-0.5 if softmax_scale is None else float(softmax_scale),
    )
    _native.call_record("wm_pool_attn", device, record)
    return out


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(dtype: int, storage: int, batch: int, heads: int, kv_heads: int, length: int, slots: int, dim: int, tree: bool) -> int:
    """What the library asks for by the sizes of a call."""
    a = _native.PoolAttnArgs()
    a.dtype, a.storage, a.batch, a.q_heads, a.kv_heads, a.q_len, a.k_len, a.head_dim = dtype, storage, batch, heads, kv_heads, length, slots, dim
    a.ancestors = 1 if tree else None  # only whether there is a tree matters
    return _native.load_library().wm_pool_attn_workspace_bytes(_native.ctypes.byref(a))


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

    Sums and soft-max statistics are fp32.  With bf16 queries the weights, times the values' scales, enter the product as two bf16 parts
    (16 bits) for up to 16 rows (tokens times heads) per KV head and as one for more.  Values above 2^118 in magnitude may
    overflow the sums although their mean does not; weights below 2^-118 of a row's largest, and products of a weight and a scale
    below 2^-126, count as nothing.
    """
    if key.dtype not in _QUANTISED:
        raise ValueError("the pool must be int8 or float8_e4m3fn")
    return pool_attention(query, key, value, key_scales, value_scales, kv_lengths, use_dummy_token, key_mask, softmax_scale)
