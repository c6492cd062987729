"""The 8-bit KV pool: refusals and layouts on the CPU; commit, read back and read against the CPU oracle on the GPU."""

import ctypes
import functools
import re
from pathlib import Path

import pytest
import torch

import test_abi
from oracle import serving_oracle as oracle
from white_matter_b200 import _native
from white_matter_b200.decode_step import DecodeStepGraph, KVPoolCache, QuantKVPoolCache
from white_matter_b200.quant_pool import STORAGE, dequantize_kv_rows, quantized_pool_append, quantized_pool_attention

HEADER = (Path(__file__).resolve().parent.parent / "include" / "wm_b200_serving.h").read_text()
STRUCTS = {
    "wm_pool_commit_args": _native.PoolCommitArgs,
    "wm_pool_dequant_args": _native.PoolDequantArgs,
    "wm_draft_tree_args": _native.DraftTreeArgs,
    "wm_pool_attn_args": _native.PoolAttnArgs,
}
on_gpu = pytest.mark.skipif(not torch.cuda.is_available(), reason="requires CUDA")


# ------------------------------------------------------------------ CPU


def test_every_struct_of_the_serving_header_is_mirrored(monkeypatch):
    assert sorted(re.findall(r"typedef struct (\w+) \{", HEADER)) == sorted(STRUCTS)
    monkeypatch.setattr(test_abi, "HEADER", HEADER)
    for struct, mirrored in STRUCTS.items():
        declared = test_abi.header_fields(struct)
        assert [name for name, _ in mirrored._fields_] == [name for name, _ in declared]
        for (name, have), (_, want) in zip(mirrored._fields_, declared):
            assert ctypes.sizeof(have) == ctypes.sizeof(want), name


def test_entry_points_refuse_before_any_cuda_call():
    lib = _native.load_library()
    for name, struct in _native.SERVING_ENTRY_POINTS:
        assert getattr(lib, name)(ctypes.byref(struct()), None) == -1, name
        assert getattr(lib, name)(None, None) == -1, name
    assert lib.wm_pool_attn_workspace_bytes(ctypes.byref(_native.PoolAttnArgs())) == 0


def fake_attn(**change):
    """Arguments that would be accepted, with made-up addresses: nothing is launched by a call that is refused."""
    a = _native.PoolAttnArgs()
    for name in ("q", "k", "v", "out", "k_scales", "v_scales", "workspace"):
        setattr(a, name, 1 << 20)
    for name in ("q_strides", "k_strides", "v_strides", "out_strides"):
        setattr(a, name, _native._Strides(4096, 1024, 64))
    a.dtype, a.storage = _native.WM_BF16, _native.WM_INT8
    a.batch, a.q_heads, a.kv_heads, a.q_len, a.k_len, a.head_dim, a.scale = 1, 2, 1, 1, 8000, 64, 1.0
    for name, value in change.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize(
    "change, status, text",
    [
        (dict(dtype=2), -1, b"dtype"),
        (dict(storage=_native.WM_F32), -1, b"queries' type"),
        (dict(k_scales=None), -1, b"scales"),
        (dict(batch=0), -1, b"sizes"),
        (dict(q_heads=3, kv_heads=2), -1, b"multiple of kv_heads"),
        (dict(lead=2), -1, b"lead"),
        (dict(depths=1 << 20), -1, b"tree tables"),
        (dict(head_dim=72), -2, b"multiple of 16 bytes"),
        (dict(head_dim=144), -2, b"at most 128"),
        (dict(k=(1 << 20) + 8), -2, b"aligned"),
        (dict(k_strides=_native._Strides(4096, 1024, 72)), -2, b"aligned"),
        (dict(q_len=513, draft_k=1 << 20, draft_v=1 << 20, ancestors=1 << 20, depths=1 << 20), -2, b"drafted tokens"),
        (dict(q_len=2**31 - 1), -2, b"too many query rows"),
        (dict(workspace=None), -4, b"workspace"),
        (dict(workspace_bytes=16), -4, b"workspace"),
    ],
)
def test_attention_refusals(change, status, text):
    lib = _native.load_library()
    assert lib.wm_pool_attn(ctypes.byref(fake_attn(**change)), None) == status
    assert text in lib.wm_last_error()


@pytest.mark.parametrize(
    "change, text",
    [
        (dict(out=(1 << 20) + 4), b"output rows"),
        (dict(out_strides=_native._Strides(4096, 1024, 33)), b"output rows"),
        (dict(workspace=(1 << 20) + 8), b"workspace must be"),
        (dict(k_len=2**31 - 1), b"too many slots"),
        (dict(k_strides=_native._Strides(4096, 1024, 1 << 24)), b"2^24"),
    ],
)
def test_attention_refuses_what_it_could_not_address(change, text):
    lib = _native.load_library()
    assert lib.wm_pool_attn(ctypes.byref(fake_attn(**change)), None) == -2
    assert text in lib.wm_last_error()


def test_read_back_refuses_more_slots_than_it_counts():
    a = _native.PoolDequantArgs()
    for name in ("codes", "scales", "out"):
        setattr(a, name, 1 << 20)
    a.code_strides = a.out_strides = _native._Strides(1 << 35, 1 << 35, 16)
    a.storage, a.dtype, a.batch, a.heads, a.slots, a.head_dim = _native.WM_INT8, _native.WM_BF16, 1, 1, 2**31 - 1, 16
    lib = _native.load_library()
    assert lib.wm_pool_dequant(ctypes.byref(a), None) == -2 and b"too many slots" in lib.wm_last_error()


@pytest.mark.parametrize(
    "change, status, text",
    [
        (dict(lengths=None), -1, b"lengths"),
        (dict(dtype=5), -1, b"new rows"),
        (dict(storage=_native.WM_F32), -1, b"rows' type"),
        (dict(key_scales=None), -1, b"scales"),
        (dict(rows=0), -1, b"positive"),
        (dict(rows=3), -1, b"more rows"),
        (dict(lead=-1), -1, b"lead"),
        (dict(head_dim=24), -2, b"multiple of 16"),
        (dict(head_dim=256), -2, b"up to 128"),
        (dict(values=(1 << 20) + 4), -2, b"aligned"),
        (dict(new_key_strides=_native._Strides(64, 64, 60)), -2, b"aligned"),
        (dict(heads=65536, rows=65536, source_rows=65536), -2, b"rows per sequence"),
    ],
)
def test_commit_refusals(change, status, text):
    a = _native.PoolCommitArgs()
    for name in ("keys", "values", "key_scales", "value_scales", "new_keys", "new_values", "lengths"):
        setattr(a, name, 1 << 20)
    for name in ("key_strides", "value_strides", "new_key_strides", "new_value_strides"):
        setattr(a, name, _native._Strides(4096, 1024, 64))
    a.storage, a.dtype = _native.WM_E4M3, _native.WM_BF16
    a.batch, a.heads, a.slots, a.rows, a.source_rows, a.head_dim = 1, 1, 8, 2, 2, 64
    for name, value in change.items():
        setattr(a, name, value)
    lib = _native.load_library()
    assert lib.wm_pool_commit(ctypes.byref(a), None) == status
    assert text in lib.wm_last_error()


@pytest.mark.parametrize("many", [2**31 - 1, 2**31 - 65535])
def test_more_sequences_than_32_bits_count_a_grid_at_a_time_are_refused(many):
    commit = _native.PoolCommitArgs()
    for name in ("keys", "values", "key_scales", "value_scales", "new_keys", "new_values", "lengths"):
        setattr(commit, name, 1 << 20)
    for name in ("key_strides", "value_strides", "new_key_strides", "new_value_strides"):
        setattr(commit, name, _native._Strides(4096, 1024, 64))
    commit.storage, commit.dtype = _native.WM_INT8, _native.WM_BF16
    commit.batch, commit.heads, commit.slots, commit.rows, commit.source_rows, commit.head_dim = many, 1, 8, 2, 2, 64
    lib = _native.load_library()
    assert lib.wm_pool_commit(ctypes.byref(commit), None) == -2 and b"too many sequences" in lib.wm_last_error()
    back = _native.PoolDequantArgs()
    for name in ("codes", "scales", "out"):
        setattr(back, name, 1 << 20)
    back.code_strides = back.out_strides = _native._Strides(4096, 1024, 64)
    back.storage, back.dtype, back.batch, back.heads, back.slots, back.head_dim = _native.WM_INT8, _native.WM_BF16, many, 1, 8, 64
    assert lib.wm_pool_dequant(ctypes.byref(back), None) == -2 and b"planes" in lib.wm_last_error()


@pytest.mark.parametrize("change, status", [(dict(lengths=None), -1), (dict(batch=0), -1), (dict(rows=0), -1), (dict(source=0), -1), (dict(capacity=0), -1), (dict(rows=2**31 - 1), -2)])
def test_advance_refusals(change, status):
    a = dict(lengths=1 << 20, batch=1, rows=4, source=4, capacity=9)
    a.update(change)
    assert _native.load_library().wm_pool_advance(a["lengths"], 0, None, None, a["batch"], a["rows"], a["source"], a["capacity"], None) == status


def test_python_refusals():
    codes, rows = torch.zeros(1, 2, 8, 64, dtype=torch.int8), torch.zeros(1, 2, 1, 64)
    scales, lengths = torch.zeros(1, 2, 8), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="requires? CUDA"):
        quantized_pool_append(codes, codes, scales, scales, lengths, rows, rows)
    with pytest.raises(ValueError, match="int8 or float8_e4m3fn"):
        quantized_pool_append(codes.float(), codes.float(), scales, scales, lengths, rows, rows)
    with pytest.raises(ValueError, match="use_dummy_token must be boolean"):
        quantized_pool_append(codes, codes, scales, scales, lengths, rows, rows, use_dummy_token=1)
    with pytest.raises(ValueError, match="int8 or float8_e4m3fn"):
        dequantize_kv_rows(rows, scales)
    with pytest.raises(ValueError, match="bfloat16 or float32"):
        dequantize_kv_rows(codes, scales, dtype=torch.float16)
    with pytest.raises(ValueError, match="requires? CUDA"):
        dequantize_kv_rows(codes, scales)
    with pytest.raises(ValueError, match="int8 or float8_e4m3fn"):
        quantized_pool_attention(rows, rows, rows, scales, scales)
    with pytest.raises(ValueError, match="requires? CUDA"):
        quantized_pool_attention(rows, codes, codes, scales, scales)
    with pytest.raises(ValueError, match="storage must be one of"):
        QuantKVPoolCache(1, 1, 1, 8, 64, storage="int4", device="cpu")
    with pytest.raises(ValueError, match="multiple of 16"):
        QuantKVPoolCache(1, 1, 1, 8, 72, device="cpu")
    with pytest.raises(ValueError, match="positive"):
        QuantKVPoolCache(1, 1, 0, 8, 64, device="cpu")
    pool = QuantKVPoolCache(2, 3, 2, 8, 64, storage="e4m3", use_dummy_token=True, device="cpu")
    assert pool.keys.shape == (2, 6, 9, 64) and pool.keys.dtype == torch.float8_e4m3fn
    with pytest.raises(ValueError, match="channel must be in"):
        pool.channel(3)


@pytest.mark.parametrize("storage", sorted(STORAGE))
def test_the_oracle_keeps_the_error_bound_of_the_format(storage):
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(40, 64, generator=gen) * torch.exp(3 * torch.randn(40, 1, generator=gen))
    codes, scales = oracle.quantise_rows(x, storage)
    assert torch.equal(codes, codes.to(STORAGE[storage]).float())  # every code is a number of the type
    if storage == "int8":
        top = x.abs().amax(-1, keepdim=True).double()
        off = top / 254 + 2.0**-22 * top  # half a step, and the roundings of both quotients, the product and code * scale
    else:
        off = torch.maximum(x.abs().double() * 2.0**-4, scales[:, None].double() * 2.0**-10)
    assert ((codes.double() * scales[:, None].double() - x.double()).abs() <= off).all()


# ------------------------------------------------------------------ GPU: commit and read back


def make_pool(batch, heads, slots, dim, storage):
    """A pool whose slots hold something already, so that a slot that should not be written shows."""
    codes = torch.full((batch, heads, slots, dim), 3.0)
    scales = torch.full((batch, heads, slots), 0.5)
    return codes, scales, codes.to(STORAGE[storage]).cuda(), scales.cuda()


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("dim", [16, 48, 64, 80, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("storage", sorted(STORAGE))
def test_commit_writes_the_rows_of_the_definition(storage, dtype, dim):
    batch, heads, slots, rows, lead = 5, 3, 13, 7, 1
    gen = torch.Generator().manual_seed(dim)
    lengths = torch.tensor([0, 5, 12, -9, 100], dtype=torch.int64)  # the last three run over the ends of the pool
    new = [(torch.randn(batch, rows, heads, dim, generator=gen) * torch.exp(2 * torch.randn(batch, rows, heads, 1, generator=gen))).to(dtype) for _ in "kv"]
    new[0][0, 0] = 0
    new[0][1, 1, 1, 3] = float("nan")
    new[0][1, 2, 0, 5] = float("-inf")
    new[1][0, 1] = 2.0**-101
    new[1][0, 2] *= 2.0**-96
    new[1][0, 3] = 3.0e38
    new[1][1, 0, :, 1:] = 0  # a single element far above the others
    for lengths_dtype, index, counts in (
        (torch.int64, None, None),
        (torch.int32, torch.tensor([[0, 2, 2, 6], [6, 5, 1, 0], [0, 1, 2, 3], [3, 3, 3, 3], [1, 2, 3, 4]]), None),
        (torch.int32, torch.tensor([[0, 2, 7, 6], [-1, 5, 1, 0], [0, 1, 2, 3], [3, 3, 3, 3], [1, 2, 3, 4]], dtype=torch.int32), torch.tensor([4, 3, 0, 2, -5])),
        (torch.int64, None, torch.tensor([7, 1, 50, 0, 3], dtype=torch.int32)),
    ):
        expected, pools = [], []
        for x in new:
            codes, scales, pool, pool_scales = make_pool(batch, heads, slots, dim, storage)
            oracle.commit(codes, scales, lengths, x.transpose(1, 2), storage, lead, index, counts)
            expected.append((codes, scales))
            pools.append((pool, pool_scales))
        on = lambda t: None if t is None else t.cuda()
        quantized_pool_append(
            pools[0][0], pools[1][0], pools[0][1], pools[1][1], lengths.to(lengths_dtype).cuda(), *(x.cuda().transpose(1, 2) for x in new),
            use_dummy_token=bool(lead), index=on(index), counts=on(counts),
        )
        for (codes, scales), (pool, pool_scales) in zip(expected, pools):
            assert torch.equal(pool.cpu().float(), codes)
            assert torch.equal(torch.nan_to_num(pool_scales.cpu(), nan=-1.0), torch.nan_to_num(scales, nan=-1.0))


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_plain_pool_commits_picked_rows(dtype):
    gen = torch.Generator().manual_seed(4)
    pool = KVPoolCache(3, 1, 2, 10, 64, use_dummy_token=True, dtype=dtype)
    pool.lengths.copy_(torch.tensor([0, 4, 9]))
    new = [torch.randn(3, 2, 6, 64, generator=gen).to(dtype) for _ in "kv"]
    index, counts = torch.tensor([[5, 0, 5], [1, 2, 3], [4, 4, 0]], dtype=torch.int32), torch.tensor([3, 2, 3])
    expected = [pool.keys.cpu().clone(), pool.values.cpu().clone()]
    for target, x in zip(expected, new):
        oracle.commit(target, None, [0, 4, 9], x, None, 1, index, counts)
    pool.append(*(x.cuda() for x in new), index=index.cuda(), counts=counts.cuda())
    assert torch.equal(pool.keys.cpu(), expected[0]) and torch.equal(pool.values.cpu(), expected[1])
    assert pool.lengths.tolist() == [3, 6, 10]


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("dim", [16, 64, 112])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("storage", sorted(STORAGE))
def test_read_back_is_code_times_scale(storage, dtype, dim):
    gen = torch.Generator().manual_seed(dim)
    codes, scales = oracle.quantise_rows(torch.randn(3, 4, 9, dim, generator=gen), storage)
    scales[0, 0, 2], scales[2, 3, 8] = float("nan"), float("nan")
    pool = codes.to(STORAGE[storage]).cuda()
    lengths = torch.tensor([5, -3, 50])
    for lengths_arg, lead in ((None, False), (lengths, False), (lengths.int(), True)):
        got = dequantize_kv_rows(pool[:, 1:3], scales.cuda()[:, 1:3], lengths=None if lengths_arg is None else lengths_arg.cuda(), use_dummy_token=lead, dtype=dtype)
        want = (codes * scales[..., None])[:, 1:3].to(dtype)  # one fp32 rounding, one to the type
        if lengths_arg is not None:
            for b in range(3):
                want[b, :, max(0, int(lengths[b]) + lead) :] = 0
        assert torch.equal(torch.nan_to_num(got.cpu(), nan=-77.0), torch.nan_to_num(want, nan=-77.0))


# ------------------------------------------------------------------ GPU: attention


def quantised_problem(seed, storage, dtype, batch, heads, kv_heads, tokens, slots, dim, lead, masked, lengths):
    """Inputs with everything that must not be used poisoned: unused capacity, and masked slots."""
    gen = torch.Generator().manual_seed(seed)
    query = torch.randn(batch, tokens, heads, dim, generator=gen).to(dtype).transpose(1, 2)
    pools = []
    for spread in (0.3, 1.0):
        x = torch.randn(batch, kv_heads, slots, dim, generator=gen) * torch.exp(spread * torch.randn(batch, kv_heads, slots, 1, generator=gen))
        codes, scales = oracle.quantise_rows(x, storage)
        pools.append((codes, scales))
    mask = None
    if masked:
        mask = torch.rand(batch, slots, generator=gen) < 0.6
        mask[0] = False  # a sequence that sees nothing
    rows = [codes * scales[..., None].double() for codes, scales in pools]
    for b in range(batch):
        n = slots if lengths is None else min(max(int(lengths[b]), 0), slots - lead) + lead
        dead = torch.arange(slots) >= n
        if mask is not None:
            dead |= ~mask[b]
        for codes, scales in pools:
            scales[b][:, dead] = float("nan")
            codes[b][:, dead] = 100.0 if storage == "int8" else float("nan")
    return query, pools, rows, mask


def check_attention(got, query, rows, lengths, lead, mask, draft=None, scale=None):
    out, mass, reach = oracle.attention(query, rows[0], rows[1], lengths, lead, mask, draft, scale)
    keys = rows[0].shape[2] + (query.shape[2] if draft is not None else 0)
    limit = oracle.bound(out, mass, reach, query.dtype, query.shape[3], keys)
    got = got.cpu().double()
    assert torch.isfinite(got).all()
    worst = ((got - out).abs() / limit).max().item()
    assert worst <= 1, f"error {worst:.3g} times the bound"


SHAPES = [  # batch, heads, kv_heads, tokens, slots, dim, lead, masked, lengths
    (1, 1, 1, 1, 1, 16, 0, False, [1]),
    (3, 4, 4, 1, 130, 64, 0, False, [0, 1, 130]),
    (3, 8, 2, 1, 300, 128, 1, True, [299, 300, 17]),
    (2, 6, 2, 5, 257, 80, 1, False, [128, 256]),
    (4, 2, 1, 9, 33, 32, 0, True, [-4, 31, 32, 999]),
    (2, 5, 1, 33, 140, 48, 0, False, None),
    (2, 16, 2, 17, 200, 96, 1, True, [200, 64]),
    (1, 3, 3, 40, 700, 64, 0, False, [650]),
    (300, 1, 1, 1, 40, 64, 0, False, [i % 41 for i in range(300)]),
    # beyond what one cluster per segment takes: shares of tiles, segments across shares
    (3, 4, 2, 1, 4300, 64, 0, False, [4300, 0, 129]),
    (2, 2, 1, 3, 4300, 128, 1, True, [4000, 77]),
    (2, 9, 1, 1, 4200, 80, 0, False, [1, 4200]),
    # many rows per KV head
    (2, 4, 1, 16, 4300, 64, 1, False, [4300, 200]),
    (1, 3, 1, 40, 1000, 112, 0, True, [990]),
    (40, 4, 2, 9, 150, 64, 0, False, [3 * i for i in range(40)]),
    (2, 16, 1, 8, 700, 64, 0, True, [700, 300]),
]


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("storage", sorted(STORAGE))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_read_matches_the_oracle(shape, storage, dtype):
    batch, heads, kv_heads, tokens, slots, dim, lead, masked, lengths = shape
    query, pools, rows, mask = quantised_problem(7, storage, dtype, *shape)
    (k, ks), (v, vs) = pools
    got = quantized_pool_attention(
        query.cuda(), k.to(STORAGE[storage]).cuda(), v.to(STORAGE[storage]).cuda(), ks.cuda(), vs.cuda(),
        kv_lengths=None if lengths is None else torch.tensor(lengths).cuda(), use_dummy_token=bool(lead),
        key_mask=None if mask is None else mask.cuda(),
    )
    assert got.shape == (batch, tokens, heads, dim) and got.dtype == dtype
    check_attention(got, query, rows, lengths, lead, mask)


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("storage", sorted(STORAGE))
def test_scores_far_from_zero_and_far_apart(storage):
    gen = torch.Generator().manual_seed(5)
    for shift in (-300.0, 300.0):
        query = torch.randn(2, 4, 3, 64, generator=gen).bfloat16()
        query[..., 0] = 8.0
        x = torch.randn(2, 2, 400, 64, generator=gen)
        x[..., 0] = shift + torch.linspace(-90, 90, 400)[torch.randperm(400, generator=gen)]
        (k, ks), (v, vs) = oracle.quantise_rows(x, storage), oracle.quantise_rows(torch.randn(2, 2, 400, 64, generator=gen), storage)
        got = quantized_pool_attention(query.cuda(), k.to(STORAGE[storage]).cuda(), v.to(STORAGE[storage]).cuda(), ks.cuda(), vs.cuda(), softmax_scale=1.0)
        check_attention(got, query, [k * ks[..., None].double(), v * vs[..., None].double()], None, 0, None, None, 1.0)


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("tokens", [1, 3, 9])
@pytest.mark.parametrize("storage", sorted(STORAGE))
def test_codes_over_the_whole_range_of_their_type(storage, tokens):
    """Elements spread over many powers of two inside a row: subnormal codes, zeros and full ones side by side."""
    gen = torch.Generator().manual_seed(13)
    x = [torch.randn(2, 2, 150, 64, generator=gen) * torch.exp2(-12 * torch.rand(2, 2, 150, 64, generator=gen)) for _ in "kv"]
    (k, ks), (v, vs) = (oracle.quantise_rows(t, storage) for t in x)
    query = torch.randn(2, 4, tokens, 64, generator=gen).bfloat16()
    got = quantized_pool_attention(query.cuda(), k.to(STORAGE[storage]).cuda(), v.to(STORAGE[storage]).cuda(), ks.cuda(), vs.cuda(), softmax_scale=1.0)
    check_attention(got, query, [k * ks[..., None].double(), v * vs[..., None].double()], None, 0, None, None, 1.0)


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("tokens", [1, 9])
def test_value_scales_far_apart(tokens):
    """A row that attends to a token whose value is a millionth of the others' still gets it exactly enough."""
    gen = torch.Generator().manual_seed(14)
    k = torch.zeros(1, 1, 200, 64)
    k[0, 0, :, 0] = -40.0
    k[0, 0, 77, 0] = 40.0
    v = torch.randn(1, 1, 200, 64, generator=gen)
    v[0, 0, 77] *= 1e-6
    (kc, ks), (vc, vs) = (oracle.quantise_rows(t, "int8") for t in (k, v))
    query = torch.zeros(1, 2, tokens, 64).bfloat16()
    query[..., 0] = 8.0
    got = quantized_pool_attention(query.cuda(), kc.to(torch.int8).cuda(), vc.to(torch.int8).cuda(), ks.cuda(), vs.cuda())
    check_attention(got, query, [kc * ks[..., None].double(), vc * vs[..., None].double()], None, 0, None)


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("tokens", [1, 3, 9, 40])
@pytest.mark.parametrize("storage", sorted(STORAGE))
def test_value_scales_of_zero_and_next_to_it(storage, tokens):
    """An element stands for code * scale whatever the code is: nothing where the scale is zero or subnormal."""
    gen = torch.Generator().manual_seed(15)
    k, v = torch.randn(2, 1, 2, 150, 64, generator=gen).unbind(0)
    (kc, ks), (vc, vs) = (oracle.quantise_rows(t, storage) for t in (k, v))
    vs[0, 0, ::3], vs[0, 1, 1::3] = 0.0, 2.0**-130
    query = torch.randn(1, 2, tokens, 64, generator=gen).bfloat16()
    got = quantized_pool_attention(query.cuda(), kc.to(STORAGE[storage]).cuda(), vc.to(STORAGE[storage]).cuda(), ks.cuda(), vs.cuda())
    check_attention(got, query, [kc * ks[..., None].double(), vc * vs[..., None].double()], None, 0, None)


@pytest.mark.gpu
@on_gpu
def test_a_poisoned_row_shows_in_the_queries_that_see_it():
    pool = QuantKVPoolCache(2, 1, 2, 40, 64)
    x = torch.randn(2, 2, 20, 64).bfloat16()
    x[1, 0, 11, 9] = float("inf")
    pool.append(x.cuda(), torch.randn(2, 2, 20, 64).bfloat16().cuda())
    out = pool.read(torch.randn(2, 4, 1, 64).bfloat16().cuda(), 0)
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1, 0, :2]).all() and torch.isfinite(out[1, 0, 2:]).all()


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("storage", sorted(STORAGE))
def test_offsets_beyond_32_bits(storage):
    gen = torch.Generator().manual_seed(6)
    span = 2**32 + 4096  # bytes between two sequences, and elements: one byte each
    flat = torch.zeros(span + 2 * 40 * 64, dtype=torch.int8, device="cuda")
    view = lambda t: t.as_strided((2, 2, 40, 64), (span, 40 * 64, 64, 1)).view(STORAGE[storage])
    keys = view(flat)
    values = torch.zeros(2, 2, 40, 64, dtype=torch.int8, device="cuda").view(STORAGE[storage])
    ks, vs = torch.zeros(2, 2, 40, device="cuda"), torch.zeros(2, 2, 40, device="cuda")
    new = [torch.randn(2, 2, 40, 64, generator=gen).bfloat16() for _ in "kv"]
    quantized_pool_append(keys, values, ks, vs, torch.zeros(2, dtype=torch.int32, device="cuda"), *(x.cuda() for x in new))
    (k, k_scales), (v, v_scales) = (oracle.quantise_rows(x, storage) for x in new)
    assert torch.equal(keys.cpu().float(), k) and torch.equal(ks.cpu(), k_scales)
    assert torch.equal(dequantize_kv_rows(keys, ks, dtype=torch.float32).cpu(), k * k_scales[..., None])
    query = torch.randn(2, 2, 1, 64, generator=gen).bfloat16()
    got = quantized_pool_attention(query.cuda(), keys, values, ks, vs)
    check_attention(got, query, [k * k_scales[..., None].double(), v * v_scales[..., None].double()], None, 0, None)


@pytest.mark.gpu
@on_gpu
def test_empty_calls():
    pool = QuantKVPoolCache(2, 1, 2, 8, 64)
    empty = torch.zeros(2, 2, 0, 64, device="cuda")
    pool.append(empty, empty)
    assert pool.lengths.tolist() == [0, 0]
    assert pool.read(torch.zeros(2, 2, 0, 64, device="cuda"), 0).shape == (2, 0, 2, 64)
    assert not pool.read(torch.ones(2, 2, 3, 64, device="cuda"), 0).any()
    assert not pool.dequantize()[0].any()
    with pytest.raises(ValueError, match="no gradients"):
        pool.read(torch.ones(2, 2, 3, 64, device="cuda", requires_grad=True), 0)
    with pytest.raises(RuntimeError, match="aligned"):
        dequantize_kv_rows(pool.keys.as_strided((2, 2, 3, 16), (512, 256, 17, 1)), pool.key_scales[:, :, :3])
    with pytest.raises(ValueError, match="queries?' type|query's dtype"):
        from white_matter_b200 import draft_tree_attention, prepare_draft_tree

        x = torch.zeros(1, 2, 1, 64, device="cuda")
        tree = prepare_draft_tree(torch.tensor([-1], device="cuda"))
        draft_tree_attention(x, x.bfloat16(), x.bfloat16(), x, x, tree)


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("storage", sorted(STORAGE))
def test_a_captured_step_over_the_8_bit_pool_replays(storage):
    torch.manual_seed(8)
    batch, channels, kv_heads, heads, capacity, dim = 4, 2, 2, 4, 300, 64
    make = lambda: QuantKVPoolCache(batch, channels, kv_heads, capacity, dim, storage=storage, use_dummy_token=True)
    rows = lambda n: torch.randn(batch, channels * kv_heads, n, dim, device="cuda", dtype=torch.bfloat16)
    cache, eager = make(), make()
    first, dummy = (rows(200), rows(200)), (rows(1)[0, :, 0], rows(1)[0, :, 0])
    for c in (cache, eager):
        c.set_dummy(*dummy)
        c.append(*first, advance=False)
        c.lengths.copy_(torch.tensor([0, 3, 127, 200]))
    queries, new = torch.randn(2, batch, heads, 1, dim, device="cuda", dtype=torch.bfloat16), (rows(1), rows(1))

    def step_on(c):
        outs = [c.read(queries[layer], layer) for layer in range(channels)]
        c.append(*new)
        return torch.stack(outs)

    graph = DecodeStepGraph(lambda: step_on(cache), cache)
    for turn in range(4):
        queries.normal_()
        for x in new:
            x.normal_()
        replayed = graph().clone()
        assert torch.equal(replayed, step_on(eager)), f"turn {turn}"
        assert torch.equal(cache.lengths, eager.lengths)
    assert torch.equal(cache.keys.float(), eager.keys.float()) and torch.equal(cache.key_scales, eager.key_scales)
    keys, values = cache.dequantize(dtype=torch.float32)
    lengths = cache.lengths.cpu()
    out = cache.read(queries[1], 1)
    check_attention(out, queries[1].cpu(), [keys[:, 2:].cpu(), values[:, 2:].cpu()], lengths, 1, None)


@pytest.mark.gpu
@on_gpu
def test_two_streams_at_once_do_not_disturb_each_other():
    torch.manual_seed(9)
    pools, queries = [], []
    for _ in range(2):
        pool = QuantKVPoolCache(8, 1, 8, 2000, 64)
        pool.append(torch.randn(8, 8, 2000, 64, device="cuda"), torch.randn(8, 8, 2000, 64, device="cuda"))
        pools.append(pool)
        queries.append(torch.randn(8, 8, 1, 64, device="cuda", dtype=torch.bfloat16))
    alone = [p.read(q, 0) for p, q in zip(pools, queries)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                results[i].append(pools[i].read(queries[i], 0))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(r, alone[i]) for r in results[i])


@pytest.mark.gpu
@on_gpu
def test_nothing_that_requires_grad_is_taken():
    pool = QuantKVPoolCache(1, 1, 2, 16, 64)
    rows = torch.randn(1, 2, 3, 64, device="cuda").bfloat16()
    pool.append(rows, rows)
    query, scales = torch.randn(1, 2, 1, 64, device="cuda").bfloat16(), pool.key_scales.clone().requires_grad_()
    with pytest.raises(ValueError, match="no gradients"):
        quantized_pool_attention(query, pool.keys, pool.values, scales, pool.value_scales)
    with pytest.raises(ValueError, match="no gradients"):
        quantized_pool_append(pool.keys, pool.values, scales, pool.value_scales, pool.lengths, rows, rows)
    with pytest.raises(ValueError, match="no gradients"):
        dequantize_kv_rows(pool.keys, scales)
    with torch.no_grad():
        quantized_pool_attention(query, pool.keys, pool.values, scales, pool.value_scales)


@pytest.mark.gpu
@on_gpu
def test_a_captured_step_notices_replaced_scales():
    pool = QuantKVPoolCache(1, 1, 2, 16, 64)
    rows = torch.randn(1, 2, 3, 64, device="cuda").bfloat16()
    pool.append(rows, rows)
    query = torch.randn(1, 2, 1, 64, device="cuda").bfloat16()
    step = DecodeStepGraph(lambda: pool.read(query, 0), pool)
    step()
    pool.key_scales = pool.key_scales.clone()
    with pytest.raises(ValueError, match="capture the step again"):
        step()


# ------------------------------------------------------------------ GPU: values of zero, codes that are no number


@functools.lru_cache
def leading_key_rows(storage, slots, dim):
    """Codes and scales of the keys and values of the test below."""
    gen = torch.Generator().manual_seed(21)
    k, v = torch.zeros(1, 1, slots, dim), torch.zeros(1, 1, slots, dim)
    k[..., 0], k[..., 1] = -5.5, 5.5  # exact in both storages
    k[0, 0, 0, 0], k[0, 0, 0, 1] = 5.5, 0.0
    v[0, 0, 0] = torch.randn(dim, generator=gen)
    v[0, 0, 1::3] = 2.0**-98 * torch.randn(len(range(1, slots, 3)), dim, generator=gen).clamp(-2, 2)
    return tuple(oracle.quantise_rows(t, storage) for t in (k, v))


def expanded(codes, scales, storage, batch):
    """One sequence's rows as the pool of a whole batch, without copies: enough segments that a share holds a long run of keys."""
    codes, scales = codes.to(STORAGE[storage]).cuda(), scales.cuda()
    return codes.expand(batch, -1, -1, -1), scales.expand(batch, -1, -1)


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("dim", [64, 128, 48])
@pytest.mark.parametrize("tokens", [1, 9, 20, 40, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("storage", sorted(STORAGE))
def test_keys_with_values_of_zero_stay_in_the_sum(storage, dtype, tokens, dim):
    """One key leads 8 000 others by 11.2 (a weight of 2^-16.2 each, 0.11 together); the others' values are zeros, or so small that
    their scale times such a weight is no normal fp32 number."""
    batch, slots = (300, 8000) if dtype == torch.bfloat16 else (300, 2000)
    (kc, ks), (vc, vs) = leading_key_rows(storage, slots, dim)
    query = torch.zeros(1, 1, tokens, dim).to(dtype)
    query[..., 0], query[..., 1] = 1.0, -0.04
    (keys, key_scales), (values, value_scales) = expanded(kc, ks, storage, batch), expanded(vc, vs, storage, batch)
    got = quantized_pool_attention(query.cuda().expand(batch, -1, -1, -1), keys, values, key_scales, value_scales, softmax_scale=1.0)
    rows = [kc * ks[..., None].double(), vc * vs[..., None].double()]
    out, mass, reach = oracle.attention(query[:, :, :1], *rows, None, 0, None, None, 1.0)
    limit = oracle.bound(out, mass, reach, dtype, dim, slots)
    worst = ((got.cpu().double() - out).abs() / limit).max().item()
    assert worst <= 1, f"error {worst:.3g} times the bound"


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 128])
@pytest.mark.parametrize("batch, slots, tokens", [(1, 300, 1), (2, 300, 5), (2, 300, 20), (2, 4400, 1), (2, 4400, 3), (2, 4400, 17), (2, 4400, 40)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_e4m3_codes_that_are_no_number(dtype, batch, slots, tokens, dim):
    """A pool that was quantised elsewhere may hold the two NaN codes: in a visible key they reach everything of the queries that see
    it, in a visible value their element alone, and nothing else."""
    gen = torch.Generator().manual_seed(22)
    heads, kv_heads = 4, 2
    kc, vc = (torch.randn(batch, kv_heads, slots, dim, generator=gen).mul(64).to(torch.float8_e4m3fn).float() for _ in "kv")
    ks, vs = (torch.exp(0.3 * torch.randn(batch, kv_heads, slots, generator=gen)) / 64 for _ in "kv")
    query = torch.randn(batch, heads, tokens, dim, generator=gen).to(dtype)
    mask = torch.rand(batch, slots, generator=gen) < 0.7
    lengths = torch.tensor([slots - 3, slots // 2][:batch])
    seen = torch.tensor([[7, slots - 9], [3, slots // 2 - 1]])
    mask[torch.arange(2)[:batch, None], seen[:batch]] = True
    mask[:, 5] = False
    codes = [t.to(torch.float8_e4m3fn).view(torch.uint8) for t in (kc, vc)]
    for which in codes:  # not seen: masked, or behind the last token
        which[:, :, 5], which[:, :, int(lengths[0]) :] = 0x7F, 0xFF
        for b in range(batch):
            which[b, :, int(lengths[b]) :] = 0x7F
    places = [(batch - 1, 1, int(seen[batch - 1, 0]), 0, 0x7F), (batch - 1, 1, int(seen[batch - 1, 1]), dim - 1, 0xFF), (batch - 1, 1, int(seen[batch - 1, 0]), dim // 2 + 1, 0xFF)]
    clean = oracle.attention(query, kc * ks[..., None].double(), vc * vs[..., None].double(), lengths, 0, mask)
    for kind in (0, 1):
        spoilt = [c.clone() for c in codes]
        want = torch.zeros(batch, tokens, heads, dim, dtype=torch.bool)
        for b, h, slot, d, code in places[:1] if kind == 0 else places:
            spoilt[kind][b, h, slot, d] = code
            want[b, :, 2 * h : 2 * h + 2, slice(None) if kind == 0 else d] = True
        got = quantized_pool_attention(
            query.cuda(), *(s.view(torch.float8_e4m3fn).cuda() for s in spoilt), ks.cuda(), vs.cuda(), kv_lengths=lengths.cuda(), key_mask=mask.cuda(),
        ).cpu()
        assert torch.equal(torch.isnan(got), want), kind
        out, mass, reach = clean
        limit = oracle.bound(out, mass, reach, dtype, dim, slots)
        # the element of the spoilt value counts elsewhere as the number it replaces: only columns without one are compared
        worst = ((got.double() - out).abs() / limit)[~want].max().item()
        assert worst <= 1, f"error {worst:.3g} times the bound"
    # without a mask, every slot up to the last in sight
    got = quantized_pool_attention(query.cuda(), *(s.view(torch.float8_e4m3fn).cuda() for s in spoilt), ks.cuda(), vs.cuda(), kv_lengths=torch.tensor([5] * batch).cuda())
    want = torch.zeros(batch, tokens, heads, dim, dtype=torch.bool)
    if batch == 2:
        want[1, :, 2:4, 0] = want[1, :, 2:4, dim // 2 + 1] = True
    assert torch.equal(torch.isnan(got.cpu()), want)


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("kind", ["plain", "int8"])
def test_lengths_stop_at_the_first_index_outside_the_new_rows(kind):
    """A padded branch: slots that the commit skipped must not come into sight."""
    make = lambda: KVPoolCache(5, 1, 2, 12, 64) if kind == "plain" else QuantKVPoolCache(5, 1, 2, 12, 64)
    rows = torch.randn(5, 2, 4, 64, device="cuda").bfloat16()
    index = torch.tensor([[0, 2, -1, -1], [3, 4, 0, 1], [-1, -1, -1, -1], [0, 1, 2, 3], [2, 2, 1, 9]], device="cuda")
    for counts, want in ((None, [2, 1, 0, 4, 3]), ([1, 4, 2, 3, -7], [1, 1, 0, 3, 0])):
        for index_dtype in (torch.int64, torch.int32):
            pool = make()
            start = torch.tensor([0, 3, 5, 10, 12], dtype=torch.int32)
            pool.lengths.copy_(start)
            pool.append(rows, rows, index=index.to(index_dtype), counts=None if counts is None else torch.tensor(counts, device="cuda"))
            assert pool.lengths.tolist() == [min(12, int(s) + n) for s, n in zip(start, want)]
    pool = make()
    pool.append(rows[:, :, :0], rows[:, :, :0], index=index)
    assert not pool.lengths.any()
    pool.append(rows, rows, index=index[:, :0])
    assert not pool.lengths.any()


@pytest.mark.gpu
@on_gpu
def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as forward_ad

    pool = QuantKVPoolCache(1, 1, 2, 16, 64)
    rows = torch.randn(1, 2, 3, 64, device="cuda").bfloat16()
    pool.append(rows, rows)
    query = torch.randn(1, 2, 1, 64, device="cuda").bfloat16()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(query, torch.ones_like(query))
        for mode in (torch.no_grad, torch.enable_grad):
            with mode(), pytest.raises(ValueError, match="derivatives"):
                pool.read(dual, 0)
        dual_rows = forward_ad.make_dual(rows, torch.ones_like(rows))
        with pytest.raises(ValueError, match="derivatives"):
            pool.append(dual_rows, rows)
        with pytest.raises(ValueError, match="derivatives"):
            dequantize_kv_rows(pool.keys, forward_ad.make_dual(pool.key_scales, torch.ones_like(pool.key_scales)))
        pool.read(query, 0)  # nothing in it has a tangent


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("rows", [1, 31, 32, 33, 100])
def test_long_branches_and_strided_lengths_advance_alike(rows):
    gen = torch.Generator().manual_seed(rows)
    batch, capacity = 70, 90
    index = torch.randint(0, rows + 1, (batch, rows), generator=gen)  # `rows` is the first number outside
    index[:10] = index[:10].clamp(max=rows - 1)
    counts = torch.randint(-2, rows + 3, (batch,), generator=gen)
    new = torch.randn(batch, 1, rows, 64, device="cuda").bfloat16()
    for dtype in (torch.int32, torch.int64):
        pool = QuantKVPoolCache(batch, 1, 1, capacity, 64)
        start = torch.randint(0, capacity, (batch,), generator=gen)
        pool.lengths = torch.stack((start, start), 1).to(dtype).cuda()[:, 0]  # stride 2
        pool.append(new, new, index=index.cuda(), counts=counts.cuda())
        want = []
        for b in range(batch):
            n = 0
            while n < min(rows, int(counts[b])) and index[b, n] < rows:
                n += 1
            want.append(min(capacity, int(start[b]) + n))
        assert pool.lengths.tolist() == want


# ------------------------------------------------------------------ GPU: masks over long sequences


def long_masked_problem(seed, storage, dtype, batch, heads, kv_heads, tokens, slots, dim, lead, lengths, blank):
    """A problem whose long sequences keep three slots of five, in runs that end inside tiles, while sequence `blank` (a short one,
    or none) sees nothing; every slot that is not seen is poisoned."""
    query, pools, rows, _ = quantised_problem(seed, storage, dtype, batch, heads, kv_heads, tokens, slots, dim, lead, False, lengths)
    gen = torch.Generator().manual_seed(seed + 2)
    mask = torch.rand(batch, slots, generator=gen) < 0.6
    mask[:, 200:330] = False  # a whole tile that nothing is left of
    mask[:, 1000:1300] = True  # and two that keep everything
    if blank is not None:
        mask[blank] = False
    for codes, scales in pools:
        for b in range(batch):
            scales[b][:, ~mask[b]] = float("nan")
            codes[b][:, ~mask[b]] = 100.0 if storage == "int8" else float("nan")
    return query, pools, rows, mask


LONG_MASKED = [  # batch, heads, kv_heads, tokens, slots, dim, lead, lengths, blank sequence
    (3, 2, 1, 3, 4300, 128, 1, [4299, 4100, 77], 2),  # up to 16 rows per KV head, shares
    (2, 4, 2, 1, 4300, 64, 0, [4300, 50], 1),
    (2, 2, 1, 7, 4200, 80, 0, [4150, 30], 1),
    (1, 3, 1, 2, 1900, 112, 0, [1890], None),  # a cluster per segment
    (2, 4, 2, 5, 1800, 96, 1, [1799, 20], 1),
    (3, 8, 1, 9, 4300, 64, 0, [4300, 4000, 60], 2),  # more rows: 32, 64 and 128 per block
    (2, 2, 1, 16, 4300, 128, 1, [4200, 40], 1),
    (1, 3, 1, 40, 1000, 112, 0, [990], None),
    (2, 4, 1, 15, 2100, 48, 1, [2000, 9], 1),
]


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("storage", sorted(STORAGE))
@pytest.mark.parametrize("shape", LONG_MASKED, ids=str)
def test_masks_over_long_sequences(shape, storage, dtype):
    batch, heads, kv_heads, tokens, slots, dim, lead, lengths, blank = shape
    query, pools, rows, mask = long_masked_problem(31, storage, dtype, *shape)
    (k, ks), (v, vs) = pools
    got = quantized_pool_attention(
        query.cuda(), k.to(STORAGE[storage]).cuda(), v.to(STORAGE[storage]).cuda(), ks.cuda(), vs.cuda(), kv_lengths=torch.tensor(lengths).cuda(),
        use_dummy_token=bool(lead), key_mask=mask.cuda(),
    )
    assert got[0].abs().amax(-1).min() > 0 and (blank is None or not got[blank].any())
    check_attention(got, query, rows, lengths, lead, mask)


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("tokens", [1, 3, 20, 100])
@pytest.mark.parametrize("storage", sorted(STORAGE))
def test_a_call_repeats_itself_bit_for_bit(storage, tokens):
    """The shares, and so the order of every sum, follow from the sizes and lengths alone."""
    torch.manual_seed(23)
    pool = QuantKVPoolCache(9, 1, 3, 3000, 64, storage=storage)
    for _ in range(3):
        pool.append(torch.randn(9, 3, 1000, 64, device="cuda"), torch.randn(9, 3, 1000, 64, device="cuda"))
    pool.lengths.copy_(torch.arange(9) * 333 + 1)
    for dtype in (torch.bfloat16, torch.float32):
        query = torch.randn(9, 6, tokens, 64, device="cuda").to(dtype)
        first = pool.read(query, 0)
        for _ in range(5):
            assert torch.equal(pool.read(query, 0), first)
