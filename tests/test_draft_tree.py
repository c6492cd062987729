"""Trees of drafted tokens: tables, attention over plain and 8-bit pools, and a drafting loop from draft to commit."""

import pytest
import torch

from oracle import serving_oracle as oracle
from test_quant_pool import LONG_MASKED, check_attention, long_masked_problem, on_gpu, quantised_problem
from white_matter_b200 import DraftTree, KVPoolCache, QuantKVPoolCache, draft_tree_attention, prepare_draft_tree
from white_matter_b200.quant_pool import STORAGE


def random_parents(gen, batch, tokens, broken=False):
    """Parents in any order: node numbers are shuffled, so a parent may come after its child."""
    rows = []
    for _ in range(batch):
        up = [int(torch.randint(-1, i, (1,), generator=gen)) if i else -1 for i in range(tokens)]
        if broken:
            for i in range(tokens):
                draw = float(torch.rand(1, generator=gen))
                if draw < 0.1:
                    up[i] = [-2, -(2**31), tokens, 2**31 - 1, i, (i + 1) % tokens][int(torch.randint(0, 6, (1,), generator=gen))]
        order = torch.randperm(tokens, generator=gen).tolist()
        row = [0] * tokens
        for i in range(tokens):
            row[order[i]] = order[up[i]] if 0 <= up[i] < tokens else up[i]
        rows.append(row)
    return torch.tensor(rows)


def test_refusals():
    with pytest.raises(ValueError, match="CUDA"):
        prepare_draft_tree(torch.zeros(1, 3, dtype=torch.int32))
    with pytest.raises(ValueError, match="integer"):
        prepare_draft_tree(torch.zeros(1, 3))
    with pytest.raises(ValueError, match="include_self must be boolean"):
        prepare_draft_tree(torch.zeros(3, dtype=torch.int32), include_self=1)
    q, kv = torch.zeros(2, 4, 3, 64), torch.zeros(2, 2, 9, 64)
    draft, tree = torch.zeros(2, 2, 3, 64), DraftTree(torch.zeros(2, 3, 1, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int32))
    with pytest.raises(ValueError, match=r"drafted K/V must be \(B,HKV,T,D\)"):
        draft_tree_attention(q, kv, kv, kv, kv, tree)
    with pytest.raises(ValueError, match="query's dtype"):
        draft_tree_attention(q, kv, kv, draft.double(), draft.double(), tree)
    with pytest.raises(ValueError, match="prepared for these"):
        draft_tree_attention(q, kv, kv, draft, draft, DraftTree(tree.ancestors[:, :2], tree.depths[:, :2]))
    with pytest.raises(ValueError, match="int32"):
        draft_tree_attention(q, kv, kv, draft, draft, DraftTree(tree.ancestors.long(), tree.depths))
    with pytest.raises(ValueError, match="at most 512"):
        big = torch.zeros(1, 1, 513, 64)
        draft_tree_attention(big, big, big, big, big, tree)
    with pytest.raises(ValueError, match="requires? CUDA"):
        draft_tree_attention(q, kv, kv, draft, draft, tree)


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("include_self", [False, True])
@pytest.mark.parametrize("tokens", [1, 2, 5, 31, 32, 33, 64, 200, 512])
def test_tables_follow_the_chains_of_parents(tokens, include_self):
    gen = torch.Generator().manual_seed(tokens)
    for broken in (False, True):
        parents = random_parents(gen, 3, tokens, broken)
        if tokens > 2:
            parents[2] = torch.arange(-1, tokens - 1)  # one long chain
        visible, depths = oracle.tree_tables(parents, include_self)
        for given in (parents, parents.int()):
            tree = prepare_draft_tree(given.cuda(), include_self=include_self)
            assert torch.equal(tree.depths.cpu(), depths)
            assert torch.equal(tree.ancestors.cpu(), oracle.pack_bits(visible))
    one = prepare_draft_tree(parents[0].cuda(), include_self=include_self)
    assert one.depths.shape == (1, tokens) and torch.equal(one.ancestors.cpu(), oracle.pack_bits(visible)[:1])


def problem(seed, storage, dtype, batch, heads, kv_heads, tokens, slots, dim, lead, masked, lengths, shared=False):
    if storage in STORAGE:
        query, pools, rows, mask = quantised_problem(seed, storage, dtype, batch, heads, kv_heads, tokens, slots, dim, lead, masked, lengths)
    else:
        query, pools, rows, mask = quantised_problem(seed, "int8", dtype, batch, heads, kv_heads, tokens, slots, dim, lead, masked, lengths)
        rows = [r.to(dtype) for r in rows]
        pools = [(torch.where(torch.isnan(s)[..., None], torch.full_like(r, float("nan")), r), None) for r, (_, s) in zip(rows, pools)]
    gen = torch.Generator().manual_seed(seed + 1)
    parents = random_parents(gen, 1 if shared else batch, tokens)
    if tokens > 3:
        parents[:, 1] = -2  # a padding node, and whatever hangs on it
    draft = [torch.randn(batch, kv_heads, tokens, dim, generator=gen).to(dtype) for _ in "kv"]
    return query, pools, rows, mask, parents, draft


SHAPES = [  # batch, heads, kv_heads, tokens, slots, dim, lead, masked, lengths
    (1, 1, 1, 1, 1, 16, 0, False, [0]),
    (2, 4, 4, 8, 130, 64, 0, False, [0, 130]),
    (3, 8, 2, 4, 300, 128, 1, True, [299, 300, 17]),
    (2, 6, 2, 21, 257, 80, 1, False, [128, 256]),
    (3, 2, 1, 64, 33, 32, 0, True, [-4, 31, 999]),
    (2, 6, 1, 33, 140, 48, 0, False, None),
    (1, 2, 2, 130, 200, 96, 1, False, [70]),
    (1, 2, 1, 300, 10, 64, 0, False, [0]),
    (2, 4, 2, 6, 4300, 64, 1, True, [4300, 40]),
    (2, 4, 1, 12, 4300, 128, 0, False, [4300, 130]),
    (30, 2, 1, 20, 140, 64, 1, False, [5 * i for i in range(30)]),
    (2, 16, 2, 20, 300, 64, 0, True, [300, 150]),  # 160 rows per KV head: two blocks of 128
    (1, 12, 1, 10, 260, 128, 1, False, [200]),
]


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("include_self", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("storage", ["plain", *sorted(STORAGE)])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention_matches_the_oracle(shape, storage, dtype, include_self):
    batch, heads, kv_heads, tokens, slots, dim, lead, masked, lengths = shape
    shared = include_self and batch > 1
    query, pools, rows, mask, parents, draft = problem(11, storage, dtype, *shape, shared=shared)
    visible, depths = oracle.tree_tables(parents, include_self)
    clean = [d.clone() for d in draft]
    query = query.clone()
    for b in range(batch):  # padding nodes may hold anything
        dead = depths[0 if shared else b] < 0
        query[b][:, dead] = float("nan")
        for d in draft:
            d[b][:, dead] = float("nan")
    (k, ks), (v, vs) = pools
    kind = STORAGE.get(storage, dtype)
    got = draft_tree_attention(
        query.cuda(), k.to(kind).cuda(), v.to(kind).cuda(), *(d.cuda() for d in draft), prepare_draft_tree(parents.cuda(), include_self=include_self),
        kv_lengths=None if lengths is None else torch.tensor(lengths, dtype=torch.int32).cuda(), use_dummy_token=bool(lead),
        key_mask=None if mask is None else mask.cuda(), key_scales=None if ks is None else ks.cuda(), value_scales=None if vs is None else vs.cuda(),
    )
    assert got.shape == (batch, tokens, heads, dim) and got.dtype == dtype
    check_attention(got, torch.nan_to_num(query), rows, lengths, lead, mask, (*clean, visible, depths))


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("tokens", [3, 30])
@pytest.mark.parametrize("dim, dtype", [(8, torch.bfloat16), (24, torch.bfloat16), (40, torch.bfloat16), (72, torch.bfloat16), (120, torch.bfloat16), (4, torch.float32), (20, torch.float32), (100, torch.float32)])
def test_head_sizes_that_fill_no_tile(dim, dtype, tokens):
    query, pools, rows, mask, parents, draft = problem(5, "plain", dtype, 2, 4, 2, tokens, 150, dim, 1, True, [149, 40])
    visible, depths = oracle.tree_tables(parents, True)
    got = draft_tree_attention(
        query.cuda(), pools[0][0].cuda(), pools[1][0].cuda(), *(d.cuda() for d in draft), prepare_draft_tree(parents.cuda(), include_self=True),
        kv_lengths=torch.tensor([149, 40]).cuda(), use_dummy_token=True, key_mask=mask.cuda(),
    )
    check_attention(got, query, rows, [149, 40], 1, mask, (*draft, visible, depths))


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("tokens", [2, 24])
def test_layouts_other_than_contiguous(tokens):
    """Pools as (B,N,HKV,D) views with gaps between the rows, queries and drafts off their 16 bytes or with strided elements, a mask
    out of a wider one: the same result as from contiguous copies."""
    torch.manual_seed(6)
    wide = torch.randn(2, 90, 3, 96, device="cuda").bfloat16()
    key, value = wide[:, :, :2, :64].transpose(1, 2), wide[:, :, 1:, 16:80].transpose(1, 2)
    query = torch.randn(2, 4, tokens, 130, device="cuda").bfloat16()[..., 1:129:2]
    draft = [torch.randn(2 * 2 * tokens * 64 + 3, device="cuda").bfloat16()[3:].view(2, 2, tokens, 64) for _ in "kv"]
    mask = (torch.rand(2, 180, device="cuda") < 0.8)[:, ::2]
    tree = prepare_draft_tree(torch.arange(-1, tokens - 1, device="cuda"))
    lengths = torch.tensor([[70, 0], [90, 0]], device="cuda")[:, 0]
    common = dict(kv_lengths=lengths, key_mask=mask)
    got = draft_tree_attention(query, key, value, *draft, tree, **common)
    plain = [t.clone(memory_format=torch.contiguous_format) for t in (query, key, value, *draft)]
    assert torch.equal(got, draft_tree_attention(*plain, tree, kv_lengths=lengths.clone(), key_mask=mask.clone(memory_format=torch.contiguous_format)))
    check_attention(got, plain[0].cpu(), [plain[1].cpu(), plain[2].cpu()], lengths.cpu(), 0, mask.cpu(), (plain[3].cpu(), plain[4].cpu(), *oracle.tree_tables(torch.arange(-1, tokens - 1)[None], False)))


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("tokens", [4, 20])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_poisoned_drafted_token_reaches_its_descendants_alone(dtype, tokens):
    gen = torch.Generator().manual_seed(2)
    parents = random_parents(gen, 2, tokens)
    visible, _ = oracle.tree_tables(parents, False)
    victim = int(visible[0].sum(0).argmax())  # the node most others descend from
    query, pool = torch.randn(2, 4, tokens, 64, generator=gen).to(dtype), torch.randn(2, 2, 50, 64, generator=gen).to(dtype)
    for which, poison in ((0, float("nan")), (1, float("inf")), (1, float("nan"))):
        draft = [torch.randn(2, 2, tokens, 64, generator=gen).to(dtype) for _ in "kv"]
        draft[which][0, 1, victim] = poison
        out = draft_tree_attention(query.cuda(), pool.cuda(), pool.cuda(), *(d.cuda() for d in draft), prepare_draft_tree(parents.cuda()))
        bad = ~torch.isfinite(out.cpu()).all(-1)
        want = torch.zeros(2, tokens, 4, dtype=torch.bool)
        want[0, :, 2:] = visible[0, :, victim, None]
        assert torch.equal(bad, want)


@pytest.mark.gpu
@on_gpu
def test_a_chain_equals_a_cached_prefix():
    """A draft that does not branch is the strict prefix: the same result as the existing operator over committed rows."""
    from white_matter_b200 import strict_causal_attention

    torch.manual_seed(3)
    tokens, past = 12, 70
    k, v = (torch.randn(2, 2, past + tokens, 64, device="cuda").bfloat16() for _ in "kv")
    q = torch.randn(2, 4, tokens, 64, device="cuda").bfloat16()
    lengths = torch.full((2,), past, dtype=torch.int32, device="cuda")
    expected = strict_causal_attention(q, k, v, query_start=past, kv_lengths=lengths + tokens)
    tree = prepare_draft_tree(torch.arange(-1, tokens - 1, device="cuda"))
    got = draft_tree_attention(q, k[:, :, :past], v[:, :, :past], k[:, :, past:], v[:, :, past:], tree, kv_lengths=lengths)
    # both within the bf16 bound of the exact result: weights and result rounded on either side
    assert (got.double() - expected.double()).abs().max() <= 2 * (2.0**-8 + 2 * 2.0**-8) * v.abs().max()


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("storage", ["plain", *sorted(STORAGE)])
def test_draft_verify_commit_loop_replayed_from_a_graph(storage):
    """Several turns of drafting: tables, attention of the drafted tokens over two channels, commit of an accepted branch, one read --
    captured once, replayed with new trees, queries and branches, and checked against the oracle over the dequantised pool."""
    gen = torch.Generator().manual_seed(12)
    batch, channels, kv_heads, heads, dim, tokens, capacity = 3, 2, 2, 4, 64, 10, 160
    make = lambda: (
        KVPoolCache(batch, channels, kv_heads, capacity, dim, use_dummy_token=True)
        if storage == "plain"
        else QuantKVPoolCache(batch, channels, kv_heads, capacity, dim, storage=storage, use_dummy_token=True)
    )
    cache = make()
    rows = lambda n: torch.randn(batch, channels * kv_heads, n, dim, generator=gen).bfloat16()
    cache.set_dummy(rows(1)[0, :, 0].cuda(), rows(1)[0, :, 0].cuda())
    cache.append(rows(90).cuda(), rows(90).cuda(), advance=False)
    cache.lengths.copy_(torch.tensor([0, 33, 90]))
    parents = torch.zeros(batch, tokens, dtype=torch.int32, device="cuda")
    queries = torch.zeros(channels, batch, heads, tokens, dim, dtype=torch.bfloat16, device="cuda")
    draft_k, draft_v = (torch.zeros(batch, channels * kv_heads, tokens, dim, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    branch, count = torch.zeros(batch, tokens, dtype=torch.int32, device="cuda"), torch.zeros(batch, dtype=torch.int32, device="cuda")

    def step():
        tree = prepare_draft_tree(parents)
        outs = []
        for c in range(channels):
            own = slice(c * kv_heads, (c + 1) * kv_heads)
            outs.append(cache.read_tree(queries[c], c, draft_k[:, own], draft_v[:, own], tree))
        cache.append(draft_k, draft_v, index=branch, counts=count)
        outs.append(cache.read(queries[0, :, :, :1], 0))
        return torch.cat([o.flatten() for o in outs])

    stream = torch.cuda.Stream()
    before = cache.lengths.clone()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    cache.lengths.copy_(before)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = step()
    cache.lengths.copy_(before)
    for turn in range(3):
        tree = random_parents(gen, batch, tokens)
        visible, depths = oracle.tree_tables(tree, False)
        parents.copy_(tree)
        queries.copy_(torch.randn(queries.shape, generator=gen))
        new_k, new_v = rows(tokens), rows(tokens)
        draft_k.copy_(new_k), draft_v.copy_(new_v)
        leaf = [int(depths[b].argmax()) for b in range(batch)]
        for b in range(batch):
            chain = sorted(visible[b, leaf[b]].nonzero()[:, 0].tolist(), key=lambda n: int(depths[b, n])) + [leaf[b]]
            branch[b, : len(chain)] = torch.tensor(chain, dtype=torch.int32)
            count[b] = len(chain) if b else 0  # nothing accepted in the first sequence
        lengths = cache.lengths.cpu().clone()
        plain = (cache.keys, cache.values) if storage == "plain" else cache.dequantize(dtype=torch.float32)
        pool_rows = [p.float().cpu() for p in plain]
        graph.replay()
        got = result.clone()
        size = batch * tokens * heads * dim
        for c in range(channels):
            own = slice(c * kv_heads, (c + 1) * kv_heads)
            check_attention(
                got[c * size : (c + 1) * size].view(batch, tokens, heads, dim), queries[c].cpu(), [r[:, own] for r in pool_rows], lengths, 1, None,
                (new_k[:, own], new_v[:, own], visible, depths),
            )
        assert torch.equal(cache.lengths.cpu(), lengths + count.cpu())
        plain = (cache.keys, cache.values) if storage == "plain" else cache.dequantize(dtype=torch.float32)
        after = [p.float().cpu() for p in plain]
        for new, old, now in zip((new_k, new_v), pool_rows, after):
            for b in range(batch):
                at, n = 1 + int(lengths[b]), int(count[b])
                assert torch.equal(now[b, :, :at], old[b, :, :at])
                picked = new[b][:, branch[b, :n].cpu().long()]
                if storage == "plain":
                    assert torch.equal(now[b, :, at : at + n], picked.float())
                elif n:
                    codes, scales = oracle.quantise_rows(picked, storage)
                    assert torch.equal(now[b, :, at : at + n], codes * scales[..., None])
        check_attention(got[channels * size :].view(batch, 1, heads, dim), queries[0, :, :, :1].cpu(), [r[:, :kv_heads] for r in after], cache.lengths.cpu(), 1, None)


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("storage", sorted(STORAGE))
def test_an_infinite_drafted_value_takes_no_bits_from_the_rows_that_do_not_see_it(storage):
    """Up to 16 rows over an 8-bit pool take the weights in two bf16 parts, 16 bits: also next to a drafted value that is infinite and
    that they do not see.  Values of alternating sign cancel, so the weights' error shows beside a small result: two parts leave
    2^-16 of the mass, one part 2^-9 (both twice, for the sum that divides them)."""
    tokens, dim = 12, 64
    gen = torch.Generator().manual_seed(44)
    query = torch.randn(1, 1, tokens, dim, generator=gen).bfloat16()
    (kc, ks), (vc, vs) = (oracle.quantise_rows(torch.randn(1, 1, 4, dim, generator=gen), storage) for _ in "kv")
    draft = [torch.randn(1, 1, tokens, dim, generator=gen).bfloat16() for _ in "kv"]
    draft[1] = torch.where(torch.arange(tokens)[:, None] % 2 == 0, 1.0, -1.0).expand(1, 1, tokens, dim).bfloat16().clone()
    parents = torch.cat((torch.arange(-1, tokens - 2), torch.tensor([-1])))[None]  # a chain, and one node beside it
    visible, depths = oracle.tree_tables(parents, True)
    out, mass, reach = oracle.attention(query, kc * ks[..., None].double(), vc * vs[..., None].double(), [0], 0, None, (*draft, visible, depths))
    draft[1][0, 0, tokens - 1] = float("inf")
    got = draft_tree_attention(
        query.cuda(), kc.to(STORAGE[storage]).cuda(), vc.to(STORAGE[storage]).cuda(), *(d.cuda() for d in draft),
        prepare_draft_tree(parents.cuda(), include_self=True), kv_lengths=torch.tensor([0]).cuda(), key_scales=ks.cuda(), value_scales=vs.cuda(),
    ).cpu().double()
    assert torch.isinf(got[0, -1]).all()
    # rounding of the result, weights in two parts, scores and exponentials in fp32 as in oracle.bound
    limit = 1.01 * (2.0**-8 * out.abs() + (2 * 2.0**-16 + 2.1 * ((dim + 8) * 2.0**-24 * reach + 2.0**-21)) * mass)
    worst = ((got - out).abs() / limit)[0, :-1].max().item()
    assert worst <= 1, f"error {worst:.3g} times the bound"


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("storage", ["plain", *sorted(STORAGE)])
@pytest.mark.parametrize("shape", LONG_MASKED, ids=str)
def test_masks_over_long_sequences_of_a_tree(shape, storage, dtype):
    batch, heads, kv_heads, tokens, slots, dim, lead, lengths, blank = shape
    query, pools, rows, mask = long_masked_problem(41, "int8" if storage == "plain" else storage, dtype, *shape)
    if storage == "plain":
        rows = [r.to(dtype) for r in rows]
        pools = [(torch.where(torch.isnan(s)[..., None], torch.full_like(r, float("nan")), r), None) for r, (_, s) in zip(rows, pools)]
    gen = torch.Generator().manual_seed(42)
    parents = random_parents(gen, batch, tokens)
    draft = [torch.randn(batch, kv_heads, tokens, dim, generator=gen).to(dtype) for _ in "kv"]
    (k, ks), (v, vs) = pools
    kind = STORAGE.get(storage, dtype)
    got = draft_tree_attention(
        query.cuda(), k.to(kind).cuda(), v.to(kind).cuda(), *(d.cuda() for d in draft), prepare_draft_tree(parents.cuda()), kv_lengths=torch.tensor(lengths).cuda(),
        use_dummy_token=bool(lead), key_mask=mask.cuda(), key_scales=None if ks is None else ks.cuda(), value_scales=None if vs is None else vs.cuda(),
    )
    assert got[0].abs().amax(-1).min() > 0
    check_attention(got, query, rows, lengths, lead, mask, (*draft, *oracle.tree_tables(parents, False)))


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("tokens", [3, 30])
@pytest.mark.parametrize("dim, dtype", [(8, torch.bfloat16), (40, torch.bfloat16), (72, torch.bfloat16), (120, torch.bfloat16), (4, torch.float32), (20, torch.float32), (100, torch.float32)])
def test_head_sizes_that_fill_no_tile_over_long_sequences(dim, dtype, tokens):
    """The same head sizes where a sequence has many steps, with and without a mask."""
    batch, heads, kv_heads, slots, lengths = 2, 4, 2, 1100, [1090, 700]
    gen = torch.Generator().manual_seed(43)
    query, k, v = (torch.randn(batch, n, t, dim, generator=gen).to(dtype) for n, t in ((heads, tokens), (kv_heads, slots), (kv_heads, slots)))
    draft = [torch.randn(batch, kv_heads, tokens, dim, generator=gen).to(dtype) for _ in "kv"]
    parents = random_parents(gen, batch, tokens)
    for mask in (None, torch.rand(batch, slots, generator=gen) < 0.6):
        got = draft_tree_attention(
            query.cuda(), k.cuda(), v.cuda(), *(d.cuda() for d in draft), prepare_draft_tree(parents.cuda()), kv_lengths=torch.tensor(lengths).cuda(),
            key_mask=None if mask is None else mask.cuda(),
        )
        check_attention(got, query, [k, v], lengths, 0, mask, (*draft, *oracle.tree_tables(parents, False)))


@pytest.mark.gpu
@on_gpu
@pytest.mark.parametrize("slots", [200, 4400])
@pytest.mark.parametrize("tokens", [4, 12, 30])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_e4m3_codes_that_are_no_number_reach_the_nodes_and_no_padding(dtype, tokens, slots):
    gen = torch.Generator().manual_seed(45)
    batch, heads, kv_heads, dim = 2, 2, 1, 64
    codes = [torch.randn(batch, kv_heads, slots, dim, generator=gen).mul(64).to(torch.float8_e4m3fn).view(torch.uint8) for _ in "kv"]
    scales = torch.full((batch, kv_heads, slots), 1 / 64)
    query, *draft = (torch.randn(batch, n, tokens, dim, generator=gen).to(dtype) for n in (heads, kv_heads, kv_heads))
    parents = random_parents(gen, batch, tokens)
    parents[:, 2] = -2
    live = oracle.tree_tables(parents, True)[1] >= 0
    for kind in (0, 1):
        spoilt = [c.clone() for c in codes]
        spoilt[kind][1, 0, slots - 7, 9] = 0xFF
        got = draft_tree_attention(
            query.cuda(), *(s.view(torch.float8_e4m3fn).cuda() for s in spoilt), *(d.cuda() for d in draft), prepare_draft_tree(parents.cuda(), include_self=True),
            key_scales=scales.cuda(), value_scales=scales.cuda(),
        ).cpu()
        want = torch.zeros(batch, tokens, heads, dim, dtype=torch.bool)
        want[1, :, :, slice(None) if kind == 0 else 9] = live[1, :, None] if kind == 1 else live[1, :, None, None]
        assert torch.equal(torch.isnan(got), want)
        assert not got[~live].any()
