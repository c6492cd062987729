"""Cases of the operators around an 8-bit KV pool and drafted tokens: what a serving step calls, in plain torch and as kernels.

Five operators, told apart by ``case["op"]``:

* ``commit``   new rows are quantised (int8 or e4m3, one scale per row) as they are written into the pool
* ``readback`` the rows that an 8-bit pool stands for
* ``read``     attention of queries behind the committed tokens over an 8-bit pool
* ``tables``   ancestor bits and depths of a tree of drafted tokens
* ``tree``     attention of drafted tokens: the committed slots of a pool (fp32, bf16, 8-bit) and their own ancestors

With ``own`` false ``run`` computes them from elementary torch operations in 32 bits, with ``own`` true through the
package's public functions.  Codes come back as the pool stores them (int8 whole numbers, e4m3 values) next to their scales.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
INT8_TOP, E4M3_TOP = 127.0, 448.0
SMALLEST = 2.0**-100  # rows whose largest magnitude is below this are held as zeros


def listed():
    return [
        # one decode step of 64 sequences: one new row per sequence and pool head (8 channels of 16 heads)
        dict(name="commit_step_int8", op="commit", storage="int8", dtype="bf16", batch=64, heads=128, rows=1, dim=64, capacity=256, lead=0, branch=False),
        # the accepted branch of 33 drafted tokens, gathered out of the draft's rows, behind a dummy slot
        dict(name="commit_branch_e4m3", op="commit", storage="e4m3", dtype="fp32", batch=16, heads=32, rows=33, dim=128, capacity=200, lead=1, branch=True),
        # a prompt of 2048 tokens enters the pool of the 8-channel model
        dict(name="commit_prompt_e4m3", op="commit", storage="e4m3", dtype="bf16", batch=8, heads=128, rows=2048, dim=64, capacity=2300, lead=0, branch=False),
        # a short channel is read back for inspection, and a whole pool is turned back into bf16
        dict(name="readback_channel_int8", op="readback", storage="int8", dtype="fp32", batch=4, heads=16, capacity=300, dim=64, lead=1),
        dict(name="readback_pool_e4m3", op="readback", storage="e4m3", dtype="bf16", batch=16, heads=128, capacity=2049, dim=64, lead=0),
        # decode: one sequence with a short history; the 64-sequence pool with ragged lengths; grouped heads, new tokens, mask
        dict(name="read_one_int8", op="read", storage="int8", dtype="bf16", batch=1, heads=16, kv_heads=16, dim=64, tokens=1, capacity=512, lead=0, masked=False),
        dict(name="read_pool_int8", op="read", storage="int8", dtype="bf16", batch=64, heads=16, kv_heads=16, dim=64, tokens=1, capacity=8192, lead=0, masked=False),
        dict(name="read_grouped_e4m3", op="read", storage="e4m3", dtype="bf16", batch=24, heads=32, kv_heads=8, dim=128, tokens=7, capacity=5000, lead=1, masked=True),
        # the tables of one small tree and of a batch of wide ones
        dict(name="tables_one", op="tables", batch=1, tokens=8, include_self=False),
        dict(name="tables_batch", op="tables", batch=128, tokens=256, include_self=True),
        # verification of drafts: the 64-sequence bf16 pool with 32 drafted tokens each, and wide trees over an int8 pool
        dict(name="tree_pool_bf16", op="tree", storage="bf16", dtype="bf16", batch=64, heads=16, kv_heads=16, dim=64, tokens=32, capacity=8192, lead=0, masked=False, include_self=False),
        dict(name="tree_grouped_int8", op="tree", storage="int8", dtype="bf16", batch=8, heads=32, kv_heads=8, dim=128, tokens=41, capacity=4100, lead=1, masked=True, include_self=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["commit", "readback", "read", "read", "tables", "tree", "tree"])
    storage, dim, lead = rng.choice(["int8", "e4m3"]), rng.choice([32, 48, 64, 64, 80, 96, 128, 128]), rng.choice([0, 1])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    if op == "tables":
        return dict(op=op, batch=_log(rng, 1, 128), tokens=_log(rng, 1, 256), include_self=rng.random() < 0.5)
    if op in ("commit", "readback"):
        batch, heads = _log(rng, 1, 48), _log(rng, 1, 128)
        most = min(2049, max(1, (200 << 20) // (batch * heads * dim)))  # no more elements than the largest listed pool
        capacity = _log(rng, 1, most)
        if op == "readback":
            return dict(op=op, storage=storage, dtype=dtype, batch=batch, heads=heads, capacity=capacity, dim=dim, lead=lead)
        rows = _log(rng, 1, capacity)
        return dict(op=op, storage=storage, dtype=dtype, batch=batch, heads=heads, rows=rows, dim=dim, capacity=capacity, lead=lead, branch=rng.random() < 0.4)
    kv_heads, group = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([1, 1, 2, 3, 4, 8])
    batch = _log(rng, 1, 32)
    tokens = rng.choice([1, 1, 1, 2, 5]) if op == "read" else _log(rng, 1, 64)
    if op == "tree":
        storage = rng.choice(["int8", "e4m3", "bf16", "bf16"])
    if dtype == "fp32":  # fp32 is the checking type: a quarter of the work at most
        tokens, storage = min(tokens, 16), storage if storage != "bf16" else "fp32"
    # neither more pool bytes nor more products than the largest listed read
    most = (1 << 29) // (batch * kv_heads * dim * (4 if storage == "fp32" else 2 if storage == "bf16" else 1))
    most = min(most, (1 << 34) // (batch * kv_heads * group * tokens * dim * (4 if dtype == "fp32" else 1)), 12000)
    capacity = _log(rng, 1, max(1, most))
    c = dict(op=op, storage=storage, dtype=dtype, batch=batch, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, tokens=tokens,
             capacity=capacity, lead=lead, masked=rng.random() < 0.3)
    if op == "tree":
        c["include_self"] = rng.random() < 0.5
    return c


# ------------------------------------------------------------------ inputs


def _lengths(case):
    """Committed tokens per sequence, spread evenly over 1 .. capacity; one sequence alone is nearly full."""
    batch, top = case["batch"], case["capacity"]
    if batch == 1:
        return [max(1, top - top // 16)]
    return [1 + round(i * (top - 1) / (batch - 1)) for i in range(batch)]


def _rows(gen, *shape, like_keys):
    """Keys after their norm and rotary embedding have channels of uneven size; values have tokens of uneven size."""
    x = torch.randn(*shape, generator=gen, device="cuda")
    if like_keys:
        return x.mul_(torch.exp(0.5 * torch.randn(shape[-1], generator=gen, device="cuda")))
    return x.mul_(torch.exp(0.4 * torch.randn(*shape[:-1], 1, generator=gen, device="cuda")))


def _parents(case, gen):
    """Trees as drafting makes them: every node hangs on the committed prefix (-1) or on one of the nodes before it, mostly a
    late one; the last nodes of some trees are padding (-2)."""
    batch, tokens = case["batch"], case["tokens"]
    place = torch.arange(tokens, device="cuda").expand(batch, tokens)
    back = 1 + (torch.rand(batch, tokens, generator=gen, device="cuda").pow(3) * place).long()
    parents = torch.clamp(place - back, min=-1)
    live = torch.randint(max(1, tokens - tokens // 8), tokens + 1, (batch, 1), generator=gen, device="cuda")
    return torch.where(place < live, parents, torch.full_like(parents, -2)).int()


def _power(exponent):
    """2^exponent in fp32, put together from its bits (normal range)."""
    return ((exponent.int() + 127) << 23).view(torch.float32)


def _quantise(x, storage):
    """(codes, scales) of rows, by the definition in the pool's documentation."""
    x = x.float()
    top = x.abs().amax(-1)
    used = top >= SMALLEST
    safe = torch.where(used, top, torch.ones_like(top))
    if storage == "int8":
        full = torch.full_like(safe, INT8_TOP)
        codes = torch.round(x * torch.div(full, safe)[..., None])
        scales = torch.div(safe, full)
    else:
        fraction, exponent = torch.frexp(safe)  # safe = fraction * 2^exponent, fraction in [0.5, 1)
        exponent = torch.where(fraction > 0.875, exponent - 8, exponent - 9)  # 448 = 0.875 * 2^9
        scales = _power(exponent)
        codes = x * _power(-exponent)[..., None]
    codes = torch.where(used[..., None], codes, torch.zeros_like(codes)).to(DTYPES[storage])
    return codes, torch.where(used, scales, torch.zeros_like(scales))


def _pool(gen, case, heads):
    """Keys, values and their scales (None where the pool is not held in 8 bits)."""
    slots = case["capacity"] + case["lead"]
    made = []
    for like_keys in (True, False):
        x = _rows(gen, case["batch"], heads, slots, case["dim"], like_keys=like_keys)
        made.append(_quantise(x, case["storage"]) if case["storage"] in ("int8", "e4m3") else (x.to(DTYPES[case["storage"]]), None))
        del x
    return made[0][0], made[1][0], made[0][1], made[1][1]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op, s = case["op"], dict(case)
    if op == "tables":
        s["parents"] = _parents(case, gen)
        return s
    batch, dim, slots = case["batch"], case["dim"], case["capacity"] + case["lead"]
    if op == "commit":
        shape = (batch, case["heads"], slots, dim)
        s["keys"] = torch.zeros(shape, dtype=torch.uint8, device="cuda").view(DTYPES[case["storage"]])
        s["values"] = torch.zeros(shape, dtype=torch.uint8, device="cuda").view(DTYPES[case["storage"]])
        s["key_scales"] = torch.zeros(shape[:3], device="cuda")
        s["value_scales"] = torch.zeros(shape[:3], device="cuda")
        rows = case["rows"]
        # a projection leaves its rows as (batch, tokens, heads, dim); the pool's heads come second
        s["new_k"] = _rows(gen, batch, rows, case["heads"], dim, like_keys=True).to(DTYPES[case["dtype"]]).transpose(1, 2)
        s["new_v"] = _rows(gen, batch, rows, case["heads"], dim, like_keys=False).to(DTYPES[case["dtype"]]).transpose(1, 2)
        s["lengths"] = torch.randint(0, case["capacity"] - rows + 1, (batch,), generator=gen, device="cuda").int()
        s["index"] = s["counts"] = None
        if case["branch"]:
            s["counts"] = torch.randint(0, rows + 1, (batch,), generator=gen, device="cuda").int()
            s["index"] = torch.randint(0, rows, (batch, rows), generator=gen, device="cuda").sort(-1).values.int()
        return s
    order = torch.randperm(batch, generator=gen, device="cuda")
    s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")[order]
    heads = case["heads"] if op == "readback" else case["kv_heads"]
    s["keys"], s["values"], s["key_scales"], s["value_scales"] = _pool(gen, case, heads)
    if op == "readback":
        return s
    tokens = case["tokens"]
    dtype = DTYPES[case["dtype"]]
    s["query"] = torch.randn(batch, tokens, case["heads"], dim, generator=gen, device="cuda").to(dtype).transpose(1, 2)
    s["key_mask"] = None
    if case["masked"]:
        s["key_mask"] = torch.rand(batch, slots, generator=gen, device="cuda") < 0.7
        s["key_mask"][:, : case["lead"]] = True
    if op == "tree":
        s["draft_k"] = _rows(gen, batch, tokens, heads, dim, like_keys=True).to(dtype).transpose(1, 2)
        s["draft_v"] = _rows(gen, batch, tokens, heads, dim, like_keys=False).to(dtype).transpose(1, 2)
        s["parents"] = _parents(case, gen)
        s["closure"], s["depths"] = _closure(s["parents"], case["include_self"])
        s["ancestors"] = _pack(s["closure"])
    return s


# ------------------------------------------------------------------ plain forms


def _closure(parents, include_self):
    """(visible (B,T,T), depths): node i sees its ancestors (and itself); padding nodes see nothing and have depth -1."""
    tokens = parents.shape[1]
    node = torch.arange(tokens, device=parents.device)
    eye = torch.eye(tokens, dtype=torch.float64, device=parents.device)
    # (I + A)^T has a positive entry wherever a path of at most T steps leads; binomials of 256 stay far below the fp64 range
    reach = torch.matrix_power((parents[..., None] == node).double() + eye, tokens) > 0
    live = parents >= -1
    depths = torch.where(live, reach.sum(-1) - 1, torch.full_like(parents, -1, dtype=torch.long)).int()
    if not include_self:
        reach = reach & (eye == 0)
    return reach & live[..., None], depths


def _pack(visible):
    """(B,T,T) truth values -> (B,T,ceil(T/32)) words, node j in bit j % 32 of word j // 32."""
    batch, tokens = visible.shape[:2]
    words = -(-tokens // 32)
    padded = torch.nn.functional.pad(visible, (0, 32 * words - tokens)).view(batch, tokens, words, 32)
    value = (padded.long() << torch.arange(32, device=visible.device)).sum(-1)
    return torch.where(value >= 2**31, value - 2**32, value).int()


def _visible_slots(s):
    """(B, slots): the dummy and the committed tokens, as far as the mask keeps them."""
    slot = torch.arange(s["keys"].shape[2], device="cuda")
    seen = slot < s["lengths"][:, None] + s["lead"]
    return seen if s["key_mask"] is None else seen & s["key_mask"]


def _plain_attention(s):
    batch, kv_heads, slots, dim = s["keys"].shape
    tokens, group = s["tokens"], s["heads"] // s["kv_heads"]
    q = s["query"].float().reshape(batch, kv_heads, group * tokens, dim) * dim**-0.5
    scores = q @ s["keys"].float().transpose(-1, -2)
    if s["key_scales"] is not None:
        scores = scores * s["key_scales"][:, :, None]
    visible = _visible_slots(s)[:, None, None, :].expand(batch, 1, group * tokens, slots)
    if s["op"] == "tree":
        scores = torch.cat((scores, q @ s["draft_k"].float().transpose(-1, -2)), -1)
        drafts = s["closure"][:, None].expand(batch, group, tokens, tokens).reshape(batch, 1, group * tokens, tokens)
        live = (s["parents"] >= -1)[:, None].expand(batch, group, tokens).reshape(batch, 1, group * tokens, 1)
        visible = torch.cat((visible & live, drafts), -1)
    scores = torch.where(visible, scores, torch.full_like(scores[..., :1], -math.inf))
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = weights.sum(-1, keepdim=True)
    weights = weights / torch.where(total > 0, total, torch.ones_like(total))
    past, drafted = weights[..., :slots], weights[..., slots:]
    if s["value_scales"] is not None:
        past = past * s["value_scales"][:, :, None]
    out = past @ s["values"].float()
    if s["op"] == "tree":
        out = out + drafted @ s["draft_v"].float()
    out = out.view(batch, kv_heads * group, tokens, dim).transpose(1, 2)
    return out.to(DTYPES[s["dtype"]])


def _plain_commit(s):
    batch, heads, rows, dim = s["new_k"].shape
    slot = s["lengths"].long()[:, None] + s["lead"] + torch.arange(rows, device="cuda")
    at = slot[:, None].expand(batch, heads, rows)  # in range: the inputs leave room for every row
    row_at = at[..., None].expand(batch, heads, rows, dim)
    new_k, new_v, keep = s["new_k"], s["new_v"], None
    if s["index"] is not None:
        keep = (torch.arange(rows, device="cuda") < s["counts"][:, None])[:, None]
        pick = s["index"].long()[:, None, :, None].expand(batch, heads, rows, dim)
        new_k, new_v = new_k.gather(2, pick), new_v.gather(2, pick)
    for new, codes, scales in ((new_k, "keys", "key_scales"), (new_v, "values", "value_scales")):
        c, x = _quantise(new, s["storage"])
        c, target = c.view(torch.uint8), s[codes].view(torch.uint8)
        if keep is not None:  # rows behind the accepted ones keep what the slot held
            c = torch.where(keep[..., None], c, target.gather(2, row_at))
            x = torch.where(keep, x, s[scales].gather(2, at))
        target.scatter_(2, row_at, c)
        s[scales].scatter_(2, at, x)
    return _stored(s)


def _stored(s):
    return {n: s[n] for n in ("keys", "values", "key_scales", "value_scales")}


def _plain_readback(s):
    live = (torch.arange(s["keys"].shape[2], device="cuda") < s["lengths"][:, None] + s["lead"])[:, None, :, None]
    out = {}
    for codes, scales in (("keys", "key_scales"), ("values", "value_scales")):
        x = s[codes].float() * s[scales][..., None]
        out[codes] = torch.where(live, x, torch.zeros_like(x[..., :1])).to(DTYPES[s["dtype"]])
    return out


def run(s):
    op = s["op"]
    if own:
        import white_matter_b200 as wm

        if op == "commit":
            wm.quantized_pool_append(
                s["keys"], s["values"], s["key_scales"], s["value_scales"], s["lengths"], s["new_k"], s["new_v"],
                use_dummy_token=bool(s["lead"]), index=s["index"], counts=s["counts"],
            )
            return _stored(s)
        if op == "readback":
            common = dict(lengths=s["lengths"], use_dummy_token=bool(s["lead"]), dtype=DTYPES[s["dtype"]])
            return {
                "keys": wm.dequantize_kv_rows(s["keys"], s["key_scales"], **common),
                "values": wm.dequantize_kv_rows(s["values"], s["value_scales"], **common),
            }
        if op == "tables":
            tree = wm.prepare_draft_tree(s["parents"], include_self=s["include_self"])
            return {"ancestors": tree.ancestors, "depths": tree.depths}
        common = dict(kv_lengths=s["lengths"], use_dummy_token=bool(s["lead"]), key_mask=s["key_mask"])
        if op == "read":
            return wm.quantized_pool_attention(s["query"], s["keys"], s["values"], s["key_scales"], s["value_scales"], **common)
        tree = wm.DraftTree(s["ancestors"], s["depths"])
        return wm.draft_tree_attention(
            s["query"], s["keys"], s["values"], s["draft_k"], s["draft_v"], tree, key_scales=s["key_scales"],
            value_scales=s["value_scales"], **common,
        )
    if op == "commit":
        return _plain_commit(s)
    if op == "readback":
        return _plain_readback(s)
    if op == "tables":
        visible, depths = _closure(s["parents"], s["include_self"])
        return {"ancestors": _pack(visible), "depths": depths}
    return _plain_attention(s)


# ------------------------------------------------------------------ floors


def work(case):
    op = case["op"]
    if op == "tables":
        n = case["batch"] * case["tokens"]
        return {"bytes": 4 * n * (2 + -(-case["tokens"] // 32)), "flops": n * case["tokens"]}
    wide, dim = 4 if case["dtype"] == "fp32" else 2, case["dim"]
    if op == "commit":
        rows = 2 * case["batch"] * case["heads"] * case["rows"] * (0.5 if case["branch"] else 1)  # half of a branch is accepted on average
        return {"bytes": rows * (dim * (wide + 1) + 4), "flops": 2 * rows * dim}
    seen = sum(_lengths(case)) + case["batch"] * case["lead"]
    if op == "readback":
        slots = case["batch"] * (case["capacity"] + case["lead"])
        return {"bytes": 2 * case["heads"] * (seen * (dim + 4) + slots * dim * wide), "flops": 2 * case["heads"] * seen * dim}
    held = {"int8": dim + 4, "e4m3": dim + 4, "bf16": 2 * dim, "fp32": 4 * dim}[case["storage"]]
    kept = seen * (0.7 if case["masked"] else 1)
    rows = case["batch"] * case["heads"] * case["tokens"]
    total = 2 * case["kv_heads"] * kept * held + 2 * rows * dim * wide
    flops = 4 * dim * case["heads"] * case["tokens"] * kept
    if case["masked"]:
        total += case["batch"] * (case["capacity"] + case["lead"])
    if op == "tree":
        total += 2 * case["batch"] * case["kv_heads"] * case["tokens"] * dim * wide
    return {"bytes": total, "flops": flops}


# ------------------------------------------------------------------ definitions in 64 bits


def _exact_rows(x, storage):
    """Codes and scales row by row from the definition; int8's two roundings to 32 bits belong to the definition."""
    x = x.double()
    a = x.abs().max(dim=-1, keepdim=True).values
    zero = a < SMALLEST
    a = a.masked_fill(zero, 1.0)
    if storage == "int8":
        inverse = (INT8_TOP / a).float().double()  # 48-bit products below: exact in 64 bits before their rounding
        codes = ((x * inverse).float().double()).round()
        scale = a / INT8_TOP
    else:
        e = torch.ceil(torch.log2(a / E4M3_TOP) - 1e-9)
        scale = torch.exp2(e)
        y = x / scale
        step = torch.exp2(torch.clamp(torch.floor(torch.log2(y.abs().clamp(min=1e-30))), min=-6) - 3)
        codes = (y / step).round() * step
    return codes.masked_fill(zero, 0.0), scale.masked_fill(zero, 0.0)[..., 0]


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    lead = case.get("lead", 0)
    if op == "tables":
        return None  # whole numbers: equality with the plain form is what counts
    if op == "commit":
        out = {}
        for name, rows in (("key", s["new_k"]), ("value", s["new_v"])):
            codes = torch.zeros(s[name + "s"].shape, dtype=torch.float64, device="cuda")
            scales = torch.zeros(s[name + "_scales"].shape, dtype=torch.float64, device="cuda")
            for b in range(case["batch"]):
                at = int(s["lengths"][b]) + lead
                mine = rows[b]
                if case["branch"]:
                    mine = mine[:, s["index"][b, : int(s["counts"][b])].long()]
                n = mine.shape[1]
                if n:
                    codes[b, :, at : at + n], scales[b, :, at : at + n] = _exact_rows(mine, case["storage"])
            out[name + "s"] = None if case["storage"] == "int8" else codes
            out[name + "_scales"] = scales
        return out
    if op == "readback":
        out = {}
        for name in ("key", "value"):
            x = s[name + "s"].double() * s[name + "_scales"].double()[..., None]
            for b in range(case["batch"]):
                x[b, :, int(s["lengths"][b]) + lead :] = 0
            out[name + "s"] = x
        return out
    batch, group, dim = case["batch"], case["heads"] // case["kv_heads"], case["dim"]
    out = torch.zeros(batch, case["tokens"], case["heads"], dim, dtype=torch.float64, device="cuda")
    for b in range(batch):
        n = int(s["lengths"][b]) + lead
        keep = torch.ones(n, dtype=torch.bool, device="cuda") if s["key_mask"] is None else s["key_mask"][b, :n]
        k, v = s["keys"][b, :, :n].double()[:, keep], s["values"][b, :, :n].double()[:, keep]
        if s["key_scales"] is not None:
            k = k * s["key_scales"][b, :, :n].double()[:, keep, None]
            v = v * s["value_scales"][b, :, :n].double()[:, keep, None]
        parents = s["parents"][b].tolist() if op == "tree" else None
        for t in range(case["tokens"]):
            kk, vv = k, v
            if parents is not None:
                if parents[t] < -1:
                    continue
                path, node = ([t] if case["include_self"] else []), parents[t]
                while node >= 0:
                    path.append(node)
                    node = parents[node]
                kk = torch.cat((k, s["draft_k"][b][:, path].double()), 1)
                vv = torch.cat((v, s["draft_v"][b][:, path].double()), 1)
            if kk.shape[1]:
                q = s["query"][b, :, t].double().view(case["kv_heads"], group, dim)
                p = torch.softmax(torch.einsum("hgd,hnd->hgn", q, kk) / math.sqrt(dim), -1)
                out[b, t] = torch.einsum("hgn,hnd->hgd", p, vv).reshape(case["heads"], dim)
    return out
