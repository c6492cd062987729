"""CPU restatement of the serving operators: quantised rows, draft trees and attention behind the committed tokens, from
their definitions (attention in 64 bits, with the sums that error bounds are made of)."""

from __future__ import annotations

import numpy as np
import torch

SMALLEST = np.float32(2.0**-100)


def quantise_row(x: np.ndarray, storage: str) -> tuple[np.ndarray, np.float32]:
    """(codes as fp32 numbers, scale) of one fp32 row; every operation below is a single IEEE fp32 rounding."""
    x = x.astype(np.float32)
    if not np.isfinite(x).all():
        return np.zeros_like(x), np.float32("nan")
    top = np.abs(x).max()
    if top < SMALLEST:
        return np.zeros_like(x), np.float32(0)
    if storage == "int8":
        return np.rint(x * (np.float32(127) / top)), top / np.float32(127)
    exponent = -200
    while float(top) > 448.0 * 2.0**exponent:
        exponent += 1
    scaled = torch.from_numpy(x.astype(np.float64) * 2.0**-exponent)  # exact
    return round_e4m3(scaled).numpy().astype(np.float32), np.float32(2.0**exponent)


def round_e4m3(y: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 number, ties to even: three fraction bits, smallest normal 2^-6."""
    power = torch.floor(torch.log2(y.abs().clamp(min=2.0**-30)))
    power = torch.where(y.abs() < torch.exp2(power), power - 1, power)
    step = torch.exp2(torch.clamp(power, min=-6) - 3)
    return torch.round(y / step) * step


def quantise_rows(x: torch.Tensor, storage: str) -> tuple[torch.Tensor, torch.Tensor]:
    flat = x.float().reshape(-1, x.shape[-1]).numpy()
    codes = np.zeros_like(flat)
    scales = np.zeros(len(flat), dtype=np.float32)
    for i, row in enumerate(flat):
        codes[i], scales[i] = quantise_row(row, storage)
    return torch.from_numpy(codes).view(x.shape), torch.from_numpy(scales).view(x.shape[:-1])


def commit(codes, scales, lengths, new, storage, lead, index=None, counts=None) -> None:
    """In-place commit to (B,H,N,D) codes held as fp32 numbers and (B,H,N) scales; storage None copies the rows."""
    batch, _, slots, _ = codes.shape
    rows = new.shape[2] if index is None else index.shape[1]
    for b in range(batch):
        for i in range(rows if counts is None else min(rows, int(counts[b]))):
            slot, source = int(lengths[b]) + lead + i, i if index is None else int(index[b, i])
            if 0 <= slot < slots and 0 <= source < new.shape[2]:
                if storage is None:
                    codes[b, :, slot] = new[b, :, source]
                else:
                    codes[b, :, slot], scales[b, :, slot] = quantise_rows(new[b, :, source], storage)


def tree_tables(parents: torch.Tensor, include_self: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """(visible (B,T,T), depths (B,T)) by walking every node's chain."""
    batch, tokens = parents.shape
    visible, depths = torch.zeros(batch, tokens, tokens, dtype=torch.bool), torch.full((batch, tokens), -1, dtype=torch.int32)
    for b in range(batch):
        up = parents[b].tolist()
        for i in range(tokens):
            chain, node = [], up[i]
            while 0 <= node < tokens and len(chain) <= tokens:
                chain.append(node)
                node = up[node]
            if node == -1 and len(chain) <= tokens:
                visible[b, i, chain] = True
                visible[b, i, i] = include_self
                depths[b, i] = len(chain)
    return visible, depths


def pack_bits(visible: torch.Tensor) -> torch.Tensor:
    batch, tokens = visible.shape[:2]
    words = torch.zeros(batch, tokens, -(-tokens // 32), dtype=torch.int64)
    for j in range(tokens):
        words[:, :, j // 32] |= visible[:, :, j].long() << (j % 32)
    return torch.where(words >= 2**31, words - 2**32, words).int()


def attention(query, keys, values, lengths, lead, key_mask=None, draft=None, scale=None):
    """query (B,H,T,D), keys/values (B,HKV,N,D) real numbers, draft = (keys, values, visible (B|1,T,T), depths).

    Returns out (B,T,H,D), mass = sum of weight * |value| per element, and reach (B,T,H,1), the largest
    sum of |q*k| * scale over the visible keys: what the rounding errors of weights and scores are proportional to.
    """
    batch, heads, tokens, dim = query.shape
    kv_heads, slots = keys.shape[1], keys.shape[2]
    scale = dim**-0.5 if scale is None else scale
    out, mass, reach = (torch.zeros(batch, tokens, heads, n, dtype=torch.float64) for n in (dim, dim, 1))
    for b in range(batch):
        n = slots if lengths is None else min(max(int(lengths[b]), 0), slots - lead) + lead
        keep = torch.ones(n, dtype=torch.bool) if key_mask is None else key_mask[b, :n]
        for t in range(tokens):
            pick, t_draft = None, 0
            if draft is not None:
                t_draft = 0 if draft[3].shape[0] == 1 else b
                if draft[3][t_draft, t] < 0:
                    continue
                pick = draft[2][t_draft, t]
            for h in range(heads):
                g = h // (heads // kv_heads)
                k, v = keys[b, g, :n][keep].double(), values[b, g, :n][keep].double()
                if pick is not None:
                    k = torch.cat((k, draft[0][b, g][pick].double()))
                    v = torch.cat((v, draft[1][b, g][pick].double()))
                if not len(k):
                    continue
                q = query[b, h, t].double()
                p = torch.softmax(k @ q * scale, 0)
                out[b, t, h], mass[b, t, h], reach[b, t, h] = p @ v, p @ v.abs(), (k.abs() @ q.abs()).max() * scale
    return out, mass, reach


def bound(out, mass, reach, dtype, dim: int, keys: int):
    """How far an operator's result may be from ``out``, element by element.

    * the result is rounded to its type: u_out * |out|;
    * scores carry (dim + 8) fp32 roundings of sums of at most ``reach``, and the exponential a relative 2^-21; a score
      that is off by e moves the weights by a factor exp(+-e), numerator and denominator alike: 2 * e * mass;
    * sums over the keys in fp32, in any order: 2 * keys * 2^-24 * mass;
    * with bf16 operands, weights (times a value scale) are rounded to bf16 before the value product: 2^-8 * mass,
      and once more at most for the sum that divides them.
    """
    u = 2.0**-8 if dtype == torch.bfloat16 else 2.0**-24
    weights = 2 * (1.01 * ((dim + 8) * 2.0**-24 * reach + 2.0**-21) + keys * 2.0**-24)
    if dtype == torch.bfloat16:
        weights = weights + 2 * 2.0**-8
    return 1.01 * (u * out.abs() + weights * mass) + 1e-30
