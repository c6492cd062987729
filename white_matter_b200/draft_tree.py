"""Attention of drafted tokens that branch: one pass over a tree of candidates behind the committed tokens of a pool.

A draft proposes several continuations at once; they share prefixes and so form a tree, given by every node's parent
(-1: the committed prefix).  ``prepare_draft_tree`` turns the parents into the tables that the attention reads, once
per draft and for all layers; ``draft_tree_attention`` lets every node attend to the committed slots and to its own
ancestors among the drafted tokens, whose K/V lie outside the pool.  After verification the accepted branch is
committed by ``append(..., index=..., counts=...)`` of the pool classes.

In the strict-past convention of this package a token does not attend to itself (``include_self=False``); with
``include_self=True`` the operator serves ordinary causal attention.  The upstream project decodes one token at a time
and has no counterpart.  Inference only.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native
from .quant_pool import pool_attention

MAX_NODES = 512


class DraftTree(NamedTuple):
    """Tables of trees of T drafted tokens: ``ancestors`` (B,T,ceil(T/32)) int32 words, bit j % 32 of word j // 32 of row
    i set where node i attends to node j; ``depths`` (B,T) int32, the number of ancestors, -1 for padding nodes.  B is 1
    for a tree that a whole batch shares.  The rotary position of node i of sequence b is ``lengths[b] + depths[b, i]``."""

    ancestors: torch.Tensor
    depths: torch.Tensor


def prepare_draft_tree(parents: torch.Tensor, *, include_self: bool = False) -> DraftTree:
    """Ancestor bits and depths of trees given by their parents, (B,T) or (T,) integers on the GPU, T <= 512.

    ``parents[b, i]`` is the node that node i hangs on, in any order, or -1 for the committed prefix.  A node whose
    chain of parents does not end in -1 -- another negative number, a number of T or more, a cycle -- is padding: it
    sees nothing and no node sees it.  Runs on the device without a host read, so it can be captured in a CUDA graph and
    replayed with other parents.
    """
    if type(include_self) is not bool:
        raise ValueError("include_self must be boolean")
    if parents.ndim not in (1, 2) or parents.dtype not in (torch.int32, torch.int64):
        raise ValueError("parents must be integer (B,T) or (T,)")
    if not parents.is_cuda:
        raise ValueError("sm100 draft trees require CUDA tensors")
    if parents.ndim == 1:
        parents = parents[None]
    batch, tokens = parents.shape
    if tokens > MAX_NODES:
        raise ValueError(f"at most {MAX_NODES} drafted tokens are supported")
    if parents.dtype != torch.int32:  # numbers outside the tree stay outside it
        parents = parents.clamp(-2, MAX_NODES).to(torch.int32)
    parents = parents.contiguous()
    ancestors = parents.new_empty((batch, tokens, -(-tokens // 32)))
    depths = torch.empty_like(parents)
    if batch and tokens:
        record = _native.pack_draft_tree(parents.data_ptr(), ancestors.data_ptr(), depths.data_ptr(), batch, tokens, include_self)
        _native.call_record("wm_draft_tree", parents.get_device(), record)
    return DraftTree(ancestors, depths)


def draft_tree_attention(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    draft_key: torch.Tensor,
    draft_value: torch.Tensor,
    tree: DraftTree,
    *,
    kv_lengths: torch.Tensor | None = None,
    use_dummy_token: bool = False,
    key_mask: torch.Tensor | None = None,
    softmax_scale: float | None = None,
    key_scales: torch.Tensor | None = None,
    value_scales: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of the nodes of a draft tree over the committed tokens of a pool and their own ancestors.

    ``query`` (B,H,T,D) holds the drafted tokens' queries, ``draft_key`` / ``draft_value`` (B,HKV,T,D) their K/V in the
    same dtype (bf16 or fp32).  ``key`` / ``value`` (B,HKV,N,D) are the pool, in the query's dtype or in 8 bits with
    ``key_scales`` / ``value_scales`` as in ``quantized_pool_attention``; the rules for ``kv_lengths``,
    ``use_dummy_token`` and ``key_mask`` are the same.  Node i also sees the drafted tokens that ``tree`` names.
    Padding nodes, and nodes that see nothing, return zero; the K/V of padding nodes, and of slots that are not seen, may
    hold anything.  Precision and range are those of ``quantized_pool_attention``; over bf16 pools the weights are one bf16
    part for any number of rows.  Returns (B,T,H,D).
    """
    if query.ndim != 4:
        raise ValueError("query must be (B,H,T,D)")
    batch, _, tokens, dim = query.shape
    if tokens > MAX_NODES:
        raise ValueError(f"at most {MAX_NODES} drafted tokens are supported")
    if draft_key.shape != draft_value.shape or draft_key.shape != (batch, key.shape[1] if key.ndim == 4 else -1, tokens, dim):
        raise ValueError("drafted K/V must be (B,HKV,T,D)")
    if any(t.dtype != query.dtype or t.device != query.device for t in (draft_key, draft_value)):
        raise ValueError("drafted K/V must have the query's dtype and device")
    ancestors, depths = tree
    if depths.ndim != 2 or depths.shape[0] not in (1, batch) or depths.shape[1] != tokens or ancestors.shape != (*depths.shape, -(-tokens // 32)):
        raise ValueError("the tree must have been prepared for these drafted tokens")
    if ancestors.dtype != torch.int32 or depths.dtype != torch.int32 or ancestors.device != query.device or depths.device != query.device:
        raise ValueError("tree tables must be int32 on the query's device")
    return pool_attention(
        query, key, value, key_scales, value_scales, kv_lengths, use_dummy_token, key_mask, softmax_scale,
        (draft_key, draft_value, ancestors, depths),
    )
