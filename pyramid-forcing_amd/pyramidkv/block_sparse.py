"""Attention over chosen blocks of the ragged cache.

``ragged_attention`` reads every cached key for every query.  Here each tile
of queries (``block_q`` tokens times the query heads that share a KV head)
reads only the blocks of ``block_k`` keys that a cheap score ranks highest:

* ``block_means``             the mean key of every block;
* ``block_select``            per tile, the blocks whose mean has the largest
                              product with the tile's summed queries, the first
                              (sink) and last (recent) ones always among them;
* ``block_sparse_attention``  softmax attention of the tile over its list;
* ``sparse_ragged_attention`` the three in a row; ``MegaCache.attend(sparse=...)``
                              runs them on the packed cache.

Layouts.  q is [total_q, heads, D] with sequence b at rows cu_seqlens_q[b] ..
[b + 1].  k and v are [total_k, D] with one sequence per (batch, KV head), in
the order b * kv_heads + h (what the cache packs: cu_seqlens_k has batches *
kv_heads + 1 entries), or [total_k, kv_heads, D] with one per batch.  Query
head h reads KV head h // (heads // kv_heads).  Where ``seqlens_k`` is given,
sequence s has that many of its rows in use: a cache that grows in place.

Block j of key sequence s is row cu_seqlens_k[s] // block_k + s + j of the
means (total_k // block_k + sequences rows), tile i of query sequence b row
cu_seqlens_q[b] // block_q + b + i of the lists (total_q // block_q + batches
rows of [kv_heads, topk] int32): no prefix sum over ragged lengths is needed
to find one.

All run on the current stream without a host synchronisation, in workspaces of
torch's allocator, and may be captured into a graph.  They have no derivatives:
a gradient or a tangent through means or attention raises; the choice of blocks,
and means written in place (out=), carry none.  Rows of the attention's results
that no sequence owns, and those past max_seqlen_q in theirs, are not written.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _ops


@dataclass
class BlockSparse:
    """How many blocks a tile of queries attends to, and of what sizes."""
    topk: int
    block_q: int = 128
    block_k: int = 64
    sink_blocks: int = 0
    recent_blocks: int = 0


def block_means(k, cu_seqlens_k, block_k=64, *, max_seqlen_k=0, seqlens_k=None, out=None, last=0):
    """Mean key of every block in fp32, shaped like k with its rows replaced
    by the blocks' (rows without keys are 0).  max_seqlen_k, a bound of a
    sequence's keys, sizes the launch (0: unknown).  With ``out`` (an earlier
    call's result) only the blocks that hold a sequence's ``last`` keys are
    computed again, in place: what a cache needs that has grown by as many."""
    if out is None:
        if last:
            raise ValueError("block_means: last needs out, the means to bring up to date")
        return _ops.ops().block_means(k, cu_seqlens_k, int(block_k), int(max_seqlen_k), seqlens_k)
    _ops.ops().block_means_(out, k, cu_seqlens_k, int(block_k), int(last), int(max_seqlen_k), seqlens_k)
    return out


def block_select(q, means, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, topk, *, block_q=128, block_k=64,
                 sink_blocks=0, recent_blocks=0, causal=False, seqlens_k=None, rank_own=False):
    """The blocks that each tile attends to, [tile rows, kv_heads, topk] int32,
    ascending and padded with -1.  A block's score is the product of the tile's
    summed queries with its mean, summed in 64 bits and rounded to fp32 (ties:
    the lower index; NaN counts as -inf).  Keys past max_seqlen_k are not
    considered, and tiles past max_seqlen_q get no block.  causal (block_q 1):
    token i of n chooses from the blocks that hold its keys up to keys - n + i.
    The last of them is taken whatever its score, as by recent_blocks 1: its mean
    may cover later keys, on which no choice depends so (where sink_blocks is topk
    there is no room for it).  rank_own: that block is ranked like the others, for
    means that hold no later keys."""
    return _ops.ops().block_select(q, means, cu_seqlens_q, cu_seqlens_k, int(max_seqlen_q), int(max_seqlen_k), int(topk),
                                   int(block_q), int(block_k), int(sink_blocks), int(recent_blocks), bool(causal),
                                   seqlens_k, bool(rank_own))


def block_sparse_attention(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, lists, *, block_q=128, block_k=64,
                           softmax_scale=None, causal=False, return_lse=False, seqlens_k=None):
    """Attention of each tile over the blocks of its list.  Entries below 0,
    past the sequence's blocks or repeated are passed over, in any order.  A row
    without keys is 0 (as ragged_attention has it, one whose keys all score
    -inf is NaN).  return_lse: also the natural logarithm of each row's
    softmax sum, [heads, total_q] fp32, by which results over different keys
    can be joined."""
    if softmax_scale is None:
        softmax_scale = q.shape[-1] ** -0.5
    out = _ops.ops().block_sparse_attention(q, k, v, cu_seqlens_q, cu_seqlens_k, int(max_seqlen_q), lists,
                                            float(softmax_scale), int(block_q), int(block_k), bool(causal),
                                            bool(return_lse), seqlens_k)
    return (out[0], out[1]) if return_lse else out[0]


def sparse_ragged_attention(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, sparse: BlockSparse, *,
                            softmax_scale=None, causal=False, seqlens_k=None, means=None):
    """Means (unless given), selection and attention in a row.  causal: no result
    depends on a later key, through the choice of blocks either."""
    if means is None:
        means = block_means(k, cu_seqlens_k, sparse.block_k, max_seqlen_k=max_seqlen_k, seqlens_k=seqlens_k)
    lists = block_select(q, means, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, sparse.topk,
                         block_q=sparse.block_q, block_k=sparse.block_k, sink_blocks=sparse.sink_blocks,
                         recent_blocks=sparse.recent_blocks, causal=causal, seqlens_k=seqlens_k)
    return block_sparse_attention(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, lists, block_q=sparse.block_q,
                                  block_k=sparse.block_k, softmax_scale=softmax_scale, causal=causal,
                                  seqlens_k=seqlens_k)
