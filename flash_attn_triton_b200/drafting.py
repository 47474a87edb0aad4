"""Decoding with trees of drafted tokens: a small model drafts a tree of tokens for each request, the large one verifies all of
them in one step over its KV cache.  No counterpart in the reference.  A step, with `flash_attn_with_kvcache(tree_mask=)` between:

    slots, cu, used = build_block_table(cache_seqlens, torch.full_like(cache_seqlens, nodes), free_pages, block_table, page_size, batch * nodes)
    q, k = qk_norm_rotary(q, k, q_weight, k_weight, cos, sin, positions=cache_seqlens[:, None] + depth)          # each layer
    out = flash_attn_with_kvcache(q, k_cache, v_cache, k, v, cache_seqlens=cache_seqlens, block_table=block_table, tree_mask=mask)
    path, accepted, token = verify_draft_tree(draft_tokens, parents, target_probs, draft_probs, accept_uniforms, sample_uniforms)
    kvcache_compact(k_caches, v_caches, cache_seqlens, path, accepted, block_table=block_table)                    # all layers
    pages, n = release_pages(cache_seqlens + nodes, cache_seqlens + accepted, block_table, page_size, num_pages)
    cache_seqlens += accepted                                     # `token` is the root of the next tree

`nodes` is the seqlen_q of the call, the nodes of the largest tree.  The call appends that many rows for every request, those of nodes that a
request does not use too, so that every request needs pages for all of them: an entry of the table that this step did not fill may name a
page that is another request's by now.
"""
from __future__ import annotations

import torch

from . import _native as N
from . import flash_attn_interface as _api

_PROB_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


def _i32(x):
    """Integers as int32; those that do not fit stay out of range."""
    return x if x.dtype == torch.int32 else x.clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32)


def _on(device, *tensors):
    if device.type != "cuda":
        raise ValueError("All tensors must be CUDA tensors")
    if any(t is not None and t.device != device for t in tensors):
        raise ValueError("All tensors must be on the same CUDA device")


def qk_norm_rotary(q, k, q_weight=None, k_weight=None, rotary_cos=None, rotary_sin=None, positions=None, eps=1e-6,
                   rotary_interleaved=False):
    """RMS norm of every head of q and k, then the rotary embedding, in one pass: y = x * rsqrt(mean(x^2) + eps) * weight over
    head_dim, rotated at the token's position.  In fp32, rounded once.  Returns (q, k) as new tensors; differentiable in q, k and the weights, once.

    q (batch, seqlen, nheads, d) or packed (tokens, nheads, d), fp16, bf16 or fp32; k the same with its own number of heads; weights (d,)
    of q's dtype or both fp32, None for ones; tables (seqlen_ro, rotary_dim / 2) of q's dtype or fp32, None for no rotation.  positions:
    integers, (batch, seqlen) or (seqlen,), packed (tokens,); None for the rows' own numbers.  The tokens of a drafted tree sit at the
    length of the context plus their depth.  A position outside the tables rotates nothing."""
    if torch._C._get_tracing_state() is not None:
        raise ValueError("qk_norm_rotary cannot be recorded by torch.jit.trace")
    return N.host().qk_norm(q, k, q_weight, k_weight, rotary_cos, rotary_sin, positions, eps, rotary_interleaved)


def verify_draft_tree(draft_tokens, parents, target_probs, draft_probs, accept_uniforms, sample_uniforms):
    """Which drafted tokens the target model accepts, and the token that follows them, so that what comes out is distributed as
    if the target alone had sampled it.

    A request's tree has up to `nodes` nodes.  Node 0 is the root, the last token that is certain; draft_tokens (batch, nodes) integers, parents
    (batch, nodes) or (nodes,) integers: the node before each one.  A node whose parent is not an earlier node (-1, say) is not used;
    the children of a node are tried in the order of their numbers.  target_probs, draft_probs (batch, nodes, vocab) fp32, fp16 or
    bf16: the distribution of the token after each node, of the target and of the draft model that the node's children were drawn from, each on its
    own.  accept_uniforms (batch, nodes) and sample_uniforms (batch,) fp32: random numbers in [0, 1).

    A child x is accepted with probability min(1, p(x) / q(x)), else the target's distribution p becomes norm(max(p - q, 0)) for the next
    one; where no child is left, the next token is sampled from p.  In 64 bits.  Returns
      path (batch, nodes) int32       the accepted nodes in order, the root first, -1 behind them
      num_accepted (batch,) int32     how many, the root among them
      next_token (batch,) int64       -1 where the probabilities hold nothing or are no finite numbers
    A chain of drafts is parents = (-1, 0, 1, ...).  The distributions are taken to sum to 1."""
    if target_probs.ndim != 3 or draft_probs.shape != target_probs.shape:
        raise ValueError("target_probs and draft_probs must have the same shape (batch, nodes, vocab)")
    if target_probs.dtype not in _PROB_DTYPES or draft_probs.dtype != target_probs.dtype:
        raise ValueError("target_probs and draft_probs must be matching FP32, FP16 or BF16 tensors")
    batch, nodes, vocab = target_probs.shape
    if not 1 <= nodes <= 1024:
        raise ValueError("a tree must have 1 to 1024 nodes")
    if not 1 <= vocab < 2 ** 31:
        raise ValueError("the vocabulary must have 1 to 2 ** 31 - 1 tokens")
    for x, name, shapes in ((draft_tokens, "draft_tokens", ((batch, nodes),)), (parents, "parents", ((batch, nodes), (nodes,)))):
        if x.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{name} must use int32 or int64")
        if x.shape not in shapes:
            raise ValueError(f"{name} must hold one value per node")
    if accept_uniforms.dtype != torch.float32 or sample_uniforms.dtype != torch.float32:
        raise ValueError("accept_uniforms and sample_uniforms must be FP32 tensors")
    if accept_uniforms.shape != (batch, nodes) or sample_uniforms.shape != (batch,):
        raise ValueError("accept_uniforms must have shape (batch, nodes) and sample_uniforms (batch,)")
    _on(target_probs.device, draft_tokens, parents, draft_probs, accept_uniforms, sample_uniforms)
    if target_probs.stride(2) != 1 and vocab > 1:
        target_probs = target_probs.contiguous()
    if draft_probs.stride(2) != 1 and vocab > 1:
        draft_probs = draft_probs.contiguous()
    return N.host().verify(draft_tokens.to(torch.int64).contiguous(), _i32(parents).contiguous(), target_probs, draft_probs,
                           accept_uniforms.contiguous(), sample_uniforms.contiguous())


_COMPACT_ERRORS = ("num_accepted must be between 0 and the length of a path",
                   "the accepted part of a path must ascend from 0 or more",
                   "the rows of a path do not lie inside the cache",
                   "block_table or cache_batch_idx contains an index that does not exist")


_CACHES_DIFFER = ("the KV caches must have the same shape (num_pages, page_size, nheads_k, headdim)",
                  "kvcache_compact supports matching FP16 or BF16 caches",
                  "the caches of all layers must have the same strides",
                  "KV caches must have a unit head-dim stride and 16-byte aligned rows",
                  "All tensors must be on the same CUDA device",
                  "the KV caches must not overlap")


def kvcache_compact(k_cache, v_cache, cache_seqlens, path, num_accepted, block_table=None, cache_batch_idx=None, cache_leftpad=None):
    """Move the rows of accepted tokens together, in place: for i < num_accepted[b], the row at position cache_seqlens[b] + i takes
    what the one at cache_seqlens[b] + path[b, i] holds.  With the path of `verify_draft_tree` and the lengths from before the drafted tokens
    were appended, the accepted ones then follow the context, and the sequence has num_accepted[b] tokens more.

    k_cache, v_cache: fp16 or bf16 caches as in flash_attn_with_kvcache, or lists of them, one per layer, of the same shape, dtype and strides,
    none of which overlaps another; all layers are moved by one launch.  path (batch, n) integers, ascending in its first num_accepted[b]
    entries; cache_seqlens, num_accepted (batch,).  The rows of drafted tokens belong to one request: requests that name the same cache row
    (cache_batch_idx), or share a page behind their contexts, may come out with either one's tokens.

    With value checks on, values that do not fit raise ValueError and nothing is moved; off (see set_validation), such requests are passed
    over."""
    k_caches, v_caches = (list(x) if isinstance(x, (list, tuple)) else [x] for x in (k_cache, v_cache))
    if not k_caches or len(k_caches) != len(v_caches):
        raise ValueError("k_cache and v_cache must be tensors, or lists of as many tensors")
    first = k_caches[0]
    if first.ndim != 4:
        raise ValueError("the KV caches must have the same shape (num_pages, page_size, nheads_k, headdim)")
    if first.dtype not in _api._KERNEL_DTYPES:
        raise ValueError("kvcache_compact supports matching FP16 or BF16 caches")
    _api._check_head_dim(first.shape[3])
    if first.shape[2] == 0:
        raise ValueError("the KV caches need at least one head")
    differs = N.host().caches_match(k_caches, v_caches)
    if differs:
        raise ValueError(_CACHES_DIFFER[differs - 1])
    if path.ndim != 2 or path.dtype not in (torch.int32, torch.int64):
        raise ValueError("path must have shape (batch, n) and use int32 or int64")
    batch, device = path.shape[0], first.device
    if block_table is not None:
        if block_table.ndim != 2 or block_table.shape[0] != batch:
            raise ValueError("block_table must have shape (batch, max_num_pages)")
        if block_table.dtype not in (torch.int32, torch.int64):
            raise ValueError("block_table must contain integer page indices")
        if cache_leftpad is not None:
            raise ValueError("cache_leftpad cannot be combined with paged KV caches")
        if cache_batch_idx is not None:
            raise ValueError("cache_batch_idx cannot be combined with paged KV caches")
    elif cache_batch_idx is None and first.shape[0] < batch:
        raise ValueError("cache_batch_idx must contain valid cache-row indices")
    _on(device, path)
    lens, accepted, rows, pads = (None if x is None else _api._as_i32(x, device) for x in (cache_seqlens, num_accepted, cache_batch_idx, cache_leftpad))
    for x, name in ((lens, "cache_seqlens"), (accepted, "num_accepted"), (rows, "cache_batch_idx"), (pads, "cache_leftpad")):
        if x is not None and x.numel() != batch:
            raise ValueError(f"{name} must contain one value per request")
    if batch == 0:
        return
    if block_table is not None:
        block_table = _i32(block_table).to(device).contiguous()
        if block_table.shape[1] == 0:                    # no pages: only paths of nothing are allowed
            block_table = block_table.new_full((batch, 1), -1)
    path = _i32(path).contiguous()
    for i in range(0, len(k_caches), N.COMPACT_LAYERS):
        failed = N.host().compact(k_caches[i:i + N.COMPACT_LAYERS], v_caches[i:i + N.COMPACT_LAYERS], lens, path, accepted, block_table, rows,
                                  pads, _api._VALIDATE)
        if failed:
            raise ValueError(_COMPACT_ERRORS[(failed & -failed).bit_length() - 1])


def release_pages(held_lens, kept_lens, block_table, page_size, num_pages):
    """Pages that requests no longer need: the counterpart of `build_block_table`.  Request b has pages for held_lens[b] tokens in its
    row of block_table (batch, max_pages) int32 and keeps those for kept_lens[b], 0 when it has ended.  Returns
      pages (num_pages,) int32     entries [ceil(kept / page_size), ceil(held / page_size)) of the rows, request by request, -1 behind the last
      pages_released () int32      how many
    to be put behind the free pages.  The table stays as it is: the next step enters its pages over these.  num_pages is a number that the
    host knows to be enough.  Pages that several requests share are named by each of them.

    With value checks on, lengths that do not fit raise ValueError; off (see set_validation), all pages are -1 and pages_released is -1."""
    if block_table.ndim != 2 or block_table.dtype != torch.int32:
        raise ValueError("block_table must be a CUDA tensor (batch, max_num_pages) of int32")
    if block_table.shape[1] > 1 and block_table.stride(1) != 1:
        raise ValueError("block_table must have rows of unit stride")
    page_size, num_pages = int(page_size), int(num_pages)
    if not 0 < page_size < 2 ** 31:
        raise ValueError("page_size must be positive")
    if not 0 <= num_pages < 2 ** 31:
        raise ValueError("num_pages must be non-negative and below 2 ** 31")
    device = block_table.device
    _on(device)
    held, kept = (_api._as_i32(x, device) for x in (held_lens, kept_lens))
    if held.numel() != block_table.shape[0] or kept.numel() != block_table.shape[0]:
        raise ValueError("held_lens and kept_lens must contain one length per row of block_table")
    made = N.host().release(held, kept, block_table, page_size, num_pages, _api._VALIDATE)
    if isinstance(made, int):
        raise ValueError(("kept_lens must not be negative, nor larger than held_lens", "a request exceeds its row of block_table",
                          "the released pages exceed num_pages")[(made & -made).bit_length() - 1])
    return made
