"""PyTorch dispatcher bindings for the B200 branchcraft kernels.

Importing this module loads the native operator library (``_C*.so`` next to
this file, which links ``lib/libbranchcraft.so``) and registers fake (meta)
kernels so ``torch.compile`` and FakeTensor tracing see every op's output.
The public API is ``torch.ops.branchcraft``; the functions below are thin
wrappers with the reference's names (python/branchcraft_torch/__init__.py).
There is no fallback: a missing extension is an ImportError.
"""
from pathlib import Path

import torch

_library = next(Path(__file__).parent.glob("_C*.so"), None)
if _library is None:
    raise ImportError("branchcraft CUDA extension is missing; run "
                      "`python branchcraft-cuda_b200/build.py`")
torch.ops.load_library(str(_library))


@torch.library.register_fake("branchcraft::tree_verify")
def _fake_tree_verify(q, prefix_k, prefix_v, pages, lengths, draft_k, draft_v, parent):
    return q.new_empty(q.shape, dtype=torch.float32)


@torch.library.register_fake("branchcraft::packed_decode_out")
def _fake_packed_decode_out(q, packed_kv, pages, lengths, output, scale):
    return output


@torch.library.register_fake("branchcraft::commit_path_")
def _fake_commit_path(cache_k, cache_v, draft_k, draft_v, path_nodes, dest_pages,
                      dest_slots, request):
    return None


@torch.library.register_fake("branchcraft::paged_decode")
def _fake_paged_decode(q, k, v, pages, lengths, splits=0):
    return q.new_empty(q.shape, dtype=torch.float32)


@torch.library.register_fake("branchcraft::tree_verify_out")
def _fake_tree_verify_out(q, prefix_k, prefix_v, pages, lengths, draft_k, draft_v, parent,
                          output):
    return output


@torch.library.register_fake("branchcraft::packed_decode_kv_out")
def _fake_packed_decode_kv_out(q, k_cache, v_cache, pages, lengths, output, scale, splits=0):
    return output


@torch.library.register_fake("branchcraft::commit_batch_")
def _fake_commit_batch(cache_k, cache_v, draft_k, draft_v, clone_src, clone_dst,
                       entry_request, entry_node, entry_page, entry_slot):
    return None


def _fake_plan_outputs(pages, max_tokens):
    batch = pages.shape[0]
    return (pages.new_empty(batch + 1), pages.new_empty(max_tokens), pages.new_empty(max_tokens),
            pages.new_empty((3, batch)), pages.new_empty(3))


@torch.library.register_fake("branchcraft::append_plan")
def _fake_append_plan(pages, lengths, new_tokens, refcount, free_stack, free_count, max_tokens,
                      max_pages=0):
    return (pages.new_empty((pages.shape[0], max_pages or pages.shape[1])),
            torch.empty_like(lengths), torch.empty_like(refcount), torch.empty_like(free_stack),
            torch.empty_like(free_count), *_fake_plan_outputs(pages, max_tokens))


@torch.library.register_fake("branchcraft::append_plan_")
def _fake_append_plan_(pages, lengths, new_tokens, refcount, free_stack, free_count, max_tokens):
    return _fake_plan_outputs(pages, max_tokens)


@torch.library.register_fake("branchcraft::append_kv_")
def _fake_append_kv(cache_k, cache_v, k, v, slot_map, clones=None, counts=None):
    return None


@torch.library.register_fake("branchcraft::chunk_attention")
def _fake_chunk_attention(q, k, v, pages, query_start, lengths, scale=None, softcap=0.0, window=0,
                          alibi_slopes=None, prefix=None, key_start=None):
    return q.new_empty(q.shape)


@torch.library.register_fake("branchcraft::chunk_attention_out")
def _fake_chunk_attention_out(q, k, v, pages, query_start, lengths, output, scale=None,
                              softcap=0.0, window=0, alibi_slopes=None, prefix=None,
                              key_start=None):
    return output


@torch.library.register_fake("branchcraft::beam_select")
def _fake_beam_select(logits, scores, k):
    out = scores.new_empty((scores.shape[0], k))
    return out, out.new_empty(out.shape, dtype=torch.int32), out.new_empty(out.shape,
                                                                          dtype=torch.int32)


def _fake_rows(pages, parents):
    batch, beams = parents.shape
    return pages.new_empty((batch, beams, pages.shape[2])), pages.new_empty((batch, beams))


@torch.library.register_fake("branchcraft::beam_reorder")
def _fake_beam_reorder(pages, lengths, parents, refcount, free_stack, free_count):
    return (*_fake_rows(pages, parents), torch.empty_like(refcount), torch.empty_like(free_stack),
            torch.empty_like(free_count))


@torch.library.register_fake("branchcraft::beam_reorder_")
def _fake_beam_reorder_(pages, lengths, parents, refcount, free_stack, free_count):
    return _fake_rows(pages, parents)


def tree_verify(q, prefix_k, prefix_v, pages, lengths, draft_k, draft_v, parent):
    """Return FP32 [batch, candidate, query head, dimension] outputs."""
    return torch.ops.branchcraft.tree_verify(
        q, prefix_k, prefix_v, pages, lengths, draft_k, draft_v, parent)


def tree_verify_out(q, prefix_k, prefix_v, pages, lengths, draft_k, draft_v, parent, output):
    """Tree verify into a preallocated FP32 or FP16 output (CUDA-graph safe)."""
    return torch.ops.branchcraft.tree_verify_out(
        q, prefix_k, prefix_v, pages, lengths, draft_k, draft_v, parent, output)


def packed_decode_out(q, packed_kv, pages, lengths, output, scale):
    """Decode into a preallocated FP16 output (safe for CUDA graph capture)."""
    return torch.ops.branchcraft.packed_decode_out(q, packed_kv, pages, lengths, output, scale)


def packed_decode_kv_out(q, k_cache, v_cache, pages, lengths, output, scale, splits=0):
    """Decode from separate K / V views [P, Hkv, 16, D] of one cache (e.g. vLLM's
    [num_blocks, 2, 16, Hkv, D] as cache[:, 0].transpose(1, 2) and cache[:, 1]...)."""
    return torch.ops.branchcraft.packed_decode_kv_out(
        q, k_cache, v_cache, pages, lengths, output, scale, splits)


def paged_decode(q, k, v, pages, lengths, splits=0):
    """Paged GQA decode, FP32 [batch, query heads, dim]; splits 0 = automatic."""
    return torch.ops.branchcraft.paged_decode(q, k, v, pages, lengths, splits)


def commit_path_(cache_k, cache_v, draft_k, draft_v, path_nodes, dest_pages, dest_slots,
                 request):
    """Write accepted draft K/V to preallocated physical destinations."""
    return torch.ops.branchcraft.commit_path_(
        cache_k, cache_v, draft_k, draft_v, path_nodes, dest_pages, dest_slots, request)


def commit_batch_(cache_k, cache_v, draft_k, draft_v, clone_src, clone_dst, entry_request,
                  entry_node, entry_page, entry_slot):
    """All page clones of a commit plan, then all of its node writes."""
    return torch.ops.branchcraft.commit_batch_(
        cache_k, cache_v, draft_k, draft_v, clone_src, clone_dst, entry_request, entry_node,
        entry_page, entry_slot)


# (resolved once: a packet's look-up of its overload costs a step's small calls)
_append_plan = torch.ops.branchcraft.append_plan.default
_append_plan_ = torch.ops.branchcraft.append_plan_.default
_append_kv_ = torch.ops.branchcraft.append_kv_.default
_chunk_attention = torch.ops.branchcraft.chunk_attention.default
_chunk_attention_out = torch.ops.branchcraft.chunk_attention_out.default
_beam_select = torch.ops.branchcraft.beam_select.default
_beam_reorder = torch.ops.branchcraft.beam_reorder.default
_beam_reorder_ = torch.ops.branchcraft.beam_reorder_.default


def append_plan(pages, lengths, new_tokens, refcount, free_stack, free_count, max_tokens,
                max_pages=0):
    """Give every sequence's new tokens their pages and slots under the pool's rules (reference
    counts, free stack, copy-on-write). Returns the new (pages [S, max_pages or as before],
    lengths, refcount, free_stack, free_count) and (query_start [S + 1], slot_map [max_tokens],
    positions [max_tokens], clones [3, S], counts [3]: tokens, clones, status). A nonzero status
    (1 bad counts, 2 pool exhausted, 3 malformed tables) plans nothing."""
    return _append_plan(pages, lengths, new_tokens, refcount, free_stack, free_count, max_tokens,
                        max_pages)


def append_plan_(pages, lengths, new_tokens, refcount, free_stack, free_count, max_tokens):
    """append_plan updating tables, lengths and pool state in place; returns (query_start,
    slot_map, positions, clones, counts)."""
    return _append_plan_(pages, lengths, new_tokens, refcount, free_stack, free_count, max_tokens)


def append_kv_(cache_k, cache_v, k, v, slot_map, clones=None, counts=None):
    """Write k, v [tokens, Hkv, D] into the slots of a plan (-1: skipped), and copy its clones'
    valid slots, in one launch. Caches [P, 16, Hkv, D], strided views included."""
    return _append_kv_(cache_k, cache_v, k, v, slot_map, clones, counts)


def chunk_attention(q, k, v, pages, query_start, lengths, scale=None, softcap=0.0, window=0,
                    alibi_slopes=None, prefix=None, key_start=None):
    """Attention of new tokens q [tokens, Hq, D] (request b: rows query_start[b] ..
    query_start[b + 1], the last of its lengths[b] keys) over the paged caches k, v
    [P, 16, Hkv, D]. Causal; `prefix` [B] opens a request's leading keys to all its tokens,
    `window` keeps the last keys, `key_start` [tokens] is a token's first key (packed documents);
    `softcap` caps scores by a tanh, `alibi_slopes` [Hq] take slope * distance off. Output of q's
    type; rows of tokens in no request are unspecified (chunk_attention_out leaves them). A token
    that sees no key gets zeros, one that sees a score of NaN or +inf, or none above -inf, NaN."""
    return _chunk_attention(q, k, v, pages, query_start, lengths, scale, softcap, window,
                            alibi_slopes, prefix, key_start)


def chunk_attention_out(q, k, v, pages, query_start, lengths, output, scale=None, softcap=0.0,
                        window=0, alibi_slopes=None, prefix=None, key_start=None):
    """chunk_attention into a preallocated output (32-byte aligned, CUDA-graph safe) of q's type
    or FP32; for FP32 probabilities are held as two 16-bit numbers at up to 1.9 times the time."""
    return _chunk_attention_out(
        q, k, v, pages, query_start, lengths, output, scale, softcap, window, alibi_slopes,
        prefix, key_start)


def beam_select(logits, scores, k):
    """The k best (beam, token) pairs of every request by scores + log_softmax(logits):
    (scores [B, k] FP32, tokens [B, k], parents [B, k]), best first, ties to the lowest
    beam * vocab + token (all pairs of a beam whose score is -inf or NaN among them, at -inf).
    logits [B, beams, vocab], scores [B, beams] FP32."""
    return _beam_select(logits, scores, k)


def beam_reorder(pages, lengths, parents, refcount, free_stack, free_count):
    """Page tables [B, beams, max_pages] after parents [B, new beams] (-1 drops a row): returns
    (pages, lengths, refcount, free_stack, free_count), every new row forked from its parent,
    every old one released, unheld pages pushed on the free stack."""
    return _beam_reorder(pages, lengths, parents, refcount, free_stack, free_count)


def beam_reorder_(pages, lengths, parents, refcount, free_stack, free_count):
    """beam_reorder updating the pool's state in place; returns (pages, lengths)."""
    return _beam_reorder_(pages, lengths, parents, refcount, free_stack, free_count)
