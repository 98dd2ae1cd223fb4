"""Plain restatements of the prompt and beam operators for the tests: the page
bookkeeping on the host pool's own primitives (bc_cow.PagePool: alloc, release,
fork), attention and beam scores in 64 bits, and bounds on what the kernels'
roundings may do to them."""
from __future__ import annotations

import copy
import math

import numpy as np
import torch

from bc_cow import PagePool


# ---------------------------------------------------------------- page plans


def append_sequential(pool: PagePool, requests, new_tokens):
    """The pool after `new_tokens`, one request after the other; returns the
    slot map, positions and clones. Raises RuntimeError where pages run out
    (the pool is then unchanged)."""
    before = copy.deepcopy(pool.__dict__)
    slots, positions, clones = [], [], []
    try:
        for r, n in zip(requests, new_tokens):
            length, row = pool.lengths[r], pool.pages[r]
            if n > 0 and length % 16 and pool.refcount[row[-1]] > 1:
                old, fresh = row[-1], pool.alloc()
                clones.append((old, fresh, length % 16))
                row[-1] = fresh
                pool.release(old)
            while len(row) * 16 < length + n:
                row.append(pool.alloc())
            for pos in range(length, length + n):
                slots.append(row[pos // 16] * 16 + pos % 16)
                positions.append(pos)
            pool.lengths[r] = length + n
    except RuntimeError:
        pool.__dict__.update(before)
        raise
    return slots, positions, clones


def reorder_sequential(pool: PagePool, beams, parents):
    """beams [batch][beams_in]: request ids of the pool; parents [batch][beams_out].
    Forks every new row, then releases every old one, in order. Returns the new
    request ids (None: an empty row)."""
    made = [[None if p < 0 else pool.fork(beams[b][p]) for p in row]
            for b, row in enumerate(parents)]
    for row in beams:
        for r in row:
            for page in pool.pages.pop(r):
                pool.release(page)
            del pool.lengths[r]
    return made


def device_state(pool: PagePool, device="cuda"):
    def t(x):
        return torch.tensor(x, dtype=torch.int32, device=device)

    return (t(pool.refcount), t(pool.free + [0] * (pool.physical_pages - len(pool.free))),
            t([len(pool.free)]))


def assert_pool(pool: PagePool, refcount, stack, count):
    assert refcount.tolist() == pool.refcount
    assert int(count.item()) == len(pool.free)
    assert stack[:len(pool.free)].tolist() == pool.free


# ------------------------------------------------------------------ attention


def visible(length, n, window=0, prefix=0, key_start=None):
    """[n, length] truth: which keys each new token sees."""
    pos = length - n + torch.arange(n)[:, None]
    j = torch.arange(length)[None]
    hi = torch.clamp(pos + 1, min=min(prefix, length))
    lo = pos + 1 - window if window else torch.zeros_like(pos)
    if key_start is not None:
        lo = torch.maximum(lo, torch.as_tensor(key_start).long()[:, None])
    return (j >= lo) & (j < hi)


def chunk_attention(q, k, v, pages, query_start, lengths, scale=None, softcap=0.0, window=0,
                    alibi_slopes=None, prefix=None, key_start=None):
    """(out, spread, score error) in float64 on the CPU: spread = sum_j p_j |v_j|
    per element, score error = the largest sum_d |q_d k_d| * scale of a row."""
    q, k, v = (t.detach().cpu() for t in (q, k, v))
    pages, query_start, lengths = (t.cpu().tolist() for t in (pages, query_start, lengths))
    hq, dim = q.shape[1:]
    group = hq // k.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64)
    spread = torch.zeros_like(out)
    big = torch.zeros(q.shape[0], hq, 1, dtype=torch.float64)
    for b, length in enumerate(lengths):
        a, e = query_start[b], query_start[b + 1]
        if e <= a or length == 0:
            continue
        ids = [p if 0 <= p < k.shape[0] else -1 for p in pages[b][:(length + 15) // 16]]
        seen = visible(length, e - a, window, int(prefix[b]) if prefix is not None else 0,
                       None if key_start is None else key_start.cpu()[a:e])

        def gather(cache, h):
            rows = [cache[p, :, h] if p >= 0 else torch.zeros(16, dim, dtype=cache.dtype)
                    for p in ids]
            x = torch.cat(rows)[:length].double()
            return torch.where(seen.any(0)[:, None], x, torch.zeros_like(x))

        dist = (length - (e - a) + torch.arange(e - a)[:, None] - torch.arange(length)).abs()
        for g in range(k.shape[2]):
            kk, vv = gather(k, g), gather(v, g)
            for h in range(g * group, (g + 1) * group):
                qq = q[a:e, h].double()
                x = qq @ kk.T * scale
                big[a:e, h, 0] = (qq.abs() @ kk.abs().T * scale).masked_fill(~seen, 0).amax(1)
                if softcap:
                    x = softcap * torch.tanh(x / softcap)
                if alibi_slopes is not None:
                    x = x - float(alibi_slopes[h]) * dist
                x = x.masked_fill(~seen, -math.inf)
                m = x.amax(1, keepdim=True)
                p = torch.where(seen, torch.exp(x - torch.where(m == -math.inf, 0.0, m)), 0.0)
                p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
                out[a:e, h] = p @ vv
                spread[a:e, h] = p @ vv.abs()
    return out, spread, big


def assert_chunk_close(got, want, dtype, out_dtype=None):
    """|error| <= the output's rounding, plus the probabilities' rounding to
    `dtype` (half a step each, weighted by |v|), plus FP32 scores: a sum of D
    products within (D + 8) 2^-23 of sum |q_d k_d| (two roundings of 2^-24 a
    term), which moves a probability and the sum by that much each; the
    exponential and the output's own arithmetic within 2^-16."""
    out, spread, big = want
    out_dtype = out_dtype or got.dtype
    u = torch.finfo(dtype).eps / 2
    uo = torch.finfo(out_dtype).eps / 2
    dim = out.shape[-1]
    score = 2 * (dim + 8) * 2.0 ** -23 * big
    tol = uo * out.abs() + spread * (1 + uo) * (u + score + 2.0 ** -16)
    # a value below the type's normal range is rounded to its smallest step
    tol = tol + torch.finfo(out_dtype).smallest_normal * uo * 2
    err = (got.detach().cpu().double() - out).abs()
    assert torch.isfinite(got).all(), "non-finite output"
    bad = err > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside; worst " \
                          f"{float((err / tol).max()):.2f} of the tolerance at " \
                          f"{np.unravel_index(int((err / tol).argmax()), err.shape)}"


# ----------------------------------------------------------------------- beams


def beam_scores(logits, scores):
    """[batch, beams, vocab] float64 candidates."""
    x = logits.detach().cpu().double()
    x = torch.where(torch.isnan(x), -math.inf, x).clamp(max=float(torch.finfo(logits.dtype).max))
    m = x.amax(-1, keepdim=True)
    safe = torch.where(m == -math.inf, 0.0, m)
    total = torch.exp(x - safe).sum(-1, keepdim=True).log()
    s = scores.detach().cpu().double()
    s = torch.where(torch.isnan(s), -math.inf, s)[:, :, None]
    c = s + (x - safe - total)
    return torch.where((m == -math.inf) | (s == -math.inf) | (x == -math.inf), -math.inf, c)


def beam_select(logits, scores, k):
    c = beam_scores(logits, scores)
    batch, beams, vocab = c.shape
    order = np.argsort(-c.reshape(batch, -1).numpy(), axis=1, kind="stable")[:, :k]
    order = torch.from_numpy(np.ascontiguousarray(order))
    return c.reshape(batch, -1).gather(1, order), order % vocab, order // vocab
