"""The serving operators of prompts and beams, measured: their cases, their plain
forms in elementary torch operations, and the same passes through the
framework's kernels (``own``).

Operators (all over a pool of 16-token pages):
  plan     append_plan      page tables, slot map and positions of new tokens
  append   append_kv_       new K/V rows and page clones into the paged cache
  chunk    chunk_attention  attention of a chunk of new tokens over that cache
  select   beam_select      the best (beam, token) pairs of every request
  reorder  beam_reorder     page tables after the beams' new parents
"""
import math
import random
import sys

import torch

own = False

PAGE = 16
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _ops():
    if "branchcraft-cuda_b200" not in sys.path:
        sys.path.insert(0, "branchcraft-cuda_b200")
    import branchcraft_torch

    return branchcraft_torch


# ---------------------------------------------------------------------- cases


def listed():
    return [
        # One new token each of four long conversations: the serving step of single tokens.
        dict(name="chunk-single-4x32768", op="chunk", batch=4, q_heads=32, kv_heads=8, dim=128,
             dtype="fp16", new_min=1, new_max=1, ctx_min=32767, ctx_max=32767, ragged=1,
             softcap=0.0, window=0, alibi=False, prefix=False, documents=0),
        # A few drafted tokens on short prefixes of a small model with distance biases: latency.
        dict(name="chunk-few-2x7", op="chunk", batch=2, q_heads=8, kv_heads=2, dim=64,
             dtype="fp16", new_min=7, new_max=7, ctx_min=150, ctx_max=250, ragged=2,
             softcap=0.0, window=0, alibi=True, prefix=False, documents=0),
        # A whole long prompt in one chunk.
        dict(name="chunk-prompt-8192", op="chunk", batch=1, q_heads=32, kv_heads=8, dim=128,
             dtype="bf16", new_min=8192, new_max=8192, ctx_min=0, ctx_max=0, ragged=3,
             softcap=0.0, window=0, alibi=False, prefix=False, documents=0),
        # Continuous batching: single tokens and chunks of prompts together, an odd group of
        # seven heads, capped scores and a sliding window.
        dict(name="chunk-mixed-capped", op="chunk", batch=12, q_heads=28, kv_heads=4, dim=128,
             dtype="bf16", new_min=1, new_max=600, ctx_min=0, ctx_max=4096, ragged=4,
             softcap=30.0, window=1024, alibi=False, prefix=False, documents=0),
        # The next token's slot for 256 beams, eight to a request, their last pages shared.
        dict(name="plan-beams-256", op="plan", batch=256, beams=8, pool=32768, new_min=1,
             new_max=1, ctx_min=100, ctx_max=2000, width=256, spare=0, ragged=5),
        # The prompts of a full batch.
        dict(name="plan-prompts-64", op="plan", batch=64, beams=1, pool=16384, new_min=1,
             new_max=2048, ctx_min=0, ctx_max=1000, width=256, spare=1000, ragged=6),
        # One row a beam, some with a cloned page.
        dict(name="append-beams-64", op="append", batch=64, beams=8, pool=2048, kv_heads=8,
             dim=128, dtype="fp16", new_min=1, new_max=1, ctx_min=100, ctx_max=2000, fused=False,
             ragged=7),
        # Rows of long prompts out of a fused QKV projection.
        dict(name="append-prompts-16x2048", op="append", batch=16, beams=1, pool=8192, kv_heads=8,
             dim=128, dtype="bf16", new_min=500, new_max=2048, ctx_min=0, ctx_max=2000, fused=True,
             ragged=8),
        # One request's four beams, a vocabulary of ordinary size.
        dict(name="select-1x4x32000", op="select", batch=1, beams=4, vocab=32000, k=8,
             dtype="fp32", masked=True),
        # A batch of requests, eight beams each, a large vocabulary of odd size.
        dict(name="select-32x8x131071", op="select", batch=32, beams=8, vocab=131071, k=16,
             dtype="bf16", masked=False),
        # Two requests early in their search.
        dict(name="reorder-2x4", op="reorder", batch=2, beams=4, pool=2048, ctx_min=60,
             ctx_max=200, tail=2, common=0, ragged=9),
        # A full batch with a common system prompt and long contexts.
        dict(name="reorder-64x8", op="reorder", batch=64, beams=8, pool=65536, ctx_min=1000,
             ctx_max=4096, tail=12, common=32, ragged=10),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["chunk", "chunk", "plan", "append", "select", "reorder"])
    ragged = rng.randrange(1 << 20)
    if op == "chunk":
        kv = rng.choice([1, 2, 3, 4, 8])
        group = rng.choice([1, 2, 3, 4, 6, 7, 8])
        dim = rng.choice([64, 128])
        batch = _log(rng, 1, 24)
        ctx = _log(rng, 1, 16384)
        new = 1 if rng.random() < 0.25 else _log(rng, 2, 2048)
        # (the plain form's padded scores stay below those of the largest listed case)
        while batch * kv * group * new * (ctx + new) > 1.5e9 or batch * (ctx + new) * kv > 1 << 20:
            batch, new, ctx = max(1, batch // 2), max(1, new * 2 // 3), max(1, ctx * 2 // 3)
        even = rng.random() < 0.3
        return dict(op=op, batch=batch, q_heads=kv * group, kv_heads=kv, dim=dim,
                    dtype=rng.choice(["fp16", "bf16"]), new_min=new if even else 1, new_max=new,
                    ctx_min=ctx if even else 0, ctx_max=ctx, ragged=ragged,
                    softcap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                    window=rng.choice([0, 0, _log(rng, 1, 4096)]), alibi=rng.random() < 0.3,
                    prefix=rng.random() < 0.25, documents=rng.choice([0, 0, rng.randint(2, 6)]))
    if op == "plan":
        beams = rng.choice([1, 1, 2, 4, 5, 8])
        batch = beams * _log(rng, 1, 512 // beams)
        new = 1 if rng.random() < 0.5 else _log(rng, 2, 1000)
        return dict(op=op, batch=batch, beams=beams, pool=65536, new_min=rng.choice([0, 1]),
                    new_max=new, ctx_min=rng.choice([0, 17]), ctx_max=_log(rng, 20, 1000),
                    width=128 + rng.randint(0, 9), spare=rng.choice([0, 0, 333]), ragged=ragged)
    if op == "append":
        beams = rng.choice([1, 1, 4, 7])
        batch = beams * _log(rng, 1, 64 // beams)
        new = 1 if rng.random() < 0.4 else _log(rng, 2, 400)
        return dict(op=op, batch=batch, beams=beams, pool=8192, kv_heads=rng.choice([1, 2, 4, 8]),
                    dim=rng.choice([64, 128]), dtype=rng.choice(["fp16", "bf16"]), new_min=1,
                    new_max=new, ctx_min=0, ctx_max=_log(rng, 20, 1000),
                    fused=rng.random() < 0.5, ragged=ragged)
    if op == "select":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
        return dict(op=op, batch=_log(rng, 1, 64 // beams), beams=beams,
                    vocab=_log(rng, 500, 200000), k=rng.choice([1, 2, 4, 7, 16, 32]),
                    dtype=rng.choice(["fp32", "fp16", "bf16"]), masked=rng.random() < 0.5)
    beams = rng.choice([1, 2, 4, 5, 8, 16])
    return dict(op=op, batch=_log(rng, 1, 256 // beams), beams=beams, pool=65536,
                ctx_min=17, ctx_max=_log(rng, 40, 2000), tail=rng.randint(0, 16),
                common=rng.choice([0, 1]), ragged=ragged)


def _pages(tokens):
    return (tokens + PAGE - 1) // PAGE


def _ragged(c):
    """New tokens and context of every sequence: lists, by the case alone."""
    r = random.Random(c["ragged"])
    beams = c.get("beams", 1)
    new, ctx = [], []
    for g in range(c["batch"] // beams):
        length = r.randint(c["ctx_min"], c["ctx_max"])
        for _ in range(beams):
            ctx.append(length)
            # (half of a mixed batch has one token)
            one = c["new_min"] == 1 < c["new_max"] and r.random() < 0.5
            new.append(1 if one else r.randint(c["new_min"], c["new_max"]))
    return new, ctx


# --------------------------------------------------------------------- states


class State:
    def __init__(self, case, **fields):
        self.case = case
        self.__dict__.update(fields)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(c, g, new, ctx):
    """Tables, reference counts and free stack of `batch` sequences, the beams of a request
    sharing every page."""
    beams, pool = c["beams"], c["pool"]
    perm = torch.randperm(pool, generator=g, device="cuda").int()
    counts = _ints([_pages(x) for x in ctx[::beams]]).long()
    first = torch.cumsum(counts, 0) - counts
    width = max(c.get("width", 1), max(_pages(n + x) for n, x in zip(new, ctx)))
    col = torch.arange(width, device="cuda")
    used = col[None] < counts[:, None]
    rows = torch.where(used, perm[(first[:, None] + col).clamp(max=pool - 1)], -1)
    table = rows.repeat_interleave(beams, 0).contiguous()
    total = sum(_pages(x) for x in ctx[::beams])
    refcount = torch.zeros(pool, dtype=torch.int32, device="cuda")
    refcount[perm[:total].long()] = beams
    stack = torch.zeros(pool, dtype=torch.int32, device="cuda")
    stack[: pool - total] = perm[total:]
    return table, refcount, stack, _ints([pool - total])


def _prepare_chunk(c, seed):
    g = _gen(seed)
    dt = DTYPES[c["dtype"]]
    new, ctx = _ragged(c)
    lens = [n + x for n, x in zip(new, ctx)]
    need = [_pages(x) for x in lens]
    width, pool = max(need), sum(need) + 5
    perm = torch.randperm(pool, generator=g, device="cuda").int()
    cnt = _ints(need).long()
    first = torch.cumsum(cnt, 0) - cnt
    col = torch.arange(width, device="cuda")
    pages = torch.where(col[None] < cnt[:, None], perm[(first[:, None] + col).clamp(max=pool - 1)], -1)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dt)

    tokens = sum(new)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    r = random.Random(c["ragged"] + 1)
    key_start = prefix = slopes = None
    if c["documents"]:  # packed documents: a token's keys begin where its document begins
        key_start = []
        for n, x in zip(new, ctx):
            cuts = sorted([0] + [r.randrange(0, n + x) for _ in range(c["documents"] - 1)])
            key_start += [max(d for d in cuts if d <= x + i) for i in range(n)]
        key_start = _ints(key_start)
    if c["prefix"]:  # a prompt's leading part attends in both directions
        prefix = _ints([r.randint(0, x) for x in lens])
    if c["alibi"]:
        slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / c["q_heads"]) for h in range(c["q_heads"])],
                              dtype=torch.float32, device="cuda")
    return State(c, q=rand(tokens, c["q_heads"], c["dim"]), k=rand(pool, PAGE, c["kv_heads"], c["dim"]),
                 v=rand(pool, PAGE, c["kv_heads"], c["dim"]), pages=pages.contiguous(),
                 query_start=_ints(starts), lengths=_ints(lens), scale=1 / math.sqrt(c["dim"]),
                 softcap=c["softcap"], window=c["window"], slopes=slopes, prefix=prefix,
                 key_start=key_start, new_max=max(new))


def _prepare_plan(c, seed):
    new, ctx = _ragged(c)
    table, refcount, stack, count = _tables(c, _gen(seed), new, ctx)
    return State(c, pages=table, lengths=_ints(ctx), new=_ints(new), refcount=refcount, stack=stack,
                 count=count, max_tokens=sum(new) + c["spare"])


def _prepare_append(c, seed):
    g = _gen(seed)
    s = _prepare_plan(dict(c, width=1, spare=0), seed)
    _, _, _, _, _, _, slot_map, _, clones, counts = _plain_plan(s)
    dt, heads, dim, tokens = DTYPES[c["dtype"]], c["kv_heads"], c["dim"], s.max_tokens

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dt)

    if c["fused"]:  # K and V out of one projection of four query heads a KV head
        x = rand(tokens, 6 * heads, dim)
        k, v = x[:, 4 * heads:5 * heads], x[:, 5 * heads:]
    else:
        k, v = rand(tokens, heads, dim), rand(tokens, heads, dim)
    return State(c, cache_k=rand(c["pool"], PAGE, heads, dim), cache_v=rand(c["pool"], PAGE, heads, dim),
                 k=k, v=v, slot_map=slot_map, clones=clones, counts=counts)


def _prepare_select(c, seed):
    g = _gen(seed)
    x = torch.randn(c["batch"], c["beams"], c["vocab"], generator=g, device="cuda") * 2.5
    if c["masked"]:  # tokens that a grammar forbids
        drop = torch.rand(c["batch"], 1, c["vocab"], generator=g, device="cuda") < 0.6
        x = x.masked_fill(drop, -math.inf)
    scores = -10 * torch.rand(c["batch"], c["beams"], generator=g, device="cuda")
    return State(c, logits=x.to(DTYPES[c["dtype"]]), scores=scores, k=c["k"])


def _prepare_reorder(c, seed):
    g = _gen(seed)
    w, batch, pool = c["beams"], c["batch"], c["pool"]
    r = random.Random(c["ragged"])
    lens = [r.randint(c["ctx_min"], c["ctx_max"]) for _ in range(batch)]
    need = _ints([_pages(x) for x in lens])[:, None, None].long()
    tail = torch.minimum(_ints([r.randint(0, c["tail"]) for _ in range(batch)])[:, None, None].long(),
                         need - c["common"])
    width = max(_pages(x) for x in lens)
    col = torch.arange(width, device="cuda")[None, None]
    beam = torch.arange(w, device="cuda")[None, :, None]
    # page identities: common to all, one a request, or one a beam (its own last pages)
    base = c["common"] + torch.arange(batch, device="cuda")[:, None, None] * width * (w + 1)
    ident = torch.where(col < c["common"], col, torch.where(
        col < need - tail, base + col, base + (beam + 1) * width + col)).expand(batch, w, width)
    used = (col < need).expand(batch, w, width)
    distinct, index = torch.unique(ident[used], return_inverse=True)
    perm = torch.randperm(pool, generator=g, device="cuda")
    table = torch.full((batch, w, width), -1, dtype=torch.int32, device="cuda")
    table[used] = perm[index].int()
    refcount = torch.zeros(pool, dtype=torch.int32, device="cuda")
    refcount.index_add_(0, table[used].long(), torch.ones_like(table[used]))
    taken = distinct.numel()
    stack = torch.zeros(pool, dtype=torch.int32, device="cuda")
    stack[: pool - taken] = perm[taken:].int()
    parents = torch.randint(0, w, (batch, w), generator=g, device="cuda").int()
    lengths = _ints(lens)[:, None].expand(batch, w).contiguous()
    return State(c, pages=table, lengths=lengths, parents=parents, refcount=refcount, stack=stack,
                 count=_ints([pool - taken]))


def prepare(case, seed):
    return {"chunk": _prepare_chunk, "plan": _prepare_plan, "append": _prepare_append,
            "select": _prepare_select, "reorder": _prepare_reorder}[case["op"]](case, seed)


# ---------------------------------------------------------------- plain forms


def _plain_chunk(s):
    batch, width = s.pages.shape
    hq, dim = s.q.shape[1:]
    hkv = s.k.shape[2]
    group, keys, dev = hq // hkv, width * PAGE, s.q.device
    start, length = s.query_start.long(), s.lengths.long()
    new = start[1:] - start[:-1]
    token = start[:-1, None] + torch.arange(s.new_max, device=dev)       # [B, n]
    inside = token < start[1:, None]
    token = token.clamp(max=s.q.shape[0] - 1)
    ids = s.pages.clamp(min=0).long()
    k = s.k[ids].reshape(batch, keys, hkv, dim).permute(0, 2, 3, 1).float()
    v = s.v[ids].reshape(batch, keys, hkv, dim).permute(0, 2, 1, 3).float()
    q = s.q[token].float().reshape(batch, s.new_max, hkv, group, dim).permute(0, 2, 3, 1, 4)
    x = torch.matmul(q.reshape(batch, hkv, group * s.new_max, dim), k)
    x = x.reshape(batch, hkv, group, s.new_max, keys).mul_(s.scale)
    pos = (length - new)[:, None] + torch.arange(s.new_max, device=dev)  # [B, n]
    j = torch.arange(keys, device=dev)
    if s.softcap:
        x = x.div_(s.softcap).tanh_().mul_(s.softcap)
    if s.slopes is not None:
        far = (pos[:, :, None] - j).abs().float()[:, None, None]
        x = x.sub_(s.slopes.reshape(hkv, group, 1, 1) * far)
    lo = torch.zeros_like(pos)
    hi = pos + 1
    if s.window:
        lo = torch.maximum(lo, pos + 1 - s.window)
    if s.key_start is not None:
        lo = torch.maximum(lo, s.key_start[token].long())
    if s.prefix is not None:
        hi = torch.maximum(hi, torch.minimum(s.prefix.long(), length)[:, None])
    seen = (j >= lo[:, :, None]) & (j < hi[:, :, None])                  # [B, n, keys]
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    x = x.sub_(m).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.reshape(batch, hkv, group * s.new_max, keys), v)
    o = o.reshape(batch, hkv, group, s.new_max, dim) / torch.where(total == 0, torch.ones_like(total), total)
    o = o.permute(0, 3, 1, 2, 4).reshape(batch, s.new_max, hq, dim)
    return o[inside].to(s.q.dtype)


def _plain_plan(s):
    batch, width = s.pages.shape
    dev = s.pages.device
    row = torch.arange(batch, device=dev)
    old, new = s.lengths.long(), s.new.long()
    have, want = (old + PAGE - 1) // PAGE, (old + new + PAGE - 1) // PAGE
    last = s.pages[row, (have - 1).clamp(min=0)].long()
    partial = (old % PAGE != 0) & (new > 0)
    # rank of a sequence among those that write into the same partial page
    key = torch.where(partial, last, s.refcount.numel() + row)
    order = torch.argsort(key, stable=True)
    head = torch.ones_like(key, dtype=torch.bool)
    head[1:] = key[order][1:] != key[order][:-1]
    begin = torch.cummax(torch.where(head, row, torch.zeros_like(row)), 0).values
    rank = torch.empty_like(row)
    rank[order] = row - begin
    clone = partial & (rank < s.refcount[last.clamp(min=0)] - 1)
    pops = want - have + clone
    first = torch.cumsum(pops, 0) - pops
    top = s.count.long() - 1

    def popped(i):
        return s.stack[(top - i).clamp(min=0)]

    col = torch.arange(width, device=dev)[None]
    fresh = popped(first[:, None] + clone[:, None] + col - have[:, None])
    table = torch.where(col < have[:, None], s.pages, torch.where(col < want[:, None], fresh, -1))
    moved = clone[:, None] & (col == have[:, None] - 1)
    table = torch.where(moved, popped(first)[:, None], table)
    refcount = s.refcount.clone()
    taken = pops.sum()
    place = torch.arange(s.stack.numel(), device=dev)
    window = (place <= top) & (place > top - taken)
    refcount.index_add_(0, s.stack.long(), window.int())
    refcount.index_add_(0, torch.where(clone, last, 0), -clone.int())
    start = torch.zeros(batch + 1, dtype=torch.int64, device=dev)
    start[1:] = torch.cumsum(new, 0)
    t = torch.arange(s.max_tokens, device=dev)
    owner = (torch.searchsorted(start, t, right=True) - 1).clamp(max=batch - 1)
    pos = old[owner] + t - start[owner]
    live = t < start[-1]
    page = table[owner, (pos // PAGE).clamp(max=width - 1)].long()
    slot_map = torch.where(live, page * PAGE + pos % PAGE, -1).int()
    positions = torch.where(live, pos, -1).int()
    at = torch.cumsum(clone, 0) - 1
    clones = torch.full((3, batch + 1), -1, dtype=torch.int32, device=dev)
    to = torch.where(clone, at, batch)
    clones[0].scatter_(0, to, last.int())
    clones[1].scatter_(0, to, popped(first))
    clones[2].scatter_(0, to, (old % PAGE).int())
    counts = torch.stack([start[-1], clone.sum(), torch.zeros_like(taken)]).int()
    return (table, (old + new).int(), refcount, s.stack.clone(), (s.count - taken).int(), start.int(),
            slot_map, positions, clones[:, :batch].contiguous(), counts)


def _plain_append(s):
    heads, dim = s.k.shape[1:]
    slot = torch.arange(PAGE, device=s.k.device)
    src, dst, valid = (x.long()[:, None] for x in s.clones)
    copied = (slot < valid) & (src >= 0)
    to, of = (dst * PAGE + slot)[copied], (src * PAGE + slot)[copied]
    live = s.slot_map >= 0
    at = s.slot_map[live].long()
    k, v = s.cache_k.view(-1, heads, dim), s.cache_v.view(-1, heads, dim)
    k[to], v[to] = k[of], v[of]
    k[at], v[at] = s.k[live], s.v[live]
    return s.cache_k, s.cache_v


def _plain_select(s):
    batch, beams, vocab = s.logits.shape
    # (64 bits: the order of two beams' candidates hangs on the last digits of their sums)
    x = s.logits.double()
    m = x.amax(-1, keepdim=True)
    x = x - m - (x - m).exp().sum(-1, keepdim=True).log()
    x = x + s.scores.double()[:, :, None]
    value, index = torch.sort(x.reshape(batch, beams * vocab), dim=1, descending=True, stable=True)
    value, index = value[:, :s.k], index[:, :s.k]
    return value.float(), (index % vocab).int(), (index // vocab).int()


def _plain_reorder(s):
    batch, w, width = s.pages.shape
    dev, pool = s.pages.device, s.refcount.numel()
    parent = s.parents.long()
    pages = torch.gather(s.pages, 1, parent[:, :, None].expand(batch, w, width))
    lengths = torch.gather(s.lengths, 1, parent)
    children = torch.zeros(batch, w, dtype=torch.int32, device=dev)
    children.scatter_add_(1, parent, torch.ones_like(s.parents))
    used = s.pages >= 0
    at = torch.where(used, s.pages.long(), pool).reshape(-1)
    change = (children - 1)[:, :, None].expand(batch, w, width).reshape(-1)
    refcount = torch.cat([s.refcount, s.refcount.new_zeros(1)]).index_add(0, at, change.contiguous())[:pool]
    # freed pages, in the order of their last release
    seen = torch.full((pool + 1,), -1, dtype=torch.int64, device=dev)
    seen.scatter_reduce_(0, at, torch.arange(at.numel(), device=dev), "amax")
    freed = (refcount == 0) & (s.refcount > 0)
    order = torch.argsort(torch.where(freed, seen[:pool], at.numel()), stable=True)
    place = s.count.long() + torch.arange(pool, device=dev)
    pushed = torch.arange(pool, device=dev) < freed.sum()
    stack = torch.cat([s.stack, s.stack.new_zeros(1)])
    stack = stack.scatter(0, torch.where(pushed, place, pool), order.int())[:pool]
    return pages, lengths, refcount, stack, (s.count + freed.sum()).int()


def run(state):
    s, op = state, state.case["op"]
    if own:
        b = _ops()
        if op == "chunk":
            return b.chunk_attention(s.q, s.k, s.v, s.pages, s.query_start, s.lengths, scale=s.scale,
                                     softcap=s.softcap, window=s.window, alibi_slopes=s.slopes,
                                     prefix=s.prefix, key_start=s.key_start)
        if op == "plan":
            return b.append_plan(s.pages, s.lengths, s.new, s.refcount, s.stack, s.count, s.max_tokens)
        if op == "append":
            b.append_kv_(s.cache_k, s.cache_v, s.k, s.v, s.slot_map, s.clones, s.counts)
            return s.cache_k, s.cache_v
        if op == "select":
            return b.beam_select(s.logits, s.scores, s.k)
        return b.beam_reorder(s.pages, s.lengths, s.parents, s.refcount, s.stack, s.count)
    return {"chunk": _plain_chunk, "plan": _plain_plan, "append": _plain_append,
            "select": _plain_select, "reorder": _plain_reorder}[op](s)


# ----------------------------------------------------------------------- work


def work(case):
    c, op = case, case["op"]
    if op == "chunk":
        new, ctx = _ragged(c)
        r = random.Random(c["ragged"] + 1)
        pairs = keys = 0
        docs = []
        if c["documents"]:
            for n, x in zip(new, ctx):
                docs.append(sorted([0] + [r.randrange(0, n + x) for _ in range(c["documents"] - 1)]))
        tops = [r.randint(0, n + x) for n, x in zip(new, ctx)] if c["prefix"] else [0] * len(new)
        for b, (n, x) in enumerate(zip(new, ctx)):
            low, high = n + x, 0
            for i in range(n):
                p = x + i
                hi = max(p + 1, tops[b])
                lo = max(0, p + 1 - c["window"]) if c["window"] else 0
                if docs:
                    lo = max(lo, max(d for d in docs[b] if d <= p))
                pairs += hi - lo
                low, high = min(low, lo), max(high, hi)
            keys += high - low
        rows = 2 * sum(new) * c["q_heads"] * c["dim"] * 2
        return {"bytes": rows + keys * c["kv_heads"] * c["dim"] * 4 + 4 * (keys // PAGE + 2 * len(new)),
                "flops": 4 * c["dim"] * c["q_heads"] * pairs}
    if op in ("plan", "append"):
        new, ctx = _ragged(c)
        shared = sum(1 for x in ctx if x % PAGE) * (c["beams"] - 1) // c["beams"]
        if op == "append":
            row = c["kv_heads"] * c["dim"] * 4
            return {"bytes": 2 * row * (sum(new) + shared * PAGE // 2) + 4 * sum(new), "flops": 0}
        width = max(c["width"], max(_pages(n + x) for n, x in zip(new, ctx)))
        table = sum(_pages(x) for x in ctx) + c["batch"] * width
        return {"bytes": 4 * (table + 4 * c["pool"] + 5 * c["batch"] + 2 * (sum(new) + c["spare"])),
                "flops": 0}
    if op == "select":
        n = c["batch"] * c["beams"] * c["vocab"]
        return {"bytes": n * DTYPES[c["dtype"]].itemsize + c["batch"] * (4 * c["beams"] + 12 * c["k"]),
                "flops": 4 * n}
    r = random.Random(c["ragged"])
    lens = [r.randint(c["ctx_min"], c["ctx_max"]) for _ in range(c["batch"])]
    rows = c["batch"] * c["beams"]
    table = sum(_pages(x) for x in lens) * c["beams"] + rows * max(_pages(x) for x in lens)
    return {"bytes": 4 * (table + 4 * c["pool"] + 3 * rows), "flops": 0}


# ---------------------------------------------------------------------- exact


def _exact_chunk(case, seed):
    s = prepare(case, seed)
    hq, dim = s.q.shape[1:]
    hkv = s.k.shape[2]
    group = hq // hkv
    starts, lens = s.query_start.tolist(), s.lengths.tolist()
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    for b, length in enumerate(lens):
        t0, t1 = starts[b], starts[b + 1]
        ids = s.pages[b, :_pages(length)].long()
        j = torch.arange(length, device="cuda")
        for a in range(t0, t1, 1024):  # rows of at most 1024 tokens at a time
            e = min(a + 1024, t1)
            p = length - (t1 - t0) + torch.arange(a - t0, e - t0, device="cuda")
            first, end = torch.zeros_like(p), p + 1
            if s.window:
                first = (p + 1 - s.window).clamp(min=0)
            if s.key_start is not None:
                first = torch.maximum(first, s.key_start[a:e].long())
            if s.prefix is not None:
                end = end.clamp(min=min(int(s.prefix[b]), length))
            hidden = (j[None] < first[:, None]) | (j[None] >= end[:, None])
            for h in range(hq):
                kk = s.k[ids, :, h // group].reshape(-1, dim)[:length].double()
                vv = s.v[ids, :, h // group].reshape(-1, dim)[:length].double()
                x = (s.q[a:e, h].double() @ kk.T) / math.sqrt(dim)
                if s.softcap:
                    x = s.softcap * torch.tanh(x / s.softcap)
                if s.slopes is not None:
                    x = x - float(s.slopes[h]) * (p[:, None] - j[None]).abs().double()
                x[hidden] = -math.inf
                out[a:e, h] = torch.nan_to_num(torch.softmax(x, -1), nan=0.0) @ vv
    return out


def _exact_select(case, seed):
    s = prepare(case, seed)
    best = []
    for b in range(case["batch"]):
        x = s.logits[b].double()
        p = torch.log_softmax(x, -1) + s.scores[b, :, None].double()
        best.append(torch.topk(p.reshape(-1), case["k"]).values)
    return torch.stack(best), None, None


def exact(case, seed):
    if case["op"] == "chunk":
        return _exact_chunk(case, seed)
    if case["op"] == "select":
        return _exact_select(case, seed)
    return None  # page ids and copied bytes: nothing is computed in floating point
