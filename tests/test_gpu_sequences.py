"""The prompt and beam operators together, as a serving loop runs them: prompts
in chunks, then a beam search, over one pool on the device. Every step's
attention is checked against the formula on the rows' own token histories, every
selection against 64-bit scores, and the pool against the host's."""
import math

import numpy as np
import pytest
import torch

import serving_oracle as S
from bc_cow import PagePool

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def bc():
    import branchcraft_torch

    return branchcraft_torch


def ints(x):
    return torch.tensor(np.asarray(x, np.int32), device="cuda")


class Toy:
    """K, V, Q of a token by table and position; logits by a random projection."""

    def __init__(self, vocab, hq, hkv, dim, dtype, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def rand(*shape):
            return torch.randn(*shape, generator=g, device="cuda")

        self.k, self.v, self.q = (rand(vocab, h, dim) for h in (hkv, hkv, hq))
        self.pos = rand(512, 1, dim) * 0.5
        self.out = rand(hq * dim, vocab) * 0.2
        self.dtype = dtype

    def rows(self, tokens, positions):
        t, p = tokens.long(), positions.long().clamp(min=0)
        return ((self.q[t] + self.pos[p]).to(self.dtype), (self.k[t] + self.pos[p]).to(self.dtype),
                self.v[t].to(self.dtype))

    def logits(self, o):
        return o.float().flatten(1) @ self.out


def dense(toy, histories, starts, q, **options):
    """The oracle's attention of each row's last tokens over its own history."""
    need = [(len(h) + 15) // 16 for h in histories]
    width = max(1, max(need))
    hkv, dim = toy.k.shape[1:]
    pool = max(1, sum(need))
    k = torch.zeros(pool, 16, hkv, dim, dtype=toy.dtype, device="cuda")
    v = torch.zeros_like(k)
    pages, at = [], 0
    for h, n in zip(histories, need):
        if h:
            _, kk, vv = toy.rows(ints(h), torch.arange(len(h), device="cuda"))
            k.view(-1, hkv, dim)[at * 16:at * 16 + len(h)] = kk
            v.view(-1, hkv, dim)[at * 16:at * 16 + len(h)] = vv
        pages.append(list(range(at, at + n)) + [-1] * (width - n))
        at += n
    return S.chunk_attention(q, k, v, ints(pages), ints(starts), ints([len(h) for h in histories]),
                             **options)


@pytest.mark.parametrize("dtype,dim,options", [
    (torch.float16, 64, {}), (torch.bfloat16, 128, dict(softcap=20.0, window=40))])
def test_beam_search(bc, dtype, dim, options):
    from branchcraft_torch.sequences import PagedSequences

    requests, beams, hq, hkv, vocab = 5, 4, 6, 2, 211
    toy = Toy(vocab, hq, hkv, dim, dtype)
    rng = np.random.default_rng(dim)
    rows = requests * beams
    seq = PagedSequences(requests, beams, 12, 300, hkv, dim, dtype)
    pool = PagePool(300)
    ids = [[pool.new(0) for _ in range(beams)] for _ in range(requests)]
    histories = [[] for _ in range(rows)]

    def step(new):  # new: row -> tokens
        counts = [len(new.get(r, [])) for r in range(rows)]
        tokens = ints([t for r in range(rows) for t in new.get(r, [])])
        spare = 3  # capacity beyond the tokens, as a captured step has
        tokens = torch.cat([tokens, ints([0] * spare)])
        for r, ts in new.items():
            histories[r] += ts
        pos = [len(histories[r]) - c + i for r, c in enumerate(counts) for i in range(c)]
        q, k, v = toy.rows(tokens, ints(pos + [0] * spare))
        start, positions = seq.append(k, v, ints(counts))
        seq.check()
        assert start.tolist() == [0, *np.cumsum(counts).tolist()]
        assert positions.tolist() == pos + [-1] * spare
        S.append_sequential(pool, [r for row in ids for r in row], counts)
        n = sum(counts)
        out = torch.full(q.shape, 3.0, dtype=dtype, device="cuda")
        bc.chunk_attention_out(q, seq.k, seq.v, seq.pages, start, seq.lengths, out, **options)
        S.assert_chunk_close(out[:n], dense(toy, histories, start.tolist(), q[:n], **options), dtype)
        assert (out[n:] == 3).all()
        assert torch.equal(seq.attend(q, start, **options)[:n], out[:n])
        return out, start

    # the prompts, in two chunks, into the first beam of each request
    prompts = [rng.integers(0, vocab, size=int(n)).tolist() for n in (1, 16, 33, 70, 5)]
    step({r * beams: p[:len(p) // 2] for r, p in enumerate(prompts)})
    out, start = step({r * beams: p[len(p) // 2:] for r, p in enumerate(prompts)})
    last = start.long()[1::beams] - 1
    logits = toy.logits(out[last])[:, None]                      # [requests, 1, vocab]
    scores = torch.zeros(requests, 1, device="cuda")
    for _ in range(20):
        want = S.beam_select(logits, scores, beams)
        scores, token, parent = bc.beam_select(logits, scores, beams)
        t, p = token.cpu(), parent.cpu()
        assert t.tolist() == want[1].tolist() and p.tolist() == want[2].tolist()
        made = S.reorder_sequential(pool, ids, parent.tolist())
        seq.reorder(parent)
        ids = made
        histories = [list(histories[r * beams + q]) for r in range(requests) for q in p[r].tolist()]
        assert seq.lengths.tolist() == [len(h) for h in histories]
        S.assert_pool(pool, seq.refcount, seq.free_stack, seq.free_count)
        out, start = step({r * beams + j: [int(t[r, j])] for r in range(requests)
                           for j in range(beams)})
        assert seq.pages.tolist() == pool.page_table([r for row in ids for r in row], 12)
        logits = toy.logits(out[:rows]).view(requests, beams, vocab)
    # the requests end: every page comes back
    seq.reorder(torch.full((requests, beams), -1, dtype=torch.int32, device="cuda"))
    S.reorder_sequential(pool, ids, [[-1] * beams] * requests)
    S.assert_pool(pool, seq.refcount, seq.free_stack, seq.free_count)
    assert int(seq.free_count) == 300


def test_exhaustion_appends_nothing(bc):
    from branchcraft_torch.sequences import PagedSequences

    seq = PagedSequences(2, 1, 8, 4, 1, 64)
    k = torch.ones(60, 1, 64, dtype=torch.float16, device="cuda")
    seq.append(k, k, ints([30, 20]))
    seq.check()
    before = [t.clone() for t in (seq.k, seq.pages, seq.lengths, seq.refcount, seq.free_count)]
    start, positions = seq.append(k + 1, k, ints([30, 20]))
    assert start.tolist() == [0, 0, 0] and (positions == -1).all()
    for a, b in zip(before, (seq.k, seq.pages, seq.lengths, seq.refcount, seq.free_count)):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="exhausted"):
        seq.check()
    seq.append(k, k, ints([70, -1]))
    with pytest.raises(ValueError):
        seq.check()


def test_captured_decode_loop(bc):
    """One captured step (rows, attention, selection, reordering), replayed: the state
    advances on the device alone and equals the same steps issued one by one."""
    from branchcraft_torch.sequences import PagedSequences

    requests, beams, hq, hkv, dim, vocab = 3, 4, 4, 2, 64, 97
    toy = Toy(vocab, hq, hkv, dim, torch.float16, seed=5)
    rows = requests * beams

    def make():
        seq = PagedSequences(requests, beams, 8, 120, hkv, dim)
        state = dict(token=torch.zeros(rows, dtype=torch.int32, device="cuda"),
                     scores=torch.zeros(requests, beams, device="cuda"), seq=seq)
        state["scores"][:, 1:] = -math.inf  # one beam at first
        return state

    ones = torch.ones(rows, dtype=torch.int32, device="cuda")

    def step(s):
        seq = s["seq"]
        q, k, v = toy.rows(s["token"], seq.lengths)
        start, _ = seq.append(k, v, ones)
        o = seq.attend(q, start)
        logits = toy.logits(o).view(requests, beams, vocab)
        scores, token, parent = bc.beam_select(logits, s["scores"], beams)
        seq.reorder(parent)
        s["scores"].copy_(scores)
        s["token"].copy_(token.view(-1))

    plain, captured = make(), make()
    step(make())  # (warm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(captured)
    for _ in range(50):
        step(plain)
        graph.replay()
    torch.cuda.synchronize()
    a, b = plain["seq"], captured["seq"]
    assert a.lengths.tolist() == [50] * rows
    for x, y in ((a.lengths, b.lengths), (a.pages, b.pages), (a.refcount, b.refcount),
                 (a.free_count, b.free_count), (plain["token"], captured["token"]),
                 (plain["scores"], captured["scores"]), (a.k, b.k), (a.v, b.v)):
        assert torch.equal(x, y)
    n = int(a.free_count)
    assert torch.equal(a.free_stack[:n], b.free_stack[:n])


def test_schemas(bc):
    """opcheck: schemas and fake kernels of the ops on real calls."""
    t = torch.library.opcheck
    pages, lengths = ints([[0, -1], [1, -1]]), ints([3, 5])
    state = ints([1, 1, 0, 0]), ints([2, 3, 0, 0]), ints([2])
    utils = ("test_schema", "test_faketensor")
    op = torch.ops.branchcraft
    t(op.append_plan.default, (pages, lengths, ints([1, 2]), *state, 4), test_utils=utils)
    t(op.append_plan_.default, (pages, lengths, ints([1, 2]), *state, 4), test_utils=utils)
    x = torch.randn(3, 2, 64, device="cuda").half()
    cache = torch.randn(4, 16, 2, 64, device="cuda").half()
    t(op.append_kv_.default, (cache, cache.clone(), x, x.clone(), ints([1, 2, 40])), test_utils=utils)
    t(op.chunk_attention.default, (x, cache, cache.clone(), pages, ints([0, 1, 3]), lengths),
      test_utils=utils)
    t(op.chunk_attention_out.default,
      (x, cache, cache.clone(), pages, ints([0, 1, 3]), lengths, torch.empty_like(x)), test_utils=utils)
    t(op.beam_select.default, (torch.randn(2, 3, 50, device="cuda"), torch.randn(2, 3, device="cuda"), 4),
      test_utils=utils)
    rows = ints([[[0, -1], [1, -1]]])
    t(op.beam_reorder.default, (rows, ints([[3, 5]]), ints([[1, 1]]), *state), test_utils=utils)
    t(op.beam_reorder_.default, (rows, ints([[3, 5]]), ints([[1, 1]]), *state), test_utils=utils)


def test_check_follows_replays(bc):
    from branchcraft_torch.sequences import PagedSequences

    seq = PagedSequences(1, 1, 4, 2, 1, 64)
    row = torch.zeros(16, 1, 64, dtype=torch.float16, device="cuda")
    new = ints([16])
    seq.append(row, row, ints([0]))  # (a first call outside the capture)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        seq.append(row, row, new)
    seq.append(row, row, new)
    seq.check()
    graph.replay()
    seq.check()
    assert seq.lengths.tolist() == [32]
    graph.replay()  # both pages are in use
    with pytest.raises(RuntimeError, match="exhausted"):
        seq.check()
    assert seq.lengths.tolist() == [32]
    seq.append(row, row, ints([0]))
    seq.check()
