"""New tokens into the paged cache: append_plan against the page pool's
sequential rules, bit for bit, and append_kv_ against plain indexing."""
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


def plan_inputs(pool, reqs, new, width):
    return ints(pool.page_table(reqs, width)), ints([pool.lengths[r] for r in reqs]), ints(new)


def check_plan(bc, pool, reqs, new, spare=0, in_place=False):
    width = max(1, max((pool.lengths[r] + n + 15) // 16 for r, n in zip(reqs, new)),
                max(len(pool.pages[r]) for r in reqs)) + 1
    pages, lengths, count = plan_inputs(pool, reqs, new, width)
    state = S.device_state(pool)
    total = sum(new)
    if in_place:
        outs = bc.append_plan_(pages, lengths, count, *state, total + spare)
        tables = (pages, lengths, *state)
    else:
        kept = [t.clone() for t in (pages, lengths, *state)]
        outs = bc.append_plan(pages, lengths, count, *state, total + spare, width + 2)
        tables, outs = outs[:5], outs[5:]
        assert all(torch.equal(a, b) for a, b in zip(kept, (pages, lengths, *state)))
    query_start, slot_map, positions, clones, counts = outs
    slots, pos, cl = S.append_sequential(pool, reqs, new)
    assert counts.tolist() == [total, len(cl), 0]
    assert tables[0].tolist() == pool.page_table(reqs, tables[0].shape[1])
    assert tables[1].tolist() == [pool.lengths[r] for r in reqs]
    S.assert_pool(pool, *tables[2:])
    assert query_start.tolist() == [0, *np.cumsum(new).tolist()]
    assert slot_map.tolist() == slots + [-1] * spare
    assert positions.tolist() == pos + [-1] * spare
    assert clones[:, :len(cl)].T.tolist() == [list(c) for c in cl]
    assert (clones[:, len(cl):] == -1).all()


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("seed", range(6))
def test_random_histories(bc, seed, in_place):
    rng = np.random.default_rng(seed)
    pool, live, snaps = PagePool(400), [], []
    for _ in range(40):
        op = rng.choice(["new", "fork", "fork", "snap", "append", "append", "rollback"])
        if op == "new" or not live:
            if len(pool.free) > 10:
                live.append(pool.new(int(rng.integers(0, 70))))
        elif op == "fork":
            live.append(pool.fork(int(rng.choice(live))))
        elif op == "snap":
            snaps.append(pool.checkpoint(int(rng.choice(live))))
        elif op == "rollback" and snaps:
            pool.rollback(snaps.pop())
        elif op == "append":
            reqs = [int(x) for x in rng.choice(live, size=int(rng.integers(1, len(live) + 1)),
                                               replace=False)]
            new = rng.integers(0, int(rng.choice([2, 40])), size=len(reqs)).tolist()
            need = sum(n // 16 + 2 for n in new)
            if need <= len(pool.free):
                check_plan(bc, pool, reqs, new, spare=int(rng.integers(0, 5)), in_place=in_place)


@pytest.mark.parametrize("batch,beams", [(1, 1), (33, 1), (1024, 8), (1500, 3), (4096, 4096),
                                         (4096, 1)])
def test_large_batches(bc, batch, beams):
    """Many sequences, groups of them sharing a partial page - up to one group of all."""
    rng = np.random.default_rng(batch)
    pool, reqs = PagePool(30000), []
    while len(reqs) < batch:
        first = pool.new(int(rng.integers(1, 60)))
        group = [first] + [pool.fork(first) for _ in range(min(beams, batch - len(reqs)) - 1)]
        if rng.random() < 0.5 and beams > 1:
            pool.checkpoint(first)  # somebody outside the batch holds the page too
        reqs += group
    check_plan(bc, pool, reqs, rng.integers(0, 3, size=batch).tolist(), spare=3)


def test_long_prompts(bc):
    pool = PagePool(20000)
    reqs = [pool.new(n) for n in (0, 5, 16, 1000)]
    check_plan(bc, pool, reqs, [100000, 1, 33333, 0], spare=5)
    check_plan(bc, pool, reqs, [7, 8, 9, 20000], in_place=True)


def test_failed_plans_change_nothing(bc):
    pool = PagePool(12)
    reqs = [pool.new(20), pool.new(40)]
    reqs.append(pool.fork(reqs[0]))
    cases = []

    def case(status, new, max_tokens=64, change=None):
        width = 9
        pages, lengths, count = plan_inputs(pool, reqs, new, width)
        state = list(S.device_state(pool))
        if change:
            change(pages, lengths, state)
        kept = [t.clone() for t in (pages, lengths, *state)]
        out = bc.append_plan(pages, lengths, count, *state, max_tokens)
        assert out[9].tolist() == [0, 0, status]
        assert torch.equal(out[1], kept[1])
        for a, b in zip(out[2:5], kept[2:]):
            assert torch.equal(a, b)
        assert (out[5] == 0).all() and (out[6] == -1).all() and (out[7] == -1).all()
        assert (out[8] == -1).all()
        res = bc.append_plan_(pages, lengths, count, *state, max_tokens)
        assert res[4].tolist() == [0, 0, status]
        assert all(torch.equal(a, b) for a, b in zip(kept, (pages, lengths, *state)))
        cases.append(status)

    case(1, [1, -1, 2])
    case(1, [30, 30, 5])
    case(1, [2 ** 31 - 1, 2 ** 31 - 1, 1])
    case(2, [100, 100, 1], 300)
    case(3, [1, 150, 1], 300)                                     # wider than the table

    def bad_len(pages, lengths, state):
        lengths[1] = 1000
    case(3, [1, 1, 1], change=bad_len)

    def neg_len(pages, lengths, state):
        lengths[1] = -7
    case(3, [1, 1, 1], change=neg_len)

    def bad_page(pages, lengths, state):
        pages[1, 2] = 99
    case(3, [1, 1, 1], change=bad_page)

    def bad_ref(pages, lengths, state):
        state[0][int(pages[1, 2])] = 0
    case(3, [1, 1, 1], change=bad_ref)

    def bad_count(pages, lengths, state):
        state[2][0] = 13
    case(3, [1, 1, 1], change=bad_count)

    def bad_stack(pages, lengths, state):
        state[1][int(state[2][0]) - 1] = 12
    case(3, [1, 1, 1], change=bad_stack)

    def two_lengths(pages, lengths, state):
        lengths[2] = 21
    case(3, [1, 1, 1], change=two_lengths)

    def more_writers(pages, lengths, state):
        lengths[1] = 20
        pages[1, :2] = pages[0, :2]
    case(3, [1, 1, 1], change=more_writers)
    assert sorted(set(cases)) == [1, 2, 3]


def test_plan_refusals(bc):
    pool = PagePool(8)
    reqs = [pool.new(5)]
    pages, lengths, count = plan_inputs(pool, reqs, [1], 3)
    state = S.device_state(pool)
    for args in ((pages.long(), lengths, count, *state, 1), (pages, lengths, count, *state, -1),
                 (pages, lengths[:0], count, *state, 1), (pages, lengths, count.cpu(), *state, 1),
                 (pages, lengths, count, state[0], state[1][:3].contiguous(), state[2], 1),
                 (torch.zeros(4097, 1, dtype=torch.int32, device="cuda"),
                  torch.zeros(4097, dtype=torch.int32, device="cuda"),
                  torch.zeros(4097, dtype=torch.int32, device="cuda"), *state, 1)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            bc.append_plan(*args)


# ------------------------------------------------------------------------ rows


def rows_case(dtype, tokens, pool, hkv, dim, seed, spread=True):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    slot = torch.randperm(pool * 16, generator=g, device="cuda")[:tokens].int()
    return (rand(pool, 16, hkv, dim), rand(pool, 16, hkv, dim), rand(tokens, hkv, dim),
            rand(tokens, hkv, dim), slot)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,hkv,dim", [(1, 1, 64), (1, 8, 128), (37, 3, 64), (1000, 8, 128),
                                            (129, 2, 128), (5, 200, 128)])
def test_rows(bc, dtype, tokens, hkv, dim):
    ck, cv, k, v, slot = rows_case(dtype, tokens, 100, hkv, dim, tokens)
    if tokens > 3:
        slot[tokens // 2] = -1
    wk, wv = ck.clone(), cv.clone()
    live = slot >= 0
    wk.view(-1, hkv, dim)[slot[live].long()] = k[live]
    wv.view(-1, hkv, dim)[slot[live].long()] = v[live]
    bc.append_kv_(ck, cv, k, v, slot)
    assert torch.equal(ck, wk) and torch.equal(cv, wv)


def test_rows_strided(bc):
    """Parts of a fused projection into vLLM's planes and an interleaved cache."""
    ck, cv, k, v, slot = rows_case(torch.float16, 50, 20, 4, 128, 1)
    fused = torch.randn(50, 12, 128, device="cuda").half()
    fused[:, 4:8], fused[:, 8:] = k, v
    bc.append_kv_(ck, cv, k, v, slot)
    planes = torch.zeros(20, 2, 16, 4, 128, device="cuda", dtype=torch.float16)
    bc.append_kv_(planes[:, 0], planes[:, 1], fused[:, 4:8], fused[:, 8:], slot)
    inter = torch.zeros(20, 4, 16, 256, device="cuda", dtype=torch.float16)
    bc.append_kv_(inter[..., :128].transpose(1, 2), inter[..., 128:].transpose(1, 2), k, v, slot)
    at = slot.long()
    for got in (planes[:, 0], inter[..., :128].transpose(1, 2)):
        assert torch.equal(got.reshape(-1, 4, 128)[at], k)
        assert int((got != 0).any(-1).any(-1).sum()) == 50
    for got in (planes[:, 1], inter[..., 128:].transpose(1, 2)):
        assert torch.equal(got.reshape(-1, 4, 128)[at], v)


def test_bits_are_kept(bc):
    """Every 16-bit pattern arrives as it is (NaN payloads included)."""
    bits = torch.arange(-32768, 32768, device="cuda").to(torch.int16)
    k = bits.view(torch.float16).view(64, 8, 128)
    ck = torch.zeros(4, 16, 8, 128, dtype=torch.float16, device="cuda")
    cv = torch.zeros_like(ck)
    bc.append_kv_(ck, cv, k, k.flip(0).contiguous(), torch.arange(64, dtype=torch.int32, device="cuda"))
    assert torch.equal(ck.view(torch.int16).reshape(-1), bits)
    assert torch.equal(cv.view(torch.int16), k.flip(0).view(torch.int16).view(4, 16, 8, 128))


def test_clones_and_rows_together(bc):
    """A clone copies the valid slots only, and rows land beside them: the last
    holder writes in place into the page that the others clone."""
    pool = PagePool(30)
    first = pool.new(21)
    reqs = [first] + [pool.fork(first) for _ in range(3)]
    pages, lengths, new = plan_inputs(pool, reqs, [3, 1, 20, 2], 4)
    state = S.device_state(pool)
    old = pages.clone()
    ck = torch.randn(30, 16, 2, 64, device="cuda").half()
    cv = torch.randn_like(ck)
    before_k, before_v = ck.clone(), cv.clone()
    _, slot_map, _, clones, counts = bc.append_plan_(pages, lengths, new, *state, 26)
    assert counts.tolist() == [26, 3, 0]
    k = torch.randn(26, 2, 64, device="cuda").half()
    v = torch.randn_like(k)
    bc.append_kv_(ck, cv, k, v, slot_map, clones, counts)
    t = 0
    for b, n in enumerate(new.tolist()):
        for pos in range(lengths[b].item()):
            page, slot = int(pages[b, pos // 16]), pos % 16
            if pos < 21:
                src = int(old[b, pos // 16])
                assert torch.equal(ck[page, slot], before_k[src, slot])
                assert torch.equal(cv[page, slot], before_v[src, slot])
            else:
                assert torch.equal(ck[page, slot], k[t]) and torch.equal(cv[page, slot], v[t])
                t += 1
    assert t == 26


def test_bad_slots_and_clones_are_skipped(bc):
    import bc_capi

    bc_capi.last_device_error(reset=True)
    ck, cv, k, v, slot = rows_case(torch.float16, 6, 10, 2, 64, 4)
    wk = ck.clone()
    slot[:] = ints([160, -2, 2 ** 31 - 1, -2 ** 31, -1, 33])
    wk.view(-1, 2, 64)[33] = k[5]
    bc.append_kv_(ck, cv, k, v, slot)
    assert torch.equal(ck, wk)
    assert bc_capi.last_device_error(reset=True) == bc_capi.ERR_COMMIT_INDEX
    for clone in ([-1, 2, 3], [10, 2, 3], [1, 10, 3], [1, 2, 17], [1, 2, -1], [2, 2, 3]):
        bc.append_kv_(ck, cv, k[:0], v[:0], slot[:0], ints(clone)[:, None].contiguous(),
                      ints([0, 1, 0]))
        assert torch.equal(ck, wk)
        assert bc_capi.last_device_error(reset=True) == bc_capi.ERR_COMMIT_INDEX
    bc.append_kv_(ck, cv, k[:0], v[:0], slot[:0])  # nothing to do


def test_row_refusals(bc):
    ck, cv, k, v, slot = rows_case(torch.float16, 6, 10, 2, 64, 5)
    one = ints([[0], [1], [2]])
    for args in ((ck, cv, k.bfloat16(), v, slot), (ck, cv, k[:5], v, slot),
                 (ck, cv, k, v, slot.long()), (ck, cv.bfloat16(), k, v, slot),
                 (ck, cv, k, v, slot, one), (ck, cv, k, v, slot, one, ints([0])),
                 (ck, cv, k.transpose(0, 1).contiguous().transpose(0, 1), v, slot),
                 (ck[:, :8].contiguous(), cv[:, :8].contiguous(), k, v, slot),
                 (ck, cv, torch.zeros(769, device="cuda").half()[1:].view(6, 2, 64), v, slot)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            bc.append_kv_(*args)


def test_plan_and_rows_in_a_graph(bc):
    """A captured step advances the state at every replay."""
    pool = PagePool(64)
    first = pool.new(30)
    reqs = [first, pool.fork(first), pool.new(3)]
    pages, lengths, new = plan_inputs(pool, reqs, [1, 1, 1], 6)
    state = S.device_state(pool)
    ck = torch.zeros(64, 16, 2, 64, device="cuda", dtype=torch.float16)
    cv, k = torch.zeros_like(ck), torch.ones(3, 2, 64, device="cuda", dtype=torch.float16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, slot_map, _, clones, counts = bc.append_plan_(pages, lengths, new, *state, 3)
        bc.append_kv_(ck, cv, k, k, slot_map, clones, counts)
        k.add_(1)
    for step in range(20):
        graph.replay()
        slots, _, cl = S.append_sequential(pool, reqs, [1, 1, 1])
        assert slot_map.tolist() == slots and counts.tolist() == [3, len(cl), 0]
        assert (ck.view(-1, 2, 64)[slot_map.long()] == step + 1).all()
    assert pages.tolist() == pool.page_table(reqs, 6)
    S.assert_pool(pool, *state)


@pytest.mark.parametrize("length", [-1, -2 ** 31, 145, 2 ** 31 - 1, 2 ** 31 - 14, 100])
def test_failed_plans_keep_rows(bc, length):
    """New tables after a plan that failed hold the rows as they were, at malformed lengths
    too (there the whole row)."""
    pages = torch.arange(27, dtype=torch.int32, device="cuda").view(3, 9).contiguous()
    lengths = ints([40, length, 144])
    state = ints([1] * 40), ints(list(range(40))), ints([40])
    for new, width in ((ints([1, 0, 1]), 9), (ints([1, 1, -1]), 12), (ints([0, 0, 200]), 9)):
        out = bc.append_plan(pages, lengths, new, *state, 300, width)
        assert out[9][2].item() != 0 and torch.equal(out[1], lengths)
        want = torch.full((3, width), -1, dtype=torch.int32, device="cuda")
        for b, x in enumerate((40, length, 144)):
            n = (x + 15) // 16 if 0 <= x <= 144 else 9
            want[b, :n] = pages[b, :n]
        assert torch.equal(out[0], want)
