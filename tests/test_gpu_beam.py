"""Beam search: beam_select against 64-bit scores with the lowest index first
among equals, beam_reorder against the page pool's forks and releases, and a
whole search over device state."""
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


def check_select(bc, logits, scores, k):
    got = bc.beam_select(logits, scores, k)
    value, token, parent = S.beam_select(logits, scores, k)
    assert got[1].tolist() == token.tolist() and got[2].tolist() == parent.tolist()
    g = got[0].cpu().double()
    assert torch.equal(torch.isinf(g), torch.isinf(value))
    fin = torch.isfinite(value)
    # the result's rounding, and a log-sum within 2^-22 (expf: 2 units of 2^-24
    # relative, a thread's 32-term sum in FP32: 31 more at 2^-24, in the mean far less)
    tol = value.abs() * 2.0 ** -23 + 34 * 2.0 ** -24
    assert ((g - value).abs()[fin] <= tol[fin]).all()
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,beams,vocab,k", [
    (1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 17, 4), (1, 4, 32000, 8), (3, 8, 16384, 16),
    (2, 5, 16385, 7), (1, 64, 500, 64), (2, 2, 50257, 64), (1, 2, 200001, 3), (5, 16, 3, 40),
    (1, 1, 1 << 20, 64)])
def test_select(bc, dtype, batch, beams, vocab, k):
    g = torch.Generator(device="cuda").manual_seed(vocab + k)
    logits = (torch.randn(batch, beams, vocab, generator=g, device="cuda") * 2.5).to(dtype)
    scores = -9 * torch.rand(batch, beams, generator=g, device="cuda")
    check_select(bc, logits, scores, k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_select_ties_and_order(bc, dtype):
    """All logits equal; sorted up and down; the best ones all in one place."""
    beams, vocab = 2, 40000
    scores = torch.tensor([[-1.0, -1.0]], device="cuda")
    x = torch.zeros(1, beams, vocab, device="cuda", dtype=dtype)
    got = check_select(bc, x, scores, 64)
    assert got[1][0].tolist() == list(range(64)) and (got[2] == 0).all()
    ramp = torch.linspace(-8, 8, vocab, device="cuda").to(dtype).expand(1, beams, vocab).contiguous()
    check_select(bc, ramp, scores, 64)
    check_select(bc, ramp.flip(-1).contiguous(), scores, 64)
    x[0, 1, 20000:20040] = 5
    check_select(bc, x, scores, 64)
    zeros = torch.zeros(1, 1, 100, device="cuda", dtype=dtype)
    zeros[0, 0, ::2] = -0.0
    assert bc.beam_select(zeros, scores[:, :1].contiguous(), 5)[1].tolist() == [[0, 1, 2, 3, 4]]


@pytest.mark.parametrize("dtype,vec", [(torch.float32, 4), (torch.float16, 8), (torch.bfloat16, 8)])
@pytest.mark.parametrize("k", [64, 33])
def test_select_best_in_few_threads(bc, dtype, vec, k):
    """The best logits in the places of k - 1 pairs of threads (16-byte loads go to 256
    threads in turn), more than a block lists at once: the second look is thinned."""
    rows, vocab = 600, 40000
    g = torch.Generator(device="cuda").manual_seed(k)
    x = torch.randn(rows, 1, vocab, generator=g, device="cuda")
    x[..., (torch.arange(vocab, device="cuda") // vec) % 256 < 2 * (k - 1)] += 40
    check_select(bc, x.to(dtype), -torch.rand(rows, 1, generator=g, device="cuda"), k)


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 4096), (torch.float32, 8192),
                                         (torch.bfloat16, 8192), (torch.float16, 16384)])
def test_select_whole_steps(bc, dtype, vocab):
    """Rows of exactly a block's step, whose last segment may be empty: the best k are
    one of each beam."""
    beams = 16
    x = torch.randn(2, beams, vocab, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    for w in range(beams):
        x[:, w, 100 * w + 3] = 30.0 + w / 4
    scores = torch.linspace(-3, 0, beams, device="cuda").repeat(2, 1).contiguous()
    got = check_select(bc, x.to(dtype), scores, beams)
    assert sorted(got[2][0].tolist()) == list(range(beams))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_select_infinities_and_nan(bc, dtype):
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(4, 3, 1000, generator=g, device="cuda").to(dtype)
    scores = -torch.rand(4, 3, generator=g, device="cuda")
    x[0, :, 5:] = -math.inf          # fewer tokens than asked for
    x[1, 1] = -math.inf              # a beam that cannot go on
    x[1, 0, 7] = math.nan
    scores[2, 0] = -math.inf         # beams that are out
    scores[2, 1] = math.nan
    x[3] = -math.inf                 # nothing possible: lowest indices
    x[3, 2, 0] = math.nan
    got = check_select(bc, x, scores, 20)
    assert got[1][3].tolist() == list(range(20)) and (got[0][3] == -math.inf).all()
    low = torch.full((1, 2, 50), torch.finfo(dtype).min, device="cuda", dtype=dtype)
    low[0, 1, 30] = 1.0
    got = check_select(bc, low, scores[:1, :2].contiguous(), 1)
    assert got[1].item() == 30 and got[2].item() == 1
    inf = torch.zeros(1, 1, 50, device="cuda", dtype=dtype)
    inf[0, 0, 9] = math.inf
    got = bc.beam_select(inf, torch.zeros(1, 1, device="cuda"), 2)
    assert got[1][0, 0].item() == 9 and not torch.isnan(got[0]).any()


def test_select_strided_and_graph(bc):
    wide = torch.randn(3, 4, 1010, device="cuda")
    x, scores = wide[:, :, :1001], -torch.rand(3, 4, device="cuda")
    check_select(bc, x, scores, 6)
    check_select(bc, wide[:, :, 3:1004], scores, 6)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = bc.beam_select(x, scores, 6)
    wide.copy_(torch.randn_like(wide))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, bc.beam_select(x, scores, 6)))


def test_select_refusals(bc):
    x, s = torch.zeros(2, 3, 50, device="cuda"), torch.zeros(2, 3, device="cuda")
    for args in ((x.double(), s, 1), (x, s.half(), 1), (x, s[:, :2].contiguous(), 1), (x, s, 0),
                 (x, s, 65), (x[:, :1, :5].contiguous(), s[:, :1].contiguous(), 6),
                 (x.transpose(1, 2), torch.zeros(2, 50, device="cuda"), 1), (x[0], s[0], 1),
                 (torch.zeros(1, 65, 4, device="cuda"), torch.zeros(1, 65, device="cuda"), 1),
                 (torch.zeros(1, 1, (1 << 20) + 1, device="cuda"), s[:1, :1].contiguous(), 1),
                 (x[:, ::2], s[:, ::2].contiguous(), 1), (x.cpu(), s, 1)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            bc.beam_select(*args)


# --------------------------------------------------------------------- reorder


def ints(x):
    return torch.tensor(np.asarray(x, np.int32), device="cuda")


def table(pool, rows, width):
    return ints([[pool.pages[r] + [-1] * (width - len(pool.pages[r])) if r is not None
                  else [-1] * width for r in row] for row in rows])


def lens(pool, rows):
    return ints([[pool.lengths[r] if r is not None else 0 for r in row] for row in rows])


def check_reorder(bc, pool, beams, parents, width, in_place):
    pages, lengths, state = table(pool, beams, width), lens(pool, beams), S.device_state(pool)
    kept = [t.clone() for t in (pages, lengths, *state)]
    if in_place:
        po, lo = bc.beam_reorder_(pages, lengths, ints(parents), *state)
        after = state
    else:
        po, lo, *after = bc.beam_reorder(pages, lengths, ints(parents), *state)
        assert all(torch.equal(a, b) for a, b in zip(kept, (pages, lengths, *state)))
        # entries past the count are left as they were
        n = int(after[2].item())
        assert torch.equal(after[1][n:], kept[3][n:])
    made = S.reorder_sequential(pool, beams, parents)
    assert po.tolist() == table(pool, made, width).tolist()
    assert lo.tolist() == lens(pool, made).tolist()
    S.assert_pool(pool, *after)
    return made


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("batch,beams", [(1, 1), (1, 4), (3, 5), (20, 8), (2, 64)])
def test_search_histories(bc, batch, beams, in_place):
    """Requests with a common prompt, branching, diverging and ending over many steps."""
    rng = np.random.default_rng(batch * 100 + beams)
    pool = PagePool(6000)
    common = pool.new(64)
    rows = []
    for _ in range(batch):
        r = pool.fork(common)
        S.append_sequential(pool, [r], [int(rng.integers(0, 60))])
        rows.append([r])
    rows = check_reorder(bc, pool, rows, np.zeros((batch, beams), int).tolist(), 40, in_place)
    for step in range(12):
        live = [r for row in rows for r in row if r is not None]
        S.append_sequential(pool, live, [int(rng.integers(1, 20)) if step % 3 == 0 else 1] * len(live))
        parents = rng.integers(0, beams, size=(batch, beams))
        if step == 9 and batch > 1:
            parents[0] = -1  # this request is done
        if step == 5:
            parents[:, 0] = -1
            parents[:, 1:] = 0
        for b in range(batch):  # parents with a row
            for j in range(beams):
                if parents[b, j] >= 0 and rows[b][parents[b, j]] is None:
                    parents[b, j] = -1
        # a dropped row is a request without pages
        rows = [[r if r is not None else pool.new(0) for r in row] for row in rows]
        rows = check_reorder(bc, pool, rows, parents.tolist(), 40, in_place)
    # everything goes: pages come back in the order of their last release
    rows = [[r if r is not None else pool.new(0) for r in row] for row in rows]
    pool_pages = pool.pages.pop(common)
    pool.lengths.pop(common)
    for p in pool_pages:
        pool.release(p)
    check_reorder(bc, pool, rows, [[-1]] * batch, 40, in_place)
    assert len(pool.free) == 6000


def test_reorder_widths(bc):
    """Rows of exactly 32 and 33 columns, and a table much wider than its rows."""
    for width, length in ((1, 10), (32, 512), (33, 513), (500, 40)):
        pool = PagePool(600)
        r = pool.new(length)
        rows = [[r, pool.fork(r), pool.new(length)]]
        S.append_sequential(pool, [rows[0][1]], [1] if width > (length + 1 + 15) // 16 else [0])
        check_reorder(bc, pool, rows, [[2, 2]], width, False)


def test_reorder_malformed(bc):
    import bc_capi

    bc_capi.last_device_error(reset=True)
    pool = PagePool(20)
    rows = [[pool.new(40), pool.new(40)]]
    pages, lengths, state = table(pool, rows, 4), lens(pool, rows), S.device_state(pool)
    for bad in (2, -2, 2 ** 31 - 1, -2 ** 31):
        po, lo, rc, *_ = bc.beam_reorder(pages, lengths, ints([[bad, 1]]), *state)
        assert lo.tolist() == [[0, 40]] and (po[0, 0] == -1).all()
        assert rc.tolist() == [0 if p in pool.pages[rows[0][0]] else c
                               for p, c in enumerate(pool.refcount)]
        assert bc_capi.last_device_error(reset=True) == bc_capi.ERR_PARENT
    for bad in (20, -1, 2 ** 31 - 1):
        broken = pages.clone()
        broken[0, 0, 1] = bad
        po, lo, rc, stack, count = bc.beam_reorder(broken, lengths, ints([[1, 1]]), *state)
        assert int(count) == len(pool.free) + 2
        assert bc_capi.last_device_error(reset=True) == bc_capi.ERR_PAGE_RANGE
    for bad in (-1, 65, 2 ** 31 - 1):
        wrong = lengths.clone()
        wrong[0, 0] = bad
        bc.beam_reorder(pages, wrong, ints([[1, 1]]), *state)
        assert bc_capi.last_device_error(reset=True) & bc_capi.ERR_LENGTH


def test_reorder_refusals(bc):
    pool = PagePool(20)
    rows = [[pool.new(40), pool.new(40)]]
    pages, lengths, state = table(pool, rows, 4), lens(pool, rows), S.device_state(pool)
    good = ints([[0, 1]])
    for args in ((pages[0], lengths, good, *state), (pages, lengths[:, :1].contiguous(), good, *state),
                 (pages, lengths, good.long(), *state), (pages, lengths, good.cpu(), *state),
                 (pages, lengths, ints([[0, 1]] * 2), *state),
                 (pages, lengths, torch.zeros(1, 65, dtype=torch.int32, device="cuda"), *state),
                 (pages, lengths, good, state[0], state[1][:3].contiguous(), state[2])):
        with pytest.raises((RuntimeError, NotImplementedError)):
            bc.beam_reorder(*args)


@pytest.mark.parametrize("out", [-math.inf, math.nan])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_select_beams_that_are_out(bc, dtype, out):
    """The pairs of a beam that is out score -inf like any other impossible pair: the
    lowest index first among all of them, whatever its logits."""
    up = torch.arange(5.0, device="cuda").to(dtype)[None, None]
    got = check_select(bc, up, torch.full((1, 1), out, device="cuda"), 2)
    assert got[1].tolist() == [[0, 1]]
    g = torch.Generator(device="cuda").manual_seed(9)
    for beams, vocab, k, allowed in ((2, 1000, 8, 3), (3, 17, 40, 5), (4, 40001, 64, 20),
                                     (2, 200001, 64, 1), (1, 33000, 64, 0), (8, 300, 64, 50)):
        for dead in ([0], list(range(beams)), list(range(1, beams)), [beams - 1]):
            x = torch.randn(2, beams, vocab, generator=g, device="cuda").to(dtype)
            x[..., torch.randperm(vocab, generator=g, device="cuda")[allowed:]] = -math.inf
            x[:, dead] = torch.randn(2, len(dead), vocab, generator=g, device="cuda").to(dtype)
            scores = -torch.rand(2, beams, generator=g, device="cuda")
            scores[0, dead] = out
            check_select(bc, x, scores, k)
            scores[1, dead] = out
            check_select(bc, x, scores, min(k, allowed + 1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab", [5, 1001, 8192, 32001, 50257, 131071, 200003])
def test_select_beams_alike(bc, dtype, vocab):
    """Beams with the same logits and scores (a first step): equal pairs by the lowest index,
    however the beams' rows lie to the memory's 16-byte pieces."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    for beams, k in ((4, 8), (8, 16), (3, 5)):
        x = (torch.randn(3, 1, vocab, generator=g, device="cuda") * 3).to(dtype)
        x = x.expand(3, beams, vocab).contiguous()
        check_select(bc, x, torch.zeros(3, beams, device="cuda"), k)
