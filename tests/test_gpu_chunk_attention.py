"""Attention of a chunk of new tokens over the paged cache (chunk_attention)
against the formula in 64 bits: types, head groups, lengths from one token to
many key tiles, masks, score caps and biases, strided inputs and caches,
malformed metadata, and what it must leave alone."""
import math

import pytest
import torch

import serving_oracle as S

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def bc():
    import branchcraft_torch

    return branchcraft_torch


@pytest.fixture(autouse=True)
def clean_error_word():
    import bc_capi

    bc_capi.last_device_error(reset=True)
    yield
    bc_capi.last_device_error(reset=True)


def error_word():
    import bc_capi

    return bc_capi.last_device_error(reset=True)


def make(new, lens, hq, hkv, dim, dtype, seed=0, extra_pages=3, width=None, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [(x + 15) // 16 for x in lens]
    pool = sum(need) + extra_pages
    perm = torch.randperm(pool, generator=g, device="cuda").tolist()
    width = width or max(1, max(need))
    pages, at = [], 0
    for n in need:
        pages.append(perm[at:at + n] + [-1] * (width - n))
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)

    def rand(*shape):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    return dict(q=rand(starts[-1], hq, dim), k=rand(pool, 16, hkv, dim), v=rand(pool, 16, hkv, dim),
                pages=ints(pages), query_start=ints(starts), lengths=ints(lens))


def check(bc, f, out_dtype=None, **options):
    if out_dtype is None:
        got = bc.chunk_attention(**f, **options)
    else:
        got = torch.full(f["q"].shape, float("nan"), dtype=out_dtype, device="cuda")
        bc.chunk_attention_out(*(f[n] for n in ("q", "k", "v", "pages", "query_start", "lengths")),
                               got, **options)
    torch.cuda.synchronize()
    S.assert_chunk_close(got, S.chunk_attention(**f, **options), f["q"].dtype)
    return got


SHAPES = [  # new tokens, lengths, query heads, KV heads
    ([1], [1], 1, 1), ([1], [17], 8, 2), ([1, 1, 1], [0 + 1, 130, 1000], 8, 2),
    ([5], [5], 4, 4), ([33], [33], 8, 2), ([64], [257], 8, 2), ([65], [129], 4, 1),
    ([128], [128], 3, 3), ([129], [640], 6, 2), ([200, 1, 0, 37], [200, 900, 40, 37], 8, 2),
    ([7, 7], [200, 16], 14, 2), ([300], [300], 7, 1), ([40], [1500], 10, 2), ([2], [2500], 64, 1),
    ([3], [40], 128, 1), ([700], [1800], 2, 1),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,lens,hq,hkv", SHAPES)
def test_causal(bc, new, lens, hq, hkv, dim, dtype):
    check(bc, make(new, lens, hq, hkv, dim, dtype))
    assert error_word() == 0


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_fp32_output(bc, dtype):
    f = make([90, 1], [300, 77], 8, 2, 128, dtype, seed=3)
    check(bc, f, out_dtype=torch.float32)


OPTIONS = [
    dict(softcap=5.0), dict(softcap=50.0), dict(window=1), dict(window=20), dict(window=128),
    dict(window=129), dict(alibi=True), dict(alibi=True, softcap=20.0, window=300),
    dict(prefix=True), dict(documents=True), dict(prefix=True, alibi=True, documents=True),
    dict(prefix=True, window=50), dict(scale=0.3),
]


def options_of(f, o, seed=1):
    o, kw = dict(o), {}
    g = torch.Generator().manual_seed(seed)
    hq = f["q"].shape[1]
    lens = f["lengths"].tolist()
    starts = f["query_start"].tolist()
    if o.pop("alibi", False):
        kw["alibi_slopes"] = torch.tensor([2.0 ** (-8 * (h + 1) / hq) for h in range(hq)],
                                          device="cuda")
    if o.pop("prefix", False):
        kw["prefix"] = torch.tensor([int(torch.randint(0, x + 3, (), generator=g)) for x in lens],
                                    dtype=torch.int32, device="cuda")
    if o.pop("documents", False):
        ks = []
        for b, x in enumerate(lens):
            n = starts[b + 1] - starts[b]
            cuts = [0] + sorted(int(c) for c in torch.randint(0, x + 1, (3,), generator=g))
            ks += [max(c for c in cuts if c <= x - n + i) for i in range(n)]
        kw["key_start"] = torch.tensor(ks, dtype=torch.int32, device="cuda")
    return kw | o


@pytest.mark.parametrize("dtype,dim", [(F16, 64), (BF16, 128)])
@pytest.mark.parametrize("o", OPTIONS, ids=str)
def test_score_options(bc, o, dtype, dim):
    f = make([70, 1, 150], [500, 333, 150], 6, 2, dim, dtype, seed=5)
    check(bc, f, **options_of(f, o))
    assert error_word() == 0


@pytest.mark.parametrize("softcap", [0.5, 30.0])
def test_large_scores(bc, softcap):
    """Scores far beyond the cap, and a softmax on few keys."""
    f = make([50], [400], 4, 2, 128, BF16, seed=6, scale=4.0)
    check(bc, f, softcap=softcap)
    check(bc, f)


def test_empty_rows_are_zero(bc):
    """Rows whose mask leaves nothing: a key_start past the token, no length, and
    more tokens than keys (reported)."""
    f = make([20], [20], 4, 2, 64, F16)
    ks = torch.arange(20, dtype=torch.int32, device="cuda")
    ks[5] = 6
    ks[7] = 2 ** 31 - 1
    got = check(bc, f, key_start=ks)
    assert (got[5] == 0).all() and (got[7] == 0).all() and (got[6] != 0).any()
    assert error_word() == 0
    f["lengths"] = torch.tensor([4], dtype=torch.int32, device="cuda")
    got = bc.chunk_attention(**f)
    torch.cuda.synchronize()
    assert (got[:16] == 0).all() and (got[16:] != 0).any()
    import bc_capi
    assert error_word() == bc_capi.ERR_LENGTH
    f["lengths"].zero_()
    assert (bc.chunk_attention(**f) == 0).all()
    assert error_word() == bc_capi.ERR_LENGTH


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_nothing_unseen_is_used(bc, dtype, bad):
    """NaN and infinities in slots past the lengths, in pages no token sees
    (before the window) and in pages of nobody change no bit."""
    f = make([60, 1], [200, 1000], 8, 2, 128, dtype, seed=7)
    want = bc.chunk_attention(**f, window=130)
    g = dict(f, k=f["k"].clone(), v=f["v"].clone())
    used = torch.zeros(f["k"].shape[0], 16, dtype=torch.bool)
    for b, (n, x) in enumerate(((60, 200), (1, 1000))):
        for j in range(max(0, x - n + 1 - 130), x):
            used[int(f["pages"][b, j // 16]), j % 16] = True
    for name in ("k", "v"):
        g[name][~used.cuda()] = bad
    got = bc.chunk_attention(**g, window=130)
    assert torch.equal(got, want)
    # keys seen by later rows only, in K: masked scores of any value
    k = f["k"].clone()
    k[int(f["pages"][0, 199 // 16]), 199 % 16] = bad
    got = bc.chunk_attention(f["q"], k, f["v"], f["pages"], f["query_start"], f["lengths"],
                             window=130)
    assert torch.equal(got[:59], want[:59])


def test_pages_out_of_range(bc):
    """A seen page outside the pool reads as zeros and is reported; one that the
    window hides is not looked at."""
    import bc_capi

    f = make([40], [300], 4, 2, 64, F16, seed=8)
    pool = f["k"].shape[0]
    for bad in (-1, pool, 2 ** 31 - 1, -2 ** 31):
        g = dict(f, pages=f["pages"].clone())
        g["pages"][0, 10] = bad
        got = bc.chunk_attention(**g)
        S.assert_chunk_close(got, S.chunk_attention(**g), F16)
        assert error_word() == bc_capi.ERR_PAGE_RANGE
        g["pages"][0, 10] = f["pages"][0, 10]
        g["pages"][0, 2] = bad
        got = bc.chunk_attention(**g, window=100)
        S.assert_chunk_close(got, S.chunk_attention(**g, window=100), F16)
        assert error_word() == 0


def test_malformed_metadata_is_brought_into_range(bc):
    import bc_capi

    f = make([30, 30], [100, 100], 4, 2, 64, F16, seed=9)
    for starts, lens in (([0, 70, 60], [100, 100]), ([-3, 30, 60], [100, 100]),
                         ([0, 30, 1000], [100, 100]), ([0, 30, 60], [100, 10 ** 9]),
                         ([0, 30, 60], [-5, 100])):
        g = dict(f, query_start=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                 lengths=torch.tensor(lens, dtype=torch.int32, device="cuda"))
        out = bc.chunk_attention(**g)
        torch.cuda.synchronize()
        assert out.shape == f["q"].shape
        assert error_word() & bc_capi.ERR_LENGTH


def test_rows_of_no_request_are_left(bc):
    f = make([9, 30], [50, 64], 8, 2, 128, BF16, seed=10)
    want = bc.chunk_attention(**f)
    g = dict(f, q=torch.cat([f["q"], torch.randn(25, 8, 128, device="cuda").to(BF16)]))
    out = torch.full(g["q"].shape, 7.0, dtype=BF16, device="cuda")
    bc.chunk_attention_out(*g.values(), out)
    assert torch.equal(out[:39], want) and (out[39:] == 7).all()
    # rows before the first request and between... the starts may begin late
    g["query_start"] = g["query_start"] + 5
    g["q"] = torch.cat([f["q"][:5], f["q"], f["q"][:20]])
    out.fill_(7.0)
    bc.chunk_attention_out(*g.values(), out)
    assert torch.equal(out[5:44], want) and (out[:5] == 7).all() and (out[44:] == 7).all()


def test_strided_inputs(bc):
    """Q out of a fused projection; caches as vLLM's planes, as interleaved
    [P, Hkv, 16, 2D] and with padded heads."""
    f = make([50, 3], [400, 90], 8, 2, 128, F16, seed=11)
    want = bc.chunk_attention(**f)
    fused = torch.zeros(53, 12, 128, dtype=F16, device="cuda")
    fused[:, :8] = f["q"]
    assert torch.equal(bc.chunk_attention(**dict(f, q=fused[:, :8])), want)
    p, _, h, d = f["k"].shape
    planes = torch.stack([f["k"], f["v"]], 1)                        # [P, 2, 16, Hkv, D]
    assert torch.equal(bc.chunk_attention(**dict(f, k=planes[:, 0], v=planes[:, 1])), want)
    inter = torch.cat([f["k"], f["v"]], 3).transpose(1, 2).contiguous()  # [P, Hkv, 16, 2D]
    got = bc.chunk_attention(**dict(f, k=inter[..., :d].transpose(1, 2),
                                    v=inter[..., d:].transpose(1, 2)))
    assert torch.equal(got, want)
    wide = torch.full((2, p, 16, h, 192), float("nan"), dtype=F16, device="cuda")
    wide[0, ..., :128], wide[1, ..., :128] = f["k"], f["v"]
    assert torch.equal(bc.chunk_attention(**dict(f, k=wide[0, ..., :128], v=wide[1, ..., :128])),
                       want)


def test_shared_pages_and_repeated_pages(bc):
    """Two requests on the same pages, and a page that a row holds twice."""
    f = make([10, 10], [100, 100], 4, 2, 64, BF16, seed=12)
    f["pages"][1] = f["pages"][0]
    f["pages"][1, 3] = f["pages"][1, 2]
    check(bc, f)


def test_long_context_splits(bc):
    """Few rows over many keys: the key range is shared by many blocks."""
    f = make([1, 3], [20000, 9001], 8, 2, 128, F16, seed=13)
    check(bc, f)
    check(bc, f, window=15000, softcap=20.0)
    f = make([1], [40000], 4, 1, 64, BF16, seed=14)
    check(bc, f)


def test_many_requests(bc):
    """More requests than blocks, empty ones among them."""
    g = torch.Generator().manual_seed(3)
    new = torch.randint(0, 4, (700,), generator=g).tolist()
    lens = [n + int(torch.randint(0, 60, (), generator=g)) for n in new]
    check(bc, make(new, lens, 4, 2, 64, F16, seed=15))


def test_offsets_past_32_bits(bc):
    """A cache of more than 2^32 bytes: pages at its far end."""
    pool, hkv, dim = 300000, 8, 128  # 16 * 8 * 128 * 2 bytes a page: 9.8 GB each
    k = torch.empty(pool, 16, hkv, dim, dtype=F16, device="cuda")
    v = torch.empty_like(k)
    f = make([5], [100], 16, hkv, dim, F16, seed=16)
    far = [pool - 1, 131072 + 5, 262143, 262144, 262145, pool - 2, 0]
    for i, page in enumerate(far):
        k[page], v[page] = f["k"][f["pages"][0, i]], f["v"][f["pages"][0, i]]
    want = bc.chunk_attention(**f)
    got = bc.chunk_attention(f["q"], k, v, torch.tensor([far], dtype=torch.int32, device="cuda"),
                             f["query_start"], f["lengths"])
    assert torch.equal(got, want)


def test_determinism_streams_and_graph(bc):
    f = make([1, 200, 1], [9000, 700, 3000], 8, 2, 128, BF16, seed=17)
    want = bc.chunk_attention(**f)
    for _ in range(5):
        assert torch.equal(bc.chunk_attention(**f), want)
    # two calls at once on two streams
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(10):
        for s, o in zip(streams, outs):
            with torch.cuda.stream(s):
                o.append(bc.chunk_attention(**f))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for o in outs for x in o)
    # captured, replayed on changed inputs
    out = torch.empty_like(f["q"])
    args = [f[n] for n in ("q", "k", "v", "pages", "query_start", "lengths")]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        bc.chunk_attention_out(*args, out)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    f["q"].mul_(-1)
    f["lengths"][0] = 4000
    want = bc.chunk_attention(**f)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_matches_decode_and_tree(bc):
    """One token per request is the decode op's result; a chain of drafted nodes
    is the tree op's, once the nodes' rows are in the cache."""
    f = make([1, 1], [500, 37], 8, 2, 128, F16, seed=18)
    got = torch.empty(2, 8, 128, device="cuda")
    bc.chunk_attention_out(*f.values(), got)
    want = bc.paged_decode(f["q"], f["k"], f["v"], f["pages"], f["lengths"])
    torch.testing.assert_close(got, want, atol=2e-3, rtol=2e-3)
    n, length = 7, 100
    f = make([n], [length], 8, 2, 128, F16, seed=19)
    at = [(int(f["pages"][0, j // 16]), j % 16) for j in range(length - n, length)]
    dk = torch.stack([f["k"][p, s] for p, s in at])[None]
    dv = torch.stack([f["v"][p, s] for p, s in at])[None]
    parent = torch.arange(-1, n - 1, dtype=torch.int32, device="cuda")[None]
    want = bc.tree_verify(f["q"][None], f["k"], f["v"], f["pages"],
                          torch.tensor([length - n], dtype=torch.int32, device="cuda"), dk, dv,
                          parent.contiguous())
    got = bc.chunk_attention(**f)
    torch.testing.assert_close(got.float(), want[0], atol=2e-3, rtol=2e-3)


def test_refusals(bc):
    f = make([4], [20], 8, 2, 64, F16)

    def refuses(**change):
        with pytest.raises((RuntimeError, NotImplementedError)):
            bc.chunk_attention(**(f | change))

    refuses(q=f["q"].bfloat16())
    refuses(q=f["q"].float())
    refuses(q=f["q"].transpose(0, 1).contiguous().transpose(0, 1))
    refuses(q=f["q"][:, :7].contiguous())
    refuses(k=f["k"].bfloat16())
    refuses(k=f["k"][:, :8].contiguous(), v=f["v"][:, :8].contiguous())
    refuses(lengths=f["lengths"].long())
    refuses(query_start=f["query_start"][:1].contiguous())
    refuses(scale=0.0)
    refuses(scale=float("nan"))
    refuses(softcap=-1.0)
    refuses(softcap=float("inf"))
    refuses(window=-1)
    refuses(alibi_slopes=torch.ones(7, device="cuda"))
    refuses(prefix=torch.ones(2, dtype=torch.int32, device="cuda"))
    refuses(key_start=torch.ones(3, dtype=torch.int32, device="cuda"))
    refuses(pages=f["pages"].cpu())
    odd = torch.zeros(4 * 8 * 64 + 1, dtype=F16, device="cuda")[1:].view(4, 8, 64)
    refuses(q=odd)
    with pytest.raises(RuntimeError):
        bc.chunk_attention_out(*f.values(), torch.empty(4, 8, 64, dtype=BF16, device="cuda"))
    empty = bc.chunk_attention(f["q"][:0], f["k"], f["v"], f["pages"], f["query_start"] * 0,
                               f["lengths"])
    assert empty.shape == (0, 8, 64)


@pytest.mark.parametrize("dtype,dim", [(F16, 64), (BF16, 128)])
def test_key_starts_in_any_order(bc, dtype, dim):
    f = make([300, 1, 77], [520, 400, 77], 4, 2, dim, dtype, seed=11)
    g = torch.Generator(device="cuda").manual_seed(3)
    start = torch.randint(-5, 560, (378,), generator=g, device="cuda", dtype=torch.int32)
    check(bc, f, key_start=start)
    check(bc, f, key_start=start, window=40)


def test_as_many_requests_as_allowed(bc):
    new = [(b * 7) % 3 for b in range(4096)]
    lens = [n + (b * 5) % 40 for b, n in enumerate(new)]
    check(bc, make(new, lens, 2, 1, 64, F16, seed=12))
