"""chunk_attention where its arithmetic can go wrong: score caps from tiny to
huge, bits that must not depend on what a row does not see, infinities and NaN
in what it does see, and probabilities far below the largest one."""
import math

import pytest
import torch

import serving_oracle as S
from test_gpu_chunk_attention import BF16, F16, check, make

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan


@pytest.fixture(scope="module")
def bc():
    import branchcraft_torch

    return branchcraft_torch


# ------------------------------------------------------- bits and unseen values


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("softcap", [4.0, 30.0])
@pytest.mark.parametrize("bad", [60.0, INF, -INF, NAN])
def test_unseen_keys_change_no_capped_bit(bc, dtype, softcap, bad):
    """Slots past the lengths, pages that no token sees and keys that only later
    tokens see, with scores capped and seven heads a group (126 of 128 rows used)."""
    f = make([60, 1], [200, 1000], 14, 2, 128, dtype, seed=7)
    want = bc.chunk_attention(**f, window=130, softcap=softcap)
    g = dict(f, k=f["k"].clone(), v=f["v"].clone())
    used = torch.zeros(f["k"].shape[0], 16, dtype=torch.bool)
    for b, (n, x) in enumerate(((60, 200), (1, 1000))):
        for j in range(max(0, x - n + 1 - 130), x):
            used[int(f["pages"][b, j // 16]), j % 16] = True
    for name in ("k", "v"):
        g[name][~used.cuda()] = bad
    assert torch.equal(bc.chunk_attention(**g, window=130, softcap=softcap), want)
    k = f["k"].clone()
    k[int(f["pages"][0, 199 // 16]), 199 % 16] = bad
    got = bc.chunk_attention(**dict(f, k=k), window=130, softcap=softcap)
    assert torch.equal(got[:59], want[:59]) and torch.equal(got[60:], want[60:])


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_other_requests_change_no_capped_bit(bc, dtype):
    """A request's last row tile also holds the next request's rows."""
    f = make([20, 41], [300, 41], 14, 2, 128, dtype, seed=8)
    want = bc.chunk_attention(**f, softcap=30.0)
    q = f["q"].clone()
    q[20:] *= 60
    got = bc.chunk_attention(**dict(f, q=q), softcap=30.0)
    assert torch.equal(got[:20], want[:20])
    # one row's scores do not change the next row's
    q = f["q"].clone()
    q[3, 5] *= 60
    got = bc.chunk_attention(**dict(f, q=q), softcap=30.0)
    same = torch.ones(61, 14, dtype=torch.bool, device="cuda")
    same[3, 5] = False
    assert torch.equal(got[same], want[same])


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_earlier_calls_change_no_capped_bit(bc, dtype):
    """With seven heads a group two rows of a tile are nobody's: what an earlier
    launch left in their place is not looked at."""
    f = make([18], [300], 7, 1, 128, dtype, seed=9)
    calm = make([2500], [2500], 8, 1, 128, dtype, seed=10)
    wild = dict(calm, q=calm["q"] * 100)
    got = []
    for before in (calm, wild, calm, wild):
        bc.chunk_attention(**before, softcap=30.0)
        got.append(bc.chunk_attention(**f, softcap=30.0))
    assert all(torch.equal(x, got[0]) for x in got)


# ------------------------------------------------------------------ score caps


def two_keys(scale, softcap, most, dtype, dim=128):
    """64 heads of one token that sees two keys. Key 1, the token's own, has score 0; head
    h's score with key 0 is near softcap * tanh(u_h), |u_h| <= most, and its distance bias
    takes about as much off: the output weighs what is left."""
    u = torch.cat([torch.linspace(-1, 1, 58), torch.tensor([0, 1e-6, -1e-6, 1e-3, -1e-3, 0.02])])
    u = u.double() * most
    q = (u * softcap / scale / dim).to(dtype)[None, :, None].expand(1, 64, dim).contiguous()
    k = torch.zeros(1, 16, 1, dim, dtype=dtype)
    k[0, 0] = 1
    v = torch.zeros(1, 16, 1, dim, dtype=dtype)
    v[0, 0], v[0, 1] = 1, -1
    score = softcap * torch.tanh(q[0, :, 0].double() * dim * scale / softcap)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    f = dict(q=q.cuda(), k=k.cuda(), v=v.cuda(), pages=ints([[0]]), query_start=ints([0, 1]),
             lengths=ints([2]))
    return f, score.float().cuda()


@pytest.mark.parametrize("dtype,scale,softcap", [
    (F16, 0.0884, 0.5), (F16, 0.0884, 50.0), (BF16, 0.0884, 50.0), (BF16, 0.001, 50.0),
    (F16, 0.0884, 3000.0), (BF16, 0.0884, 1e4), (F16, 0.0884, 1e5), (BF16, 1e-5, 1.0),
    (BF16, 1.0, 1e-4), (BF16, 1.0, 1e-7), (BF16, 1e-3, 1e-30)])
@pytest.mark.parametrize("most", [0.34, 0.745, 4.0])
def test_cap_of_any_size(bc, dtype, scale, softcap, most):
    f, score = two_keys(scale, softcap, most, dtype)
    got = check(bc, f, out_dtype=torch.float32, scale=scale, softcap=softcap, alibi_slopes=score)
    # q.k is exact here (128 equal terms of at most 11 bits), so the score is off by its own
    # arithmetic alone: some eight roundings of 2^-24 of the cap, the polynomial's 2^-26, and
    # 2^-22 for each approximate unit: below 2^-19 of the cap. The output is tanh(x / 2) of
    # what is left, whose slope is 1/2 at most.
    want = S.chunk_attention(**f, scale=scale, softcap=softcap, alibi_slopes=score)[0]
    tol = 2.0 ** -20 * softcap + torch.finfo(dtype).eps / 2 + 2.0 ** -16
    assert ((got.cpu().double() - want).abs() <= tol).all()
    # the same scores without the bias, and rows of zeros
    check(bc, f, scale=scale, softcap=softcap)
    f["q"].zero_()
    f["v"].fill_(1)
    check(bc, f, scale=scale, softcap=softcap)


@pytest.mark.parametrize("softcap", [1e3, 1e5, 1e10, 1e25, 3e38])
def test_wide_caps_leave_scores(bc, softcap):
    """A cap far beyond the scores: what there is without one (softcap * tanh(x / softcap)
    is x but for (x / softcap)^2 / 3, 1e-5 at most here)."""
    f = make([50, 1], [300, 700], 6, 2, 128, F16, seed=21)
    check(bc, f, softcap=softcap)


@pytest.mark.parametrize("softcap", [1e-3, 1e-10, 1e-38, 1e-45])
def test_narrow_caps_leave_the_mean(bc, softcap):
    f = make([50, 1], [300, 700], 6, 2, 128, F16, seed=22)
    f["q"][7] = 0
    check(bc, f, softcap=softcap)


# ------------------------------------------------- values that are not finite


def natural(f, softcap=0.0):
    """(out, tolerance) of a single request by the formula in 64 bits, where infinities
    and NaN go as they may: a row that sees a score of +inf or NaN is NaN, so is one whose
    seen scores are all -inf. The tolerance is serving_oracle.assert_chunk_close's."""
    q, k, v = (f[n].cpu().double() for n in "qkv")
    n, hq, dim = q.shape
    length = int(f["lengths"][0])
    ids = f["pages"][0, :(length + 15) // 16].cpu().long()
    k, v = (t[ids].flatten(0, 1)[:length].repeat_interleave(hq // t.shape[2], 1) for t in (k, v))
    seen = S.visible(length, n)[:, None]
    x = torch.einsum("nhd,jhd->nhj", q, k) * dim ** -0.5
    if softcap:
        x = softcap * torch.tanh(x / softcap)
    x = x.masked_fill(~seen, -INF)
    p = torch.where(seen, torch.exp(x - x.amax(-1, keepdim=True)), 0.0)
    p = p / p.sum(-1, keepdim=True)
    out = torch.einsum("nhj,jhd->nhd", p, v)
    u = torch.finfo(f["q"].dtype).eps / 2
    big = torch.einsum("nhd,jhd->nhj", q.abs(), k.abs()).masked_fill(~seen, 0)
    big = big.masked_fill(~big.isfinite(), 0).amax(-1, keepdim=True) * dim ** -0.5
    tol = u * out.abs() + torch.einsum("nhj,jhd->nhd", p, v.abs()) * (1 + u) * (
        u + 2 * (dim + 8) * 2.0 ** -23 * big + 2.0 ** -16) + torch.finfo(f["q"].dtype).smallest_normal * u * 2
    return out, tol


def check_natural(bc, f, softcap=0.0):
    got = bc.chunk_attention(**f, softcap=softcap)
    want, tol = natural(f, softcap)
    g = got.cpu().double()
    assert torch.equal(torch.isnan(g), torch.isnan(want))
    fin = ~torch.isnan(want)
    assert ((g - want).abs()[fin] <= tol[fin]).all()
    return got


@pytest.mark.parametrize("dtype,dim", [(F16, 128), (BF16, 64)])
@pytest.mark.parametrize("new,length", [(40, 300), (5, 120), (1, 20), (1, 20000), (40, 6000)])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_queries_not_finite(bc, new, length, dtype, dim, bad):
    """Whole items and items split over blocks alike: the row is NaN, the others keep
    their bits."""
    f = make([new], [length], 6, 2, dim, dtype, seed=31)
    want = bc.chunk_attention(**f)
    f["q"][new // 2, 4, 7] = bad
    got = check_natural(bc, f)
    same = torch.ones(new, 6, dtype=torch.bool, device="cuda")
    same[new // 2, 4] = False
    assert got[new // 2, 4].isnan().all() and torch.equal(got[same], want[same])


@pytest.mark.parametrize("dtype,dim", [(F16, 128), (BF16, 64)])
@pytest.mark.parametrize("new,length", [(40, 300), (5, 120), (1, 20), (1, 20000), (40, 6000)])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_keys_not_finite(bc, new, length, dtype, dim, bad, softcap):
    """A key of KV head 1 that the last tokens see: their rows follow the formula, rows
    that do not see it keep their bits."""
    f = make([new], [length], 6, 2, dim, dtype, seed=32)
    want = bc.chunk_attention(**f, softcap=softcap)
    at = length - (new + 1) // 2
    f["k"][f["pages"][0, at // 16].item(), at % 16, 1, 7] = bad
    got = check_natural(bc, f, softcap)
    first = at - (length - new)
    if not softcap:
        assert torch.equal(got[:first], want[:first]) and torch.equal(got[:, :3], want[:, :3])


@pytest.mark.parametrize("dtype,dim", [(F16, 128), (BF16, 64)])
@pytest.mark.parametrize("new,length,ends", [(3, 3, 3), (1, 1, 1), (40, 300, 300), (1, 20000, 20000),
                                             (40, 300, 140), (1, 20000, 15000), (200, 200, 70)])
def test_scores_of_minus_infinity(bc, new, length, ends, dtype, dim):
    """Keys up to `ends` with scores of -inf: of no weight beside others, NaN where a row
    sees none but such."""
    f = make([new], [length], 6, 2, dim, dtype, seed=33)
    f["q"][..., 5] = 1
    for j in range(ends):
        f["k"][f["pages"][0, j // 16].item(), j % 16, :, 5] = -INF
    got = check_natural(bc, f)
    assert got.isnan().any() == (length - new < ends)


# --------------------------------------------------------- small probabilities


@pytest.mark.parametrize("new,batch,length", [(1, 160, 60000), (100, 40, 20000)])
def test_many_small_probabilities(bc, new, batch, length):
    """One key of score 18 and tens of thousands of score 0, 2^-26 of its weight each and a
    thousandth of the output together. FP16 probabilities that small are rounded to
    2^-25 2^-7 of the largest one (its smallest step, at the kernel's scale of 2^7). All
    requests hold the same pages: enough of them that items are hardly split."""
    f = make([new], [length], 8, 1, 128, F16, seed=41)
    f["q"].fill_(18 / 128 ** 0.5)
    f["k"].zero_()
    f["v"].fill_(1)
    first = f["pages"][0, 0].item()
    f["k"][first, 0] = 1
    f["v"][first, 0] = 0
    got = bc.chunk_attention(
        f["q"].repeat(batch, 1, 1), f["k"], f["v"], f["pages"].repeat(batch, 1),
        torch.arange(batch + 1, dtype=torch.int32, device="cuda") * new, f["lengths"].repeat(batch))
    got = got.cpu().double().view(batch, new, 8, 128)
    want, spread, big = S.chunk_attention(**f)
    u = 2.0 ** -11
    tol = u * want + spread * (u + 2 * 136 * 2.0 ** -23 * big + 2.0 ** -16) + length * 2.0 ** -32
    assert (want > 2e-4).all() and ((got - want).abs() <= tol).all()


# ----------------------------------------------------------------- FP32 output


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,lens,hq,hkv", [
    ([1], [1], 1, 1), ([1, 1, 1], [1, 130, 1000], 8, 2), ([129], [640], 6, 2),
    ([200, 1, 0, 37], [200, 900, 40, 37], 8, 2), ([7, 7], [200, 16], 14, 2), ([300], [300], 7, 1),
    ([1, 3], [20000, 9001], 8, 2), ([700], [1800], 2, 1)])
def test_fp32_output_keeps_probabilities(bc, new, lens, hq, hkv, dim, dtype):
    """For FP32 output a probability is two 16-bit numbers: what the first rounds off, 2^-9
    of it at most, the second holds to 2^-9 of that (2^-12 and 2^-24 for FP16): 2^-18
    together, within assert_chunk_close's 2^-16 for the exponential; no rounding of 2^-9 or
    2^-12 is left. Sixteen additions to the output a tile of 128 keys, of two products of
    eight steps each, may cut 2^-23 of the sum."""
    f = make(new, lens, hq, hkv, dim, dtype, seed=51)
    for options in ({}, dict(softcap=20.0, window=300), dict(scale=0.3)):
        got = torch.full(f["q"].shape, NAN, device="cuda")
        bc.chunk_attention_out(*(f[n] for n in ("q", "k", "v", "pages", "query_start", "lengths")),
                               got, **options)
        want, spread, big = S.chunk_attention(**f, **options)
        tiles = torch.tensor([(x + 127) // 128 for n, x in zip(new, lens) for _ in range(n)])
        tol = 2.0 ** -24 * want.abs() + spread * (
            2 * (dim + 8) * 2.0 ** -23 * big + 2.0 ** -16 + 2.0 ** -19 * tiles[:, None, None])
        assert ((got.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_fp32_output_is_the_rounded_output_unrounded(bc, dtype):
    """Empty rows, masked rows, NaN and rows of nobody as with 16-bit output."""
    f = make([40, 30], [300, 64], 14, 2, 128, dtype, seed=52)
    ks = torch.zeros(70, dtype=torch.int32, device="cuda")
    ks[5], ks[50] = 2 ** 31 - 1, 60
    f["q"][9, 3, 4] = NAN
    f["q"] = torch.cat([f["q"], f["q"][:6]])
    ks = torch.cat([ks, ks[:6]])
    a = torch.full(f["q"].shape, 7.0, device="cuda")
    b = a.to(dtype)
    for out in (a, b):
        bc.chunk_attention_out(*(f[n] for n in ("q", "k", "v", "pages", "query_start", "lengths")),
                               out, key_start=ks)
    assert torch.equal(a.isnan(), b.isnan()) and a[9, 3].isnan().all()
    assert (a[5] == 0).all() and (b[5] == 0).all() and (a[70:] == 7).all()
    fin = ~a.isnan()
    # both within 2^-9 (2^-12) of the weights times |v| < 6 and the output's own rounding
    eps = torch.finfo(dtype).eps
    assert ((a - b.float()).abs()[fin] <= eps * (6 + a.abs()[fin])).all()


# ------------------------------------------------------------- very large scores


@pytest.mark.parametrize("dtype,dim,size", [
    (F16, 128, 200.0), (F16, 64, 3000.0), (F16, 128, 60000.0), (BF16, 128, 200.0),
    (BF16, 64, 3e9), (BF16, 128, 1e18)])
@pytest.mark.parametrize("new,length", [(1, 17), (40, 300), (1, 20000), (150, 3000)])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_any_finite_size(bc, new, length, sign, dtype, dim, size):
    """Scores from 10^5 to 10^38, whose last place is many powers of e. All equal: the mean of
    the seen values. One key a 64th above the others: that key's value alone."""
    f = make([new], [length], 4, 2, dim, dtype, seed=61)
    f["q"].fill_(sign * size)
    f["k"].fill_(size)
    ids = f["pages"][0, :(length + 15) // 16].long()
    v = f["v"][ids].flatten(0, 1)[:length].cpu().double().repeat_interleave(2, 1)
    at = length - new + torch.arange(new)
    got = bc.chunk_attention(**f).cpu().double()
    want = v.cumsum(0)[at] / (at + 1.0)[:, None, None]
    spread = v.abs().cumsum(0)[at] / (at + 1.0)[:, None, None]
    # equal weights, each rounded to 16 bits; the sums' FP32 additions (sixteen a tile at most,
    # 2^-23 each) and the output's rounding
    u = torch.finfo(dtype).eps / 2
    tol = u * want.abs() + spread * (1 + u) * (u + 2.0 ** -16 + 2.0 ** -19 * ((length + 127) // 128))
    assert ((got - want).abs() <= tol).all()
    first = length // 2
    f["k"][ids[first // 16], first % 16] *= 1 + sign / 64
    seen = at >= first
    got = bc.chunk_attention(**f).cpu().double()
    # Its weight need not be 1: up to 2^20 (in log2 units) the exponent is the unrounded
    # product less its rounded value, up to 2^-5 apart, so the weight 2^(2^-5) at most. That
    # is rounded to 16 bits (u) in the product and not in the sum; then the output's u.
    alone = v[first].expand(int(seen.sum()), -1, -1)
    assert ((got[seen] - alone).abs() <= 2 * u * (1 + u) * alone.abs()).all()
