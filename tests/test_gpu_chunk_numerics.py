"""chunk_attention where its arithmetic can go wrong: infinities and NaN in what
a row sees."""
import math

import pytest
import torch

import serving_oracle as S
from test_gpu_chunk_attention import BF16, F16, make

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan


@pytest.fixture(scope="module")
def bc():
    import branchcraft_torch

    return branchcraft_torch


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
