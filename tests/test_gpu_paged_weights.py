"""What happens to the softmax weights of paged attention: small ones beside a large one, NaN, long sums, the kernels'
different row counts.  Every operator against its definition in 64 bits; tolerances beside each test."""

import math

import pytest
import torch

from kiv_b200 import paged
from tests.gpu_helpers import DEV
from tests.test_gpu_paged import BF, FP, HALF, HF, Case, ref_attend

pytestmark = pytest.mark.gpu


def shared_pages(L, S, hkv, D, dtype, batch):
    """One run of pages in order that every sequence of the batch owns: (k_pages, v_pages, block_table), zeros."""
    N = -(-L // S)
    kp = torch.zeros(N, hkv, S, D, dtype=dtype, device=DEV)
    return kp, torch.zeros_like(kp), torch.arange(N, dtype=torch.int32, device=DEV).repeat(batch, 1)


def ints(*lists):
    return [torch.tensor(x, dtype=torch.int32, device=DEV) for x in lists]


@pytest.mark.parametrize("dtype,D,S,tile", [(FP, 64, 32, 32), (BF, 80, 32, 64)])
def test_sums_of_like_weights_do_not_drift(dtype, D, S, tile):
    """Equal scores but one, 1 above, over 262144 keys that one block walks: 888 sequences of 64 heads, a multiple of the
    blocks.  Adding a weight e^-1 at a time in fp32 is off by 4.2e-4 (every addition rounds the same way); the sums of
    key tiles by at most half a step of the running sum at each of n = 262144 / tile additions, n 2^-25, 2.5e-4 and 1.3e-4.
    The exponential and the logarithm add 1e-5; the output, whose sum is formed alike, twice that bound."""
    L = 262144
    kp, vp, table = shared_pages(L, S, 1, D, dtype, 888)
    vp.fill_(1)
    kp[0, 0, 0, 0] = 1
    q = torch.zeros(888, 64, D, dtype=dtype, device=DEV)
    q[..., 0] = 1
    out, lse = paged.paged_attend(q, kp, vp, table, *ints([L] * 888, range(889)), 1.0, max_query_len=1, return_lse=True)
    bound = L / tile * 2.0 ** -25 + 1e-5
    assert (lse.double() - math.log(math.e + L - 1)).abs().max() <= bound
    half = HALF[dtype] * (2 if dtype != FP else 1)              # the output's rounding and, 16 bits, the weights'
    assert (out.double() - 1).abs().max() <= 2 * bound + half


@pytest.mark.parametrize("dtype,D,S,tile", [(FP, 64, 32, 32), (FP, 256, 32, 32), (BF, 80, 32, 64), (HF, 128, 10, 64)])
@pytest.mark.parametrize("heads", [8, 64])
def test_small_weights_reach_the_sum_of_a_large_one(dtype, D, S, tile, heads):
    """One key scores 17.5 above 60000 others, whose weights, 2.5e-8 each, are below half a step of the sum 1 that they
    are added to: 1.5e-3 in all.  Added by key tiles (16 to 64 of them at a time), each addition is off by at most half a
    step, 2^-24 (2^-25 below 1): 60000 / tile of them, 1.2e-4 and 6e-5; scores and logarithm, 2e-5 of 17.5 as elsewhere."""
    L, n = 60000, 450
    kp, vp, table = shared_pages(L, S, 1, D, dtype, n)
    kp[0, 0, 0, 0] = 17.5
    vp[0, 0, 0, 0] = 1
    q = torch.zeros(n, heads, D, dtype=dtype, device=DEV)
    q[..., 0] = 1
    out, lse = paged.paged_attend(q, kp, vp, table, *ints([L] * n, range(n + 1)), 1.0, max_query_len=1, return_lse=True)
    off = L / tile * 2.0 ** -24
    want = 17.5 + math.log1p((L - 1) * math.exp(-17.5))
    assert (lse.double() - want).abs().max() <= off + 2e-6 * 17.5
    assert (out[..., 0].double() * math.exp(want - 17.5) - 1).abs().max() <= off + 2e-5 + HALF[dtype]


@pytest.mark.parametrize("D,S,hq,new", [
    (128, 128, 8, [1] * 200), (64, 16, 7, [18, 1, 5] * 60), (96, 48, 1, [40000]), (128, 16, 8, [5000, 1, 900]),   # tcgen05
    (256, 64, 8, [3] * 90), (256, 128, 8, [2900, 100]),
    (80, 16, 8, [1] * 500), (80, 16, 8, [3] * 300), (128, 10, 8, [40] * 300)])                                    # warp-level MMAs
def test_fp16_weights_far_below_the_largest_count(D, S, hq, new):
    """One key with value 0 scores 17.5 above a tail of 60000 whose values are around 1: the result is the tail's share,
    1.5e-3.  Each weight is rounded to fp16, at most half a step h = 2^-11 of itself while it is a normal number (2 h for
    the few that are not), the output to h of itself, the tensor cores' cutting sums over at most 128 key tiles 1e-4 (as in the drift
    tests), and the sum of the weights, near 1, is off by at most half a step at each of up to 940 key tiles, 6e-5; scores
    near 17.5 in fp32 and the exponential, 1e-5."""
    L = 60000
    g = torch.Generator(device=DEV).manual_seed(7)
    kp, vp, table = shared_pages(L, S, 1, D, HF, len(new))
    k, v = (x.view(-1, S, D)[:, :, :].reshape(-1, D) for x in (kp, vp))
    k[:, 1] = (torch.randn(k.shape[0], generator=g, device=DEV) * 0.5).to(HF)
    v.copy_((torch.randn(v.shape, generator=g, device=DEV) / 4 + 1).to(HF))
    k[0], v[0] = 0, 0
    k[0, 0] = 17.5
    q = torch.zeros(sum(new), hq, D, dtype=HF, device=DEV)
    q[..., 0] = 1
    q[..., 1] = torch.rand(q.shape[:2], generator=g, device=DEV).to(HF)
    lens = [L - 37 * (b % 5) for b in range(len(new))]
    starts = [sum(new[:b]) for b in range(len(new) + 1)]
    errors = torch.zeros(1, dtype=torch.int64, device=DEV)
    out, lse = paged.paged_attend(q, kp, vp, table, *ints(lens, starts), 1.0, max_query_len=max(new), return_lse=True, errors=errors)
    h = HALF[HF]
    for b in sorted({0, 1, len(new) // 2, len(new) - 1} & set(range(len(new)))):
        for i in sorted({0, new[b] // 2, new[b] - 1}):
            t, n = starts[b] + i, lens[b] - new[b] + i + 1
            x = q[t].double() @ k[:n].double().T
            want = torch.softmax(x, -1) @ v[:n].double()
            assert want.abs().max() < 5e-3
            assert ((out[t].double() / want - 1).abs() <= 3 * h + 2e-4).all(), (t, (out[t].double() / want - 1).abs().max())
            assert (lse[t].double() - x.logsumexp(-1)).abs().max() <= 2e-5 * 17.5
    assert int(errors) == 0


@pytest.mark.parametrize("dtype,D,S", [(BF, 128, 16), (HF, 64, 16), (BF, 256, 32), (BF, 80, 16), (HF, 128, 10), (FP, 64, 16), (FP, 40, 8)])
@pytest.mark.parametrize("n,L", [(1, 300), (3, 70), (90, 200), (1, 30000), (200, 20000)])
def test_nan_in_a_live_row_reaches_the_results_it_belongs_to(dtype, D, S, n, L):
    """A NaN query gives a NaN row, a NaN key a NaN for every row that sees it; nothing else changes."""
    c = Case([n, n], [L, L], 4, 2, D, S, dtype, seed=n)
    t = n // 2
    clean, clse = paged.paged_attend(c.q, *c.args(), D ** -0.5, return_lse=True)
    c.q[t, 1, 3] = math.nan                                     # sequence 0, one token, one head
    j = L - n + t                                               # sequence 1: the key of its new token t, key head 1
    pg = int(c.table[1, j // S])
    c.kp[pg, 1, j % S, 5] = math.nan
    out, lse = paged.paged_attend(c.q, *c.args(), D ** -0.5, return_lse=True, errors=c.errors)
    bad = torch.zeros(2 * n, 4, dtype=torch.bool, device=DEV)
    bad[t, 1] = True
    bad[n + t:, 2:] = True
    assert torch.isnan(out[bad]).all() and torch.isnan(lse[bad]).all()
    assert torch.equal(out[~bad], clean[~bad]) and torch.equal(lse[~bad], clse[~bad])
    assert int(c.errors) == 0


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D,S", [(80, 16), (192, 16), (128, 10), (64, 7), (256, 12)])
def test_the_hint_of_the_longest_query_changes_no_precision(dtype, D, S):
    """The warp-level kernels go by max_query_len (16, 32 or 64 rows) or the mean.  Whatever it says, few keys or many:
    the weights keep twice the rows' bits, so an output is off by its own rounding, half a step, and 2e-5 of the largest
    value for fp32 sums (a weight rounded once would be off by up to half a step of the largest value)."""
    for new, lens in (([1, 2, 1], [3, 2, 5]), ([5, 1, 40], [9, 300, 77])):
        c = Case(new, lens, 8, 2, D, S, dtype, seed=D)
        want, _ = ref_attend(c.q, c.kp, c.vp, c.table, c.lens, c.starts, D ** -0.5)
        for hint in (0, 1, 5, 12, 40, 4000):
            got = paged.paged_attend(c.q, *c.args(), D ** -0.5, max_query_len=hint, errors=c.errors).double()
            err = (got - want).abs() - HALF[dtype] * want.abs() - 2e-5 * c.v_live
            assert (err <= 0).all(), (hint, err.max())
        assert int(c.errors) == 0
