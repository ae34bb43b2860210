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
