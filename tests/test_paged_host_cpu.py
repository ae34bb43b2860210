"""The host side of the rotation and paged-cache operators, without a GPU."""

import pytest
import torch
from torch.autograd import forward_ad

from kiv_b200 import _native as nat
from kiv_b200 import paged


def test_inputs_with_a_tangent_are_refused():
    q, k, w = torch.zeros(1, 2, 1, 64), torch.zeros(1, 1, 1, 64), torch.ones(64)
    rows, pages, ints = torch.zeros(1, 1, 64), torch.zeros(1, 1, 8, 64), torch.zeros(1, 1, dtype=torch.int32)
    calls = [lambda d: paged.qk_norm_rope(d(q), k, eps=1e-6), lambda d: paged.qk_norm_rope(q, k, eps=1e-6, k_weight=d(w)),
             lambda d: paged.paged_append(rows, d(rows), pages, pages, ints, ints[0], ints[0]),
             lambda d: paged.paged_attend(d(rows), pages, pages, ints, ints[0], ints[0], 1.0)]

    def dual(x):
        return forward_ad.make_dual(x, torch.ones_like(x))

    with forward_ad.dual_level():
        for call in calls:
            with pytest.raises(nat.KIVNativeError, match="tangent"):
                call(dual)
            with torch.no_grad(), pytest.raises(nat.KIVNativeError, match="tangent"):     # which keeps tangents
                call(dual)
            with pytest.raises(nat.KIVNativeError, match="CUDA device"):                  # passes on to the next check
                call(lambda x: x)
    with pytest.raises(nat.KIVNativeError, match="tangent"):
        torch.func.jvp(lambda x: paged.qk_norm_rope(x, None, eps=1e-6)[0], (q,), (q,))
