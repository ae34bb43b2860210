"""Calls of the rotation and paged-cache operators that their documentation allows: rows at any address, steps of a cache
whose sequences come and go, capture before the first token."""

import pytest
import torch

from kiv_b200 import PagedKVCache, paged
from kiv_b200.middleware import fused_rotary
from tests.gpu_helpers import DEV
from tests.test_gpu_paged import BF, FP, HF, Case

pytestmark = pytest.mark.gpu


def _shifted(x):
    """The same values, contiguous, one element behind an aligned address."""
    flat = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)
    y = flat[1:].view(x.shape)
    y.copy_(x)
    assert y.is_contiguous() and y.data_ptr() % 16
    return y


@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_contiguous_rows_off_a_16_byte_boundary(dtype):
    """Such rows are copied by the operators; results are those of aligned ones, to the bit."""
    g = torch.Generator(device=DEV).manual_seed(1)
    q, k = (torch.randn(2, h, 5, 64, generator=g, device=DEV).to(dtype) for h in (4, 2))
    cos, sin = paged.rotary_table(1e4 ** (-torch.arange(32, dtype=torch.float64, device=DEV) / 32), 10)
    w = torch.randn(64, generator=g, device=DEV).to(dtype)
    want = paged.qk_norm_rope(q, k, cos, sin, eps=1e-6, q_weight=w, k_weight=w)
    got = paged.qk_norm_rope(_shifted(q), _shifted(k), _shifted(cos), _shifted(sin), eps=1e-6, q_weight=_shifted(w), k_weight=_shifted(w))
    assert all(torch.equal(a, b) for a, b in zip(want, got))

    c = Case([3, 40], [30, 90], 8, 2, 64, 16, dtype)
    want = paged.paged_attend(c.q, *c.args(), 0.1)
    assert torch.equal(paged.paged_attend(_shifted(c.q), *c.args(), 0.1), want)
    pages = [x.clone() for x in (c.kp, c.vp)]
    paged.paged_append(c.k, c.v, *c.args(), cos=cos.repeat(9, 1), sin=sin.repeat(9, 1))
    paged.paged_append(_shifted(c.k), _shifted(c.v), *pages, *c.args()[2:], cos=cos.repeat(9, 1), sin=sin.repeat(9, 1))
    assert all(torch.equal(a.nan_to_num(7), b.nan_to_num(7)) for a, b in zip(pages, (c.kp, c.vp)))


@torch.no_grad()
def test_fused_rotation_of_rows_off_a_16_byte_boundary():
    """Where the model's own function works, the one in its place does too."""
    def fail(*args, **kwargs):
        raise AssertionError("the kernel takes these")

    q, k = torch.randn(1, 4, 3, 64, device=DEV, dtype=BF), torch.randn(1, 2, 3, 64, device=DEV, dtype=BF)
    ang = torch.rand(1, 3, 32, device=DEV) * 6
    cos, sin = (torch.cat([f, f], -1).to(BF) for f in (ang.cos(), ang.sin()))
    turn = fused_rotary(fail)
    want, got = turn(q, k, cos, sin), turn(_shifted(q), _shifted(k), _shifted(cos), _shifted(sin))
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_fused_rotation_of_rows_with_a_tangent():
    """The kernel has no derivative: the model's own function answers, tangent and all."""
    def plain(q, k, cos, sin):
        calls.append(1)
        return q * cos[:, None], k * cos[:, None]

    calls = []
    turn = fused_rotary(plain)
    q, k = torch.randn(1, 4, 3, 64, device=DEV), torch.randn(1, 2, 3, 64, device=DEV)
    cos, sin = torch.rand(1, 3, 64, device=DEV), torch.rand(1, 3, 64, device=DEV)
    got, tangent = torch.func.jvp(lambda x: turn(x, k, cos, sin)[0], (q,), (torch.ones_like(q),))
    assert calls == [1] and torch.equal(got, q * cos[:, None]) and torch.equal(tangent, cos[:, None].expand_as(q))
    turn(q, k, cos, sin)
    assert calls == [1]


def test_the_table_of_a_cache_follows_its_sequences():
    """Sequences that come, go, change places and take an old name: the device table is each step's sequences' pages, and a
    step waits for nothing on the device."""
    cache = PagedKVCache(40, 4, 1, 64, device=DEV, max_batch=4, max_pages_per_seq=9)
    steps = [[("a", 9), ("b", 30)], [("a", 1), ("b", 1)], [("b", 1), ("a", 3)], "b", [("c", 5), ("a", 1), ("b", 2)], [("a", 1)], "a",
             [("a", 4), ("d", 36), ("c", 0), ("b", 3)], [("a", 1), ("c", 8), ("b", 1)], "d", [("c", 1), ("d", 1)]]
    for new in steps:
        if isinstance(new, str):
            cache.free(new)
            continue
        torch.cuda.set_sync_debug_mode("error")
        try:
            rows = cache.step(new)
        finally:
            torch.cuda.set_sync_debug_mode("default")
        table, lens, starts = (x.tolist() for x in cache.arrays())
        assert rows == starts[-1] and lens == [cache.length(s) for s, _ in new]
        seen = set()
        for row, n, (s, _) in zip(table, lens, new):
            held = -(-n // 4)
            assert all(p >= 0 for p in row[:held]) and row[held:] == [-1] * (9 - held) and not seen & set(row[:held])
            seen |= set(row[:held])


@pytest.mark.parametrize("D,S", [(128, 16), (80, 10)])
def test_capture_before_the_first_token_and_steps_of_fewer_rows(D, S):
    """A layer captured over a step without tokens serves steps of up to the captured rows; the rows of the captured call
    behind a step's tokens stay as they are."""
    caches = [PagedKVCache(64, S, 2, D, dtype=BF, device=DEV, max_batch=3) for _ in range(2)]
    g = torch.Generator(device=DEV).manual_seed(2)
    q, k, v = (torch.zeros(6, h, D, device=DEV, dtype=BF) for h in (8, 2, 2))
    out = torch.zeros_like(q)
    caches[0].step([(s, 0) for s in "xyz"])
    before = caches[0].k.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        caches[0].append(0, k, v)
        caches[0].attend(0, q, 0.1, out=out)
    assert torch.equal(caches[0].k, before)
    for new in ([2, 1, 3], [1, 1, 1], [0, 5, 0], [2, 2, 2], [1, 0, 1]):
        for t in (q, k, v):
            t.normal_(generator=g)
        out.fill_(7)
        rows = [c.step(list(zip("xyz", new))) for c in caches]
        assert rows == [sum(new)] * 2
        graph.replay()
        caches[1].append(0, k[:rows[0]], v[:rows[0]])
        want = caches[1].attend(0, q[:rows[0]], 0.1)
        if D == 128:
            assert torch.equal(out[:rows[0]], want)
        else:       # other row counts, other order of sums: each within half a step and 2e-5 of the values' largest
            assert ((out[:rows[0]] - want).abs() <= 2.0 ** -7 * want.abs() + 4e-5 * 6).all()
        assert (out[rows[0]:] == 7).all() and torch.equal(*[c.k for c in caches])
    assert int(caches[0].errors) == 0
