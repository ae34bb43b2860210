"""Paged-cache operators and the query/key turn against their definitions in 64 bits.

Tolerances.  Rows: the turn is computed in fp32 (a norm of D squares, two products and a sum) and rounded once, so an
element is off by half a step of its type plus a few fp32 steps of the row's largest element (1e-6 of it).  Attention:
the output is a mean of values with weights that sum to 1.  Its own rounding is half a step of itself.  With 16-bit rows
the weights are rounded to the rows' type before the product: sum of p_j d_j v_j with |d_j| at most half a step, at most
half a step of the largest value.  Scores are fp32 sums of D products of 16- or 32-bit numbers and the exponential and
the sums over keys are fp32: together below 2e-5 of the largest value.  lse: scores up to ~20 in fp32, 2e-5.
"""

import math

import pytest
import torch

from kiv_b200 import _native as nat
from kiv_b200 import paged
from tests.gpu_helpers import DEV

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
HALF = {BF: 2.0 ** -8, HF: 2.0 ** -11, FP: 2.0 ** -24}


# ------------------------------------------------------------------ definitions
def ref_turn(x, w, eps, cos, sin, interleaved, offset=0.0):
    """x [..., D] float64; cos, sin [..., half] float64 or None."""
    if eps is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
        if w is not None:
            x = x * (offset + w.double())
    if cos is None:
        return x
    half = cos.shape[-1]
    y = x.clone()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    return y


def ref_attend(q, kp, vp, table, lens, starts, scaling, causal=True, window=0, softcap=0.0):
    T, Hq, D = q.shape
    N, Hkv, S, _ = kp.shape
    out = torch.zeros(T, Hq, D, dtype=torch.float64, device=q.device)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64, device=q.device)
    for b in range(len(lens)):
        lo, hi, L = starts[b], starts[b + 1], lens[b]
        n = hi - lo
        if n == 0 or L == 0:
            continue
        j = torch.arange(L, device=q.device)
        pg = table[b].long()[j // S]
        ok = (pg >= 0) & (pg < N)
        pg = pg.clamp(0, N - 1)
        k = torch.where(ok[:, None, None], kp[pg, :, j % S].double(), 0.0).repeat_interleave(Hq // Hkv, 1)
        v = torch.where(ok[:, None, None], vp[pg, :, j % S].double(), 0.0).repeat_interleave(Hq // Hkv, 1)
        s = torch.einsum("nhd,lhd->hnl", q[lo:hi].double(), k) * scaling
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        place = (L - n + torch.arange(n, device=q.device))[:, None]
        seen = (j <= place) if causal else torch.ones(n, L, dtype=torch.bool, device=q.device)
        if window:
            seen = seen & (j > place - window)
        s = s.masked_fill(~seen, -math.inf)
        z = torch.logsumexp(s, -1)
        p = torch.where(seen, torch.exp(s - z[..., None]), 0.0)
        out[lo:hi] = torch.einsum("hnl,lhd->nhd", p, v)
        lse[lo:hi] = z.T
    return out, lse


class Case:
    """A batch in pages: random page order, garbage (NaN) in every row that no token owns."""

    def __init__(self, new, lens, hq, hkv, D, S, dtype, seed=0, spare=2, engine_layout=False, pad=0):
        g = torch.Generator().manual_seed(seed)
        self.new, self.lens, self.S = new, lens, S
        need = [-(-x // S) for x in lens]
        width = max(1, max(need) + 1)
        N = sum(need) + spare
        perm = torch.randperm(N, generator=g).tolist()
        table = torch.full((len(lens), width), -1, dtype=torch.int32)
        at = 0
        for b, m in enumerate(need):
            table[b, :m] = torch.tensor(perm[at:at + m], dtype=torch.int32)
            at += m
        self.starts = [0]
        for n in new:
            self.starts.append(self.starts[-1] + n)
        T = self.starts[-1] + pad

        def rows(*shape):
            return torch.randn(shape, generator=g).to(dtype).to(DEV)

        shape = (N, S, hkv, D) if engine_layout else (N, hkv, S, D)
        self.kp, self.vp = torch.full(shape, math.nan, dtype=dtype, device=DEV), torch.full(shape, math.nan, dtype=dtype, device=DEV)
        if engine_layout:
            self.kp, self.vp = self.kp.transpose(1, 2), self.vp.transpose(1, 2)
        for b, L in enumerate(lens):
            j = torch.arange(L)
            pg = table[b].long()[j // S].to(DEV)
            off = (j % S).to(DEV)
            self.kp[pg, :, off] = rows(L, hkv, D)
            self.vp[pg, :, off] = rows(L, hkv, D)
        self.table, self.q = table.to(DEV), rows(T, hq, D) * 1.5
        self.k, self.v = rows(T, hkv, D), rows(T, hkv, D)
        self.d_lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.d_starts = torch.tensor(self.starts, dtype=torch.int32, device=DEV)
        self.errors = torch.zeros(1, dtype=torch.int64, device=DEV)
        self.v_live = self.vp.nan_to_num(0).abs().max().item()     # the largest value any row can average

    def args(self):
        return self.kp, self.vp, self.table, self.d_lens, self.d_starts


def check_attend(c, **kw):
    D = c.q.shape[-1]
    out, lse = paged.paged_attend(c.q, *c.args(), D ** -0.5, return_lse=True, errors=c.errors, **kw)
    kw.pop("max_query_len", None)
    want, wlse = ref_attend(c.q, c.kp, c.vp, c.table, c.lens, c.starts, D ** -0.5, **kw)
    T = c.starts[-1]
    assert int(c.errors) == 0
    close(out[:T], want[:T], c)
    fin = torch.isfinite(wlse[:T])
    assert torch.equal(torch.isfinite(lse[:T]), fin)
    assert (lse[:T].double() - wlse[:T])[fin].abs().max().item() <= 2e-5 * max(1.0, wlse[:T][fin].abs().max().item()) if fin.any() else True
    return out, lse


def close(got, want, c):
    got, dtype = got.double(), c.q.dtype
    assert torch.isfinite(got).all()
    live = c.v_live
    half = HALF[dtype]
    # the output's rounding, the weights' rounding (16-bit rows), fp32 sums
    tol = half * want.abs() + (half if dtype != FP else 0.0) * live + 2e-5 * live
    err = (got - want).abs()
    assert (err <= tol).all(), f"max error {err.max().item():.3g}, tolerance {tol.min().item():.3g}"


# ------------------------------------------------------------------ the turn
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("hq,hkv,D,rot,inter,norm,axes", [
    (8, 1, 256, 256, False, True, 1), (28, 4, 128, 128, False, False, 1), (32, 8, 128, 96, True, True, 3),
    (4, 4, 96, 96, False, True, 1), (32, 4, 64, 32, False, True, 1), (3, 1, 64, 20, False, True, 2), (5, 1, 40, 6, True, False, 1),
    (2, 2, 8, 8, False, True, 1), (1, 1, 256, 2, False, True, 1), (7, 7, 80, 40, False, True, 3),
])
def test_turn_matches_its_definition(dtype, hq, hkv, D, rot, inter, norm, axes):
    g = torch.Generator().manual_seed(D + rot)
    B, Q, P = 2, 5, 3000
    half = rot // 2
    q = (torch.randn(B, Q, hq, D, generator=g) * 2).to(dtype).to(DEV).transpose(1, 2)
    k = torch.randn(B, hkv, Q, D, generator=g).to(dtype).to(DEV)
    cos, sin = paged.rotary_table(1e4 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half), P)
    pos = torch.randint(0, P, (axes, B, Q) if axes > 1 else (B, Q), generator=g).to(DEV)
    pair = torch.randint(0, axes, (half,), generator=g).to(torch.int32).to(DEV) if axes > 1 else None
    qw = torch.randn(D, generator=g).to(dtype).to(DEV) if norm else None
    kw = torch.randn(D, generator=g).to(dtype).to(DEV) if norm else None
    eps = 1e-6 if norm else None
    qo, ko = paged.qk_norm_rope(q, k, cos, sin, positions=pos if axes == 1 else pos.int(), pair_axes=pair, interleaved=inter,
                                eps=eps, q_weight=qw, k_weight=kw, weight_offset=1.0)
    j = torch.arange(half, device=DEV)
    at = pos[..., None].expand(B, Q, half) if axes == 1 else pos[pair.long()].permute(1, 2, 0)
    c, s = cos.double()[at, j][:, None], sin.double()[at, j][:, None]
    for got, x, w in ((qo, q, qw), (ko, k, kw)):
        want = ref_turn(x.double(), w, eps, c, s, inter, 1.0)
        tol = HALF[dtype] * want.abs() + 1e-6 * want.abs().amax(-1, keepdim=True) + 1e-30
        assert ((got.double() - want).abs() <= tol).all()


def test_turn_in_place_without_keys_and_without_rotation():
    q = torch.randn(2, 4, 3, 64, device=DEV, dtype=BF)
    w = torch.randn(64, device=DEV)                    # float32 weights beside 16-bit rows
    want = ref_turn(q.double(), w, 1e-5, None, None, False)
    got, none = paged.qk_norm_rope(q, None, eps=1e-5, q_weight=w, out=(q, None))
    assert none is None and got is q
    assert ((q.double() - want).abs() <= HALF[BF] * want.abs() + 1e-6 * want.abs().amax(-1, keepdim=True)).all()


def test_turn_rows_of_gathered_tables_and_16_bit_tables():
    """The tables a model hands its layers: [B, Q, rot], a row per token, in the rows' type."""
    q, k = torch.randn(2, 4, 7, 64, device=DEV, dtype=BF), torch.randn(2, 2, 7, 64, device=DEV, dtype=BF)
    ang = torch.rand(2, 7, 32, device=DEV) * 6
    cos, sin = torch.cat([ang, ang], -1).cos().to(BF), torch.cat([ang, ang], -1).sin().to(BF)
    qo, ko = paged.qk_norm_rope(q, k, cos.view(14, 64)[:, :32], sin.view(14, 64)[:, :32])
    for got, x in ((qo, q), (ko, k)):
        want = ref_turn(x.double(), None, None, cos[..., :32].double()[:, None], sin[..., :32].double()[:, None], False)
        assert ((got.double() - want).abs() <= HALF[BF] * want.abs() + 1e-6 * want.abs().amax(-1, keepdim=True)).all()


def test_turn_far_positions_and_positions_outside_the_table():
    P = 1 << 20
    inv = 1e6 ** (-torch.arange(32, dtype=torch.float64, device=DEV) / 32)
    cos, sin = paged.rotary_table(inv, P)
    q = torch.randn(1, 2, 4, 64, device=DEV)
    pos = torch.tensor([[P - 1, P, -1, 12345]], device=DEV)
    err = torch.zeros(1, dtype=torch.int64, device=DEV)
    got, _ = paged.qk_norm_rope(q, None, cos, sin, positions=pos, errors=err)
    ang = pos.double()[..., None] * inv
    want = ref_turn(q.double(), None, None, ang.cos()[:, None], ang.sin()[:, None], False)
    for t in (0, 3):
        assert (got[:, :, t].double() - want[:, :, t]).abs().max() <= 2e-6
    assert got[:, :, 1:3].isnan().all() and int(err) == nat.ERRBIT_POSITION


def test_turn_of_nothing():
    q = torch.empty(2, 4, 0, 64, device=DEV, dtype=BF)
    qo, ko = paged.qk_norm_rope(q, q[:, :2], eps=1e-6)
    assert qo.shape == q.shape and ko.shape == (2, 2, 0, 64)


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("new,lens,hkv,D,S,rot,inter,engine", [
    ([1], [1], 1, 64, 16, 64, False, False), ([3, 0, 1, 70], [3, 9, 33, 200], 2, 128, 16, 64, True, True),
    ([129], [300], 1, 256, 128, 256, False, False), ([5, 5], [5, 12], 3, 96, 7, 96, False, True),
    ([1] * 300, list(range(1, 301)), 1, 64, 10, 64, False, False),
])
def test_append_writes_its_rows_and_no_others(dtype, new, lens, hkv, D, S, rot, inter, engine):
    c = Case(new, lens, hkv, hkv, D, S, dtype, engine_layout=engine, pad=2)
    cos, sin = paged.rotary_table(1e4 ** (-torch.arange(rot // 2, dtype=torch.float64, device=DEV) * 2 / rot), 400)
    w = torch.randn(D, device=DEV).to(dtype)
    k0, v0 = c.kp.clone(), c.vp.clone()
    paged.paged_append(c.k, c.v, *c.args(), cos=cos, sin=sin, interleaved=inter, eps=1e-6, k_weight=w, errors=c.errors)
    assert int(c.errors) == 0
    for b, (n, L) in enumerate(zip(new, lens)):
        for i in range(n):
            place, t = L - n + i, c.starts[b] + i
            pg, off = int(c.table[b, place // S]), place % S
            want = ref_turn(c.k[t].double(), w, 1e-6, cos[place].double(), sin[place].double(), inter)
            got = c.kp[pg, :, off].double()
            assert ((got - want).abs() <= HALF[dtype] * want.abs() + 1e-6 * want.abs().amax(-1, keepdim=True)).all()
            assert torch.equal(c.vp[pg, :, off], c.v[t])
            k0[pg, :, off], v0[pg, :, off] = c.kp[pg, :, off], c.vp[pg, :, off]
    assert torch.equal(k0.view(torch.uint8), c.kp.view(torch.uint8)) if k0.is_contiguous() else torch.equal(k0.nan_to_num(7), c.kp.nan_to_num(7))
    assert torch.equal(v0.nan_to_num(7), c.vp.nan_to_num(7))


def test_append_plain_copy_and_explicit_positions():
    c = Case([4, 2], [9, 2], 2, 2, 64, 4, BF)
    paged.paged_append(c.k, c.v, *c.args())
    assert torch.equal(c.kp[c.table[0, 8 // 4].long(), :, 0], c.k[3])
    cos, sin = paged.rotary_table(1e4 ** (-torch.arange(32, dtype=torch.float64, device=DEV) / 32), 50)
    pos = torch.tensor([40, 3, 2, 1, 0, 49], device=DEV)
    paged.paged_append(c.k, c.v, *c.args(), cos=cos, sin=sin, positions=pos)
    want = ref_turn(c.k[5].double(), None, None, cos[49].double(), sin[49].double(), False)
    got = c.kp[c.table[1, 0].long(), :, 1].double()
    assert ((got - want).abs() <= HALF[BF] * want.abs() + 1e-6 * want.abs().amax(-1, keepdim=True)).all()


def test_append_skips_tokens_without_a_place():
    c = Case([2, 2, 2], [2, 2, 2], 1, 1, 64, 4, FP)
    k0 = c.kp.clone()
    c.table[0, 0] = 1000                      # past the pages
    c.table[1, 0] = -5
    c.d_lens[2] = 1                           # shorter than its new tokens: the first has place -1
    paged.paged_append(c.k, c.v, *c.args(), errors=c.errors)
    assert int(c.errors) == nat.ERRBIT_BLOCK_TABLE | nat.ERRBIT_SEQ_LEN
    pg = int(c.table[2, 0])
    assert torch.equal(c.kp[pg, :, 0], c.k[5])
    k0[pg, :, 0] = c.kp[pg, :, 0]
    assert torch.equal(k0.nan_to_num(7), c.kp.nan_to_num(7))


# ------------------------------------------------------------------ attention
SHAPES = [
    # new, lens, hq, hkv, D, S
    ([1], [1], 8, 1, 256, 128),
    ([1], [2048], 8, 1, 256, 128),
    ([1, 1, 1], [1, 65, 1000], 32, 8, 128, 16),
    ([1] * 33, [17 * i + 1 for i in range(33)], 32, 4, 64, 32),
    ([5, 1, 3], [70, 1, 900], 28, 4, 128, 64),
    ([200], [200], 4, 4, 96, 48),
    ([129, 0, 1, 64], [500, 10, 1, 64], 8, 2, 128, 128),
    ([300], [1300], 8, 1, 256, 128),
    ([257, 3], [257, 700], 28, 4, 128, 16),
    ([2, 40], [9, 41], 6, 2, 64, 7),
    ([100], [333], 32, 8, 128, 24),
    ([17], [40], 3, 3, 40, 5),
    ([3, 90], [200, 90], 40, 1, 128, 16),
    ([1, 2], [300, 310], 96, 1, 64, 32),
]


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("shape", SHAPES, ids=[str(i) for i in range(len(SHAPES))])
def test_attend_matches_its_definition(dtype, shape):
    check_attend(Case(*shape, dtype, seed=len(shape[0])))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("kw", [dict(causal=False), dict(window=1), dict(window=77), dict(window=5000), dict(softcap=3.0),
                                dict(window=40, softcap=2.0), dict(max_query_len=1), dict(max_query_len=4000)],
                         ids=lambda d: "-".join(d))
@pytest.mark.parametrize("shape", [SHAPES[2], SHAPES[4], SHAPES[6], SHAPES[7], SHAPES[9], SHAPES[10]], ids=["a", "b", "c", "d", "e", "f"])
def test_attend_masks_and_caps(dtype, kw, shape):
    check_attend(Case(*shape, dtype, seed=3), **kw)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FP, 64), (BF, 256)])
def test_attend_engine_layout_strided_queries_and_padding(dtype, D):
    c = Case([3, 150, 1], [400, 150, 77], 8, 2, D, 16, dtype, engine_layout=True, pad=5)
    packed = torch.zeros(c.q.shape[0], 3 * 8, D, dtype=dtype, device=DEV)
    packed[:, 8:16] = c.q
    c.q = packed[:, 8:16]
    out = torch.full_like(c.q.contiguous(), 7.0)
    got = paged.paged_attend(c.q, *c.args(), D ** -0.5, out=out, errors=c.errors)
    want, _ = ref_attend(c.q, c.kp, c.vp, c.table, c.lens, c.starts, D ** -0.5)
    assert got is out and int(c.errors) == 0
    close(out[:154], want[:154], c)
    assert (out[154:] == 7.0).all()                        # rows behind the last sequence


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FP, 64)])
@pytest.mark.parametrize("n", [1, 150])
def test_attend_rows_that_see_nothing_and_bad_pages(dtype, D, n):
    c = Case([n, n, n], [n + 60, n + 60, n + 60], 4, 2, D, 16, dtype)
    c.d_lens[0] = 0                                        # an empty sequence with new tokens
    c.lens[0] = 0
    c.table[1, 1] = 10 ** 6                                # reads as zeros
    c.table[2, 0] = -1
    out, lse = paged.paged_attend(c.q, *c.args(), D ** -0.5, return_lse=True, errors=c.errors)
    want, wlse = ref_attend(c.q, c.kp, c.vp, c.table, c.lens, c.starts, D ** -0.5)
    assert int(c.errors) == nat.ERRBIT_BLOCK_TABLE | nat.ERRBIT_SEQ_LEN
    assert (out[:n] == 0).all() and (lse[:n] == -math.inf).all()
    close(out, want, c)
    assert (lse[n:].double() - wlse[n:]).abs().max() <= 2e-5 * max(1.0, wlse[n:].abs().max().item())


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FP, 64)])
def test_attend_window_over_pages_given_back(dtype, D):
    """Pages wholly before every row's window may be anybody's: table entries out of range, NaN rows."""
    c = Case([3, 140], [700, 900], 4, 2, D, 16, dtype)
    want, _ = ref_attend(c.q, c.kp, c.vp, c.table, c.lens, c.starts, D ** -0.5, window=100)
    for b, (n, L) in enumerate(zip(c.new, c.lens)):
        gone = (L - n - 99) // 16
        pages = c.table[b, :gone].long()
        c.kp[pages], c.vp[pages] = math.nan, math.nan
        c.table[b, :gone // 2] = -1
    out = paged.paged_attend(c.q, *c.args(), D ** -0.5, window=100, errors=c.errors)
    assert int(c.errors) == 0
    close(out, want, c)


@pytest.mark.parametrize("dtype,D,n", [(BF, 128, 1), (BF, 128, 200), (FP, 64, 3), (BF, 256, 200)])
def test_attend_repeats_bit_for_bit_and_in_graphs(dtype, D, n):
    """Two graphs and an eager call in flight together; lengths changed between replays."""
    c = Case([n, n], [n + 2000, n + 900], 8, 2, D, 32, dtype)
    first = paged.paged_attend(c.q, *c.args(), D ** -0.5)
    outs = [torch.zeros_like(c.q) for _ in range(2)]
    graphs = []
    torch.cuda.synchronize()
    for o in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            paged.paged_attend(c.q, *c.args(), D ** -0.5, out=o)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        again = paged.paged_attend(c.q, *c.args(), D ** -0.5)
    torch.cuda.synchronize()
    assert torch.equal(first, again) and torch.equal(first, outs[0]) and torch.equal(first, outs[1])
    c.d_lens.copy_(torch.tensor([n + 5, n + 333], dtype=torch.int32))
    c.lens = [n + 5, n + 333]
    graphs[0].replay()
    want, _ = ref_attend(c.q, c.kp, c.vp, c.table, c.lens, c.starts, D ** -0.5)
    torch.cuda.synchronize()
    close(outs[0], want, c)


def test_attend_on_another_stream():
    c = Case([1, 1], [500, 900], 8, 2, 128, 32, BF)
    want = paged.paged_attend(c.q, *c.args(), 0.1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = paged.paged_attend(c.q, *c.args(), 0.1)
    s.synchronize()
    assert torch.equal(got, want)


def test_attend_pages_past_two_gigabytes():
    """Element offsets of the pages pass 2^31 (and 2^32 bytes)."""
    S, D, hkv = 128, 128, 8
    N = (1 << 32) // (S * D * hkv * 2) + 40
    kp = torch.empty(N, hkv, S, D, dtype=BF, device=DEV)
    vp = torch.empty(N, hkv, S, D, dtype=BF, device=DEV)
    table = torch.arange(N - 3, N, dtype=torch.int32, device=DEV).view(1, 3)
    k, v = torch.randn(300, hkv, D, device=DEV).to(BF), torch.randn(300, hkv, D, device=DEV).to(BF)
    for n in (1, 150):
        lens, starts = torch.tensor([300], dtype=torch.int32, device=DEV), torch.tensor([0, 300], dtype=torch.int32, device=DEV)
        paged.paged_append(k, v, kp, vp, table, lens, starts)
        q = torch.randn(n, 32, D, device=DEV).to(BF)
        qs = torch.tensor([0, n], dtype=torch.int32, device=DEV)
        out = paged.paged_attend(q, kp, vp, table, lens, qs, D ** -0.5)
        want, _ = ref_attend(q, kp, vp, table, [300], [0, n], D ** -0.5)
        tol = HALF[BF] * want.abs() + (HALF[BF] + 2e-5) * v.abs().max().item()
        assert ((out.double() - want).abs() <= tol).all()


def test_nothing_to_do():
    c = Case([0, 0], [5, 6], 4, 2, 64, 16, BF)
    out = paged.paged_attend(c.q, *c.args(), 0.1)
    assert out.shape == (0, 4, 64)
    paged.paged_append(c.k, c.v, *c.args())


def test_turn_by_sections_of_axes_and_mixed_pairs():
    """Lanes whose pairs share an axis, lanes whose pairs do not, five axes, and an axis out of range."""
    g = torch.Generator().manual_seed(5)
    q = torch.randn(1, 3, 9, 128, generator=g).to(BF).to(DEV)
    cos, sin = paged.rotary_table(1e4 ** (-torch.arange(64, dtype=torch.float64, device=DEV) / 64), 500)
    pos = torch.randint(0, 500, (5, 1, 9), generator=g).to(DEV)
    for pair in ([j // 13 for j in range(64)], [j // 16 for j in range(64)], [4 - j % 5 for j in range(64)], [4] * 64):
        for inter in (False, True):
            axes = torch.tensor(pair, dtype=torch.int32, device=DEV)
            got, _ = paged.qk_norm_rope(q, None, cos, sin, positions=pos, pair_axes=axes, interleaved=inter)
            at = pos[axes.long()].permute(1, 2, 0)
            j = torch.arange(64, device=DEV)
            want = ref_turn(q.double(), None, None, cos.double()[at, j][:, None], sin.double()[at, j][:, None], inter)
            assert ((got.double() - want).abs() <= HALF[BF] * want.abs() + 1e-6 * want.abs().amax(-1, keepdim=True)).all()
    axes = torch.zeros(64, dtype=torch.int32, device=DEV)
    axes[7] = 5
    err = torch.zeros(1, dtype=torch.int64, device=DEV)
    got, _ = paged.qk_norm_rope(q, None, cos, sin, positions=pos, pair_axes=axes, errors=err)
    assert got.isnan().all() and int(err) == nat.ERRBIT_POSITION


def test_attend_windows_and_chunks_of_many_lengths_in_one_batch():
    """Many items per block, most with dead rows at both ends of their keys, some of one row tile and some of two."""
    new = [1021, 1, 300, 130, 64, 65, 700, 256, 33]
    lens = [7000, 5, 300, 2000, 6001, 1999, 3333, 256, 4000]
    for window, softcap in ((1500, 30.0), (200, 0.0), (0, 0.0)):
        check_attend(Case(new, lens, 16, 16, 96, 48, HF, seed=1), window=window, softcap=softcap)
        check_attend(Case(new[1:6], lens[1:6], 8, 1, 256, 24, BF, seed=2), window=window, softcap=softcap)


def test_rows_of_any_strides():
    """Misaligned and transposed rows are read through a copy; expanded ones as they are."""
    base = torch.randn(2, 3, 5, 129, device=DEV, dtype=BF)
    for q in (base[..., 1:], torch.randn(2, 3, 128, 5, device=DEV, dtype=BF).transpose(2, 3),
              torch.randn(2, 1, 5, 128, device=DEV, dtype=BF).expand(2, 3, 5, 128)):
        got, k = paged.qk_norm_rope(q, q, eps=1e-6)
        want = ref_turn(q.double(), None, 1e-6, None, None, False)
        for x in (got, k):
            assert ((x.double() - want).abs() <= HALF[BF] * want.abs() + 1e-6 * want.abs().amax(-1, keepdim=True)).all()
    c = Case([3, 40], [30, 90], 8, 2, 128, 16, BF)
    want = paged.paged_attend(c.q, *c.args(), 0.1)
    odd = torch.empty(43, 8, 129, device=DEV, dtype=BF)[..., 1:].copy_(c.q)
    assert torch.equal(paged.paged_attend(odd, *c.args(), 0.1), want)
    assert torch.equal(paged.paged_attend(c.q.transpose(1, 2).contiguous().transpose(1, 2), *c.args(), 0.1), want)
    k1, v1 = (torch.randn(43, 2, 129, device=DEV, dtype=BF)[..., 1:] for _ in range(2))
    paged.paged_append(k1, v1, *c.args())
    assert torch.equal(c.kp[c.table[0, 29 // 16].long(), :, 29 % 16], k1[2])


def test_refusals_of_tensors():
    c = Case([3, 40], [30, 90], 8, 2, 128, 16, BF)
    bad = [
        lambda: paged.paged_attend(c.q, c.kp, c.vp, c.table.long(), c.d_lens, c.d_starts, 0.1),
        lambda: paged.paged_attend(c.q, c.kp, c.vp, c.table, c.d_lens[:1], c.d_starts, 0.1),
        lambda: paged.paged_attend(c.q, c.kp.float(), c.vp, c.table, c.d_lens, c.d_starts, 0.1),
        lambda: paged.paged_attend(c.q, c.kp, c.vp, c.table.cpu(), c.d_lens, c.d_starts, 0.1),
        lambda: paged.paged_attend(c.q[:, :7], *c.args(), 0.1),
        lambda: paged.paged_attend(c.q, *c.args(), 0.1, window=-3),
        lambda: paged.paged_attend(c.q, *c.args(), 0.1, window=3, causal=False),
        lambda: paged.paged_attend(c.q, *c.args(), 0.1, out=c.q.float()),
        lambda: paged.paged_attend(c.q[..., :64], *c.args(), 0.1),
        lambda: paged.paged_append(c.k, c.v[:-1], *c.args()),
        lambda: paged.paged_append(c.k, c.v, *c.args(), cos=torch.zeros(9, 64, device=DEV)),
        lambda: paged.qk_norm_rope(c.q[None], None, torch.zeros(9, 65, device=DEV), torch.zeros(9, 65, device=DEV),
                                   positions=torch.zeros(1, 8, device=DEV, dtype=torch.int64)),
        lambda: paged.qk_norm_rope(c.q[None], None, torch.zeros(9, 64, device=DEV), torch.zeros(9, 64, device=DEV)),
        lambda: paged.qk_norm_rope(c.q[None], None, q_weight=torch.zeros(128, device=DEV)),
        lambda: paged.qk_norm_rope(c.q[None].double(), None, eps=1e-6),
    ]
    for f in bad:
        with pytest.raises(nat.KIVNativeError):
            f()


@pytest.mark.parametrize("D", [64, 256])
def test_fp32_sums_over_many_keys_do_not_drift(D):
    """Values around 1 over 20000 keys.  Sums that cut instead of rounding lose 2^-24 of themselves at each of thousands
    of steps (1e-4).  Rounded ones walk: about 600 additions of at most 2^-24, four standard deviations 6e-6; with the
    weights' own errors (scores of D products, exponential: below 3e-6, of both signs) 1e-5 covers them."""
    c = Case([1, 3], [20000, 19000], 8, 1, D, 32, FP)
    c.vp += 1
    out = paged.paged_attend(c.q, *c.args(), D ** -0.5)
    want, _ = ref_attend(c.q, c.kp, c.vp, c.table, c.lens, c.starts, D ** -0.5)
    assert ((out.double() - want).abs() <= 1e-5 * want.abs().clamp(min=0.5)).all()


@pytest.mark.parametrize("dtype,D,S,hq,hkv", [(HF, 128, 128, 8, 1), (HF, 64, 16, 8, 2), (HF, 256, 64, 8, 1), (BF, 96, 128, 4, 4), (HF, 128, 10, 8, 1)])
def test_outputs_over_many_keys_do_not_drift(dtype, D, S, hq, hkv):
    """Values around 1 over 60000 keys, cut between the blocks.  The tensor cores cut their sums by about 2^-23 with
    every 16 keys (4e-4 in one sum of all, most of an fp16 half step); over at most 128 key tiles that is 1e-4.  The rounded weights add a walk, not a drift: of 60000
    weights with errors of half a step of either sign, below 1e-4; the output's rounding is half a step.  In the mean of n outputs the drift stays, while n roundings, each
    at most half a step h and even over it, leave a deviation of h / sqrt(3 n) (1.15e-4 for the 384 bf16 outputs of a
    row here, 1e-5 for fp16): five of those are added."""
    L = 60000
    c = Case([700, 1, 5], [L, L - 3, L - 700], hq, hkv, D, S, dtype)
    c.vp.mul_(0.25).add_(1)
    out = paged.paged_attend(c.q, *c.args(), D ** -0.5, errors=c.errors)
    rows = [0, 350, 699, 700, 701, 705]
    at = [b for b, n in enumerate(c.new) for _ in range(n)]
    for t in rows:
        b = at[t]
        n = c.lens[b] - c.starts[b + 1] + t + 1
        j = torch.arange(n, device=DEV)
        pg = c.table[b].long()[j // S]
        k, v = (x[pg, :, j % S].double().repeat_interleave(hq // hkv, 1) for x in (c.kp, c.vp))
        w = torch.softmax(torch.einsum("hd,lhd->hl", c.q[t].double(), k) * D ** -0.5, -1)
        want = torch.einsum("hl,lhd->hd", w, v)
        assert ((out[t].double() / want - 1).abs() <= HALF[dtype] + 2e-4).all(), t
        assert (out[t].double() / want - 1).mean().abs() <= 1.5e-4 + 5 * HALF[dtype] / (3 * want.numel()) ** 0.5, t
    assert int(c.errors) == 0


@pytest.mark.parametrize("dtype,D,S,hq,hkv,new", [(HF, 128, 128, 8, 1, [5000, 1, 1000]), (HF, 256, 64, 8, 1, [2900, 100]), (BF, 96, 128, 1, 1, [40000]),
                                                  (HF, 64, 16, 7, 1, [1, 5, 18] * 60), (HF, 128, 128, 4, 1, [1] * 200), (HF, 256, 64, 4, 2, [3] * 90)])
def test_long_stretches_of_one_block_do_not_drift(dtype, D, S, hq, hkv, new):
    """As above, with work for stretches of more than 128 key tiles in every block (256 where two groups of warps share
    a sequence's tiles), whole items among them, and batches of few rows.  The sequences share their pages."""
    L = 60000
    g = torch.Generator(device=DEV).manual_seed(3)

    def rows(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    N = -(-L // S)
    kp, vp, q = rows(N, hkv, S, D).to(dtype), (rows(N, hkv, S, D) / 4 + 1).to(dtype), rows(sum(new), hq, D).to(dtype)
    lens = [L - 37 * (b % 5) for b in range(len(new))]
    starts = [sum(new[:b]) for b in range(len(new) + 1)]
    table = torch.arange(N, dtype=torch.int32, device=DEV).repeat(len(new), 1)
    errors = torch.zeros(1, dtype=torch.int64, device=DEV)
    ints = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (lens, starts)]
    out, lse = paged.paged_attend(q, kp, vp, table, *ints, D ** -0.5, return_lse=True, errors=errors)
    k, v = (x.transpose(1, 2).reshape(-1, hkv, D)[:L].double().repeat_interleave(hq // hkv, 1) for x in (kp, vp))
    for b in sorted({0, 1, 2, len(new) // 2, len(new) - 1} & set(range(len(new)))):
        for i in sorted({0, new[b] // 2, new[b] - 1}):
            t, n = starts[b] + i, lens[b] - new[b] + i + 1
            x = torch.einsum("hd,lhd->hl", q[t].double(), k[:n]) * D ** -0.5
            want = torch.einsum("hl,lhd->hd", torch.softmax(x, -1), v[:n])
            off = out[t].double() / want - 1
            assert (off.abs() <= HALF[dtype] + 2e-4).all(), (t, off.abs().max())
            assert off.mean().abs() <= 1.5e-4 + 5 * HALF[dtype] / (3 * want.numel()) ** 0.5, (t, off.mean())
            assert (lse[t].double() - x.logsumexp(-1)).abs().max() <= 2e-5 * 12      # of values around 11.5
    assert int(errors) == 0
