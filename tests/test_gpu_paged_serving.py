"""The rotation and paged operators together, as a serving step uses them, and the fused rotation in the HF path."""

import pytest
import torch
from transformers import LlamaConfig, LlamaForCausalLM

from kiv_b200 import KIVConfig, KIVMiddleware, PagedKVCache
from kiv_b200 import _native as nat
from kiv_b200 import paged
from tests.gpu_helpers import DEV
from tests.test_gpu_paged import HALF, ref_turn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,hq,hkv,D,S", [(torch.bfloat16, 8, 2, 128, 16), (torch.float16, 8, 1, 256, 128),
                                             (torch.float32, 4, 4, 64, 10), (torch.bfloat16, 6, 2, 80, 24)])
def test_serving_steps_match_a_dense_computation(dtype, hq, hkv, D, S):
    """Prompts, decode, drafts, a sequence that leaves and one that takes its pages; two layers, queries and keys normed
    and turned.  The dense side keeps its own keys from the same projections and attends in 64 bits."""
    g = torch.Generator().manual_seed(D)
    L = 2
    cache = PagedKVCache(200, S, hkv, D, layers=L, dtype=dtype, device=DEV, max_batch=6)
    cos, sin = paged.rotary_table(1e4 ** (-torch.arange(D // 2, dtype=torch.float64, device=DEV) * 2 / D), 1024)
    qw, kw = torch.randn(D, generator=g).to(dtype).to(DEV), torch.randn(D, generator=g).to(dtype).to(DEV)
    dense = {}
    steps = [[("a", 200), ("b", 3)], [("a", 1), ("b", 1)], [("b", 5), ("c", 140), ("a", 1)], [("c", 1), ("b", 0), ("a", 17)],
             "free a", [("d", 333), ("c", 1), ("b", 2)], [("b", 1), ("c", 1), ("d", 1)]]
    for new in steps:
        if new == "free a":
            cache.free("a")
            dense.pop("a")
            continue
        T = cache.step(new)
        pos = torch.cat([torch.arange(cache.length(s) - n, cache.length(s)) for s, n in new]).to(DEV)
        for layer in range(L):
            q, k, v = (torch.randn(T, h, D, generator=g).to(dtype).to(DEV) for h in (hq, hkv, hkv))
            qt, _ = paged.qk_norm_rope(q.transpose(0, 1)[None], None, cos, sin, positions=pos[None], eps=1e-6, q_weight=qw)
            cache.append(layer, k, v, cos=cos, sin=sin, eps=1e-6, k_weight=kw)
            out = cache.attend(layer, qt[0].transpose(0, 1), D ** -0.5)
            kt = ref_turn(k.double(), kw, 1e-6, cos.double()[pos][:, None], sin.double()[pos][:, None], False).to(dtype)
            assert ((qt[0].transpose(0, 1).double() - ref_turn(q.double(), qw, 1e-6, cos.double()[pos][:, None],
                                                               sin.double()[pos][:, None], False)).abs()
                    <= HALF[dtype] * 20 + 1e-5).all()
            at = 0
            for s, n in new:
                held = dense.setdefault(s, [None] * L)
                kv = (kt[at:at + n], v[at:at + n])
                held[layer] = kv if held[layer] is None else tuple(torch.cat(p) for p in zip(held[layer], kv))
                kk, vv = (x.double().repeat_interleave(hq // hkv, 1) for x in held[layer])
                x = torch.einsum("nhd,lhd->hnl", qt[0].transpose(0, 1)[at:at + n].double(), kk) * D ** -0.5
                seen = torch.arange(kk.shape[0], device=DEV) <= (kk.shape[0] - n + torch.arange(n, device=DEV))[:, None]
                want = torch.einsum("hnl,lhd->nhd", x.masked_fill(~seen, -torch.inf).softmax(-1), vv)
                # two roundings of at most half a step each (weights of 16-bit rows, output), and a key whose fp32 turn
                # rounds to the other neighbour than the 64-bit one's: a step of one of up to 333 keys
                tol = 4 * HALF[dtype] * 5 + 4e-5
                assert ((out[at:at + n].double() - want).abs() <= tol).all()
                at += n
    assert int(cache.errors) == 0 and cache.free_pages == 200 - sum(-(-cache.length(s) // S) for s in "bcd")


def test_steps_in_a_graph():
    """append and attend captured once serve later steps: lengths and pages move underneath."""
    cache = PagedKVCache(64, 16, 2, 128, dtype=torch.bfloat16, device=DEV, max_batch=3)
    twin = PagedKVCache(64, 16, 2, 128, dtype=torch.bfloat16, device=DEV, max_batch=3)
    seqs = ["x", "y", "z"]
    prompt = [torch.randn(60, 2, 128, device=DEV).to(torch.bfloat16) for _ in range(2)]
    for c in (cache, twin):
        c.step([("x", 15), ("y", 32), ("z", 13)])
        c.append(0, *prompt)
    q, k, v = (torch.zeros(3, h, 128, device=DEV, dtype=torch.bfloat16) for h in (8, 2, 2))
    out = torch.zeros_like(q)

    def layer(c, o):
        c.append(0, k, v)
        c.attend(0, q, 0.1, out=o)

    cache.step([(s, 0) for s in seqs])                      # same batch; nothing appended while capturing
    cache._tokens = 3
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(cache, out)
    for i in range(20):
        for t in (q, k, v):
            t.normal_()
        cache.step([(s, 1) for s in seqs])
        graph.replay()
        twin.step([(s, 1) for s in seqs])
        want = torch.zeros_like(q)
        layer(twin, want)
        assert torch.equal(out, want), i
    assert int(cache.errors) == 0 and cache.length("x") == 35


def test_running_out_of_pages_changes_nothing():
    cache = PagedKVCache(4, 8, 1, 64, device=DEV, max_batch=2, max_pages_per_seq=3)
    cache.step([("a", 10)])
    with pytest.raises(nat.KIVNativeError, match="out of pages"):
        cache.step([("a", 7), ("b", 16)])
    with pytest.raises(nat.KIVNativeError, match="at most 3"):
        cache.step([("a", 20)])
    with pytest.raises(ValueError):
        cache.step([("a", 1), ("a", 1)])
    assert cache.length("a") == 10 and cache.length("b") == 0 and cache.free_pages == 2
    with pytest.raises(nat.KIVNativeError, match="rows"):
        cache.append(0, torch.zeros(9, 1, 64, device=DEV, dtype=torch.bfloat16), torch.zeros(9, 1, 64, device=DEV, dtype=torch.bfloat16))


def _model(dtype):
    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=64, max_position_embeddings=4096, attn_implementation="eager")
    return LlamaForCausalLM(cfg).to(DEV, dtype).eval()


@torch.no_grad()
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_fused_rotation_in_a_model(dtype):
    """The same tokens through the model with and without the fused rotation, prompt and decode."""
    model = _model(dtype)
    ids = torch.randint(0, 512, (1, 700), generator=torch.Generator().manual_seed(1)).to(DEV)
    logits, calls = [], []
    import kiv_b200.paged as mod
    real = mod.qk_norm_rope
    for fused in (False, True):
        mw = KIVMiddleware(model, KIVConfig(hot_budget=128, page_size=128, top_pages=64, top_p=4096, telemetry=False))
        mod.qk_norm_rope = lambda *a, **k: (calls.append(fused), real(*a, **k))[1]
        try:
            mw.install(fused_rotary=fused)
        finally:
            mod.qk_norm_rope = real
        cache = mw.create_cache()
        got = [mw.chunked_prefill(ids[:, :697], cache, chunk_size=256)]
        for t in range(697, 700):
            got.append(model(input_ids=ids[:, t:t + 1], past_key_values=cache, use_cache=True).logits[:, -1])
        logits.append(torch.cat(got).double())
        mw.uninstall()
    assert calls == [True] * (2 * 6)                        # two layers, three prompt chunks and three tokens
    # fp32: the rotation's rounding order is all that differs; bf16: a few roundings of the keys and queries
    tol = 1e-4 if dtype == torch.float32 else 0.05
    assert (logits[0] - logits[1]).abs().max() <= tol * logits[0].abs().max()
