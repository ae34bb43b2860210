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


def _llama():
    from transformers import LlamaConfig, LlamaForCausalLM
    return LlamaForCausalLM(LlamaConfig(vocab_size=64, hidden_size=64, intermediate_size=64, num_hidden_layers=1,
                                        num_attention_heads=2, num_key_value_heads=1, head_dim=32,
                                        attn_implementation="eager")).eval()


@pytest.mark.parametrize("first", [0, 1])
def test_fused_rotation_stays_until_the_last_model_leaves(first):
    """Two models of one family ask for the kernel: the one that leaves first does not take it from the other."""
    import sys
    from kiv_b200 import KIVConfig, KIVMiddleware

    users = [KIVMiddleware(_llama(), KIVConfig()) for _ in range(2)]
    module = sys.modules[type(users[0].model.model.layers[0].self_attn).__module__]
    before = module.apply_rotary_pos_emb
    for _ in range(2):                                      # and again after both have left
        for mw in users:
            mw.install(fused_rotary=True)
        fused = module.apply_rotary_pos_emb
        assert fused._kiv_original is before                # not stacked
        users[first].uninstall()
        assert module.apply_rotary_pos_emb is fused
        users[1 - first].uninstall()
        assert module.apply_rotary_pos_emb is before


def test_a_model_without_the_fused_rotation_does_not_hold_it():
    import sys
    from kiv_b200 import KIVConfig, KIVMiddleware

    asks, does_not = (KIVMiddleware(_llama(), KIVConfig()) for _ in range(2))
    module = sys.modules[type(asks.model.model.layers[0].self_attn).__module__]
    before = module.apply_rotary_pos_emb
    asks.install(fused_rotary=True)
    does_not.install()
    asks.uninstall()
    assert module.apply_rotary_pos_emb is before
    does_not.uninstall()
    assert module.apply_rotary_pos_emb is before


@torch.no_grad()
def test_fused_rotation_leaves_what_the_kernel_would_answer_otherwise():
    """Mixed dtypes (the model's products are then in the wider one), and shapes and layouts that only broadcasting takes."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from kiv_b200 import ops
    from kiv_b200.middleware import fused_rotary

    ops.load()
    calls = []

    def plain(q, k, cos, sin):
        calls.append(1)
        c, s = cos[:, None], sin[:, None]
        half = q.shape[-1] // 2
        return tuple(x * c + torch.cat([-x[..., half:], x[..., :half]], -1) * s for x in (q, k))

    turn = fused_rotary(plain)
    with FakeTensorMode():
        def t(*shape, dtype=torch.bfloat16):
            return torch.empty(shape, dtype=dtype, device="cuda")

        q, k, cs = t(2, 4, 3, 64), t(2, 2, 3, 64), t(2, 3, 64)
        f32 = t(2, 3, 64, dtype=torch.float32)
        for args, taken in [((q, k, cs, cs), True), ((q, k, cs[:1], cs[:1]), True), ((q, k, f32, f32), False),
                            ((q, k, cs, f32), False), ((q, t(2, 2, 1, 64), cs, cs), False), ((q, t(1, 2, 3, 64), cs, cs), False),
                            ((q, k, cs, t(3, 2, 64).transpose(0, 1)), False), ((q, k, *[t(2, 64, 3).mT] * 2), False)]:
            calls.clear()
            got, want = turn(*args), plain(*args)
            assert len(calls) == (1 if taken else 2)
            assert [(x.dtype, x.shape) for x in got] == [(x.dtype, x.shape) for x in want]
