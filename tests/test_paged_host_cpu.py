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


def _random_steps(rng, book, names, pages):
    """A step's list: some of the sequences in any order, with tokens that fit."""
    some = rng.sample(names, rng.randint(1, min(len(names), book.max_batch)))
    free, out = len(book.unused), []
    for s in some:
        n = rng.choice([0, 1, 1, 5, 3 * book.page_size])
        have = book.lengths.get(s, 0)
        need = -(-(have + n) // book.page_size) - len(book.held.get(s, ()))
        if need <= free and -(-(have + n) // book.page_size) <= pages:
            free -= need
            out.append((s, n))
    return out


def test_the_changed_cells_make_the_block_table():
    """Steps of random sequences in random order, some given back, some under an old name: the cells applied one step after
    the other give each row its sequence's pages and -1 behind them, and no page has two owners."""
    import random

    rng = random.Random(5)
    book = paged._PageBook(40, 4, 5, 12)
    table = [-1] * (5 * 12)
    names = list("abcdefg")
    for _ in range(400):
        new = _random_steps(rng, book, names, 12)
        starts, lens, runs, pages = book.step(new)
        cells = [at for first, count in runs for at in range(first, first + count)]
        assert len(set(cells)) == len(cells) == len(pages)
        for at, page in zip(cells, pages):
            table[at] = page
        for i, (s, n) in enumerate(new):
            held = list(book.held[s])
            assert len(held) == -(-lens[i] // 4) and starts[i + 1] - starts[i] == n and lens[i] == book.lengths[s]
            assert table[i * 12:i * 12 + 12] == held + [-1] * (12 - len(held))
        owned = [p for held in book.held.values() for p in held]
        assert sorted(owned + book.unused) == list(range(40))
        if rng.random() < 0.3:
            book.free(rng.choice(names))


def test_a_decode_step_costs_the_new_pages_not_the_held_ones():
    """64 sequences of 2048 pages: a token each changes a cell where a page begins, none elsewhere, and takes no longer
    than with one page per sequence (a step that walked every page held would take hundreds of times as long)."""
    import time

    def decode(held):
        book = paged._PageBook(64 * (held + 8), 16, 64, 64 * (held + 8))
        step = [(s, 1) for s in range(64)]
        book.step([(s, 16 * (held - 1) + s % 16) for s in range(64)])
        took = []
        for _ in range(64):
            t = time.perf_counter()
            _, lens, _, pages = book.step(step)
            took.append(time.perf_counter() - t)
            assert len(pages) == sum((n - 1) % 16 == 0 for n in lens)
        return min(took)

    decode(1)
    assert decode(2048) < 10 * decode(1)


def test_a_step_that_does_not_fit_changes_nothing_of_the_book():
    book = paged._PageBook(4, 8, 2, 3)
    book.step([("a", 10)])
    for new, error in [([("a", 7), ("b", 16)], nat.KIVNativeError), ([("a", 20)], nat.KIVNativeError),
                       ([("a", 1), ("a", 1)], ValueError), ([("b", -1)], ValueError), ([(s, 0) for s in "abc"], ValueError)]:
        with pytest.raises(error):
            book.step(new)
        assert book.lengths == {"a": 10} and list(book.held) == ["a"] and len(book.unused) == 2
