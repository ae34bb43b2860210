"""Paged-cache operators without a GPU: registration, struct layouts, refusals before any launch, tracing."""

import ctypes
import os
import subprocess

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from kiv_b200 import _native as nat
from kiv_b200 import ops, paged

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "kiv_b200.h")
ARG, CAPACITY, UNSUPPORTED = 1, 2, 4


def test_operators_are_registered_and_declare_what_they_write():
    K = ops.kiv()
    schemas = {n: str(getattr(K, n).default._schema) for n in ops.PAGED_OP_NAMES}
    assert "Tensor(a!) q_out" in schemas["qk_norm_rope"] and "Tensor(b!)? k_out" in schemas["qk_norm_rope"]
    assert "Tensor(a!) k_pages" in schemas["paged_append"] and "Tensor(b!) v_pages" in schemas["paged_append"]
    assert "Tensor(a!) out" in schemas["paged_attend"] and "Tensor(b!)? lse" in schemas["paged_attend"]


def test_struct_layouts_match_the_header(tmp_path):
    structs = {"kiv_paged": nat.PagedDesc, "kiv_turn": nat.TurnDesc, "kiv_rows": nat.RowsDesc,
               "kiv_paged_query": nat.PagedQueryDesc}
    lines = [f'printf("{s} %zu\\n", sizeof({s}));' for s in structs]
    lines += [f'printf("{s}.{f} %zu\\n", offsetof({s}, {f}));' for s, c in structs.items() for f, _ in c._fields_]
    src = tmp_path / "l.c"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "{HEADER}"\nint main(void) {{ {" ".join(lines)} return 0; }}')
    subprocess.run(["gcc", "-std=c11", str(src), "-o", str(tmp_path / "l")], check=True)
    for line in subprocess.check_output([str(tmp_path / "l")], text=True).splitlines():
        key, val = line.split()
        s, _, f = key.partition(".")
        assert int(val) == (getattr(structs[s], f).offset if f else ctypes.sizeof(structs[s])), key


def _paged(**kw):
    D, S, H = 128, 16, 2
    d = dict(batch=2, num_kv_heads=H, head_dim=D, page_size=S, dtype=1, max_query_len=0, num_pages=8, k=4096, v=8192,
             k_stride_p=H * S * D, k_stride_h=S * D, k_stride_t=D, v_stride_p=H * S * D, v_stride_h=S * D, v_stride_t=D,
             block_table=256, table_stride=4, table_width=4, seq_lens=512, q_starts=768, num_tokens=2, errors=None)
    d.update(kw)
    return nat.PagedDesc(**d)


def _query(**kw):
    d = dict(q=4096, stride_t=512, stride_h=128, out=8192, out_stride_t=512, out_stride_h=128, lse=None,
             num_query_heads=4, causal=1, window=0, scaling=0.1, softcap=0.0)
    d.update(kw)
    return nat.PagedQueryDesc(**d)


def _turn(**kw):
    d = dict(cos=4096, sin=8192, cs_stride=64, cs_rows=100, cs_dtype=0, rot_dim=128, axes=1)
    d.update(kw)
    return nat.TurnDesc(**d)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=3), UNSUPPORTED), (dict(head_dim=12, k_stride_t=16), UNSUPPORTED), (dict(head_dim=264), UNSUPPORTED),
    (dict(page_size=0), ARG), (dict(num_kv_heads=0), ARG), (dict(batch=-1), ARG), (dict(num_tokens=-1), ARG),
    (dict(seq_lens=None), ARG), (dict(q_starts=None), ARG), (dict(block_table=None), ARG), (dict(k=None), ARG),
    (dict(k=4100), ARG), (dict(v_stride_t=129), ARG), (dict(k_stride_p=-128), ARG), (dict(num_tokens=1 << 31), UNSUPPORTED),
    (dict(table_width=1 << 28), UNSUPPORTED), (dict(batch=(1 << 20) + 1), UNSUPPORTED),
])
def test_bad_caches_are_refused(kw, code):
    lib = nat.load_library()
    p, q = _paged(**kw), _query()
    assert lib.kiv_paged_attend(ctypes.byref(p), ctypes.byref(q), 4096, 1 << 40, None) == code, lib.kiv_last_error()
    assert lib.kiv_last_error()
    if "head_dim" not in kw or kw["head_dim"] != 264:
        assert lib.kiv_paged_append(ctypes.byref(p), 4096, 256, 128, 8192, 256, 128, None, None) == code
        assert lib.kiv_paged_workspace_bytes(ctypes.byref(p), ctypes.byref(q)) == 0


@pytest.mark.parametrize("kw,code", [
    (dict(num_query_heads=3), ARG), (dict(num_query_heads=0), ARG), (dict(window=-1), ARG), (dict(window=5, causal=0), ARG),
    (dict(softcap=-1.0), ARG), (dict(softcap=float("nan")), ARG), (dict(q=None), ARG), (dict(q=4104), ARG), (dict(out=None), ARG),
    (dict(stride_t=513), ARG), (dict(out_stride_h=1), ARG),
])
def test_bad_queries_are_refused(kw, code):
    lib = nat.load_library()
    p, q = _paged(), _query(**kw)
    assert lib.kiv_paged_attend(ctypes.byref(p), ctypes.byref(q), 4096, 1 << 40, None) == code


def test_workspace_is_checked():
    lib = nat.load_library()
    p, q = _paged(), _query()
    need = lib.kiv_paged_workspace_bytes(ctypes.byref(p), ctypes.byref(q))
    assert need > 0
    assert lib.kiv_paged_attend(ctypes.byref(p), ctypes.byref(q), None, need, None) == CAPACITY
    assert lib.kiv_paged_attend(ctypes.byref(p), ctypes.byref(q), 4096, need - 1, None) == CAPACITY
    assert lib.kiv_paged_attend(ctypes.byref(p), ctypes.byref(q), 4097, need, None) == CAPACITY


def test_null_descriptors_are_refused():
    lib = nat.load_library()
    p, q, t, r = _paged(), _query(), _turn(), nat.RowsDesc(4096, 0, 128, 128, 2, 0)
    assert lib.kiv_paged_attend(None, ctypes.byref(q), 4096, 1 << 40, None) == ARG
    assert lib.kiv_paged_attend(ctypes.byref(p), None, 4096, 1 << 40, None) == ARG
    assert lib.kiv_paged_append(None, 4096, 256, 128, 8192, 256, 128, None, None) == ARG
    assert lib.kiv_qk_norm_rope(1, 1, 1, 128, None, None, ctypes.byref(r), None, ctypes.byref(t), None, None) == ARG
    assert lib.kiv_qk_norm_rope(1, 1, 1, 128, ctypes.byref(r), ctypes.byref(r), ctypes.byref(r), None, ctypes.byref(t), None, None) == ARG
    assert lib.kiv_qk_norm_rope(1, 1, 1, 128, ctypes.byref(r), None, ctypes.byref(r), None, None, None, None) == ARG


@pytest.mark.parametrize("kw", [dict(sin=None), dict(rot_dim=3), dict(rot_dim=0), dict(rot_dim=130), dict(cs_dtype=2),
                                dict(axes=0), dict(cs_rows=-1), dict(norm=1, eps=-1.0), dict(norm=1, eps=float("nan")),
                                dict(norm=1, q_weight=4096, weight_dtype=2)])
def test_bad_turns_are_refused(kw):
    lib = nat.load_library()
    r, t, p = nat.RowsDesc(4096, 0, 128, 128, 2, 0), _turn(**kw), _paged()
    args = (1, 1, 1, 128, ctypes.byref(r), None, ctypes.byref(r), None, ctypes.byref(t), None, None)
    assert lib.kiv_qk_norm_rope(*args) == ARG
    assert lib.kiv_paged_append(ctypes.byref(p), 4096, 256, 128, 8192, 256, 128, ctypes.byref(t), None) == ARG


@pytest.mark.parametrize("rows", [(4104, 0, 128, 128), (4096, 0, 129, 128), (4096, 4, 128, 128), (None, 0, 128, 128)])
def test_misaligned_rows_are_refused(rows):
    lib = nat.load_library()
    r, ok, t = nat.RowsDesc(*rows, 2, 0), nat.RowsDesc(4096, 0, 128, 128, 2, 0), _turn()
    for a, b in ((r, ok), (ok, r)):
        assert lib.kiv_qk_norm_rope(1, 1, 1, 128, ctypes.byref(a), None, ctypes.byref(b), None, ctypes.byref(t), None, None) == ARG


def test_rows_and_heads_without_a_kernel_are_refused():
    lib = nat.load_library()
    r, t = nat.RowsDesc(4096, 0, 1024, 1024, 2, 0), _turn()
    for dtype, D in ((5, 128), (1, 12), (1, 520), (0, 260), (1, 0)):
        assert lib.kiv_qk_norm_rope(dtype, 1, 1, D, ctypes.byref(r), None, ctypes.byref(r), None, ctypes.byref(t), None, None) == UNSUPPORTED


def test_empty_calls_launch_nothing():
    lib = nat.load_library()
    p, q, t = _paged(num_tokens=0), _query(q=None, out=None), _turn()
    assert lib.kiv_paged_attend(ctypes.byref(p), ctypes.byref(q), None, 0, None) == 0
    assert lib.kiv_paged_append(ctypes.byref(p), None, 0, 0, None, 0, 0, None, None) == 0
    r = nat.RowsDesc(None, 0, 128, 128, 2, 0)
    assert lib.kiv_qk_norm_rope(1, 3, 0, 128, ctypes.byref(r), None, ctypes.byref(r), None, ctypes.byref(t), None, None) == 0


def test_tensors_on_the_cpu_are_refused():
    x = torch.zeros(1, 2, 3, 64)
    with pytest.raises(nat.KIVNativeError, match="CUDA device"):
        paged.qk_norm_rope(x, x)
    with pytest.raises(nat.KIVNativeError, match="CUDA device"):
        paged.paged_append(x[0], x[0], x, x, None, None, None)
    with pytest.raises(nat.KIVNativeError, match="CUDA device"):
        paged.paged_attend(x[0], x, x, None, None, None, 1.0)


def test_a_layer_step_traces_with_fake_tensors():
    ops.load()
    with FakeTensorMode():
        dev, bf = torch.device("cuda"), torch.bfloat16
        q, k = torch.empty(1, 8, 4, 64, dtype=bf, device=dev), torch.empty(1, 2, 4, 64, dtype=bf, device=dev)
        cos = torch.empty(4, 32, device=dev)
        qo, ko = torch.empty_like(q), torch.empty_like(k)
        torch.ops.kiv.qk_norm_rope(q, k, cos, cos, None, None, False, 1e-6, None, None, 0.0, qo, ko, None)
        pages = torch.empty(4, 2, 16, 64, dtype=bf, device=dev)
        ints = [torch.empty(s, dtype=torch.int32, device=dev) for s in ((1, 4), (1,), (2,))]
        rows = torch.empty(4, 2, 64, dtype=bf, device=dev)
        torch.ops.kiv.paged_append(rows, rows, pages, pages, *ints, None, None, None, None, False, None, None, 0.0, None)
        qr = torch.empty(4, 8, 64, dtype=bf, device=dev)
        out = torch.empty_like(qr)
        torch.ops.kiv.paged_attend(qr, pages, pages, *ints, 0.1, True, 0, 0.0, 0, out, None, None)


def test_rotary_tables_are_exact_at_far_positions():
    inv = torch.tensor([1.0, 1e-4], dtype=torch.float64)
    cos, sin = paged.rotary_table(inv, 1 << 20, scaling=2.0)
    far = torch.tensor([(1 << 20) - 1.0], dtype=torch.float64)
    assert cos.dtype == torch.float32 and cos.shape == (1 << 20, 2)
    assert torch.equal(cos[-1], (2 * torch.cos(far * inv)).float()) and torch.equal(sin[-1], (2 * torch.sin(far * inv)).float())


def test_paged_cache_needs_a_gpu():
    from kiv_b200 import PagedKVCache
    with pytest.raises(nat.KIVNativeError, match="CUDA devices only"):
        PagedKVCache(4, 16, 1, 64, device="cpu")
    with pytest.raises(ValueError):
        PagedKVCache(0, 16, 1, 64, device="cpu")


def test_fused_rotation_stands_in_and_leaves_again():
    """On the CPU the model's own function answers, to the bit; another convention is left alone."""
    import sys
    from transformers import LlamaConfig, LlamaForCausalLM
    from kiv_b200 import KIVConfig, KIVMiddleware
    from kiv_b200 import middleware as mid

    torch.manual_seed(0)
    model = LlamaForCausalLM(LlamaConfig(vocab_size=64, hidden_size=64, intermediate_size=64, num_hidden_layers=1,
                                         num_attention_heads=2, num_key_value_heads=1, head_dim=32,
                                         attn_implementation="eager")).eval()
    module = sys.modules[type(model.model.layers[0].self_attn).__module__]
    before = module.apply_rotary_pos_emb
    ids = torch.arange(10)[None]
    want = model(input_ids=ids, use_cache=False).logits
    mw = KIVMiddleware(model, KIVConfig())
    mw.install()
    assert module.apply_rotary_pos_emb is before            # off by default
    mw.uninstall()
    mw.install(fused_rotary=True)
    assert module.apply_rotary_pos_emb is not before
    other = KIVMiddleware(model, KIVConfig())
    other._text_model, other.topology = mw._text_model, mw.topology
    other._fuse_rotary()                                    # already there: neither stacked nor taken out by another
    assert module.apply_rotary_pos_emb._kiv_original is before and other._rotary_module is None
    assert torch.equal(model(input_ids=ids, use_cache=False).logits, want)
    mw.uninstall()
    assert module.apply_rotary_pos_emb is before

    def adjacent(q, k, cos, sin, unsqueeze_dim=1):
        c, s = cos.unsqueeze(unsqueeze_dim), sin.unsqueeze(unsqueeze_dim)
        turn = lambda x: x * c + torch.stack([-x[..., 1::2], x[..., ::2]], -1).flatten(-2) * s
        return turn(q), turn(k)

    assert mid._turns_half_split(before, 32) and not mid._turns_half_split(adjacent, 32)
    module.apply_rotary_pos_emb = adjacent
    try:
        mw.install(fused_rotary=True)
        assert module.apply_rotary_pos_emb is adjacent
        mw.uninstall()
    finally:
        module.apply_rotary_pos_emb = before


def test_inputs_that_need_gradients_are_refused():
    q, k = torch.zeros(1, 2, 1, 64), torch.zeros(1, 1, 1, 64)
    w = torch.nn.Parameter(torch.ones(64))
    rows, pages, ints = torch.zeros(1, 1, 64), torch.zeros(1, 1, 8, 64), torch.zeros(1, 1, dtype=torch.int32)
    need = rows.clone().requires_grad_()
    calls = [lambda: paged.qk_norm_rope(q.clone().requires_grad_(), k, eps=1e-6), lambda: paged.qk_norm_rope(q, k, eps=1e-6, k_weight=w),
             lambda: paged.paged_append(rows, need, pages, pages, ints, ints[0], ints[0]),
             lambda: paged.paged_attend(need, pages, pages, ints, ints[0], ints[0], 1.0)]
    for call in calls:
        with pytest.raises(nat.KIVNativeError, match="no backward"):
            call()
        with torch.no_grad(), pytest.raises(nat.KIVNativeError, match="CUDA device"):     # passes on to the next check
            call()
