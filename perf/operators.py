"""The rotation and paged-cache operators: the calls that are timed, and the same results in elementary torch operations.

Three operators, as one attention layer of a serving step uses them:

* ``rope``    norms of the queries and keys of each head and their position rotation, in one pass;
* ``append``  new keys (normed and rotated on the way) and values into the pages of a paged cache;
* ``attend``  attention of each sequence's new tokens over its pages, the new tokens included.

Sizes are those of the benchmark configurations (head layouts 8/1 x 256, 28/4 x 128, 32/8 x 128, 32/32 x 96 and
32/4 x 64, pages of 128 tokens, chunks of 4096) beside pages of 16 to 64 tokens and generic ragged batches.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
BASE = 1e6          # base of the rotation frequencies
FAR = 131072        # rows of the cos / sin tables


def listed():
    return [
        # one decode token of the MQA configuration: launch latency
        dict(name="rope one token 8/1x256", op="rope", dtype="bf16", batch=1, tokens=1, hq=8, hkv=1, dim=256, rot=256,
             norm=True, axes=1, interleaved=False),
        # prompt chunks of two sequences, no norm
        dict(name="rope chunk 28/4x128", op="rope", dtype="bf16", batch=2, tokens=4099, hq=28, hkv=4, dim=128, rot=128,
             norm=False, axes=1, interleaved=False),
        # image and video tokens: three position axes, adjacent pairs, part of the head rotated
        dict(name="rope three axes 32/8x128", op="rope", dtype="f16", batch=3, tokens=1021, hq=32, hkv=8, dim=128, rot=96,
             norm=True, axes=3, interleaved=True),
        # one token of each of 64 sequences into small pages
        dict(name="append decode 8x128", op="append", dtype="bf16", batch=64, most=1, cached=1024, hkv=8, dim=128, rot=128,
             page=16, norm=True, interleaved=False),
        # ragged prompts into large pages, 32-bit rows
        dict(name="append prompts 4x64 f32", op="append", dtype="f32", batch=5, most=3001, cached=2048, hkv=4, dim=64, rot=64,
             page=128, norm=False, interleaved=False),
        # one token over a hot window of the MQA configuration: latency
        dict(name="attend one token 8/1x256", op="attend", dtype="bf16", batch=1, most=1, cached=2047, hq=8, hkv=1, dim=256,
             page=128, even=True, window=0, softcap=0.0),
        # a decode batch of unequal lengths: bandwidth
        dict(name="attend decode 32/8x128", op="attend", dtype="bf16", batch=64, most=1, cached=32767, hq=32, hkv=8, dim=128,
             page=16, even=False, window=0, softcap=0.0),
        # a few drafted tokens of each sequence to be checked
        dict(name="attend drafts 28/4x128", op="attend", dtype="bf16", batch=16, most=5, cached=16001, hq=28, hkv=4, dim=128,
             page=64, even=True, window=0, softcap=0.0),
        # a prompt chunk over a long cache: matrix products
        dict(name="attend chunk 32/8x128", op="attend", dtype="bf16", batch=1, most=4096, cached=32768, hq=32, hkv=8, dim=128,
             page=128, even=True, window=0, softcap=0.0),
        # the same for one key head of 256
        dict(name="attend chunk 8/1x256", op="attend", dtype="bf16", batch=2, most=2047, cached=16384, hq=8, hkv=1, dim=256,
             page=128, even=False, window=0, softcap=0.0),
        # prompts and single tokens in one batch, a sliding window and capped scores
        dict(name="attend mixed 32/32x96", op="attend", dtype="f16", batch=9, most=1021, cached=6000, hq=32, hkv=32, dim=96,
             page=48, even=False, window=1500, softcap=30.0),
        # 32-bit rows
        dict(name="attend chunk 32/4x64 f32", op="attend", dtype="f32", batch=3, most=130, cached=4096, hq=32, hkv=4, dim=64,
             page=128, even=False, window=0, softcap=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(8, 1, 256), (28, 4, 128), (32, 8, 128), (32, 32, 96), (32, 4, 64)]


def draw(rng: random.Random):
    hq, hkv, dim = rng.choice(HEADS)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    op = rng.choice(["rope", "append", "attend", "attend", "attend"])
    if op == "rope":
        batch = rng.choice([1, 2, 3, 8])
        return dict(op=op, dtype=dtype, batch=batch, tokens=_log(rng, 1, 8192 // batch), hq=hq, hkv=hkv, dim=dim,
                    rot=rng.choice([dim, dim, dim // 2]), norm=rng.random() < 0.5, axes=rng.choice([1, 1, 3]),
                    interleaved=rng.random() < 0.4)
    page = rng.choice([16, 32, 48, 64, 128])
    if op == "append":
        batch = _log(rng, 1, 96)
        return dict(op=op, dtype=dtype, batch=batch, most=_log(rng, 1, 8192 // batch), cached=_log(rng, 1, 4096), hkv=hkv, dim=dim,
                    rot=rng.choice([dim, dim, dim // 2]), page=page, norm=rng.random() < 0.5, interleaved=rng.random() < 0.4)
    while True:
        batch, cached = _log(rng, 1, 64), _log(rng, 1, 32768)
        most = rng.choice([1, _log(rng, 2, 16), _log(rng, 17, 4096)])
        case = dict(op=op, dtype=dtype, batch=batch, most=most, cached=cached, hq=hq, hkv=hkv, dim=dim, page=page,
                    even=rng.random() < 0.5, window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]),
                    softcap=rng.choice([0.0, 0.0, 0.0, 30.0]))
        scores = batch * hq * most * (cached + most)
        flops = 4 * scores * dim * (8 if dtype == "f32" else 1)
        held = batch * hkv * (cached + most) * dim
        if flops < 2.0e12 and scores < 4e9 and held < 3e9:
            return case


def _lengths(case):
    """(new tokens, tokens in all) of each sequence: even batches have them alike, ragged ones from 1 (new) and 0 (cached) up."""
    n, c, b = case["most"], case["cached"], case["batch"]
    if case.get("even", False):
        return [n] * b, [n + c] * b
    rng = random.Random(b * 7919 + n * 31 + c)
    new = [n] + [max(1, round(n * rng.random() ** 2)) for _ in range(b - 1)]
    old = [c] + [round(c * rng.random()) for _ in range(b - 1)]
    return new, [x + y for x, y in zip(new, old)]


def _table(rot, device):
    freq = BASE ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    angle = torch.arange(FAR, dtype=torch.float64, device=device)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    t = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=dev, dtype=torch.float32) * scale).to(t)

    s = dict(case)
    hkv, dim = case["hkv"], case["dim"]
    if case["op"] != "attend":
        s["cos"], s["sin"] = _table(case["rot"], dev)
        s["eps"] = EPS if case["norm"] else None
        s["kw"] = (1 + 0.2 * torch.randn(dim, generator=g, device=dev)).to(t) if case["norm"] else None
    if case["op"] == "rope":
        b, n, hq = case["batch"], case["tokens"], case["hq"]
        # a projection's output: [tokens, heads, dim] rows, seen as [batch, heads, tokens, dim]
        s["q"] = normal(b, n, hq, dim, scale=1.5).transpose(1, 2)
        s["k"] = normal(b, n, hkv, dim, scale=1.5).transpose(1, 2)
        s["qw"] = (1 + 0.2 * torch.randn(dim, generator=g, device=dev)).to(t) if case["norm"] else None
        first = torch.randint(0, FAR - n, (b, 1), generator=g, device=dev)
        pos = first + torch.arange(n, device=dev)
        if case["axes"] > 1:   # frames, rows and columns of a grid 32 wide
            i = torch.arange(n, device=dev).expand(b, n)
            s["positions"] = torch.stack([first + i // 1024, first // 2 + i // 32 % 32, first // 2 + i % 32])
            half = case["rot"] // 2
            s["pair_axes"] = torch.tensor([j * 3 // half for j in range(half)], dtype=torch.int32, device=dev)
        else:
            s["positions"], s["pair_axes"] = pos, None
        return s
    new, lens = _lengths(case)
    b, page = case["batch"], case["page"]
    width = -(-max(lens) // page)
    need = [-(-x // page) for x in lens]
    pages = sum(need) + 3
    perm = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    start = torch.tensor([0] + [sum(need[:i + 1]) for i in range(b)], device=dev)
    col = torch.arange(width, device=dev)
    at = (start[:-1, None] + col).clamp_(max=pages - 1)
    s["block_table"] = torch.where(col < (start[1:] - start[:-1])[:, None], perm[at], 0)
    s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    s["q_starts"] = torch.tensor([0] + [sum(new[:i + 1]) for i in range(b)], dtype=torch.int32, device=dev)
    s["total"], s["longest"], s["most_new"] = sum(new), max(lens), max(new)
    s["k_pages"] = normal(pages, hkv, page, dim)
    s["v_pages"] = normal(pages, hkv, page, dim)
    if case["op"] == "append":
        s["k"] = normal(s["total"], hkv, dim, scale=1.5)
        s["v"] = normal(s["total"], hkv, dim)
    else:
        s["q"] = normal(s["total"], case["hq"], dim, scale=1.5)
        s["scaling"] = dim ** -0.5
    return s


def run(state):
    if own:
        return _own(state)
    return {"rope": _rope, "append": _append, "attend": _attend}[state["op"]](state)


def _own(s):
    from kiv_b200 import paged
    if s["op"] == "rope":
        return paged.qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], positions=s["positions"], pair_axes=s["pair_axes"],
                                  interleaved=s["interleaved"], eps=s["eps"], q_weight=s["qw"], k_weight=s["kw"])
    if s["op"] == "append":
        paged.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["block_table"], s["seq_lens"], s["q_starts"],
                           cos=s["cos"], sin=s["sin"], interleaved=s["interleaved"], eps=s["eps"], k_weight=s["kw"])
        return s["k_pages"], s["v_pages"]
    return paged.paged_attend(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["seq_lens"], s["q_starts"], s["scaling"],
                              window=s["window"], softcap=s["softcap"], max_query_len=s["most_new"], return_lse=True)


# ------------------------------------------------------------------ plain forms
def _turn(x, w, eps, cos, sin, interleaved):
    """RMS norm of the rows of ``x`` (fp32) and rotation of their first 2 * cos.shape[-1] elements."""
    if eps is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w.float()
    half = cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _rope(s):
    pos = s["positions"]
    if s["pair_axes"] is None:
        cos, sin = s["cos"][pos], s["sin"][pos]                       # [B, Q, half]
    else:
        pair = torch.arange(s["cos"].shape[1], device=pos.device)
        at = pos[s["pair_axes"].long()].permute(1, 2, 0)               # [B, Q, half]
        cos, sin = s["cos"][at, pair], s["sin"][at, pair]
    cos, sin = cos[:, None], sin[:, None]
    return (_turn(s["q"].float(), s["qw"], s["eps"], cos, sin, s["interleaved"]).to(s["q"].dtype),
            _turn(s["k"].float(), s["kw"], s["eps"], cos, sin, s["interleaved"]).to(s["k"].dtype))


def _places(s):
    """(sequence, place in the sequence) of every new token."""
    row = torch.arange(s["total"], device=s["q_starts"].device)
    seq = torch.searchsorted(s["q_starts"], row, right=True) - 1
    return seq, s["seq_lens"][seq] - s["q_starts"][seq + 1] + row


def _append(s):
    seq, place = _places(s)
    page = s["block_table"][seq, place // s["page"]].long()
    cos, sin = s["cos"][place][:, None], s["sin"][place][:, None]
    s["k_pages"][page, :, place % s["page"]] = _turn(s["k"].float(), s["kw"], s["eps"], cos, sin, s["interleaved"]).to(s["k"].dtype)
    s["v_pages"][page, :, place % s["page"]] = s["v"]
    return s["k_pages"], s["v_pages"]


def _attend(s):
    b, hq, hkv, d, n, longest = s["batch"], s["hq"], s["hkv"], s["dim"], s["most_new"], s["longest"]
    grp = hq // hkv
    key = torch.arange(longest, device=s["q"].device)
    page = s["block_table"][:, key // s["page"]].long()                # [B, L]
    k = s["k_pages"][page, :, key % s["page"]].float()                 # [B, L, Hkv, D]
    v = s["v_pages"][page, :, key % s["page"]].float()
    seq, place = _places(s)
    row = torch.arange(s["total"], device=seq.device) - s["q_starts"][seq]
    q = torch.zeros(b, n, hq, d, device=seq.device)
    q[seq, row] = s["q"].float() * s["scaling"]
    at = torch.full((b, n), -1, device=seq.device)
    at[seq, row] = place
    sc = torch.matmul(q.view(b, n, hkv, grp, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, grp * n, d), k.permute(0, 2, 3, 1))
    del k
    sc = sc.view(b, hkv, grp, n, longest)
    if s["softcap"]:
        sc.div_(s["softcap"]).tanh_().mul_(s["softcap"])
    hidden = key > at[:, :, None]
    if s["window"]:
        hidden |= key <= at[:, :, None] - s["window"]
    sc.masked_fill_(hidden[:, None, None], -math.inf)
    top = sc.amax(-1, keepdim=True).clamp_(min=-1e30)
    sc.sub_(top).exp_()
    total = sc.sum(-1, keepdim=True)
    o = torch.matmul(sc.view(b, hkv, grp * n, longest), v.permute(0, 2, 1, 3)).view(b, hkv, grp, n, d) / total.clamp(min=1e-38)
    lse = (top + total.log()).squeeze(-1)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, n, hq, d)[seq, row]
    return o.to(s["q"].dtype), lse.permute(0, 3, 1, 2).reshape(b, n, hq)[seq, row]


# ------------------------------------------------------------------ definition in 64 bits
def _exact_turn(x, w, eps, cos, sin, interleaved):
    x, cos, sin = x.double(), cos.double(), sin.double()
    if eps is not None:
        x = x / ((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + eps).sqrt() * w.double()
    rot = 2 * cos.shape[-1]
    pairs = x[..., :rot].unflatten(-1, (-1, 2)) if interleaved else x[..., :rot].unflatten(-1, (2, -1)).transpose(-1, -2)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.complex(cos, sin))
    out = x.clone()
    out[..., :rot] = turned.flatten(-2) if interleaved else turned.transpose(-1, -2).flatten(-2)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        pos, axes = s["positions"], s["pair_axes"]
        half = s["cos"].shape[1]
        rows = [pos if axes is None else pos[int(axes[j])] for j in range(half)]
        cos = torch.stack([s["cos"][rows[j], j] for j in range(half)], -1)[:, None]
        sin = torch.stack([s["sin"][rows[j], j] for j in range(half)], -1)[:, None]
        return (_exact_turn(s["q"], s["qw"], s["eps"], cos, sin, s["interleaved"]),
                _exact_turn(s["k"], s["kw"], s["eps"], cos, sin, s["interleaved"]))
    starts, lens, page = s["q_starts"].tolist(), s["seq_lens"].tolist(), s["page"]
    if case["op"] == "append":
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
        for i in range(case["batch"]):
            lo, hi = starts[i], starts[i + 1]
            place = torch.arange(lens[i] - (hi - lo), lens[i], device=kp.device)
            pg = s["block_table"][i].long()[place // page]
            kp[pg, :, place % page] = _exact_turn(s["k"][lo:hi], s["kw"], s["eps"], s["cos"][place][:, None], s["sin"][place][:, None],
                                                  s["interleaved"])
            vp[pg, :, place % page] = s["v"][lo:hi].double()
        return kp, vp
    hq, hkv, d = case["hq"], case["hkv"], case["dim"]
    grp = hq // hkv
    out = torch.zeros(s["total"], hq, d, dtype=torch.float64, device=s["q"].device)
    lse = torch.full((s["total"], hq), -math.inf, dtype=torch.float64, device=s["q"].device)
    for i in range(case["batch"]):
        lo, hi, length = starts[i], starts[i + 1], lens[i]
        key = torch.arange(length, device=out.device)
        pg = s["block_table"][i].long()[key // page]
        place = torch.arange(length - (hi - lo), length, device=out.device)[:, None]
        seen = key <= place
        if case["window"]:
            seen &= key > place - case["window"]
        for h in range(hkv):
            k = s["k_pages"][pg, h, key % page].double()
            v = s["v_pages"][pg, h, key % page].double()
            x = torch.einsum("ngd,ld->gnl", s["q"][lo:hi, h * grp:(h + 1) * grp].double(), k) * s["scaling"]
            if case["softcap"]:
                x = torch.tanh(x / case["softcap"]) * case["softcap"]
            x = x.masked_fill(~seen, -math.inf)
            z = torch.logsumexp(x, -1)
            x = torch.exp(x - z[..., None])
            out[lo:hi, h * grp:(h + 1) * grp] = torch.einsum("gnl,ld->ngd", x, v)
            lse[lo:hi, h * grp:(h + 1) * grp] = z.T
    return out, lse


def _seen(case):
    """Query-key pairs that the mask lets through, and keys that some query sees, over all sequences."""
    pairs = keys = 0
    new, lens = _lengths(case)
    for n, length in zip(new, lens):
        first, w = length - n, case["window"]
        if w:
            pairs += sum(min(first + i + 1, w) for i in range(n))
            keys += length - max(0, first + 1 - w)
        else:
            pairs += n * first + n * (n + 1) // 2
            keys += length
    return pairs, keys


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    hkv, d = case["hkv"], case["dim"]
    if case["op"] == "rope":
        rows = case["batch"] * case["tokens"]
        per = (case["hq"] + hkv) * d
        return {"bytes": rows * (2 * per * e + case["rot"] * 4 + 8 * case["axes"]), "flops": rows * per * (3 + (4 if case["norm"] else 0))}
    new, lens = _lengths(case)
    total = sum(new)
    if case["op"] == "append":
        return {"bytes": total * (4 * hkv * d * e + case["rot"] * 4) + 12 * case["batch"],
                "flops": total * hkv * d * (3 + (4 if case["norm"] else 0))}
    pairs, keys = _seen(case)
    return {"bytes": 2 * keys * hkv * d * e + total * case["hq"] * (2 * d * e + 4), "flops": 4 * pairs * case["hq"] * d}
