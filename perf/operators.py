"""Workloads of the rotary and block-sparse attention operators.

Each case names its ``kind``:

* ``rotary``  rotation of q (and k) heads by their positions, out of slices of
              one fused projection; forwards and backwards (``inverse``);
* ``means``   the mean key of every block of a ragged cache;
* ``select``  the blocks that each tile of queries attends to, by the product
              of the tile's summed queries with the block means;
* ``attend``  attention of each tile of queries over its listed blocks.

``run`` computes them in plain torch where ``own`` is false, and through the
framework's entry points where it is true.  ``exact`` restates them in 64
bits from their definitions.

Layouts.  Queries are ``[tokens, heads, dim]`` with sequence b at rows
``cu_q[b] .. cu_q[b + 1]``.  Keys and values are either one flat
``[rows, dim]`` with a sequence for each (batch, KV head), the layout in which
the pyramid cache packs them (``per_head``), or ``[rows, KV heads, dim]`` with
a sequence for each batch.  A sequence s that starts at row c has its blocks
at rows ``c // block + s`` and following of the means, and a query sequence
its tiles likewise, so that no prefix sum over ragged lengths is needed.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    # the packed cache of one layer: 12 heads with a key length each, 1,560 tokens per latent frame, 3 frames a chunk
    cache = dict(dtype="bf16", dim=128, heads=12, kv_heads=12, per_head=True, batch=3, q_lo=1560, q_hi=1560,
                 k_lo=6240, k_hi=32760, block=64, causal=False, lens=0)
    # a batch of single tokens over their contexts, 4 query heads to a KV head
    decode = dict(dtype="bf16", dim=128, heads=32, kv_heads=8, per_head=False, batch=16, q_lo=1, q_hi=1, k_lo=4000,
                  k_hi=32760, block=64, block_q=1, causal=False, lens=1)
    # a prompt in which every token has blocks of its own, 16 query heads to a KV head
    prompt = dict(dtype="fp16", dim=128, heads=32, kv_heads=2, per_head=False, batch=1, q_lo=2047, q_hi=2047, k_lo=2047,
                  k_hi=2047, block=64, block_q=1, causal=True, lens=2)
    # one short request on a small grouped-head model
    single = dict(dtype="fp16", dim=64, heads=8, kv_heads=2, per_head=False, batch=1, q_lo=1, q_hi=1, k_lo=1000,
                  k_hi=1000, block=64, block_q=1, causal=False, lens=3)
    return [
        # queries of a chunk of latent frames: three position axes, pairs interleaved
        dict(name="rotary_frames", kind="rotary", dtype="bf16", rows=4680, heads=12, kv_heads=0, dim=128, rotary_dim=128,
             axes=3, interleaved=True, inverse=False, far=120, scaled=False),
        # single tokens far out in scaled contexts, q and k of one projection
        dict(name="rotary_tokens", kind="rotary", dtype="bf16", rows=16, heads=32, kv_heads=8, dim=128, rotary_dim=128,
             axes=1, interleaved=False, inverse=False, far=1 << 20, scaled=True),
        # gradients of a prompt whose heads are rotated in part, in 32 bits
        dict(name="rotary_grad_part", kind="rotary", dtype="fp32", rows=8191, heads=16, kv_heads=4, dim=80, rotary_dim=32,
             axes=1, interleaved=False, inverse=True, far=8191, scaled=False),
        # block means of the packed cache, and of a few short contexts
        dict(name="means_cache", kind="means", **cache),
        dict(name="means_short", kind="means", **dict(single, batch=3, k_lo=300)),
        # the blocks of a chunk's query tiles: sink and recent frames forced
        dict(name="select_cache", kind="select", **cache, block_q=120, topk=100, sink=8, recent=16),
        # of single tokens over long contexts
        dict(name="select_tokens", kind="select", **decode, topk=32, sink=1, recent=2),
        # of every token of a prompt
        dict(name="select_prompt", kind="select", **prompt, topk=16, sink=1, recent=2),
        # attention over those lists
        dict(name="attend_cache", kind="attend", **cache, block_q=120, topk=100, sink=8, recent=16, lse=False),
        dict(name="attend_tokens", kind="attend", **decode, topk=32, sink=1, recent=2, lse=True),
        dict(name="attend_prompt", kind="attend", **prompt, topk=16, sink=1, recent=2, lse=False),
        # the smallest: one token, one short context
        dict(name="attend_single", kind="attend", **single, topk=8, sink=1, recent=1, lse=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng: random.Random):
    kind = rng.choice(["rotary", "means", "select", "select", "attend", "attend", "attend"])
    if kind == "rotary":
        dim = rng.choice([64, 80, 96, 128, 256])
        axes = rng.choice([1, 1, 3])
        rows, heads = _log(rng, 1, 16384), rng.choice([1, 3, 8, 12, 16, 32])
        kv = rng.choice([0, max(1, heads // 4)])
        rows = min(rows, 13_000_000 // ((heads + kv) * dim))
        return dict(kind=kind, dtype=rng.choice(["bf16", "fp16", "fp32"]), rows=rows, heads=heads, kv_heads=kv, dim=dim,
                    rotary_dim=dim if axes == 3 else rng.choice([dim, dim // 2, 2 * rng.randint(1, dim // 2)]), axes=axes,
                    interleaved=rng.random() < 0.5, inverse=rng.random() < 0.3,
                    far=_log(rng, 16, 1 << 20), scaled=axes == 1 and rng.random() < 0.5)
    case = dict(kind=kind, dtype=rng.choice(["bf16", "fp16"]), dim=rng.choice([64, 128, 128]),
                block=rng.choice([64, 64, 128, 256]), lens=rng.randrange(1 << 20))
    shape = rng.choice(["tiles", "tokens", "prompt"])
    if shape == "tiles":
        kv = rng.choice([1, 5, 8, 12])
        group = rng.choice([1, 1, 2])
        bq = rng.randint(32, 256 // group)
        k_hi = _log(rng, 200, 32760)
        q = _log(rng, 30, 1560)
        case.update(heads=kv * group, kv_heads=kv, per_head=rng.random() < 0.6, batch=rng.randint(1, 3), q_lo=max(1, q // 3),
                    q_hi=q, k_lo=max(1, k_hi // 4), k_hi=k_hi, block_q=bq, causal=False)
    elif shape == "tokens":
        kv = rng.choice([1, 2, 4, 8])
        k_hi = _log(rng, 100, 65000)
        case.update(heads=kv * rng.choice([1, 4, 7, 16]), kv_heads=kv, per_head=rng.random() < 0.3, batch=_log(rng, 1, 24),
                    q_lo=1, q_hi=1, block_q=1, causal=rng.random() < 0.3)
        k_hi = max(1, min(k_hi, (600_000 if kind == "means" else 4_000_000) // (case["batch"] * kv)))
        case.update(k_lo=max(1, k_hi // 8), k_hi=k_hi)
    else:
        kv = rng.choice([1, 2])
        n = _log(rng, 40, 2000)
        case.update(heads=kv * rng.choice([2, 8, 16]), kv_heads=kv, per_head=False, batch=1, q_lo=n, q_hi=n, k_lo=n,
                    k_hi=n + rng.choice([0, rng.randint(1, 2000)]), block_q=1, causal=True)
    if kind != "means":
        most = {"prompt": 16, "tokens": 64, "tiles": 100}[shape]
        if shape == "tiles":  # as many lists of keys as the largest listed case
            most = max(1, min(most, 3 * 13 * 12 * 100 // (case["batch"] * kv * -(-case["q_hi"] // case["block_q"]))))
        case["topk"] = max(1, _log(rng, 1, most) * 64 // case["block"])
        room = case["topk"]
        if kind == "select":  # contexts of more blocks than are chosen, and more chosen than forced
            case["k_lo"] = max(case["k_lo"], 4 * case["block"])
            case["k_hi"] = max(case["k_hi"], case["k_lo"])
            case["topk"] = min(case["topk"], case["k_lo"] // case["block"] - 2)
            room = case["topk"] - 1
        case["sink"] = rng.randint(0, min(2, room))
        case["recent"] = rng.randint(0, min(2, room - case["sink"]))
    if kind == "attend":
        case["lse"] = rng.random() < 0.5
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lens(case):
    """Rows of every query sequence and keys of every key sequence."""
    rng = random.Random(case["lens"])
    n = case["batch"] * (case["kv_heads"] if case["per_head"] else 1)
    ks = [rng.randint(case["k_lo"], case["k_hi"]) for _ in range(n)]
    qs = [rng.randint(case["q_lo"], case["q_hi"]) for _ in range(case["batch"])]
    return qs, ks


def _cu(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device=DEV)


def _rotary_frequencies(case):
    """(frequencies of the pairs in 64 bits, pairs of each axis, scale)."""
    pairs = case["rotary_dim"] // 2
    third = pairs // 3
    axes = (pairs - 2 * third, third, third) if case["axes"] == 3 else (pairs,)
    f = torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64) / max(n, 1)) for n in axes])
    if case["scaled"]:  # slow pairs slowed further, for contexts 16 times as long
        turns = f * 4096 / (2 * math.pi)
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        return f * keep + f / 16 * (1 - keep), axes, 0.1 * math.log(16) + 1
    return f, axes, 1.0


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rnd = lambda *shape, dtype=torch.float32: torch.randn(shape, generator=g, device=DEV, dtype=dtype)
    dtype = TYPES[case["dtype"]]
    if case["kind"] == "rotary":
        heads = case["heads"] + 2 * case["kv_heads"]
        qkv = rnd(case["rows"], heads, case["dim"]).to(dtype)  # the projection that q and k are slices of
        f, axes, scale = _rotary_frequencies(case)
        pos = torch.randint(0, case["far"], (case["rows"], case["axes"]), generator=g, device=DEV)
        return dict(case=case, q=qkv[:, :case["heads"]],
                    k=qkv[:, case["heads"]:case["heads"] + case["kv_heads"]] if case["kv_heads"] else None,
                    pos=pos[:, 0].contiguous() if case["axes"] == 1 else pos, freqs=f.to(DEV), axes=axes, scale=scale)
    qs, ks = _lens(case)
    s = dict(case=case, cu_q=_cu(qs), cu_k=_cu(ks), q_max=max(qs), k_max=max(ks))
    D, nk = case["dim"], sum(ks)
    kv_shape = (nk, D) if case["per_head"] else (nk, case["kv_heads"], D)
    if case["kind"] in ("means", "attend"):
        s["k"] = rnd(*kv_shape, dtype=dtype)
    if case["kind"] == "attend":
        s["v"] = rnd(*kv_shape, dtype=dtype)
    if case["kind"] != "means":
        s["q"] = rnd(sum(qs), case["heads"], D, dtype=dtype)
    if case["kind"] == "select":
        rows = nk // case["block"] + len(ks)
        s["means"] = rnd(rows, D) / 8 if case["per_head"] else rnd(rows, case["kv_heads"], D) / 8
    if case["kind"] == "attend":  # lists as a selection writes them: sink and recent blocks, the others at random
        p = _plan(s)
        j = torch.arange(p["blocks"], device=DEV)
        there = j < p["n"][..., None]                                       # [B, tiles, KV heads, blocks]
        r = torch.rand(there.shape, generator=g, device=DEV)
        r = torch.where((j < case["sink"]) | (j >= p["n"][..., None] - case["recent"]), 2.0, r)
        r = torch.where(there, r, -1.0)
        v, i = r.topk(min(case["topk"], p["blocks"]), dim=-1)
        i = torch.where(v >= 0, i, 1 << 30).sort(dim=-1).values
        i = torch.nn.functional.pad(torch.where(i < 1 << 30, i, -1), (0, case["topk"] - i.shape[-1]), value=-1)
        s["lists"] = _place(p, i.to(torch.int32), s["q"].shape[0] // case["block_q"] + case["batch"], -1)
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _plan(s):
    """Where the tiles and blocks lie, padded to [batch, tiles] and [KV sequences, blocks]."""
    case, B = s["case"], s["case"]["batch"]
    bq, bk, hk = case["block_q"], case["block"], case["kv_heads"]
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    lq = cu_q[1:] - cu_q[:-1]
    tiles = -(-s["q_max"] // bq)
    t = torch.arange(tiles, device=DEV)
    tile = cu_q[:-1, None] // bq + torch.arange(B, device=DEV)[:, None] + t  # [B, tiles]
    lk = (cu_k[1:] - cu_k[:-1]).view(B, -1).expand(B, hk)                    # [B, KV heads]
    begin = cu_k[:-1].view(B, -1).expand(B, hk)
    seq = torch.arange(cu_k.numel() - 1, device=DEV)
    first = (cu_k[:-1] // bk + seq).view(B, -1).expand(B, hk)
    limit = lk[:, None, :].expand(B, tiles, hk)                              # keys that a tile may see
    if case["causal"]:
        limit = (lk[:, None, :] - lq[:, None, None] + t[:, None] + 1).clamp(min=0)
    here = t[None] * bq < lq[:, None]
    limit = torch.where(here[..., None], limit, 0)
    row = (t[:, None] * bq + torch.arange(bq, device=DEV))[None].expand(B, -1, -1)  # [B, tiles, block_q]
    return dict(tile=tile, here=here, row=cu_q[:-1, None, None] + row, row_here=row < lq[:, None, None], begin=begin,
                first=first, limit=limit, n=(limit + bk - 1) // bk, blocks=-(-s["k_max"] // bk))


def _place(p, x, rows, fill):
    """x [B, tiles, ...] at its tiles' rows."""
    out = torch.full((rows,) + x.shape[2:], fill, dtype=x.dtype, device=DEV)
    out[p["tile"][p["here"]]] = x[p["here"]]
    return out


def _query_tiles(s, p, dtype):
    """[B, tiles, KV heads, block_q * group, dim], rows past a sequence's end as zero."""
    case, hk = s["case"], s["case"]["kv_heads"]
    q = s["q"][p["row"].clamp(max=s["q"].shape[0] - 1)].to(dtype)
    q = torch.where(p["row_here"][..., None, None], q, 0)
    B, T, bq = p["row"].shape
    q = q.view(B, T, bq, hk, case["heads"] // hk, case["dim"]).permute(0, 1, 3, 2, 4, 5)
    return q.reshape(B, T, hk, -1, case["dim"])


def _plain_rotary(s):
    case = s["case"]
    R, P = case["rotary_dim"], case["rotary_dim"] // 2
    pos = s["pos"].view(case["rows"], -1)
    axis = torch.repeat_interleave(torch.arange(len(s["axes"]), device=DEV), torch.tensor(s["axes"], device=DEV),
                                   output_size=P)
    angle = pos.double()[:, axis] * s["freqs"]
    c = (torch.cos(angle) * s["scale"]).float()[:, None]
    n = (torch.sin(angle) * (-s["scale"] if case["inverse"] else s["scale"])).float()[:, None]

    def turn(x):
        y = x.float()
        if case["interleaved"]:
            a, b = y[..., 0:R:2], y[..., 1:R:2]
            z = torch.stack([a * c - b * n, a * n + b * c], dim=-1).flatten(-2)
        else:
            a, b = y[..., :P], y[..., P:R]
            z = torch.cat([a * c - b * n, a * n + b * c], dim=-1)
        return torch.cat([z, y[..., R:]], dim=-1).to(x.dtype)

    return dict(q=turn(s["q"])) if s["k"] is None else dict(q=turn(s["q"]), k=turn(s["k"]))


def _plain_means(s):
    bk = s["case"]["block"]
    cu = s["cu_k"].long()
    S = cu.numel() - 1
    rows = s["k"].shape[0] // bk + S
    first = cu[:-1] // bk + torch.arange(S, device=DEV)
    r = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(first, r, right=True) - 1
    begin = cu[seq] + (r - first[seq]) * bk
    key = begin[:, None] + torch.arange(bk, device=DEV)
    ok = key < cu[seq + 1][:, None]
    ok = ok.view(rows, bk, *[1] * (s["k"].dim() - 1))
    x = torch.where(ok, s["k"][key.clamp(max=s["k"].shape[0] - 1)].float(), 0)
    return x.sum(dim=1) / ok.sum(dim=1).clamp(min=1)


def _plain_select(s):
    case = s["case"]
    p = _plan(s)
    q = _query_tiles(s, p, torch.float64).sum(dim=3)                          # [B, tiles, KV heads, dim]
    row = (p["first"][..., None] + torch.arange(p["blocks"], device=DEV)).clamp(max=s["means"].shape[0] - 1)
    if case["per_head"]:
        m = s["means"][row]                                                   # [B, KV heads, blocks, dim]
    else:
        m = s["means"][row, torch.arange(case["kv_heads"], device=DEV)[None, :, None]]
    score = torch.matmul(q.transpose(1, 2), m.double().transpose(-1, -2).contiguous()).float().transpose(1, 2)
    j, n = torch.arange(p["blocks"], device=DEV), p["n"][..., None]
    forced = (j < case["sink"]) | (j >= n - case["recent"])
    score = torch.where(forced, math.inf, score)
    score = torch.where(j < n, score, -math.inf)
    k = min(case["topk"], p["blocks"])
    i = score.sort(dim=-1, descending=True, stable=True).indices[..., :k]
    i = torch.where(i < n, i, 1 << 30).sort(dim=-1).values
    i = torch.where(i < 1 << 30, i, -1).to(torch.int32)
    i = torch.nn.functional.pad(i, (0, case["topk"] - k), value=-1)
    return _place(p, i, s["q"].shape[0] // case["block_q"] + case["batch"], -1)


def _plain_attend(s):
    case = s["case"]
    B, hk, bk, D = case["batch"], case["kv_heads"], case["block"], case["dim"]
    p = _plan(s)
    q = _query_tiles(s, p, torch.float32)
    lists = s["lists"][p["tile"].clamp(max=s["lists"].shape[0] - 1)].long()  # [B, tiles, KV heads, topk]
    key = lists[..., None] * bk + torch.arange(bk, device=DEV)
    ok = ((lists[..., None] >= 0) & (key < p["limit"][..., None, None])).flatten(-2)
    key = (p["begin"][:, None, :, None] + key.flatten(-2)).clamp(0, s["k"].shape[0] - 1)
    head = torch.arange(hk, device=DEV)[:, None]
    pick = lambda x: (x[key] if case["per_head"] else x[key, head]).float()
    score = torch.matmul(q, pick(s["k"]).transpose(-1, -2)) * D ** -0.5
    score = torch.where(ok[..., None, :], score, -math.inf)
    top = score.amax(dim=-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    e = torch.exp(score - top)
    l = e.sum(dim=-1, keepdim=True)
    o = torch.matmul(e, pick(s["v"])) / torch.where(l > 0, l, 1)
    G = case["heads"] // hk
    unpack = lambda x: x.view(B, -1, hk, case["block_q"], G, x.shape[-1]).permute(0, 1, 3, 2, 4, 5).flatten(3, 4)
    out = torch.zeros_like(s["q"])
    out[p["row"][p["row_here"]]] = unpack(o)[p["row_here"]].to(out.dtype)
    if not case["lse"]:
        return dict(out=out)
    lse = torch.empty(s["q"].shape[0], case["heads"], dtype=torch.float32, device=DEV)
    lse[p["row"][p["row_here"]]] = unpack(top + torch.log(l))[p["row_here"]][..., 0]
    return dict(out=out, lse=lse.t().contiguous())


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        package = os.path.join(ROOT, "pyramid-forcing_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        from pyramidkv import block_sparse, rope
        if kind == "rotary":
            out = rope.rotary(state["q"], state["pos"], state["freqs"], k=state["k"], axes=state["axes"],
                              interleaved=case["interleaved"], scale=state["scale"], inverse=case["inverse"])
            return dict(q=out) if state["k"] is None else dict(q=out[0], k=out[1])
        if kind == "means":
            return block_sparse.block_means(state["k"], state["cu_k"], case["block"], max_seqlen_k=state["k_max"])
        if kind == "select":
            # the formula ranks a token's own block by its mean like the others
            ranked = dict(rank_own=True) if case["causal"] and not case["recent"] else {}
            return block_sparse.block_select(state["q"], state["means"], state["cu_q"], state["cu_k"], state["q_max"],
                                             state["k_max"], case["topk"], block_q=case["block_q"],
                                             block_k=case["block"], sink_blocks=case["sink"],
                                             recent_blocks=case["recent"], causal=case["causal"], **ranked)
        out = block_sparse.block_sparse_attention(state["q"], state["k"], state["v"], state["cu_q"], state["cu_k"],
                                                  state["q_max"], state["lists"], block_q=case["block_q"],
                                                  block_k=case["block"], causal=case["causal"], return_lse=case["lse"])
        return dict(out=out[0], lse=out[1]) if case["lse"] else dict(out=out)
    return {"rotary": _plain_rotary, "means": _plain_means, "select": _plain_select, "attend": _plain_attend}[kind](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def _limits(case, ks, b, h, lq, i):
    n = ks[b * case["kv_heads"] + h] if case["per_head"] else ks[b]
    return max(0, n - lq + i + 1) if case["causal"] else n


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "rotary":
        n = case["rows"] * (case["heads"] + case["kv_heads"])
        return dict(bytes=2 * n * case["dim"] * size + 8 * case["rows"] * case["axes"] + 4 * case["rotary_dim"],
                    flops=3 * n * case["rotary_dim"])
    qs, ks = _lens(case)
    D, bk, hk = case["dim"], case["block"], case["kv_heads"]
    wide = 1 if case["per_head"] else hk
    blocks = sum(-(-n // bk) for n in ks) * wide
    if case["kind"] == "means":
        return dict(bytes=sum(ks) * wide * D * size + blocks * D * 4, flops=sum(ks) * wide * D)
    rows = sum(qs) * case["heads"]
    pairs = listed_keys = read_keys = tiles = 0
    for b, lq in enumerate(qs):
        nt = -(-lq // case["block_q"])
        tiles += nt * hk
        for h in range(hk):
            mine, most = 0, 0
            for i in range(nt):
                limit = _limits(case, ks, b, h, lq, i)
                pairs += -(-limit // bk)
                keys = min(limit, case["topk"] * bk)
                inside = min(case["block_q"], lq - i * case["block_q"])
                listed_keys += keys * inside * (case["heads"] // hk)
                mine, most = mine + keys, max(most, limit)
            read_keys += min(mine, most)
    if case["kind"] == "select":
        return dict(bytes=rows * D * size + blocks * D * 4 + 4 * tiles * case["topk"], flops=2 * D * pairs + rows * D)
    return dict(bytes=2 * rows * D * size + 2 * read_keys * D * size + 4 * tiles * case["topk"] + (4 * rows if case["lse"] else 0),
                flops=4 * D * listed_keys)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        P = case["rotary_dim"] // 2
        pos = s["pos"].view(case["rows"], -1).double()
        cols, at = [], 0
        for a, n in enumerate(s["axes"]):
            cols.append(pos[:, a:a + 1] * s["freqs"][None, at:at + n])
            at += n
        z = torch.polar(torch.full((case["rows"], P), s["scale"], dtype=torch.float64, device=DEV),
                        torch.cat(cols, dim=1) * (-1 if case["inverse"] else 1))[:, None]
        first = slice(0, 2 * P, 2) if case["interleaved"] else slice(0, P)
        second = slice(1, 2 * P, 2) if case["interleaved"] else slice(P, 2 * P)
        out = {}
        for name in ("q", "k"):
            if s[name] is not None:
                y = s[name].double().clone()
                w = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * z
                y[..., first], y[..., second] = w.real, w.imag
                out[name] = y
        return out
    qs, ks = _lens(case)
    D, bk, hk = case["dim"], case["block"], case["kv_heads"]
    if case["kind"] == "means":
        out = torch.zeros((sum(ks) // bk + len(ks),) + s["k"].shape[1:], dtype=torch.float64, device=DEV)
        c = 0
        for i, n in enumerate(ks):
            x = s["k"][c:c + n].double()
            full = n // bk
            out[c // bk + i:c // bk + i + full] = x[:full * bk].view(full, bk, *x.shape[1:]).mean(dim=1)
            if n % bk:
                out[c // bk + i + full] = x[full * bk:].mean(dim=0)
            c += n
        return out
    if case["kind"] == "select":
        return None
    bq, G = case["block_q"], case["heads"] // hk
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full((case["heads"], s["q"].shape[0]), -math.inf, dtype=torch.float64, device=DEV)
    cq = ck = 0
    kc = [0]
    for n in ks:
        kc.append(kc[-1] + n)
    for b, lq in enumerate(qs):
        nt = -(-lq // bq)
        tile0 = cq // bq + b
        for h in range(hk):
            seq = b * hk + h if case["per_head"] else b
            pick = lambda x: x[kc[seq]:kc[seq + 1]].double() if case["per_head"] else x[kc[seq]:kc[seq + 1], h].double()
            k, v, n = pick(s["k"]), pick(s["v"]), ks[seq]
            lists = s["lists"][tile0:tile0 + nt, h].long()
            allowed = torch.zeros(nt, -(-n // bk) + 1, dtype=torch.bool, device=DEV)
            allowed.scatter_(1, torch.where(lists < 0, allowed.shape[1] - 1, lists), True)
            allowed = allowed[:, :-1].repeat_interleave(bk, dim=1)[:, :n]
            if case["causal"]:
                limit = torch.arange(lq, device=DEV) + (n - lq + 1)
                allowed &= torch.arange(n, device=DEV)[None] < limit[:, None]
            for g in range(G):
                head = h * G + g
                x = s["q"][cq:cq + lq, head].double() @ k.t() * D ** -0.5
                x = x.masked_fill(~allowed.repeat_interleave(bq, dim=0)[:lq], -math.inf)
                some = ~torch.isinf(x.amax(dim=1))
                out[cq:cq + lq, head] = torch.where(some[:, None], torch.softmax(x, dim=1).nan_to_num(0) @ v, 0)
                lse[head, cq:cq + lq] = torch.logsumexp(x, dim=1)
        cq += lq
    return dict(out=out, lse=lse) if case["lse"] else dict(out=out)
