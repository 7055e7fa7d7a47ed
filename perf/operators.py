"""The cases that the operators around a shrinking, quantised KV cache are measured on, with their plain forms.

Six kinds of case, all with 32 query heads, 8 KV heads and head dimension 128 over a paged cache with 16-token pages:

* ``append4``      new K / V rows are quantised into a 4-bit cache, and the sequences are read back in 16 bits, as a prompt that
                   arrives in chunks needs its earlier rows
* ``anchor4``      layer 0 of a decode step over a 4-bit cache: dense attention, and the attention weight that every row drew
                   is added to the weight it has collected
* ``reuse4``       a reuse layer of a decode step over a 4-bit cache: attention over given index rows
* ``rope``         new rows with positions of their own on three axes (time, height, width) are normalised, rotated and
                   appended, queries rotated with them
* ``prompt_mass``  the attention weight that the tiles of a prompt gave to every earlier row
* ``evict``        the rows of least collected weight leave the caches of several layers

A 4-bit row is 128 codes in 64 bytes and eight fp16 parameters: the scales and the zeros of its four groups of 32 values.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

H, G, D, TILE, PAGE = 32, 8, 128, 32, 16
HG = H // G
SCALE = D ** -0.5
LOG2E = math.log2(math.e)
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
SEQUENCES_SEED = 91          # lengths belong to the case, not to the seed of its values
HEAD_MAP = [1, 0, 3, 3, 4, 6, 6, 2]
SECTIONS = (16, 24, 24)      # pairs of a head that turn with time, height and width


def listed():
    return [
        # a short chunk of four running conversations, behind some 450 rows each; launches and host time count
        {"name": "append4_chunk_4x61", "kind": "append4", "batch": 4, "start": 451, "tokens": 61, "dtype": "fp16"},
        # the rows of a whole long prompt
        {"name": "append4_prompt_32k", "kind": "append4", "batch": 1, "start": 0, "tokens": 32768, "dtype": "bf16"},
        # three short conversations
        {"name": "anchor4_3x777", "kind": "anchor4", "batch": 3, "context": 777, "ragged": False, "dtype": "fp16"},
        # a server's batch with contexts spread over a factor of sixteen
        {"name": "anchor4_ragged_16x32k", "kind": "anchor4", "batch": 16, "context": 32768, "ragged": True, "dtype": "bf16"},
        # one short conversation: the smallest budget
        {"name": "reuse4_1x500", "kind": "reuse4", "batch": 1, "context": 500, "ragged": False, "pct": 10, "dtype": "bf16"},
        # the benchmark's decode step, batch 64 at context 32768
        {"name": "reuse4_64x32k", "kind": "reuse4", "batch": 64, "context": 32768, "ragged": False, "pct": 10, "dtype": "fp16"},
        # the new token of every running sequence
        {"name": "rope_64x1", "kind": "rope", "batch": 64, "tokens": 1, "start": 511, "norm": False, "dtype": "fp16"},
        # the tokens of a long video, QK-norm model
        {"name": "rope_video_16k", "kind": "rope", "batch": 1, "tokens": 16384, "start": 45, "norm": True, "dtype": "bf16"},
        # a short prompt of odd length
        {"name": "prompt_mass_2x1001", "kind": "prompt_mass", "batch": 2, "length": 1001},
        # the benchmark's prompt
        {"name": "prompt_mass_32k", "kind": "prompt_mass", "batch": 1, "length": 32768},
        # a conversation that has just outgrown its share
        {"name": "evict_1x600", "kind": "evict", "batch": 1, "context": 600, "budget": 512, "recent": 64, "layers": 4,
         "ragged": False, "dtype": "fp16"},
        # long contexts halved
        {"name": "evict_4x32k", "kind": "evict", "batch": 4, "context": 32768, "budget": 16384, "recent": 1024, "layers": 8,
         "ragged": False, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: a kind, sizes spread over the logarithm of its range (odd ones among them), and the options."""
    kind = rng.choice(["append4", "anchor4", "anchor4", "reuse4", "reuse4", "rope", "prompt_mass", "evict"])
    dtype = rng.choice(["fp16", "bf16"])
    if kind == "append4":
        tokens = _log_int(rng, 1, 32768)
        return {"kind": kind, "batch": _log_int(rng, 1, max(1, min(64, 24576 // tokens))),
                "start": _log_int(rng, 1, 500) if tokens < 8192 else 0, "tokens": tokens, "dtype": dtype}
    if kind == "anchor4":
        context = _log_int(rng, 150, 131072)
        batch = _log_int(rng, 1, max(1, min(128, 2 ** 18 // context)))
        return {"kind": kind, "batch": batch, "context": context, "ragged": batch > 1 and rng.random() < 0.5, "dtype": dtype}
    if kind == "reuse4":
        context = _log_int(rng, 150, 131072)
        batch = _log_int(rng, 1, max(1, min(128, 2 ** 20 // context)))
        return {"kind": kind, "batch": batch, "context": context, "ragged": batch > 1 and rng.random() < 0.5,
                "pct": rng.choice([5, 10, 10, 20]), "dtype": dtype}
    if kind == "rope":
        tokens = _log_int(rng, 1, 16384)
        return {"kind": kind, "batch": _log_int(rng, 1, max(1, min(256, 16384 // tokens))), "tokens": tokens,
                "start": _log_int(rng, 1, 700), "norm": rng.random() < 0.5, "dtype": dtype}
    if kind == "prompt_mass":
        length = _log_int(rng, 33, 32768)
        return {"kind": kind, "batch": _log_int(rng, 1, max(1, min(16, (16384 // length) ** 2))), "length": length}
    context = _log_int(rng, 64, 65536)
    batch = _log_int(rng, 1, max(1, min(32, 2 ** 16 // context)))
    budget = max(1, int(context * rng.uniform(0.2, 0.95)))
    return {"kind": kind, "batch": batch, "context": context, "budget": budget, "recent": rng.randint(0, budget // 2),
            "layers": rng.randint(1, 8), "ragged": batch > 1 and rng.random() < 0.5, "dtype": dtype}


# ---- sizes -----------------------------------------------------------------------------------------------------------
def _lengths(case):
    """Cached rows of every sequence of the case."""
    batch, longest = case["batch"], case["context"]
    if not case["ragged"]:
        return [longest] * batch
    g = torch.Generator().manual_seed(SEQUENCES_SEED + batch + longest)
    lens = torch.randint(max(1, longest // 16), longest + 1, (batch,), generator=g).tolist()
    lens[batch // 2] = longest
    return lens


def _budget(case, n):
    """Keys that a reuse layer attends to in a sequence of n."""
    return n if n <= 128 else min(max(128, int(case["pct"] / 100 * n)), n) - TILE


# ---- 4-bit rows ------------------------------------------------------------------------------------------------------
def _codes(x):
    """Rows [..., 128] -> codes [..., 4, 32] and parameters fp16 [..., 8]: four scales, four zeros."""
    x = x.float().unflatten(-1, (4, 32))
    zero = x.amin(-1).half()
    scale = ((x.amax(-1) - zero.float()) / 15).half()
    c = (x.double() - zero.double()[..., None]) / scale.double()[..., None]     # in 64 bits: values next to a border
    c = torch.where(scale[..., None] > 0, c, torch.zeros_like(c))
    return c.round().clamp(0, 15).to(torch.uint8), torch.cat([scale, zero], -1)


# A row's nibbles, low one of a byte first.  K: four pieces of 16 bytes, piece q holds values 8q .. 8q+7 of every group.
# V: eight pieces of 8 bytes, piece r holds values 4r .. 4r+3 of every group.
def _pack(codes, pieces):
    n = codes.unflatten(-1, (pieces, 32 // pieces)).transpose(-3, -2).flatten(-3)
    return n[..., 0::2] | (n[..., 1::2] << 4)


def _unpack(packed, params, pieces):
    """Rows [..., 128] that packed codes [..., 64] and parameters [..., 8] stand for, in the parameters' type."""
    n = torch.stack([packed & 15, packed >> 4], -1).flatten(-2)
    n = n.unflatten(-1, (pieces, 4, 32 // pieces)).transpose(-3, -2).flatten(-2)
    return (n.to(params.dtype) * params[..., :4, None] + params[..., 4:, None]).flatten(-2)


K_PIECES, V_PIECES = 4, 8


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _unit_rms(x):
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6)


def _keys(shape, u, gen, dev):
    """Rows of N(0, 1) with 1 % of them moved along the direction `u` that the queries share; unit RMS."""
    k = torch.randn(*shape, generator=gen, device=dev) / D ** 0.5
    hot = torch.rand(*shape[:-1], 1, generator=gen, device=dev) < 0.01
    return _unit_rms(k + 2.5 * u * hot)


def _queries(shape, u, gen, dev):
    return _unit_rms(torch.randn(*shape, generator=gen, device=dev) / D ** 0.5 + 0.5 * u)


def _direction(gen, dev):
    u = torch.randn(D, generator=gen, device=dev)
    return u / u.norm()


def _table(lens, dev):
    """Block table [B, pages of the longest] over pages in a shuffled order."""
    per_seq = [-(-n // PAGE) for n in lens]
    order = torch.randperm(sum(per_seq), generator=torch.Generator().manual_seed(SEQUENCES_SEED)).to(torch.int32)
    table = torch.zeros(len(lens), max(per_seq), dtype=torch.int32)
    at = 0
    for b, n in enumerate(per_seq):
        table[b, :n] = order[at:at + n]
        at += n
    return table.to(dev), sum(per_seq)


def _cache4(pages, gen, dev, u):
    """Codes [pages, 16, G, 64] and parameters [pages, 16, G, 8] of K and of V; the parameters of a row's K and V lie beside
    each other."""
    k, v = (torch.empty(pages, PAGE, G, D // 2, dtype=torch.uint8, device=dev) for _ in range(2))
    params = torch.empty(pages, PAGE, G, 16, dtype=torch.float16, device=dev)
    kp, vp = params[..., :8], params[..., 8:]
    for s in range(0, pages, 4096):
        e = min(pages, s + 4096)
        for rows, cache, par, pieces in ((_keys((e - s, PAGE, G, D), u, gen, dev), k, kp, K_PIECES),
                                         (torch.randn(e - s, PAGE, G, D, generator=gen, device=dev), v, vp, V_PIECES)):
            codes, p = _codes(rows)
            cache[s:e], par[s:e] = _pack(codes, pieces), p
    return k, v, kp, vp


def _prepare_append4(case, gen, dev):
    dtype, B, T, start = DTYPES[case["dtype"]], case["batch"], case["tokens"], case["start"]
    lens = [start + T] * B
    table, pages = _table(lens, dev)
    u = _direction(gen, dev)
    k, v, kp, vp = _cache4(pages, gen, dev, u)
    new = torch.randn(B, T, 2 * G, D, generator=gen, device=dev)
    new[..., :G, :] = _keys((B, T, G, D), u, gen, dev)
    new = new.to(dtype)                                      # k and v as slices of one row per token
    return {"k": k, "v": v, "kp": kp, "vp": vp, "table": table, "k_new": new[:, :, :G], "v_new": new[:, :, G:],
            "start": torch.full((B,), start, dtype=torch.int32, device=dev),
            "lens": torch.tensor(lens, dtype=torch.int32, device=dev), "max_len": max(lens), "dtype": dtype}


def _prepare_decode4(case, gen, dev):
    lens = _lengths(case)
    table, pages = _table(lens, dev)
    u = _direction(gen, dev)
    k, v, kp, vp = _cache4(pages, gen, dev, u)
    B, longest = case["batch"], max(lens)
    state = {"k": k, "v": v, "kp": kp, "vp": vp, "table": table, "max_len": longest,
             "lens": torch.tensor(lens, dtype=torch.int32, device=dev), "mean_len": sum(lens) / B if case["ragged"] else None,
             "q": _queries((B, H, D), u, gen, dev).to(DTYPES[case["dtype"]])}
    if case["kind"] == "anchor4":
        weight = torch.rand(B, longest, generator=gen, device=dev) * 0.1
        state["mass"] = weight * (torch.arange(longest, device=dev)[None] < state["lens"][:, None])
        return state
    budgets = [_budget(case, n) for n in lens]
    score = torch.rand(B, G, longest, generator=gen, device=dev)
    score.masked_fill_(torch.arange(longest, device=dev) >= state["lens"][:, None, None], -1.0)
    rows = score.topk(max(budgets), dim=-1).indices
    counts = torch.tensor(budgets, dtype=torch.int32, device=dev)[:, None].expand(B, G).contiguous()
    rows.masked_fill_(torch.arange(max(budgets), device=dev) >= counts[..., None], longest)
    state["rows"] = rows.sort(-1).values.clamp_(max=longest - 1).to(torch.int32)
    state["counts"] = counts
    return state


def _prepare_rope(case, gen, dev):
    dtype, B, T, start = DTYPES[case["dtype"]], case["batch"], case["tokens"], case["start"]
    table, pages = _table([start + T] * B, dev)
    qkv = torch.randn(B, T, H + 2 * G, D, generator=gen, device=dev).to(dtype)
    cache = torch.randn(2, pages, PAGE, G, D, generator=gen, device=dev, dtype=dtype)
    gains = [(1 + 0.1 * torch.randn(D, generator=gen, device=dev)).to(dtype) for _ in range(2)] if case["norm"] else [None, None]
    # frames of 16 x 24 patches: the time moves on by one a frame, and every axis begins behind what came before
    t = torch.arange(T, device=dev)
    grid = torch.stack([t // 384, t // 24 % 16, t % 24])
    first = torch.randint(1, 60000, (1, B, 1), generator=gen, device=dev)
    axes = torch.repeat_interleave(torch.arange(3), torch.tensor(SECTIONS))
    return {"q": qkv[:, :, :H], "k_new": qkv[:, :, H:H + G], "v_new": qkv[:, :, H + G:], "k": cache[0], "v": cache[1],
            "table": table, "gains": gains, "start": torch.full((B,), start, dtype=torch.int32, device=dev),
            "positions": (first + grid[:, None]).to(torch.int32).contiguous(), "axes": axes.to(torch.int32).to(dev),
            "inv_freq": 1000000.0 ** (-torch.arange(0, D, 2, dtype=torch.float32, device=dev) / D)}


def _prepare_prompt_mass(case, gen, dev):
    B, L = case["batch"], case["length"]
    tiles, stride = -(-L // TILE), -(-L // 128) * 128
    pooled = torch.rand(B, G, tiles, stride, generator=gen, device=dev).pow_(4)
    at = torch.arange(stride, device=dev)
    # a tile's row holds scores of the keys before it only, and whatever was there before behind them
    pooled.masked_fill_(at[None] >= TILE * torch.arange(tiles, device=dev)[:, None], math.nan)
    return {"pooled": pooled, "mass": torch.rand(B, L, generator=gen, device=dev)}


def _prepare_evict(case, gen, dev):
    lens = _lengths(case)
    B, longest = case["batch"], max(lens)
    table, pages = _table(lens, dev)
    caches = torch.randn(case["layers"], 2, pages, PAGE, G, D, generator=gen, device=dev, dtype=DTYPES[case["dtype"]])
    mass = torch.rand(B, longest, generator=gen, device=dev).pow_(6)          # few rows draw most of the weight
    # rows in the order that an earlier eviction left
    order = torch.rand(B, longest, generator=gen, device=dev)
    lens_dev = torch.tensor(lens, dtype=torch.int32, device=dev)
    outside = torch.arange(longest, device=dev)[None] >= lens_dev[:, None]
    positions = order.masked_fill(outside, 2.0).argsort(-1).argsort(-1).to(torch.int32)
    return {"caches": caches, "table": table, "lens": lens_dev, "mass": mass.masked_fill(outside, 0.0),
            "positions": positions.masked_fill(outside, -1), "budget": case["budget"], "recent": case["recent"], "sinks": 4}


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    make = {"append4": _prepare_append4, "anchor4": _prepare_decode4, "reuse4": _prepare_decode4, "rope": _prepare_rope,
            "prompt_mass": _prepare_prompt_mass, "evict": _prepare_evict}[case["kind"]]
    return {"kind": case["kind"], **make(case, gen, dev)}


# ---- one pass, plain -------------------------------------------------------------------------------------------------
def _places(table, pos):
    """Physical page and slot of the rows `pos` [B, n]."""
    return table.long().gather(1, pos // PAGE), pos % PAGE


def _plain_append4(s):
    B, T = s["k_new"].shape[:2]
    pos = s["start"].long()[:, None] + torch.arange(T, device=s["k"].device)
    page, slot = _places(s["table"], pos)
    for new, cache, params, pieces in ((s["k_new"], s["k"], s["kp"], K_PIECES), (s["v_new"], s["v"], s["vp"], V_PIECES)):
        codes, par = _codes(new)
        cache[page, slot], params[page, slot] = _pack(codes, pieces), par
    page, slot = _places(s["table"], torch.arange(s["max_len"], device=s["k"].device).expand(B, -1))
    return [_unpack(cache[page, slot], params[page, slot].float(), pieces).to(s["dtype"])
            for cache, params, pieces in ((s["k"], s["kp"], K_PIECES), (s["v"], s["vp"], V_PIECES))]


def _attend(q, k, v, valid):
    """q [B, G, 4, D], k / v [B, G, n, D], valid [B, 1 or G, n] -> out [B, G, 4, D], probabilities [B, G, 4, n]."""
    x = torch.matmul(q, k.transpose(-1, -2)) * SCALE
    x = x.masked_fill(~valid[:, :, None], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    return torch.matmul(p, v), p


def _plain_anchor4(s):
    B = s["q"].shape[0]
    n = s["max_len"]
    page, slot = _places(s["table"], torch.arange(n, device=s["k"].device).expand(B, -1))
    k = _unpack(s["k"][page, slot], s["kp"][page, slot].float(), K_PIECES).transpose(1, 2)
    v = _unpack(s["v"][page, slot], s["vp"][page, slot].float(), V_PIECES).transpose(1, 2)
    valid = torch.arange(n, device=k.device) < s["lens"][:, None]
    out, p = _attend(s["q"].float().view(B, G, HG, D), k, v, valid[:, None])
    return out.reshape(B, H, D).to(s["q"].dtype), s["mass"] + p.sum((1, 2))


def _plain_reuse4(s):
    B = s["q"].shape[0]
    rows = s["rows"].long()[:, HEAD_MAP]                                        # [B, G, n]
    counts = s["counts"][:, HEAD_MAP]
    page = s["table"].long()[:, None].expand(-1, G, -1).gather(2, rows // PAGE)
    slot, head = rows % PAGE, torch.arange(G, device=rows.device)[None, :, None]
    k = _unpack(s["k"][page, slot, head], s["kp"][page, slot, head].float(), K_PIECES)
    v = _unpack(s["v"][page, slot, head], s["vp"][page, slot, head].float(), V_PIECES)
    valid = torch.arange(rows.shape[-1], device=rows.device) < counts[..., None]
    out, _ = _attend(s["q"].float().view(B, G, HG, D), k, v, valid)
    return out.reshape(B, H, D).to(s["q"].dtype)


def _plain_rope(s):
    T = s["k_new"].shape[1]
    angle = (s["positions"].double()[s["axes"].long()] * s["inv_freq"].double()[:, None, None]).permute(1, 2, 0)[:, :, None]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()               # [B, T, 1, 64]

    def turned(x, gain):
        x = x.float()
        if gain is not None:
            x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * gain.float()
        lo, hi = x[..., :D // 2], x[..., D // 2:]
        return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1).to(s["k"].dtype)

    page, slot = _places(s["table"], s["start"].long()[:, None] + torch.arange(T, device=cos.device))
    s["k"][page, slot], s["v"][page, slot] = turned(s["k_new"], s["gains"][1]), s["v_new"]
    return turned(s["q"], s["gains"][0]), s["k"], s["v"]


def _plain_prompt_mass(s):
    pooled, L = s["pooled"], s["mass"].shape[1]
    tiles = pooled.shape[2]
    seen = torch.arange(L, device=pooled.device)[None] < TILE * torch.arange(tiles, device=pooled.device)[:, None]
    x = torch.where(seen, pooled[..., :L], torch.zeros((), device=pooled.device))
    return (s["mass"] + x.double().sum((1, 2))).float()


def _evicted(s):
    """(sequence, source row), (sequence, target row) of the moves, and the rows that are left per sequence."""
    at = torch.arange(s["mass"].shape[1], device=s["mass"].device)
    lens, pos, budget = s["lens"].long(), s["positions"], s["budget"]
    inside = at < lens[:, None]
    newest = pos.masked_fill(~inside, -1).amax(-1, keepdim=True)
    key = s["mass"].masked_fill((pos < s["sinks"]) | (pos > newest - s["recent"]), math.inf).masked_fill(~inside, -1.0)
    best = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :budget]
    kept = torch.zeros_like(inside).scatter_(1, best, True) & inside
    return (kept & (at >= budget)).nonzero(as_tuple=True), (inside & ~kept & (at < budget)).nonzero(as_tuple=True), \
        lens.clamp(max=budget)


def _plain_evict(s):
    (b, source), (b2, target), left = _evicted(s)
    kept = left[:, None] > torch.arange(s["mass"].shape[1], device=left.device)
    mass, positions, caches, table = s["mass"].clone(), s["positions"].clone(), s["caches"], s["table"].long()
    mass[b2, target], positions[b2, target] = mass[b, source], positions[b, source]
    caches[:, :, table[b2, target // PAGE], target % PAGE] = caches[:, :, table[b, source // PAGE], source % PAGE]
    return left.to(torch.int32), mass.masked_fill(~kept, 0.0), positions.masked_fill(~kept, -1), caches


PLAIN = {"append4": _plain_append4, "anchor4": _plain_anchor4, "reuse4": _plain_reuse4, "rope": _plain_rope,
         "prompt_mass": _plain_prompt_mass, "evict": _plain_evict}


# ---- one pass, through the library -------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _strategy():
    from kascade_b200 import EfficientKascadeStrategy
    return EfficientKascadeStrategy([0], "synthetic/model", k=10, tile_size=TILE, head_mapping=[list(range(G)), HEAD_MAP],
                                    register=False)


def _own(s):
    strategy, kind = _strategy(), s["kind"]
    if kind == "append4":
        strategy.append_kv(s["k_new"], s["v_new"], s["k"], s["v"], s["table"], s["start"], k_scale=s["kp"], v_scale=s["vp"])
        return strategy.read_kv(s["k"], s["v"], s["table"], s["lens"], s["max_len"], k_scale=s["kp"], v_scale=s["vp"],
                                dtype=s["dtype"])
    if kind == "anchor4":
        mass = s["mass"].clone()
        out = strategy.paged_decode_forward(0, s["q"], s["k"], s["v"], s["table"], s["lens"], SCALE, s["max_len"], s["kp"], s["vp"],
                                            mean_seq_len=s["mean_len"], attention_mass=mass)
        return out, mass
    if kind == "reuse4":
        return strategy.paged_decode_forward(1, s["q"], s["k"], s["v"], s["table"], s["lens"], SCALE, s["max_len"], s["kp"],
                                             s["vp"], mean_seq_len=s["mean_len"], index_rows=(s["rows"], s["counts"]))
    if kind == "rope":
        q = strategy.append_kv(s["k_new"], s["v_new"], s["k"], s["v"], s["table"], s["start"], query=s["q"],
                               q_norm_weight=s["gains"][0], k_norm_weight=s["gains"][1], norm_eps=EPS, inv_freq=s["inv_freq"],
                               positions=s["positions"], rope_axes=s["axes"])
        return q, s["k"], s["v"]
    if kind == "prompt_mass":
        return strategy.prompt_mass(s["pooled"], s["mass"])
    caches = [(layer[0], layer[1]) for layer in s["caches"]]
    return *strategy.evict_kv(caches, s["table"], s["lens"], s["mass"], s["budget"], recent=s["recent"], sinks=s["sinks"],
                              token_positions=s["positions"]), s["caches"]


def run(state):
    return _own(state) if own else PLAIN[state["kind"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    row4 = D // 2 + 16                                       # codes and parameters of a row
    if kind == "append4":
        new, all_rows = case["batch"] * case["tokens"], case["batch"] * (case["start"] + case["tokens"])
        return {"bytes": 2.0 * G * (new * (2 * D + row4) + all_rows * (row4 + 2 * D)), "flops": 2.0 * G * D * (4 * new + 2 * all_rows)}
    if kind == "anchor4":
        rows, B = sum(_lengths(case)), case["batch"]
        return {"bytes": rows * (2.0 * G * row4 + 8) + 4.0 * B * H * D, "flops": 4.0 * H * D * rows}
    if kind == "reuse4":
        rows, B = sum(_budget(case, n) for n in _lengths(case)), case["batch"]
        return {"bytes": rows * G * (2.0 * row4 + 4) + 4.0 * B * H * D, "flops": 4.0 * H * D * rows}
    if kind == "rope":
        tokens = case["batch"] * case["tokens"]
        return {"bytes": tokens * ((H + 2 * G) * D * 4.0 + 12), "flops": tokens * (H + G) * D * (7.0 if case["norm"] else 3.0)}
    if kind == "prompt_mass":
        L = case["length"]
        scores = sum(min(t * TILE, L) for t in range(-(-L // TILE)))
        return {"bytes": case["batch"] * 4.0 * (G * scores + 2 * L), "flops": case["batch"] * 1.0 * G * scores}
    moved = sum(max(0, n - case["budget"]) * case["budget"] / n for n in _lengths(case))     # as many as kept rows lie behind the budget
    return {"bytes": moved * case["layers"] * 2 * G * 2 * D * 2.0 + 16.0 * sum(_lengths(case)), "flops": 1.0 * sum(_lengths(case))}


# ---- the same in 64 bits ---------------------------------------------------------------------------------------------
def _rows4(cache, params, pieces, page, slot, head=None):
    """Values of 4-bit rows in 64 bits, written from the layout of a row: nibble n of it is value `order[n]`."""
    order = [32 * g + (32 // pieces) * p + i for p in range(pieces) for g in range(4) for i in range(32 // pieces)]
    codes, par = (cache[page, slot], params[page, slot]) if head is None else (cache[page, slot, head], params[page, slot, head])
    out = torch.empty(*codes.shape[:-1], D, dtype=torch.float64, device=codes.device)
    out[..., order[0::2]] = (codes & 15).double()
    out[..., order[1::2]] = (codes >> 4).double()
    return out * par[..., :4].double().repeat_interleave(32, -1) + par[..., 4:].double().repeat_interleave(32, -1)


def _exact_append4(case, s):
    start, T = case["start"], case["tokens"]
    outs = []
    for cache, params, pieces, new in ((s["k"], s["kp"], K_PIECES, s["k_new"]), (s["v"], s["vp"], V_PIECES, s["v_new"])):
        x = new.double()
        least = torch.stack([x[..., 32 * g:32 * g + 32].amin(-1) for g in range(4)], -1).half().double()
        most = torch.stack([x[..., 32 * g:32 * g + 32].amax(-1) for g in range(4)], -1)
        step = ((most - least).float() / 15).half().double()                 # the scale is a quotient in 32 bits, kept in fp16
        least, step = (v.repeat_interleave(32, -1) for v in (least, step))
        new_rows = torch.where(step > 0, ((x - least) / step.clamp(min=1e-300)).round().clamp(0, 15), step) * step + least
        at = torch.arange(start, device=x.device).expand(case["batch"], -1)
        page, slot = _places(s["table"], at)
        outs.append(torch.cat([_rows4(cache, params, pieces, page, slot), new_rows], 1))
        assert outs[-1].shape[1] == start + T
    return outs


def _exact_decode4(case, s):
    outs, masses = [], []
    for b, n in enumerate(_lengths(case)):
        q = s["q"][b].double().view(G, HG, D)
        if case["kind"] == "anchor4":
            at = torch.arange(n, device=q.device)[None].expand(G, -1)
        else:
            at = s["rows"][b].long()[HEAD_MAP, :_budget(case, n)]
        page, slot, head = s["table"][b].long()[at // PAGE], at % PAGE, torch.arange(G, device=q.device)[:, None]
        p = torch.softmax(q @ _rows4(s["k"], s["kp"], K_PIECES, page, slot, head).transpose(1, 2) * SCALE, -1)
        outs.append((p @ _rows4(s["v"], s["vp"], V_PIECES, page, slot, head)).reshape(H, D))
        if case["kind"] == "anchor4":
            masses.append(s["mass"][b].double().index_add(0, at[0], p.sum((0, 1))))
    return (torch.stack(outs), torch.stack(masses)) if masses else torch.stack(outs)


def _exact_rope(case, s):
    at = s["positions"].double().permute(1, 2, 0)[..., s["axes"].long()] * s["inv_freq"].double()
    turn = torch.polar(torch.ones_like(at), at)[:, :, None]

    def turned(x, gain):
        x = x.double()
        if gain is not None:
            x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * gain.double()
        z = torch.complex(x[..., :D // 2].contiguous(), x[..., D // 2:].contiguous()) * turn
        return torch.cat([z.real, z.imag], -1)

    pos = s["start"].long()[:, None] + torch.arange(case["tokens"], device=at.device)
    page, slot = _places(s["table"], pos)
    k, v = s["k"].double(), s["v"].double()
    k[page, slot], v[page, slot] = turned(s["k_new"], s["gains"][1]), s["v_new"].double()
    return turned(s["q"], s["gains"][0]), k, v


def _exact_prompt_mass(case, s):
    mass, L = s["mass"].double(), case["length"]
    for t in range(1, -(-L // TILE)):
        n = min(t * TILE, L)
        mass[:, :n] += s["pooled"][:, :, t, :n].double().sum(1)
    return mass


def _exact_evict(case, s):
    mass, positions, caches = s["mass"].double(), s["positions"].clone(), s["caches"].double()
    left = []
    for b, n in enumerate(_lengths(case)):
        budget, pos = case["budget"], s["positions"][b, :n]
        left.append(min(n, budget))
        if n > budget:
            key = mass[b, :n].clone()
            key[(pos < s["sinks"]) | (pos > pos.max() - case["recent"])] = math.inf
            kept = torch.sort(key, descending=True, stable=True).indices[:budget].sort().values
            stays = torch.zeros(n, dtype=torch.bool, device=key.device)
            stays[kept] = True
            source, target = kept[kept >= budget], (~stays[:budget]).nonzero()[:, 0]
            pages = s["table"][b].long()
            caches[:, :, pages[target // PAGE], target % PAGE] = caches[:, :, pages[source // PAGE], source % PAGE]
            mass[b, target], positions[b, target] = mass[b, source], positions[b, source]
        mass[b, left[-1]:], positions[b, left[-1]:] = 0.0, -1
    return torch.tensor(left, dtype=torch.int32, device=mass.device), mass, positions, caches


def exact(case, seed):
    """What `run` returns for these inputs, from the definitions in 64 bits."""
    state = prepare(case, seed)
    return {"append4": _exact_append4, "anchor4": _exact_decode4, "reuse4": _exact_decode4, "rope": _exact_rope,
            "prompt_mass": _exact_prompt_mass, "evict": _exact_evict}[case["kind"]](case, state)
