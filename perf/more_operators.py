"""The operators of a cache held in 8 bits: their calls and their plain forms.

The cache: codes ``[slots, heads, D]`` of 8-bit floats and fp32 scales
``[slots / B, heads]``, one for each block of B slots and head, for K and for
V; a value is its code times its block's scale.

``listed()`` names the cases, ``draw(rng)`` gives another of the same ranges.
Lengths, layouts, dropped spans and trees follow from the case (``events``);
slots, K/V, queries and sinks are drawn from the seed given to ``prepare``.

Kinds:

* ``write``  new K/V rows rotated, rounded to 8 bits and stored at their slots,
             q rotated along (``kv8.append_kv8``);
* ``move``   kept rows of all layers moved to fresh slots and new positions
             (``kv8.reposition_kv8_layers``);
* ``read``   attention of one layer's new tokens over the cache
             (``kv8.attention_kv8``).

``own`` false computes each from its definition with elementary torch
operations; true calls the framework.
"""

import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FORMATS = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
LEAST_SCALE = 2.0 ** -100
POSITIONS = 40960


def listed():
    return [
        # one chat of ~4k tokens decodes a token of a GPT-OSS-shaped layer (64 q /
        # 8 KV heads x 64): latency and the launch
        dict(name="write-decode-1", kind="write", requests=1, len_lo=4101, len_hi=4101, new_lo=1, new_hi=1, q_heads=64,
             heads=8, head_dim=64, rotary=64, neox=True, dtype="bf16", format="e4m3", page=16, block=16, events=1),
        # 64 requests decode a token each (32 / 8 heads x 128)
        dict(name="write-decode-64", kind="write", requests=64, len_lo=100, len_hi=30000, new_lo=1, new_hi=1,
             q_heads=32, heads=8, head_dim=128, rotary=128, neox=True, dtype="bf16", format="e4m3", page=16, block=16,
             events=2),
        # drafted tokens and short extends of a partial-rotary fp16 model with
        # interleaved pairs, blocks of 4 tokens
        dict(name="write-ragged-fp16", kind="write", requests=24, len_lo=50, len_hi=20000, new_lo=1, new_hi=333,
             q_heads=16, heads=4, head_dim=128, rotary=64, neox=False, dtype="fp16", format="e5m2", page=16, block=4,
             events=3),
        # a whole 32k-token GPT-OSS prompt in one forward
        dict(name="write-prefill-32k", kind="write", requests=1, len_lo=0, len_hi=0, new_lo=32768, new_hi=32768,
             q_heads=64, heads=8, head_dim=64, rotary=64, neox=True, dtype="bf16", format="e4m3", page=16, block=16,
             events=4),
        # the smallest turn end: a 4k-token chat of a two-layer model
        dict(name="move-tiny-4k", kind="move", layers=2, heads=2, head_dim=64, rotary=64, neox=True, format="e4m3",
             requests=1, n_lo=4096, n_hi=4096, spans=3, fraction=0.25, page=1, block=1, events=5),
        # one 32k-token GPT-OSS-120B agent request (36 layers, 8 KV heads x 64)
        # drops 12 tool results, a scale for each token
        dict(name="move-gpt-oss-32k", kind="move", layers=36, heads=8, head_dim=64, rotary=64, neox=True,
             format="e4m3", requests=1, n_lo=32768, n_hi=32768, spans=12, fraction=0.40, page=1, block=1, events=6),
        # page-16 copy-on-write of two Llama-3-8B requests (32 layers, 8 KV heads x 128)
        dict(name="move-paged-llama3-2", kind="move", layers=32, heads=8, head_dim=128, rotary=128, neox=True,
             format="e4m3", requests=2, n_lo=9000, n_hi=14000, spans=4, fraction=0.25, page=16, block=16, events=7),
        # one fp16 request of 4k keys decodes a token: latency
        dict(name="read-fp16-1", kind="read", requests=1, q_heads=16, heads=4, head_dim=128, dtype="fp16",
             format="e5m2", sinks=False, window=0, first=0, page=1, block=1, tree=False, len_lo=4096, len_hi=4096,
             new_lo=1, new_hi=1, events=8),
        # 32 GPT-OSS requests holding ~20k keys each decode a token: a full layer
        dict(name="read-gpt-oss-32x20k", kind="read", requests=32, q_heads=64, heads=8, head_dim=64, dtype="bf16",
             format="e4m3", sinks=True, window=0, first=0, page=1, block=1, tree=False, len_lo=19000, len_hi=20500,
             new_lo=1, new_hi=1, events=9),
        # a sliding-window layer that keeps its first 4 keys, trees of up to 8
        dict(name="read-window-32x8", kind="read", requests=32, q_heads=64, heads=8, head_dim=64, dtype="bf16",
             format="e4m3", sinks=True, window=128, first=4, page=16, block=16, tree=True, len_lo=100, len_hi=20500,
             new_lo=1, new_hi=8, events=10),
        # 12 ragged Llama-3-8B requests (32 / 8 x 128) on pages of 16, ragged trees
        dict(name="read-llama3-12-paged", kind="read", requests=12, q_heads=32, heads=8, head_dim=128, dtype="bf16",
             format="e4m3", sinks=False, window=0, first=0, page=16, block=16, tree=True, len_lo=2000, len_hi=20000,
             new_lo=5, new_hi=32, events=11),
        # a chunk of 512 new tokens over 16k GPT-OSS keys: bound by the arithmetic
        dict(name="read-extend-512", kind="read", requests=1, q_heads=64, heads=8, head_dim=64, dtype="bf16",
             format="e4m3", sinks=True, window=0, first=0, page=16, block=16, tree=False, len_lo=16000, len_hi=16000,
             new_lo=512, new_hi=512, events=12),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(("write", "move", "read", "read"))
    page = rng.choice((1, 16, 16, 64))
    c = dict(kind=kind, events=rng.randrange(1 << 20), page=page,
             block=1 if page == 1 else rng.choice((1, 4, 16, 16, page)), format=rng.choice(("e4m3", "e4m3", "e5m2")))
    if kind == "move":
        head_dim = rng.choice((64, 64, 80, 96, 128))
        requests = rng.randint(1, 4)
        c.update(layers=_log_int(rng, 1, 36), heads=rng.choice((2, 4, 8)), head_dim=head_dim,
                 rotary=rng.choice((head_dim, head_dim, head_dim // 2)), neox=rng.random() < 0.7, requests=requests,
                 spans=rng.randint(1, 12), fraction=round(rng.uniform(0.1, 0.5), 3))
        c["n_hi"] = _log_int(rng, 1000, 32768 // requests)
        c["n_lo"] = max(700, c["n_hi"] // rng.randint(1, 4))
        c["n_hi"] = max(c["n_hi"], c["n_lo"])
        # no larger than the 32k request of 36 layers
        c["layers"] = max(1, min(c["layers"], 36 * 32768 * 512 // (c["heads"] * head_dim * c["n_hi"] * requests)))
        return c
    heads = rng.choice((1, 2, 4, 8))
    if kind == "write":
        head_dim = rng.choice((64, 64, 80, 96, 128, 128))
        new = _log_int(rng, 1, 8192)
        hi = _log_int(rng, 1, 30000)
        c.update(requests=_log_int(rng, 1, 64), q_heads=heads * rng.choice((1, 2, 4, 7, 8)), heads=heads,
                 head_dim=head_dim, rotary=rng.choice((head_dim, head_dim, head_dim // 2, 0)), neox=rng.random() < 0.7,
                 dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), len_lo=hi // rng.randint(1, 32), len_hi=hi,
                 new_lo=max(1, new // rng.randint(1, 32)), new_hi=new)
        # no larger than the 32k prompt
        row = (c["q_heads"] + 2 * heads) * head_dim * DTYPES[c["dtype"]].itemsize
        c["requests"] = max(1, min(c["requests"], 32768 * 80 * 64 * 2 // (row * new), 32768 * 32 // (hi + new)))
        return c
    head_dim = rng.choice((64, 64, 64, 80, 96, 128, 128))
    group = rng.choice((1, 4, 7, 8, 8))
    new = rng.choice((1, 1, _log_int(rng, 1, 64), _log_int(rng, 1, 64), _log_int(rng, 1, 600)))
    hi = _log_int(rng, 80, 32000)
    c.update(requests=_log_int(rng, 1, 48), q_heads=heads * group, heads=heads, head_dim=head_dim,
             dtype=rng.choice(("bf16", "bf16", "fp16")), sinks=rng.random() < 0.5, window=rng.choice((0, 0, 128)),
             tree=new <= 128 and rng.random() < 0.5, len_lo=max(1, hi // rng.randint(1, 8)), len_hi=hi,
             new_lo=max(1, new // rng.randint(1, 8)), new_hi=new)
    c["first"] = rng.choice((0, 4, 17)) if c["window"] else 0
    # neither more K/V than 32 x 20k keys of 8 x 64 nor more products than
    # 512 tokens over 16k keys
    keys = (min(hi, 400) if c["window"] else hi) + new
    kv = 32 * 19750 * 8 * 64 // ((hi + new) * heads * head_dim)
    mul = 512 * 16256 * 64 * 64 // (keys * new * c["q_heads"] * head_dim)
    c["requests"] = max(1, min(c["requests"], kv, mul))
    return c


# ---------------------------------------------------------------------------
# What follows from the case alone: lengths, trees, dropped spans.


def _lengths(c):
    """Per request: keys before the call, and new tokens."""
    rng = random.Random(c["events"])
    old = [rng.randint(c["len_lo"], c["len_hi"]) for _ in range(c["requests"])]
    return old, [rng.randint(c["new_lo"], c["new_hi"]) for _ in range(c["requests"])]


def _parents(c):
    """One draft tree per request: node 0 hangs on the cache (-1), the others
    on an earlier node, mostly a recent one; without trees each on the last."""
    rng = random.Random(c["events"] + 1)
    if not c["tree"]:
        return [list(range(-1, n - 1)) for n in _lengths(c)[1]]
    return [[-1] + [max(0, i - 1 - int(rng.expovariate(0.7))) for i in range(1, n)] for n in _lengths(c)[1]]


def _depths(parents):
    depth = []
    for p in parents:
        depth.append(0 if p < 0 else depth[p] + 1)
    return np.array(depth)


def _ancestors(parents, limit):
    """bool [nodes, nodes]: itself and its ancestors at most ``limit`` levels up."""
    n = len(parents)
    seen = np.zeros((n, n), dtype=bool)
    for i in range(n):
        a, up = i, 0
        while a >= 0 and up <= limit:
            seen[i, a] = True
            a, up = parents[a], up + 1
    return seen


def _pack(seen, words):
    bits = np.zeros((len(seen), 64 * words), dtype=np.uint8)
    bits[:, : seen.shape[1]] = seen
    return np.packbits(bits, axis=1, bitorder="little").view(np.int64)


def _kept(c):
    """Per request: its length and the raw indices that its dropped spans leave."""
    rng = random.Random(c["events"])
    out = []
    for _ in range(c["requests"]):
        n = rng.randint(c["n_lo"], c["n_hi"])
        keep = np.ones(n, dtype=bool)
        size = max(1, int(n * c["fraction"]) // c["spans"])
        for _ in range(c["spans"]):
            at = rng.randint(n // 20, n - size)
            keep[at: at + size] = False
        out.append((n, np.flatnonzero(keep)))
    return out


def _moves(c):
    """Per request: pages, then of its moved tokens the raw index and the rank
    (their new position).  Pages before the first dropped token stay."""
    P, out = c["page"], []
    for n, raw in _kept(c):
        rank = np.arange(len(raw))
        dropped = raw != rank
        first = int(np.argmax(dropped)) // P * P if dropped.any() else len(raw)
        out.append((-(-n // P), raw[first:], rank[first:]))
    return out


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _dev(a, dtype):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).to("cuda")


def _rope_table(rotary):
    inv = 10000.0 ** (-np.arange(0, rotary, 2) / rotary)
    angle = np.arange(POSITIONS)[:, None] * inv
    return _dev(np.concatenate((np.cos(angle), np.sin(angle)), 1), np.float32)


def _cache(c, g, *shape):
    """Codes [..., slots, heads, D] and scales [..., slots / B, heads] of normal values."""
    F = LARGEST[c["format"]]
    codes = torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)
    codes = codes.mul_(F / 5).clamp_(-F, F).to(FORMATS[c["format"]])
    power = torch.randint(0, 3, (*shape[:-3], shape[-3] // c["block"], shape[-2]), generator=g, device="cuda")
    return codes, torch.exp2(power - (8.0 if c["format"] == "e4m3" else 15.0))


# ---------------------------------------------------------------------------
# Inputs.


def prepare(case, seed):
    return {"write": _prepare_write, "move": _prepare_move, "read": _prepare_read}[case["kind"]](case, seed)


def _prepare_write(c, seed):
    g, dt, d, hk, hq, P = _gen(seed), DTYPES[c["dtype"]], c["head_dim"], c["heads"], c["q_heads"], c["page"]
    old, new = _lengths(c)
    pages = [-(-(o + n) // P) for o, n in zip(old, new)]
    ids = np.random.default_rng(seed).permutation(sum(pages) + 1)
    ends = np.concatenate(([0], np.cumsum(pages)))
    slots, positions = [], []
    for b, (o, n) in enumerate(zip(old, new)):
        rank = np.arange(o, o + n)
        slots.append(ids[ends[b] + rank // P] * P + rank % P)
        positions.append(rank)
    total = sum(new)
    qkv = torch.randn((total, (hq + 2 * hk) * d), generator=g, device="cuda").to(dt)
    # keys of real models have a few dims that are larger than the others
    wide = 1 + 3 * (torch.rand(hk * d, generator=g, device="cuda") < 0.03).to(dt)
    qkv[:, hq * d: (hq + hk) * d] *= wide
    k, k_scales = _cache(c, g, (sum(pages) + 1) * P, hk, d)
    v, v_scales = _cache(c, g, (sum(pages) + 1) * P, hk, d)
    return dict(
        case=c, qkv=qkv, slots=_dev(np.concatenate(slots), np.int64), positions=_dev(np.concatenate(positions), np.int64),
        table=_rope_table(c["rotary"]) if c["rotary"] else None, k=k, v=v, k_scales=k_scales, v_scales=v_scales,
        q_out=torch.empty((total, hq, d), dtype=dt, device="cuda") if c["rotary"] else None,
    )


def _prepare_move(c, seed):
    g, P = _gen(seed), c["page"]
    moves = _moves(c)
    fresh = [-(-len(rank) // P) for _, _, rank in moves]
    total = sum(m[0] for m in moves) + sum(fresh)
    ids = np.random.default_rng(seed).permutation(total + 1)
    src, dst, pairs, at = [], [], [], 0
    for (pages, raw, rank), n in zip(moves, fresh):
        own_pages, new_pages = ids[at: at + pages], ids[at + pages: at + pages + n]
        at += pages + n
        first = rank[0] if len(rank) else 0
        src.append(own_pages[raw // P] * P + raw % P)
        dst.append(new_pages[(rank - first) // P] * P + rank % P)
        pairs.append(np.stack((raw, rank), 1))
    k, k_scales = _cache(c, g, c["layers"], (total + 1) * P, c["heads"], c["head_dim"])
    v, v_scales = _cache(c, g, c["layers"], (total + 1) * P, c["heads"], c["head_dim"])
    pointers = [_dev([layer.data_ptr() for layer in t], np.int64) for t in (k, v, k_scales, v_scales)]
    return dict(case=c, k=k, v=v, k_scales=k_scales, v_scales=v_scales, pointers=pointers,
                src=_dev(np.concatenate(src), np.int32), dst=_dev(np.concatenate(dst), np.int32),
                pairs=_dev(np.concatenate(pairs), np.int32), table=_rope_table(c["rotary"]))


def _prepare_read(c, seed):
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    old, new = _lengths(c)
    B, P, W, d, hk = len(old), c["page"], c["window"], c["head_dim"], c["heads"]
    seq = [o + n for o, n in zip(old, new)]
    pages = [-(-s // P) for s in seq]
    free = np.random.default_rng(seed).permutation(sum(pages) + 1)
    ends = np.concatenate(([0], np.cumsum(pages)))
    tables = np.full((B, max(pages)), -1, dtype=np.int32)
    for b in range(B):
        tables[b, : pages[b]] = free[ends[b]: ends[b + 1]]
    indices = _dev(free[: sum(seq)] if P == 1 else tables, np.int32)
    trees = _parents(c)
    words = (c["new_hi"] + 63) // 64
    limit = W if W else max(new)
    masked = c["tree"] or W
    mask = np.concatenate([_pack(_ancestors(p, limit), words) for p in trees]) if masked else None
    starts = np.concatenate([np.clip(o + _depths(p) - W, 0, o) for o, p in zip(old, trees)]) if W else None
    k, k_scales = _cache(c, g, (sum(pages) + 1) * P, hk, d)
    v, v_scales = _cache(c, g, (sum(pages) + 1) * P, hk, d)
    total = sum(new)
    s = dict(
        case=c, q=torch.randn((total, c["q_heads"], d), generator=g, device="cuda", dtype=dt), k=k, v=v,
        k_scales=k_scales, v_scales=v_scales, qo_indptr=_dev(np.concatenate(([0], np.cumsum(new))), np.int32),
        kv_indptr=_dev(np.concatenate(([0], np.cumsum(seq))), np.int32), indices=indices,
        mask=None if mask is None else _dev(mask, np.int64), starts=None if starts is None else _dev(starts, np.int32),
        sinks=torch.randn(c["q_heads"], generator=g, device="cuda") if c["sinks"] else None,
        out=torch.empty((total, c["q_heads"], d), dtype=dt, device="cuda"), tables=_dev(tables, np.int64),
        scale=d ** -0.5, max_new=max(new),
        max_len=min(max(seq), c["first"] + W + max(new) + 1) if W else max(seq),
        # the batch as a rectangle, for the plain form
        token=_dev(np.concatenate([np.arange(n) for n in new]), np.int64),
        request=_dev(np.repeat(np.arange(B), new), np.int64), old=_dev(old, np.int64), new=_dev(new, np.int64),
        low=_dev([max(0, o - W - 1) if W else 0 for o in old], np.int64),
    )
    if own:
        from akv_amd import kv8

        need = kv8.attention_kv8_workspace_bytes(total, B, c["q_heads"], hk, d, s["max_len"], s["max_new"])
        s["workspace"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    return s


# ---------------------------------------------------------------------------
# One pass.


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"write": _own_write, "move": _own_move, "read": _own_read}[kind](state)
    return {"write": _plain_write, "move": _plain_move, "read": _plain_read}[kind](state)


def _cache_outputs(s):
    return dict(k=s["k"], v=s["v"], k_scales=s["k_scales"], v_scales=s["v_scales"], q=s.get("q_out"))


def _rows(s):
    """q, k and v of the fused projection."""
    c = s["case"]
    return s["qkv"].view(len(s["qkv"]), -1, c["head_dim"]).split((c["q_heads"], c["heads"], c["heads"]), 1)


def _own_write(s):
    from akv_amd import kv8

    c = s["case"]
    q, k, v = _rows(s)
    turned = dict(positions=s["positions"], cos_sin_cache=s["table"], rotary_dim=c["rotary"], is_neox_style=c["neox"],
                  q=q, q_out=s["q_out"]) if c["rotary"] else {}
    kv8.append_kv8(k, v, s["slots"], s["k"], s["v"], s["k_scales"], s["v_scales"], scale_block=c["block"], **turned)
    return _cache_outputs(s)


def _own_move(s):
    from akv_amd import kv8

    c = s["case"]
    kv8.reposition_kv8_layers(*s["pointers"], s["k"][0], s["v"][0], s["k_scales"][0], s["v_scales"][0], s["src"], s["dst"],
                              s["pairs"], s["table"], scale_block=c["block"], is_neox_style=c["neox"],
                              rotary_dim=c["rotary"])
    return _cache_outputs(s)


def _own_read(s):
    from akv_amd import kv8

    c = s["case"]
    kv8.attention_kv8(
        s["q"], s["k"], s["v"], s["k_scales"], s["v_scales"], s["qo_indptr"], s["kv_indptr"], s["indices"], s["out"],
        scale=s["scale"], max_len=s["max_len"], max_new=s["max_new"], page_size=c["page"], scale_block=c["block"],
        tree_mask=s["mask"], key_starts=s["starts"], first_keys=c["first"], sinks=s["sinks"], workspace=s["workspace"])
    return s["out"]


def _turn(c, x, cos, sin):
    """x [..., heads, D], its first ``rotary`` dims turned by cos / sin [..., 1, rotary / 2]."""
    r = c["rotary"]
    rot, rest = x[..., :r], x[..., r:]
    if c["neox"]:
        a, b = rot[..., : r // 2], rot[..., r // 2:]
        rot = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = rot[..., ::2], rot[..., 1::2]
        rot = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((rot, rest), -1)


def _store(c, codes, scales, rows, slots):
    """Rows [..., tokens, heads, D] in fp32 into codes [..., slots, heads, D] and
    scales [..., blocks, heads], over the whole pool: blocks without new rows keep
    their largest value 0 and their scale."""
    F, B = LARGEST[c["format"]], c["block"]
    lead, (n, heads, d) = codes.shape[:-3], codes.shape[-3:]
    block = slots // B
    at = block[:, None].expand(-1, heads).expand(*lead, -1, -1)
    top = torch.zeros_like(scales).scatter_reduce_(-2, at, rows.abs().amax(-1), "amax")
    offset = torch.full((n // B,), B, dtype=slots.dtype, device=slots.device)
    offset = offset.scatter_reduce_(0, block, slots % B, "amin")  # of a block's first new row; B: none
    # the smallest power of two that holds a block's values
    mantissa, exponent = torch.frexp(top)
    fit = torch.ldexp(torch.ones_like(top), exponent - (9 if F == 448.0 else 16) + (mantissa > 0.875))
    fit = torch.where(top > 0, fit, 0).clamp_min(LEAST_SCALE)
    begun = (offset == 0)[:, None]
    # (a block that was begun grows to it: its scale is a power of two, too)
    after = torch.where(begun, fit, torch.maximum(fit, scales))
    live = torch.arange(n, device=slots.device) % B < offset.repeat_interleave(B)
    ratio = torch.where(begun, 1.0, scales / after).repeat_interleave(B, -2)
    ratio = torch.where(live[:, None], ratio, 1.0)
    codes.copy_((codes.float() * ratio[..., None]).to(codes.dtype))
    by = after.gather(-2, at)
    codes.view(torch.uint8)[..., slots, :, :] = (rows / by[..., None]).to(codes.dtype).view(torch.uint8)
    scales.copy_(after)


def _plain_write(s):
    c = s["case"]
    q, k, v = (x.float() for x in _rows(s))
    if c["rotary"]:
        row = s["table"][s["positions"]]
        cos, sin = row[:, None, : c["rotary"] // 2], row[:, None, c["rotary"] // 2:]
        s["q_out"].copy_(_turn(c, q, cos, sin))
        k = _turn(c, k, cos, sin)
    _store(c, s["k"], s["k_scales"], k, s["slots"])
    _store(c, s["v"], s["v_scales"], v, s["slots"])
    return _cache_outputs(s)


def _plain_move(s):
    c = s["case"]
    src, dst, half = s["src"].long(), s["dst"].long(), c["rotary"] // 2
    rows = []
    for codes, scales in ((s["k"], s["k_scales"]), (s["v"], s["v_scales"])):
        rows.append(codes.view(torch.uint8)[:, src].view(codes.dtype).float() * scales[:, src // c["block"], :, None])
    old, new = s["table"][s["pairs"][:, 0].long()], s["table"][s["pairs"][:, 1].long()]
    co, so, cn, sn = old[:, :half], old[:, half:], new[:, :half], new[:, half:]
    norm = co * co + so * so
    cos, sin = (cn * co + sn * so) / norm, (sn * co - cn * so) / norm
    same = (s["pairs"][:, 0] == s["pairs"][:, 1])[:, None, None]
    k = torch.where(same, rows[0], _turn(c, rows[0], cos[:, None], sin[:, None]))
    _store(c, s["k"], s["k_scales"], k, dst)
    _store(c, s["v"], s["v_scales"], rows[1], dst)
    return _cache_outputs(s)


def _plain_read(s):
    c = s["case"]
    P, hk, hq, d, dev = c["page"], c["heads"], c["q_heads"], c["head_dim"], s["q"].device
    B, N, group = c["requests"], s["max_new"], c["q_heads"] // c["heads"]
    # the ranks that some token sees: the first keys, and those from `low` on
    first = torch.clamp(s["low"], max=c["first"])[:, None]
    width = s["max_len"]
    rank = torch.arange(width, device=dev)[None].expand(B, -1)
    rank = torch.where(rank < first, rank, rank - first + s["low"][:, None])
    there = rank < (s["old"] + s["new"])[:, None]
    at = torch.minimum(rank, (s["old"] + s["new"])[:, None] - 1)
    slot = s["tables"].gather(1, at // P) * P + at % P
    if P == 1:
        slot = s["indices"].long()[s["kv_indptr"][:-1].long()[:, None] + at]
    k, v = (codes.view(torch.uint8)[slot].view(codes.dtype).float() * scales[slot // c["block"]][..., None]
            for codes, scales in ((s["k"], s["k_scales"]), (s["v"], s["v_scales"])))
    # [requests, new, width]
    seen = torch.zeros((B, N, width), dtype=torch.bool, device=dev)
    before = (rank < s["old"][:, None])[s["request"]]
    if s["starts"] is not None:
        before = before & ((rank[s["request"]] >= s["starts"][:, None]) | (rank[s["request"]] < c["first"]))
    node = (rank - s["old"][:, None])[s["request"]]
    mine = (node >= 0) & there[s["request"]]
    if s["mask"] is None:
        mine = mine & (node <= s["token"][:, None])
    else:
        word = s["mask"].gather(1, node.clamp(0, 64 * s["mask"].shape[1] - 1) // 64)
        mine = mine & (word >> (node.clamp(0) % 64) & 1).bool()
    seen[s["request"], s["token"]] = before | mine
    q = torch.zeros((B, N, hq, d), device=dev)
    q[s["request"], s["token"]] = s["q"].float()
    q = q.view(B, N, hk, group, d).permute(0, 2, 3, 1, 4).reshape(B * hk, group * N, d)
    k = k.permute(0, 2, 3, 1).reshape(B * hk, d, width).contiguous()
    v = v.permute(0, 2, 1, 3).reshape(B * hk, width, d).contiguous()
    score = (torch.bmm(q, k) * s["scale"]).view(B, hk, group, N, width)
    score.masked_fill_(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True).clamp_min(-1e30)
    if s["sinks"] is not None:
        sink = s["sinks"].view(1, hk, group, 1, 1)
        top = torch.maximum(top, sink)
    weight = torch.exp(score - top)
    total = weight.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(sink - top)
    out = torch.bmm(weight.view(B * hk, group * N, width), v).view(B, hk, group, N, d) / total.clamp_min(1e-30)
    out = out.permute(0, 3, 1, 2, 4).reshape(B, N, hq, d)
    s["out"].copy_(out[s["request"], s["token"]])
    return s["out"]


# ---------------------------------------------------------------------------
# The definitions in 64 bits.


def exact(case, seed):
    return {"write": _exact_write, "move": _exact_move, "read": _exact_read}[case["kind"]](case, prepare(case, seed))


def _complex_turn(c, y, turn):
    """y [tokens, heads, D], its pairs multiplied by the complex numbers turn [tokens, rotary / 2]."""
    half = torch.arange(c["rotary"] // 2, device=y.device)
    one, two = (half, half + c["rotary"] // 2) if c["neox"] else (2 * half, 2 * half + 1)
    z = torch.complex(y[..., one], y[..., two]) * turn[:, None]
    out = y.clone()
    out[..., one], out[..., two] = z.real, z.imag
    return out


def _blocks_of(c, slots):
    """The touched blocks, and of each the tokens at its offsets ([blocks, B], -1: none)."""
    blocks, which = np.unique(slots // c["block"], return_inverse=True)
    token = np.full((len(blocks), c["block"]), -1)
    token[which, slots % c["block"]] = np.arange(len(slots))
    return blocks, token


def _rounded(c, x):
    """Values in 64 bits to the nearest that 8 bits hold, ties to the even one."""
    digits, smallest = (3, -6) if c["format"] == "e4m3" else (2, -14)
    exponent = torch.frexp(x)[1] - 1
    step = torch.exp2((exponent.clamp_min(smallest) - digits).double())
    return torch.round(x / step) * step


def _exact_store(c, codes, scales, rows, blocks, token):
    """One layer's codes and scales."""
    F, B, dev = LARGEST[c["format"]], c["block"], codes.device
    out, scale = codes.double(), scales.double().cpu().numpy()
    at = torch.from_numpy(np.maximum(token, 0)).to(dev)
    fresh = torch.from_numpy(token >= 0).to(dev)[..., None, None]
    x = torch.where(fresh, rows[at], 0.0)  # [blocks, B, heads, D]
    need = x.abs().amax((1, 3)).cpu().numpy() / F
    least = np.ldexp(1.0, np.ceil(np.log2(np.maximum(need, LEAST_SCALE))).astype(int))
    before = scale[blocks]
    grown = before * np.exp2(np.maximum(0, np.ceil(np.log2(np.maximum(need, 1e-300) / before))))
    begun = token[:, 0] >= 0
    after = np.where(begun[:, None], least, grown)
    scale[blocks] = after
    by = torch.from_numpy(after).to(dev)[:, None, :, None]
    held = torch.from_numpy(np.where(begun[:, None], 1.0, before / after)).to(dev)[:, None, :, None]
    offset = np.argmax(token >= 0, 1)
    live = torch.from_numpy(np.arange(B)[None] < offset[:, None]).to(dev)[..., None, None]
    slot = torch.from_numpy(blocks[:, None] * B + np.arange(B)[None]).to(dev)
    kept = out[slot]
    out[slot] = torch.where(fresh, _rounded(c, x / by), torch.where(live, _rounded(c, kept * held), kept))
    return out, torch.from_numpy(scale).to(dev)


def _exact_write(c, s):
    q, k, v = (x.double() for x in _rows(s))
    out = {"q": None}
    if c["rotary"]:
        row = s["table"].double()[s["positions"]]
        turn = torch.complex(row[:, : c["rotary"] // 2], row[:, c["rotary"] // 2:])
        out["q"], k = _complex_turn(c, q, turn), _complex_turn(c, k, turn)
    blocks, token = _blocks_of(c, s["slots"].cpu().numpy())
    for name, rows in (("k", k), ("v", v)):
        out[name], out[name + "_scales"] = _exact_store(c, s[name], s[name + "_scales"], rows, blocks, token)
    return out


def _exact_move(c, s):
    if s["k"].numel() > 3 << 30:
        return None
    src, dst = s["src"].long(), s["dst"].cpu().numpy()
    half = c["rotary"] // 2
    table = s["table"].double()
    phase = torch.complex(table[:, :half], table[:, half:])
    old, new = s["pairs"][:, 0].long(), s["pairs"][:, 1].long()
    turn = torch.where((old == new)[:, None], 1.0 + 0.0j, phase[new] / phase[old])
    blocks, token = _blocks_of(c, dst)
    out = {"q": None}
    for name in ("k", "v"):
        layers = []
        for codes, scales in zip(s[name], s[name + "_scales"]):
            rows = codes.double()[src] * scales.double()[src // c["block"]][..., None]
            if name == "k":
                rows = _complex_turn(c, rows, turn)
            layers.append(_exact_store(c, codes, scales, rows, blocks, token))
        out[name] = torch.stack([codes for codes, _ in layers])
        out[name + "_scales"] = torch.stack([scales for _, scales in layers])
    return out


def _exact_read(c, s):
    """Request by request and head by head, through the log of the sum."""
    P, hk, group = c["page"], c["heads"], c["q_heads"] // c["heads"]
    dev = s["q"].device
    out = torch.zeros(tuple(s["out"].shape), dtype=torch.float64, device=dev)
    q0 = at = 0
    limit = c["window"] if c["window"] else c["new_hi"]
    tables = s["tables"]
    for b, (old, new, parents) in enumerate(zip(*_lengths(c), _parents(c))):
        rank = torch.arange(old + new, device=dev)
        slot = s["indices"][at: at + old + new].long() if P == 1 else tables[b][rank // P] * P + rank % P
        seen = np.ones((new, old + new), dtype=bool)
        if c["window"]:
            lo = old + _depths(parents) - c["window"]
            seen[:, :old] = (np.arange(old)[None] >= lo[:, None]) | (np.arange(old)[None] < c["first"])
        seen[:, old:] = _ancestors(parents, limit)
        hidden = torch.from_numpy(~seen).to(dev)
        for g in range(hk):
            k, v = (codes[:, g].double()[slot] * scales[:, g].double()[slot // c["block"]][:, None]
                    for codes, scales in ((s["k"], s["k_scales"]), (s["v"], s["v_scales"])))
            for h in range(g * group, (g + 1) * group):
                score = s["q"][q0: q0 + new, h].double() @ k.T.contiguous() * s["scale"]
                score.masked_fill_(hidden, float("-inf"))
                total = torch.logsumexp(score, -1, keepdim=True)
                if s["sinks"] is not None:
                    total = torch.logaddexp(total, s["sinks"][h].double())
                out[q0: q0 + new, h] = torch.exp(score - total) @ v
        q0, at = q0 + new, at + old + new
    return out


# ---------------------------------------------------------------------------
# What a pass cannot do without.


def work(case):
    c = case
    d, hk = c["head_dim"], c["heads"]
    if c["kind"] == "move":
        moved = [len(rank) for _, _, rank in _moves(c)]
        blocks = sum(-(-n // c["block"]) for n in moved)
        rows = c["layers"] * sum(moved) * hk
        # codes in and out, scales in and out, the lists, two table rows a token
        bytes_ = 4 * rows * d + 16 * c["layers"] * blocks * hk + sum(moved) * 16 + sum(moved) * 8 * c["rotary"]
        return {"bytes": bytes_, "flops": rows * (6 * d + 3 * c["rotary"])}
    old, new = _lengths(c)
    total = sum(new)
    if c["kind"] == "write":
        e = DTYPES[c["dtype"]].itemsize
        blocks = sum(-(-(o % c["block"] + n) // c["block"]) for o, n in zip(old, new))
        turned = 2 * c["q_heads"] if c["rotary"] else 0
        bytes_ = total * d * (e * (turned + 2 * hk) + 2 * hk) + 8 * blocks * hk + 8 * total
        bytes_ += (8 * total + 4 * c["rotary"] * min(total, POSITIONS)) if c["rotary"] else 0
        return {"bytes": bytes_, "flops": total * (2 * hk * 3 * d + (c["q_heads"] + hk) * 3 * c["rotary"])}
    W, trees, seen, keys = c["window"], _parents(c), 0, 0
    for o, n, p in zip(old, new, trees):
        depth = _depths(p)
        first = np.clip(o + depth - W, 0, o) if W else np.zeros(n, dtype=np.int64)
        kept = np.minimum(first, c["first"])
        seen += int((o - first + kept).sum()) + int(np.minimum(depth + 1, W + 1 if W else n).sum())
        keys += o + n - int(first.min()) + int(min(first.min(), c["first"]))
    rows = total * c["q_heads"] * d * DTYPES[c["dtype"]].itemsize
    bytes_ = keys * hk * (2 * d + 8 / c["block"]) + 2 * rows + 4 * keys / c["page"]
    return {"bytes": bytes_, "flops": 4 * d * c["q_heads"] * seen}
