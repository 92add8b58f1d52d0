"""The operators of a step that verifies drafted tokens: their calls and their plain forms.

``listed()`` names the cases, ``draw(rng)`` gives another of the same ranges.
Lengths, layouts and trees follow from the case (``events``); slots, K/V,
queries, weights and sinks are drawn from the seed given to ``prepare``.

Kinds:

* ``maps``  the step's metadata from request lengths: indptrs, slots and
            positions of the new tokens, block tables, tree masks and the
            window's first keys (``page_table.context_step_maps``);
* ``norm``  per-head RMS norms of q and k, rotation, and the new K/V rows
            written to the pool (``qk_norm.qk_norm_rope``);
* ``tree``  attention of one layer's drafted tokens over the cache
            (``attention.tree_attention``).

``own`` false computes each from its definition with elementary torch
operations; true calls the framework.
"""

import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # one chat of 4k tokens decodes a token: latency and the launch
        dict(name="maps-decode-1", kind="maps", requests=1, len_lo=4096, len_hi=4096, new_lo=1, new_hi=1, page=1,
             kept=False, reposition=True, tree=False, window=0, events=1),
        # 32 GPT-OSS requests of ~20k kept keys each verify trees of 16 tokens:
        # slot tables, masks, and the window of the sliding-window layers
        dict(name="maps-tree-32x20k", kind="maps", requests=32, len_lo=19000, len_hi=20500, new_lo=16, new_hi=16,
             page=1, kept=True, reposition=True, tree=True, window=128, events=2),
        # a full server on pages of 16: 64 ragged requests, short chains of
        # drafted tokens, dropped spans not repositioned yet (positions with gaps)
        dict(name="maps-paged-64", kind="maps", requests=64, len_lo=2048, len_hi=65536, new_lo=1, new_hi=8, page=16,
             kept=True, reposition=False, tree=False, window=0, events=3),
        # one decoded token of a GPT-OSS-shaped layer (64 q / 8 KV heads x 64)
        dict(name="norm-decode-1", kind="norm", tokens=1, q_heads=64, heads=8, head_dim=64, rotary=64, neox=True,
             dtype="bf16"),
        # the drafted tokens of 12 requests, 32 each, of a 32 / 8 x 128 layer
        dict(name="norm-tree-384", kind="norm", tokens=384, q_heads=32, heads=8, head_dim=128, rotary=128, neox=True,
             dtype="bf16"),
        # a prefill chunk of a partial-rotary fp16 model with interleaved pairs
        dict(name="norm-partial-fp16", kind="norm", tokens=8191, q_heads=16, heads=4, head_dim=128, rotary=64,
             neox=False, dtype="fp16"),
        # a whole 32k-token GPT-OSS prompt in one forward
        dict(name="norm-prefill-32k", kind="norm", tokens=32768, q_heads=64, heads=8, head_dim=64, rotary=64,
             neox=True, dtype="bf16"),
        # one fp16 request of 4k keys verifies 8 drafted tokens: latency
        dict(name="tree-fp16-1x8", kind="tree", requests=1, q_heads=16, heads=4, head_dim=128, dtype="fp16",
             sinks=False, window=0, page=1, len_lo=4096, len_hi=4096, new_lo=8, new_hi=8, events=4),
        # 32 GPT-OSS requests holding ~20k keys each, trees of 16: a full layer
        dict(name="tree-gpt-oss-32x16", kind="tree", requests=32, q_heads=64, heads=8, head_dim=64, dtype="bf16",
             sinks=True, window=0, page=1, len_lo=19000, len_hi=20500, new_lo=16, new_hi=16, events=5),
        # the same batch on a sliding-window layer
        dict(name="tree-gpt-oss-32x16-window", kind="tree", requests=32, q_heads=64, heads=8, head_dim=64,
             dtype="bf16", sinks=True, window=128, page=1, len_lo=19000, len_hi=20500, new_lo=16, new_hi=16, events=5),
        # 12 ragged Llama-3-8B requests (32 / 8 x 128) on pages of 16, ragged trees
        dict(name="tree-llama3-12-paged", kind="tree", requests=12, q_heads=32, heads=8, head_dim=128, dtype="bf16",
             sinks=False, window=0, page=16, len_lo=2000, len_hi=20000, new_lo=5, new_hi=32, events=6),
        # wide trees of 64 over 8 long GPT-OSS requests: bound by the arithmetic
        dict(name="tree-gpt-oss-8x64", kind="tree", requests=8, q_heads=64, heads=8, head_dim=64, dtype="bf16",
             sinks=True, window=0, page=1, len_lo=18000, len_hi=32000, new_lo=64, new_hi=64, events=7),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(("maps", "norm", "norm", "tree", "tree", "tree"))
    c = dict(kind=kind)
    if kind == "norm":
        head_dim = rng.choice((64, 64, 80, 96, 128, 128))
        heads = rng.choice((1, 2, 4, 8))
        c.update(tokens=_log_int(rng, 1, 32768), q_heads=heads * rng.choice((1, 2, 4, 7, 8)), heads=heads,
                 head_dim=head_dim, rotary=rng.choice((head_dim, head_dim, head_dim // 2)), neox=rng.random() < 0.7,
                 dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")))
        # no larger than the 32k prompt
        row = (c["q_heads"] + 2 * heads) * head_dim * DTYPES[c["dtype"]].itemsize
        c["tokens"] = max(1, min(c["tokens"], 32768 * 80 * 64 * 2 // row))
        return c
    c["events"] = rng.randrange(1 << 20)
    new = _log_int(rng, 1, 64)
    c.update(new_lo=max(1, new // rng.randint(1, 8)), new_hi=new, page=rng.choice((1, 1, 16)))
    if kind == "maps":
        hi = _log_int(rng, 100, 65536)
        c.update(requests=_log_int(rng, 1, 64), len_lo=max(80, hi // rng.randint(1, 32)), kept=rng.random() < 0.7,
                 reposition=rng.random() < 0.7, tree=rng.random() < 0.6, window=rng.choice((0, 128)))
        c["len_hi"] = max(hi, c["len_lo"])
        # no more tables than 32 x 20k slots
        c["requests"] = max(1, min(c["requests"], 32 * 20500 * (4 if c["page"] > 1 else 1) // c["len_hi"]))
    else:
        head_dim = rng.choice((64, 64, 64, 96, 128, 128))
        heads = rng.choice((2, 4, 8))
        group = rng.choice((1, 4, 7, 8, 8))
        hi = _log_int(rng, 80, 32000)
        c.update(requests=_log_int(rng, 1, 32), q_heads=heads * group, heads=heads, head_dim=head_dim,
                 dtype=rng.choice(("bf16", "bf16", "fp16")), sinks=rng.random() < 0.5,
                 window=rng.choice((0, 0, 128)), len_lo=max(70, hi // rng.randint(1, 8)))
        c["len_hi"] = max(hi, c["len_lo"])
        # neither more K/V than 32 x 20k keys of 8 x 64 nor more products than
        # the trees of 64 over 8 x 25k keys
        kv = 32 * 19750 * 8 * 64 // (c["len_hi"] * heads * head_dim)
        mul = 8 * 25000 * 64 * 64 * 64 // (c["len_hi"] * c["new_hi"] * c["q_heads"] * head_dim)
        c["requests"] = max(1, min(c["requests"], kv, mul))
    return c


# ---------------------------------------------------------------------------
# What follows from the case alone: lengths, trees, kept ranks.


def _lengths(c):
    """Per request: keys before the step, and new tokens."""
    rng = random.Random(c["events"])
    old = [rng.randint(c["len_lo"], c["len_hi"]) for _ in range(c["requests"])]
    return old, [rng.randint(c["new_lo"], c["new_hi"]) for _ in range(c["requests"])]


def _parents(c):
    """One draft tree per request: node 0 hangs on the cache (-1), the others
    on an earlier node, mostly a recent one."""
    rng = random.Random(c["events"] + 1)
    return [[-1] + [max(0, i - 1 - int(rng.expovariate(0.7))) for i in range(1, n)] for n in _lengths(c)[1]]


def _words(c):
    return (c["new_hi"] + 63) // 64


def _keep(c, b, n):
    """Raw indices of n kept tokens among spans of dropped ones."""
    rng = np.random.default_rng((c["events"], b))
    gaps = np.where(rng.random(n) < 0.002, rng.integers(50, 400, n), 0)
    gaps[0] = 0
    return np.arange(n) + np.cumsum(gaps)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _dev(a, dtype):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).to("cuda")


# ---------------------------------------------------------------------------
# Inputs.


def prepare(case, seed):
    return {"maps": _prepare_maps, "norm": _prepare_norm, "tree": _prepare_tree}[case["kind"]](case, seed)


def _prepare_maps(c, seed):
    old, new = _lengths(c)
    B, P = len(old), c["page"]
    pages = [-(-(o + n) // P) for o, n in zip(old, new)]
    free = np.random.default_rng(seed).permutation(sum(pages)) + 1
    width = 8
    raws, rows, at = [], [], 0
    for b, (o, n) in enumerate(zip(old, new)):
        # kept prompt tokens, then the new ones; slots are dense by rank
        raw = _keep(c, b, o) if c["kept"] else np.arange(o)
        columns = np.concatenate((raw, raw[-1] + 1 + np.arange(n)))
        rank = np.arange(o + n)
        slots = free[at + rank // P] * P + rank % P
        at += pages[b]
        raws.append(raw)
        rows.append((columns, slots))
        width = max(width, int(columns[-1]) + 1)
    table = np.full((B, width), -1, dtype=np.int32)
    for b, (columns, slots) in enumerate(rows):
        table[b, columns] = slots
    raw_ids = _dev(np.concatenate(raws), np.int32)
    pos_ids = _dev(np.concatenate([np.arange(len(r)) for r in raws]) if c["reposition"] else np.concatenate(raws),
                   np.int32)
    off = np.concatenate(([0], np.cumsum(old)))
    registry = np.zeros((B, 6), dtype=np.int64)
    if c["kept"]:
        for b, raw in enumerate(raws):
            nxt = len(raw) if c["reposition"] else raw[-1] + 1
            registry[b] = (raw_ids.data_ptr() + 4 * off[b], pos_ids.data_ptr() + 4 * off[b], raw[-1] + 1, len(raw),
                           nxt, 0)
    total, words = sum(new), _words(c)
    i32 = dict(dtype=torch.int32, device="cuda")
    i64 = dict(dtype=torch.int64, device="cuda")
    return dict(
        case=c, registry=_dev(registry, np.int64), raw_ids=raw_ids, pos_ids=pos_ids, off=_dev(off[:-1], np.int64),
        table=_dev(table, np.int32), rows=torch.arange(B, **i64),
        seq=_dev([o + n for o, n in zip(old, new)], np.int64), new=_dev(new, np.int64),
        parents=_dev(np.concatenate(_parents(c)), np.int32) if c["tree"] else None, max_new=max(new),
        qo_indptr=torch.empty(B + 1, **i32), kv_indptr=torch.empty(B + 1, **i32),
        slot_map=torch.empty(total, **i64), positions=torch.empty(total, **i64),
        block_tables=torch.empty((B, max(pages)), **i32),
        tree_mask=torch.empty((total, words), **i64) if c["tree"] else None,
        window_mask=torch.empty((total, words), **i64) if c["window"] else None,
        window_starts=torch.empty(total, **i32) if c["window"] else None,
    )


def _rope_table(rotary, positions):
    inv = 10000.0 ** (-np.arange(0, rotary, 2) / rotary)
    angle = np.arange(positions)[:, None] * inv
    return _dev(np.concatenate((np.cos(angle), np.sin(angle)), 1), np.float32)


def _prepare_norm(c, seed):
    g, dt, d = _gen(seed), DTYPES[c["dtype"]], c["head_dim"]
    n, hq, hk = c["tokens"], c["q_heads"], c["heads"]
    qkv = torch.randn((n, (hq + 2 * hk) * d), generator=g, device="cuda").to(dt)
    slots = n + n // 4 + 8
    return dict(
        case=c, qkv=qkv, q_weight=(1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dt),
        k_weight=(1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dt),
        positions=torch.randint(0, 40960, (n,), generator=g, device="cuda"), table=_rope_table(c["rotary"], 40960),
        slot_map=torch.randperm(slots, generator=g, device="cuda")[:n].contiguous(),
        q_out=torch.empty((n, hq, d), dtype=dt, device="cuda"),
        k_pool=torch.zeros((slots, hk, d), dtype=dt, device="cuda"),
        v_pool=torch.zeros((slots, hk, d), dtype=dt, device="cuda"),
    )


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


def _depths(parents):
    depth = []
    for p in parents:
        depth.append(0 if p < 0 else depth[p] + 1)
    return np.array(depth)


def _prepare_tree(c, seed):
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    old, new = _lengths(c)
    B, P, W, d, hk = len(old), c["page"], c["window"], c["head_dim"], c["heads"]
    seq = [o + n for o, n in zip(old, new)]
    pages = [-(-s // P) for s in seq]
    free = np.random.default_rng(seed).permutation(sum(pages) + 1)
    free = free[free > 0]  # page 0 is padding
    ends = np.concatenate(([0], np.cumsum(pages)))
    if P == 1:
        indices = _dev(free, np.int32)
    else:
        tables = np.full((B, max(pages)), -1, dtype=np.int32)
        for b in range(B):
            tables[b, : pages[b]] = free[ends[b]: ends[b + 1]]
        indices = _dev(tables, np.int32)
    trees = _parents(c)
    limit = W if W else max(new)
    mask = np.concatenate([_pack(_ancestors(p, limit), _words(c)) for p in trees])
    starts = np.concatenate([np.clip(o + _depths(p) - W, 0, o) for o, p in zip(old, trees)]) if W else None
    slots, total = (sum(pages) + 1) * P, sum(new)
    pool = [torch.randn((slots, hk, d), generator=g, device="cuda", dtype=dt) for _ in range(2)]
    s = dict(
        case=c, q=torch.randn((total, c["q_heads"], d), generator=g, device="cuda", dtype=dt), k=pool[0], v=pool[1],
        qo_indptr=_dev(np.concatenate(([0], np.cumsum(new))), np.int32),
        kv_indptr=_dev(np.concatenate(([0], np.cumsum(seq))), np.int32), indices=indices, mask=_dev(mask, np.int64),
        starts=None if starts is None else _dev(starts, np.int32),
        sinks=torch.randn(c["q_heads"], generator=g, device="cuda") if c["sinks"] else None,
        out=torch.empty((total, c["q_heads"], d), dtype=dt, device="cuda"), old=old, new=new, scale=d ** -0.5,
        max_len=min(max(seq), W + max(new) + 1) if W else max(seq), max_new=max(new),
    )
    if own:
        from akv_amd import attention

        need = attention.tree_workspace_bytes(total, B, c["q_heads"], hk, d, s["max_len"], s["max_new"])
        s["workspace"] = torch.empty(max(need, 4), dtype=torch.uint8, device="cuda")
    return s


# ---------------------------------------------------------------------------
# One pass.


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"maps": _own_maps, "norm": _own_norm, "tree": _own_tree}[kind](state)
    return {"maps": _plain_maps, "norm": _plain_norm, "tree": _plain_tree}[kind](state)


def _map_outputs(s):
    names = ("qo_indptr", "kv_indptr", "slot_map", "positions", "block_tables", "tree_mask", "window_mask",
             "window_starts")
    return [s[n] for n in names if s[n] is not None]


def _own_maps(s):
    from akv_amd import page_table

    page_table.context_step_maps(
        s["registry"], s["table"], s["rows"], s["seq"], s["new"], s["qo_indptr"], s["kv_indptr"], s["slot_map"],
        s["positions"], block_tables=s["block_tables"], page_size=s["case"]["page"], parents=s["parents"],
        tree_mask=s["tree_mask"], window=s["case"]["window"] or None, window_mask=s["window_mask"],
        window_starts=s["window_starts"])
    return _map_outputs(s)


def _own_norm(s):
    from akv_amd import qk_norm

    c = s["case"]
    n, d = c["tokens"], c["head_dim"]
    q, k, v = s["qkv"].view(n, -1, d).split((c["q_heads"], c["heads"], c["heads"]), 1)
    qk_norm.qk_norm_rope(q, k, v, s["q_weight"], s["k_weight"], s["positions"], s["table"], s["q_out"], eps=EPS,
                         slot_map=s["slot_map"], k_buffer=s["k_pool"], v_buffer=s["v_pool"], rotary_dim=c["rotary"],
                         is_neox_style=c["neox"])
    return s["q_out"], s["k_pool"], s["v_pool"]


def _own_tree(s):
    from akv_amd import attention

    attention.tree_attention(
        s["q"], s["k"], s["v"], s["qo_indptr"], s["kv_indptr"], s["indices"], s["out"], scale=s["scale"],
        max_len=s["max_len"], max_new=s["max_new"], page_size=s["case"]["page"], tree_mask=s["mask"],
        key_starts=s["starts"], sinks=s["sinks"], workspace=s["workspace"])
    return s["out"]


def _indptr(lengths):
    return torch.cat((lengths.new_zeros(1), torch.cumsum(lengths, 0))).to(torch.int32)


def _bits_to_words(seen, words):
    """bool [tokens, 64 words] -> int64 [tokens, words]."""
    one = torch.ones((), dtype=torch.int64, device=seen.device) << torch.arange(64, device=seen.device)
    return (seen.view(-1, words, 64).to(torch.int64) * one).sum(-1)


def _plain_maps(s):
    c = s["case"]
    P, W, dev = c["page"], c["window"], s["seq"].device
    seq, new, reg = s["seq"], s["new"], s["registry"][s["rows"]]
    kept = reg[:, 0] != 0
    prompt, active, nxt = reg[:, 2], reg[:, 3], reg[:, 4]

    def slot_and_position(b, i):
        """Slot and position of rank i of request b (vectors)."""
        behind = i >= active[b]
        at = (s["off"][b] + torch.minimum(i, active[b] - 1)).clamp(0)
        raw = torch.where(kept[b], torch.where(behind, prompt[b] + i - active[b], s["raw_ids"][at].long()), i)
        pos = torch.where(kept[b], torch.where(behind, nxt[b] + i - active[b], s["pos_ids"][at].long()), i)
        return s["table"][s["rows"][b], raw].long(), pos

    B, width = s["block_tables"].shape
    b = torch.arange(B, device=dev)[:, None]
    first = torch.arange(width, device=dev)[None] * P
    page_slot, _ = slot_and_position(b, torch.minimum(first, seq[:, None] - 1))
    tables = torch.where(first < seq[:, None], page_slot // P, -1).to(torch.int32)

    qo = _indptr(new)
    token = torch.arange(s["slot_map"].numel(), device=dev)
    tb = torch.searchsorted(qo[1:].long(), token, right=True)
    i = token - qo[tb]
    slots, _ = slot_and_position(tb, (seq - new)[tb] + i)
    _, root = slot_and_position(tb, (seq - new)[tb])
    words = (s["max_new"] + 63) // 64
    # every node walks to its root, one ancestor a step
    depth = torch.zeros_like(i)
    tree = torch.zeros((len(token), 64 * words), dtype=torch.bool, device=dev)
    near = torch.zeros_like(tree)
    node = i
    for up in range(s["max_new"]):
        on = node >= 0
        at = node.clamp(0)[:, None]
        tree.scatter_(1, at, tree.gather(1, at) | on[:, None])
        if up <= W:
            near.scatter_(1, at, near.gather(1, at) | on[:, None])
        above = s["parents"][qo[tb] + node.clamp(0)].long() if s["parents"] is not None else node - 1
        node = torch.where(on, above, -1)
        depth = depth + (node >= 0)
    positions = root + depth
    out = [qo, _indptr(seq), slots, positions, tables]
    if s["tree_mask"] is not None:
        out.append(_bits_to_words(tree, words))
    if W:
        out.append(_bits_to_words(near, words))
        before = (seq - new)[tb]
        lo, hi = torch.zeros_like(before), before
        for _ in range(17):
            mid = (lo + hi) // 2
            _, pos = slot_and_position(tb, torch.minimum(mid, before - 1))
            less = (mid < hi) & (pos < positions - W)
            lo, hi = torch.where(less, mid + 1, lo), torch.where(less, hi, mid)
        out.append(lo.to(torch.int32))
    return out


def _plain_norm(s):
    c = s["case"]
    n, d, r = c["tokens"], c["head_dim"], c["rotary"]
    q, k, v = s["qkv"].view(n, -1, d).split((c["q_heads"], c["heads"], c["heads"]), 1)
    row = s["table"][s["positions"]]
    cos, sin = row[:, None, : r // 2], row[:, None, r // 2:]

    def norm_rotate(x, w):
        x = x.float()
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        rot, rest = y[..., :r], y[..., r:]
        if c["neox"]:
            a, b = rot[..., : r // 2], rot[..., r // 2:]
            rot = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        else:
            a, b = rot[..., ::2], rot[..., 1::2]
            rot = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        return torch.cat((rot, rest), -1).to(DTYPES[c["dtype"]])

    s["q_out"].copy_(norm_rotate(q, s["q_weight"]))
    s["k_pool"][s["slot_map"]] = norm_rotate(k, s["k_weight"])
    s["v_pool"][s["slot_map"]] = v
    return s["q_out"], s["k_pool"], s["v_pool"]


def _request_keys(s, b, at):
    """Slots of request b's keys, whose ranks begin at ``at`` of the flat list."""
    n, P = s["old"][b] + s["new"][b], s["case"]["page"]
    if P == 1:
        return s["indices"][at: at + n].long()
    rank = torch.arange(n, device=s["q"].device)
    return s["indices"][b][rank // P].long() * P + rank % P


def _visible(s, b, q0):
    """bool [new tokens, keys] of request b."""
    old, new = s["old"][b], s["new"][b]
    dev = s["q"].device
    seen = torch.ones((new, old + new), dtype=torch.bool, device=dev)
    if s["starts"] is not None:
        seen[:, :old] = torch.arange(old, device=dev)[None] >= s["starts"][q0: q0 + new, None]
    node = torch.arange(new, device=dev)
    seen[:, old:] = (s["mask"][q0: q0 + new][:, node // 64] >> (node % 64)[None] & 1).bool()
    return seen


def _plain_tree(s):
    c = s["case"]
    hk, d = c["heads"], c["head_dim"]
    group = c["q_heads"] // hk
    q0 = at = 0
    for b, (old, new) in enumerate(zip(s["old"], s["new"])):
        keys = _request_keys(s, b, at)
        first = 0
        if s["starts"] is not None:  # the keys that any of its rows sees
            first = max(0, old - c["window"] - 1)
            keys = keys[first:]
        k = s["k"][keys].float().permute(1, 2, 0).contiguous()  # [heads, dim, keys]
        v = s["v"][keys].float().transpose(0, 1).contiguous()  # [heads, keys, dim]
        q = s["q"][q0: q0 + new].float().view(new, hk, group, d).permute(1, 2, 0, 3).reshape(hk, group * new, d)
        score = (torch.bmm(q, k) * s["scale"]).view(hk, group, new, -1)
        score.masked_fill_(~_visible(s, b, q0)[:, first:], float("-inf"))
        top = score.amax(-1, keepdim=True)
        if s["sinks"] is not None:
            sink = s["sinks"].view(hk, group, 1, 1)
            top = torch.maximum(top, sink)
        weight = torch.exp(score - top)
        total = weight.sum(-1, keepdim=True)
        if s["sinks"] is not None:
            total = total + torch.exp(sink - top)
        out = torch.bmm(weight.view(hk, group * new, -1), v).view(hk, group, new, d) / total
        s["out"][q0: q0 + new] = out.permute(2, 0, 1, 3).reshape(new, -1, d).to(s["out"].dtype)
        q0, at = q0 + new, at + old + new
    return s["out"]


# ---------------------------------------------------------------------------
# The definitions in 64 bits.


def exact(case, seed):
    return {"maps": _exact_maps, "norm": _exact_norm, "tree": _exact_tree}[case["kind"]](case, prepare(case, seed))


def _exact_maps(c, s):
    """Request by request on the host, from the case's own layout."""
    old, new = _lengths(c)
    P, W, words = c["page"], c["window"], _words(c)
    table = s["table"].cpu().numpy().astype(np.int64)
    trees = _parents(c) if c["tree"] else [list(range(-1, n - 1)) for n in new]
    blocks = np.full(tuple(s["block_tables"].shape), -1, dtype=np.int32)
    slots, positions, tree, near, starts = [], [], [], [], []
    for b, (o, n) in enumerate(zip(old, new)):
        raw = _keep(c, b, o) if c["kept"] else np.arange(o)
        columns = np.concatenate((raw, raw[-1] + 1 + np.arange(n)))
        pos = np.arange(o + n) if c["reposition"] or not c["kept"] else columns
        row = table[b, columns]
        blocks[b, : -(-(o + n) // P)] = row[::P] // P
        slots.append(row[o:])
        at = pos[o] + _depths(trees[b])
        positions.append(at)
        tree.append(_pack(_ancestors(trees[b], n), words))
        near.append(_pack(_ancestors(trees[b], W), words))
        starts.append(np.searchsorted(pos[:o], at - W, side="left"))
    out = [np.concatenate(([0], np.cumsum(new))), np.concatenate(([0], np.cumsum(np.add(old, new)))),
           np.concatenate(slots), np.concatenate(positions), blocks]
    dtypes = [np.int32, np.int32, np.int64, np.int64, np.int32]
    if c["tree"]:
        out.append(np.concatenate(tree))
        dtypes.append(np.int64)
    if c["window"]:
        out += [np.concatenate(near), np.concatenate(starts)]
        dtypes += [np.int64, np.int32]
    return [o.astype(t) for o, t in zip(out, dtypes)]


def _exact_norm(c, s):
    n, d, r, hq, hk = c["tokens"], c["head_dim"], c["rotary"], c["q_heads"], c["heads"]
    x = s["qkv"].double().view(n, hq + 2 * hk, d)
    half = torch.arange(r // 2, device=x.device)
    # the dims of pair i
    one, two = (half, half + r // 2) if c["neox"] else (2 * half, 2 * half + 1)
    row = s["table"].double()[s["positions"]]
    turn = torch.complex(row[:, : r // 2], row[:, r // 2:])[:, None]
    out = torch.empty_like(x[:, : hq + hk])
    for at, count, w in ((0, hq, s["q_weight"]), (hq, hk, s["k_weight"])):
        y = x[:, at: at + count]
        y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / d + EPS) * w.double()
        z = torch.complex(y[..., one], y[..., two]) * turn
        out[:, at: at + count] = y
        out[:, at: at + count, one] = z.real
        out[:, at: at + count, two] = z.imag
    pools = []
    for rows in (out[:, hq:], x[:, hq + hk:]):
        pool = torch.zeros(tuple(s["k_pool"].shape), dtype=torch.float64, device=x.device)
        pool[s["slot_map"]] = rows
        pools.append(pool)
    return out[:, :hq], pools[0], pools[1]


def _exact_tree(c, s):
    """Row by row of (head, token), through the log of the sum."""
    hk, d = c["heads"], c["head_dim"]
    group = c["q_heads"] // hk
    out = torch.zeros(tuple(s["out"].shape), dtype=torch.float64, device=s["q"].device)
    q0 = at = 0
    for b, (old, new) in enumerate(zip(s["old"], s["new"])):
        keys = _request_keys(s, b, at)
        hidden = ~_visible(s, b, q0)
        for g in range(hk):
            k, v = s["k"][keys, g].double(), s["v"][keys, g].double()
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
    if c["kind"] == "norm":
        e, d = DTYPES[c["dtype"]].itemsize, c["head_dim"]
        elements = c["tokens"] * (c["q_heads"] + 2 * c["heads"]) * d
        rotated = c["tokens"] * (c["q_heads"] + c["heads"])
        rows = min(c["tokens"], 40960) * c["rotary"] * 4
        return {"bytes": 2 * e * elements + rows + 16 * c["tokens"] + 2 * e * d,
                "flops": rotated * (5 * d + 3 * c["rotary"])}
    old, new = _lengths(c)
    total = sum(new)
    if c["kind"] == "maps":
        P, words = c["page"], _words(c)
        pages = sum(-(-(o + n) // P) for o, n in zip(old, new))
        # a page: its row entry, its raw id where tokens were dropped, its table entry
        bytes_ = pages * (12 if c["kept"] else 8) + 4 * (c["requests"] * max(-(-(o + n) // P) for o, n in zip(old, new))
                                                          - pages)
        bytes_ += c["requests"] * (24 + 48 + 8) + total * (4 + 16)  # lengths, registry, indptrs; slots, positions
        bytes_ += total * (4 + 8 * words) if c["tree"] else 0
        bytes_ += total * (8 * words + 4 + 4) if c["window"] else 0
        return {"bytes": bytes_, "flops": 0}
    e, d, W = DTYPES[c["dtype"]].itemsize, c["head_dim"], c["window"]
    trees, seen, keys = _parents(c), 0, 0
    for o, n, p in zip(old, new, trees):
        depth = _depths(p)
        first = np.clip(o + depth - W, 0, o) if W else np.zeros(n, dtype=np.int64)
        seen += int((o - first).sum()) + int(np.minimum(depth + 1, W + 1 if W else n).sum())
        keys += o + n - int(first.min())
    rows = total * c["q_heads"] * d
    return {"bytes": 2 * e * keys * c["heads"] * d + 2 * e * rows + 4 * keys // c["page"] + 8 * total * _words(c),
            "flops": 4 * d * c["q_heads"] * seen}
