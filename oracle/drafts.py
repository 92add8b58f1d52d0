"""CPU restatement, in 64 bits, of the step that verifies drafted tokens.

``step_maps``, ``qk_norm_rope`` and ``tree_attention`` follow the definitions
in ``include/akv_amd.h`` request by request and row by row.  The reference has
no counterpart (it rejects speculative decoding); the registry rows are those
of ``akv/system/sglang/srt/layers/attention/context_backend.py:666-740``, the
sinks those of ``context_backend.py:254-272``.

Pinned by (``tests/test_oracle_drafts.py``): a chain without new tokens' masks
equals ``oracle.decode``'s indices; causal trees equal
``oracle.attention.context_attention``; the rotation equals the published
complex form and keeps norms; masks equal reachability by matrix powers.
"""

import numpy as np


def depths(parents):
    """Depth of each node; a parent that is no earlier node is none."""
    out = []
    for i, p in enumerate(parents):
        out.append(out[p] + 1 if 0 <= p < i else 0)
    return np.array(out, dtype=np.int64)


def ancestors(parents, limit=None):
    """bool [n, n]: node j is i or an ancestor of i (at most ``limit`` levels up)."""
    n = len(parents)
    seen = np.zeros((n, n), dtype=bool)
    for i in range(n):
        a, up = i, 0
        while limit is None or up <= limit:
            seen[i, a] = True
            p = int(parents[a])
            if not 0 <= p < a:
                break
            a, up = p, up + 1
    return seen


def pack_bits(seen, words):
    """bool [n, m] -> int64 words [n, words] (bits past 64 words are dropped)."""
    seen = np.asarray(seen, dtype=bool)
    bits = np.zeros((len(seen), 64 * words), dtype=np.uint8)
    m = min(seen.shape[1], 64 * words)
    bits[:, :m] = seen[:, :m]
    return np.packbits(bits, axis=1, bitorder="little").view(np.int64).reshape(len(seen), words)


def step_maps(requests, new_lens, *, page_size=1, pages=0, parents=None, words=1, window=None, capacity=None,
              chunk=False):
    """``requests``: per request (slots, positions) of all its ranks, slots -1
    where it has none; ``parents``: per request, or None for chains.  A node's
    position is the first new rank's plus its depth; with ``chunk`` a chain's
    tokens have their own ranks' (the same wherever those ascend by one, as they
    do behind a registry row's active ranks)."""
    new = [max(0, min(int(n), len(s))) for (s, _), n in zip(requests, new_lens)]
    total = sum(new)
    capacity = total if capacity is None else capacity
    out = dict(
        qo_indptr=np.concatenate(([0], np.cumsum(new))).astype(np.int64),
        kv_indptr=np.concatenate(([0], np.cumsum([len(s) for s, _ in requests]))).astype(np.int64),
        slot_map=np.full(capacity, -1, dtype=np.int64), positions=np.zeros(capacity, dtype=np.int64),
        block_tables=np.full((len(requests), pages), -1, dtype=np.int32),
        tree_mask=np.zeros((capacity, words), dtype=np.int64), window_mask=np.zeros((capacity, words), dtype=np.int64),
        window_starts=np.zeros(capacity, dtype=np.int32),
    )
    at = 0
    for b, ((slots, positions), n) in enumerate(zip(requests, new)):
        slots, positions = np.asarray(slots, dtype=np.int64), np.asarray(positions, dtype=np.int64)
        old = len(slots) - n
        heads = slots[::page_size][:pages]
        out["block_tables"][b, : len(heads)] = np.where(heads < 0, -1, heads // page_size)
        if n == 0:
            continue
        tree = list(range(-1, n - 1)) if parents is None else parents[b]
        here = slice(at, at + n)
        out["slot_map"][here] = slots[old:]
        at_pos = positions[old:] if chunk and parents is None else positions[old] + depths(tree)
        out["positions"][here] = at_pos
        out["tree_mask"][here] = pack_bits(ancestors(tree), words)
        if window is not None:
            inside = at_pos[:, None] - at_pos[None] <= window
            out["window_mask"][here] = pack_bits(ancestors(tree) & inside, words)
            out["window_starts"][here] = np.searchsorted(positions[:old], out["positions"][here] - window, side="left")
        at += n
    return out


def qk_norm_rope(x, weight, eps, rows, rotary_dim, neox):
    """Normed and rotated head rows ``[N, heads, D]`` and, per element, the sum
    of magnitudes its rotation adds (what fp32 errors are relative to);
    ``rows``: the tokens' cos | sin rows, or NaN rows."""
    x = np.asarray(x, dtype=np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    if weight is not None:
        y = y * np.asarray(weight, dtype=np.float64)
    half = rotary_dim // 2
    one = np.arange(half) if neox else 2 * np.arange(half)
    two = one + half if neox else one + 1
    rows = np.asarray(rows, dtype=np.float64)
    cos, sin = rows[:, None, :half], rows[:, None, half:]
    out, size = y.copy(), np.abs(y)
    a, b = y[..., one], y[..., two]
    out[..., one], out[..., two] = a * cos - b * sin, b * cos + a * sin
    size[..., one] = np.abs(a * cos) + np.abs(b * sin)
    size[..., two] = np.abs(b * cos) + np.abs(a * sin)
    unknown = np.isnan(rows).any(-1)
    out[unknown] = np.nan
    return out, size


def tree_attention(q, k_pool, v_pool, requests, scale, sinks=None):
    """Per token of each request: softmax with sink over the keys it sees.

    ``q`` ``[N, Hq, D]``; ``requests``: per request (first token, slots of its
    keys (-1: a hole), bool [n, keys] of what each token sees).  Returns the
    outputs, ``sum_j w_j |v_j|`` with the weights w (what errors are relative
    to), and the largest ``scale sum |q k|`` of each row's scores.
    """
    q = np.asarray(q, dtype=np.float64)
    out, size = np.zeros_like(q), np.zeros_like(q)
    spread = np.zeros(q.shape[:2])
    group = q.shape[1] // k_pool.shape[1]
    for first, slots, seen in requests:
        slots = np.asarray(slots, dtype=np.int64)
        there = (slots >= 0) & (slots < len(k_pool))
        for i in range(len(seen)):
            keys = slots[np.asarray(seen[i]) & there]
            if len(keys) == 0:
                continue
            k, v = np.asarray(k_pool[keys], dtype=np.float64), np.asarray(v_pool[keys], dtype=np.float64)
            for h in range(q.shape[1]):
                g = h // group
                s = scale * (k[:, g] @ q[first + i, h])
                spread[first + i, h] = scale * (np.abs(k[:, g]) @ np.abs(q[first + i, h])).max()
                top = s.max() if sinks is None else max(s.max(), float(sinks[h]))
                w = np.exp(s - top)
                w /= w.sum() + (0.0 if sinks is None else np.exp(float(sinks[h]) - top))
                out[first + i, h] = w @ v[:, g]
                size[first + i, h] = w @ np.abs(v[:, g])
    return out, size, spread
