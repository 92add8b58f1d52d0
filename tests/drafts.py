"""Seeded batches for the tests of the drafted-token step."""

import numpy as np
import torch

from oracle import drafts

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # finfo.eps / 2


def random_tree(rng, n):
    """Parents: mostly a recent node, now and then another root."""
    return [-1] + [int(-1 if rng.random() < 0.05 else max(0, i - 1 - rng.integers(0, 4))) for i in range(1, n)]


def f64(t):
    return t.detach().cpu().double().numpy()


class Cache:
    """A pool whose requests' keys lie at random slots or on random pages, with
    drafted tokens' queries; ``slots[b]`` are request b's, -1 for a hole."""

    def __init__(self, device, seed, old, new, *, q_heads, kv_heads, head_dim, dtype, page=1, holes=0, spread=1.0,
                 capacity=None, words=None):
        self.rng = rng = np.random.default_rng(seed)
        gen = torch.Generator().manual_seed(seed)
        self.old, self.new, self.page, self.device = list(old), list(new), page, device
        seq = [o + n for o, n in zip(old, new)]
        pages = [-(-s // page) for s in seq]
        ids = rng.permutation(sum(pages) + 3)[: sum(pages)]
        self.slots, tables, at = [], np.full((len(seq), max(pages + [1]) + 2), -7, dtype=np.int32), 0
        for b, s in enumerate(seq):
            own = ids[at: at + pages[b]].copy()
            at += pages[b]
            for _ in range(holes):
                if len(own) > 1:
                    own[rng.integers(0, len(own))] = rng.choice([-1, sum(pages) + 3, 2 ** 31 - 1])
            tables[b, : pages[b]] = own
            rank = np.arange(s)
            page_of = own[rank // page].astype(np.int64)
            bad = (page_of < 0) | (page_of >= sum(pages) + 3)
            self.slots.append(np.where(bad, -1, page_of * page + rank % page))
        n_slots, total = (sum(pages) + 3) * page, sum(new)
        self.total, capacity = total, total if capacity is None else capacity
        make = lambda *shape: (spread * torch.randn(shape, generator=gen)).to(dtype)  # noqa: E731
        self.q = make(capacity, q_heads, head_dim).to(device)
        self.k, self.v = make(n_slots, kv_heads, head_dim), make(n_slots, kv_heads, head_dim)
        self.qo = torch.tensor(np.concatenate(([0], np.cumsum(new))), dtype=torch.int32, device=device)
        self.kv = torch.tensor(np.concatenate(([0], np.cumsum(seq))), dtype=torch.int32, device=device)
        if page == 1:
            flat = [tables[b, :s] for b, s in enumerate(seq)]
            self.indices = torch.from_numpy(np.concatenate(flat + [np.zeros(1, np.int32)])).to(device)
        else:
            self.indices = torch.from_numpy(tables).to(device)
        self.trees = [random_tree(rng, n) if n else [] for n in new]
        self.words = words or max(1, -(-max(list(new) + [1]) // 64))
        self.capacity = capacity
        self.max_len, self.max_new = max(seq + [0]), max(list(new) + [0])

    def masks(self, kind):
        """bool [n, n] per request, and the words to pass (None for a chain)."""
        if kind == "chain":
            return [np.tril(np.ones((n, n), dtype=bool)) for n in self.new], None
        if kind == "tree":
            seen = [drafts.ancestors(t) for t in self.trees]
        else:  # any bits, rows without a bit among them
            seen = [self.rng.random((n, n)) < 0.4 for n in self.new]
            for s in seen:
                s[::3] = False
        words = np.zeros((self.capacity, self.words), dtype=np.int64)
        if self.total:
            words[: self.total] = np.concatenate([drafts.pack_bits(s, self.words) for s in seen])
        return seen, torch.from_numpy(words).to(self.device)

    def visible(self, seen, starts=None):
        """Requests as ``oracle.drafts.tree_attention`` takes them."""
        out, at = [], 0
        for b, (o, n) in enumerate(zip(self.old, self.new)):
            keys = np.ones((n, o + n), dtype=bool)
            if starts is not None:
                keys[:, :o] = np.arange(o)[None] >= np.asarray(starts[at: at + n])[:, None]
            keys[:, o:] = seen[b]
            out.append((at, self.slots[b], keys))
            at += n
        return out


def attention_tolerance(dtype, out_dtype, keys, want, size, spread, v_max):
    """How far a row may be off.  A weight is rounded once to ``dtype`` (the sum
    takes the same rounded weights) and its exponent carries the fp32 errors of
    a product of up to 128 terms, one scaling and exp2: 2^-24 (128 + 3) spread +
    2^-22.  Weights with errors d_j move o by at most max|d_j| (sum w|v| + |o|).
    fp32 sums over the keys add keys 2^-23 sum w|v|; fp16 weights below its
    smallest step are off by 2^-25 each, next to a weight of at least 1."""
    delta = HALF[dtype] + 131 * 2.0 ** -24 * spread[..., None] + 2.0 ** -22
    tol = delta * (size + np.abs(want)) + keys * 2.0 ** -23 * size + HALF[out_dtype] * np.abs(want)
    if dtype == torch.float16:
        tol = tol + keys * 2.0 ** -25 * 2 * v_max + 2.0 ** -25
    return tol * 1.01 + 1e-30
