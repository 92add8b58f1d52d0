"""Serving steps over an 8-bit cache, its operators one behind the other as a
loop calls them: metadata, norms, rows appended, attention of a full and of a
sliding-window layer with first keys, and at a turn's end the compaction and the
Reposition; eagerly, on another stream, in a captured graph."""

import numpy as np
import pytest
import torch

from akv_amd import kv8, page_table, qk_norm, rope, synth, tables, transfer
from oracle import drafts
from oracle import kv8 as oracle
from tests.drafts import f64, random_tree
from tests.kv8 import kv8_tolerance, layer, values

pytestmark = pytest.mark.gpu
WINDOW, FIRST = 24, 4


class Step:
    """Requests with plain rows over one layer's 8-bit pool, buffers of a fixed capacity."""

    def __init__(self, device, seed, old, new, *, page=16, block=16, q_heads=8, kv_heads=2, d=64, capacity=None,
                 requests=None, max_new=16, max_len=400, norms=False):
        self.device, self.page, self.block, self.d, self.hq, self.hk = device, page, block, d, q_heads, kv_heads
        self.batch, self.capacity = requests or len(old), capacity or sum(new)
        self.max_len, self.max_new, self.norms = max_len, max_new, norms
        gen = torch.Generator().manual_seed(seed)
        make = lambda *shape: torch.randn(shape, generator=gen).to(torch.bfloat16).to(device)  # noqa: E731
        self.slots = 1024 * page if page == 1 else 160 * page
        self.cache = layer(device, seed, self.slots, kv_heads, d, "e4m3", block)
        self.qkv = make(self.capacity, q_heads + 2 * kv_heads, d)
        self.weights = [1 + 0.1 * make(d) for _ in range(2)]
        self.sinks = torch.randn(q_heads, generator=gen).to(device)
        self.rope = rope.make_table("plain", d, 2000, base=10000.0, device=device)
        self.table = torch.full((self.batch, max_len * 3), -1, dtype=torch.int32, device=device)
        self.rows = torch.arange(self.batch, device=device)
        i32, i64 = dict(dtype=torch.int32, device=device), dict(dtype=torch.int64, device=device)
        self.registry = torch.zeros((self.batch, 6), **i64)
        self.seq, self.fresh = torch.zeros(self.batch, **i64), torch.zeros(self.batch, **i64)
        self.parents = torch.zeros(self.capacity, **i32)
        self.qo, self.kv = torch.zeros(self.batch + 1, **i32), torch.zeros(self.batch + 1, **i32)
        self.slot_map, self.positions = torch.zeros(self.capacity, **i64), torch.zeros(self.capacity, **i64)
        self.blocks = torch.zeros((self.batch, -(-max_len // page)), **i32)
        self.mask, self.near = torch.zeros((self.capacity, 1), **i64), torch.zeros((self.capacity, 1), **i64)
        self.starts = torch.zeros(self.capacity, **i32)
        self.q = torch.zeros((self.capacity, q_heads, d), dtype=torch.bfloat16, device=device)
        self.normed = torch.zeros((self.capacity, kv_heads, d), dtype=torch.bfloat16, device=device)
        self.out, self.win = torch.zeros_like(self.q), torch.zeros_like(self.q)
        need = kv8.attention_kv8_workspace_bytes(self.capacity, self.batch, q_heads, kv_heads, d, max_len, max_new)
        self.workspace = torch.empty(need, dtype=torch.uint8, device=device)
        self.set(seed, old, new)

    def set(self, seed, old, new):
        """Another batch in the same buffers (padded with empty requests)."""
        rng = np.random.default_rng(seed)
        self.old = list(old) + [0] * (self.batch - len(old))
        self.new = list(new) + [0] * (self.batch - len(new))
        ids = rng.permutation(self.slots // self.page)
        self.requests, at = [], 0
        table = np.full(tuple(self.table.shape), -1, dtype=np.int32)
        for b, (o, n) in enumerate(zip(self.old, self.new)):
            rank = np.arange(o + n)
            own = ids[at: at + -(-(o + n) // self.page)]
            at += len(own)
            slots = own[rank // self.page] * self.page + rank % self.page if o + n else rank
            table[b, rank] = slots
            self.requests.append((slots, rank))
        self.trees = [random_tree(rng, n) if n else [] for n in self.new]
        parents = np.zeros(self.capacity, np.int32)
        flat = np.concatenate([np.asarray(t, np.int32) for t in self.trees] + [np.zeros(0, np.int32)])
        parents[: len(flat)] = flat
        for to, a in ((self.table, table), (self.seq, np.add(self.old, self.new)), (self.fresh, self.new),
                      (self.parents, parents)):
            to.copy_(torch.from_numpy(np.ascontiguousarray(a)).to(to.dtype))
        gen = torch.Generator().manual_seed(seed + 7)
        self.qkv.copy_(torch.randn(tuple(self.qkv.shape), generator=gen).to(torch.bfloat16))

    def run(self):
        hq, hk = self.hq, self.hk
        (kc, ks), (vc, vs) = self.cache
        page_table.context_step_maps(
            self.registry, self.table, self.rows, self.seq, self.fresh, self.qo, self.kv, self.slot_map, self.positions,
            block_tables=self.blocks, page_size=self.page, parents=self.parents, tree_mask=self.mask, window=WINDOW,
            window_mask=self.near, window_starts=self.starts)
        q, k, v = self.qkv.split((hq, hk, hk), 1)
        if self.norms:
            qk_norm.qk_norm_rope(q, k, None, *self.weights, self.positions, self.rope, self.q, k_out=self.normed)
            kv8.append_kv8(self.normed, v, self.slot_map, kc, vc, ks, vs, scale_block=self.block)
        else:
            kv8.append_kv8(k, v, self.slot_map, kc, vc, ks, vs, scale_block=self.block, positions=self.positions,
                           cos_sin_cache=self.rope, q=q, q_out=self.q)
        args = (self.q, kc, vc, ks, vs, self.qo, self.kv, self.blocks)
        common = dict(scale=self.d ** -0.5, max_new=self.max_new, page_size=self.page, scale_block=self.block,
                      sinks=self.sinks, workspace=self.workspace)
        kv8.attention_kv8(*args, self.out, max_len=self.max_len, tree_mask=self.mask, **common)
        kv8.attention_kv8(*args, self.win, max_len=FIRST + WINDOW + self.max_new + 1, tree_mask=self.near,
                          key_starts=self.starts, first_keys=FIRST, **common)

    def check(self, before):
        """``before``: the cache's values as the step found them."""
        want = drafts.step_maps(self.requests, self.new, page_size=self.page, pages=self.blocks.shape[1],
                                parents=self.trees, window=WINDOW, capacity=self.capacity)
        total, hq, hk = int(want["qo_indptr"][-1]), self.hq, self.hk
        pos, table = want["positions"][:total], self.rope.cpu().numpy()
        rows = self.qkv[:total].cpu().float().numpy()
        if self.norms:
            k = self.normed[:total].cpu().float().numpy()
        else:
            q, k = (oracle.rows_at(rows[:, part], pos, table, self.d, True, np.float32)
                    for part in (slice(0, hq), slice(hq, hq + hk)))
            np.testing.assert_array_equal(f64(self.q[:total]), f64(torch.from_numpy(q).to(torch.bfloat16)))
        for (codes, scales), (c, s), x in zip(self.cache, before, (k, rows[:, hq + hk:])):
            oracle.store(c, s, x, want["slot_map"][:total], self.block, "e4m3")
            np.testing.assert_array_equal(values(codes), c)
            np.testing.assert_array_equal(f64(scales), s)
        dense = [c * np.repeat(s, self.block, 0)[..., None] for c, s in before]
        for out, limit in ((self.out, None), (self.win, WINDOW)):
            requests, first = [], 0
            for (slots, _), o, n, tree in zip(self.requests, self.old, self.new, self.trees):
                seen = np.ones((n, o + n), dtype=bool)
                if limit is not None:
                    seen[:, :o] = np.arange(o)[None] >= want["window_starts"][first: first + n, None]
                    seen[:, : min(FIRST, o)] = True
                seen[:, o:] = drafts.ancestors(tree, limit)
                requests.append((first, slots, seen))
                first += n
            y, size, spread = drafts.tree_attention(f64(self.q), *dense, requests, self.d ** -0.5, f64(self.sinks))
            tol = kv8_tolerance(torch.bfloat16, torch.bfloat16, self.max_len, y, size, spread)
            assert (np.abs(f64(out) - y)[:total] <= tol[:total]).all(), limit

    def held(self):
        return [(values(c), f64(s).copy()) for c, s in self.cache]


@pytest.mark.parametrize("page,block", [(1, 1), (16, 16), (16, 4), (64, 64)])
@pytest.mark.parametrize("norms", [False, True])
@pytest.mark.parametrize("max_len", [400, 4000])
def test_step_in_order(device, page, block, norms, max_len):
    s = Step(device, 1, [200, 0, 33, 90], [9, 4, 16, 1], page=page, block=block, norms=norms, max_len=max_len)
    before = s.held()
    s.run()
    s.check(before)


def test_padded_batches_in_a_row(device):
    """Buffers for more tokens and requests than a step has; the cache goes from step to step."""
    s = Step(device, 2, [40, 77], [3, 5], capacity=40, requests=6)
    for seed, old, new in ((3, [43, 82, 0], [1, 1, 7]), (4, [5], [2]), (5, [100, 3, 0, 9, 60, 1], [16, 1, 2, 1, 12, 8])):
        s.set(seed, old, new)
        before = s.held()
        s.run()
        s.check(before)


def test_other_streams_beside_each_other(device):
    steps = [Step(device, 10 + i, [120, 30 * i, 60], [4, 9, 16]) for i in range(3)]
    before = [s.held() for s in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    for s, stream in zip(steps, streams):
        with torch.cuda.stream(stream):
            s.run()
    torch.cuda.synchronize()
    for s, b in zip(steps, before):
        s.check(b)


@pytest.mark.parametrize("max_len", [400, 3000])
def test_captured_steps_share_a_workspace(device, max_len):
    """Two graphs of steps over one workspace, replayed in turn over changing
    batches, with eager work between."""
    steps = [Step(device, 20 + i, [120, 60], [4, 9], capacity=40, requests=4, max_len=max_len) for i in range(2)]
    steps[1].workspace = steps[0].workspace
    torch.cuda.synchronize()
    graphs, stream = [], torch.cuda.Stream()
    for s in steps:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            s.run()
        graphs.append(graph)
    for i, (old, new) in enumerate((([120, 60], [4, 9]), ([0, 5, 300], [16, 1, 7]), ([33], [12]), ([16, 15, 1], [1, 1, 16]))):
        for s in steps:
            s.set(30 + i, old, new)
        before = [s.held() for s in steps]
        for graph in graphs:
            graph.replay()
        if i % 2:
            torch.cuda.synchronize()
        for s, b in zip(steps, before):
            s.check(b)


@pytest.mark.parametrize("page,block", [(1, 1), (16, 16)])
def test_turn_end_over_an_8_bit_cache(device, page, block):
    """The compaction's own lists drive the Reposition of two layers, behind its
    status word; the moved rows are the oracle's, and a decode over the
    compacted request reads them."""
    w = synth.workload("tiny")
    layouts = synth.compile_layouts(w)
    n = len(layouts[0].positions)
    rng = np.random.default_rng(3)
    hk, d = 2, 64
    total = 3 * (n + page)
    total -= total % 64
    caches = [layer(device, 50 + i, total, hk, d, "e4m3", block) for i in range(2)]
    before = [[(values(c), f64(s).copy()) for c, s in cache] for cache in caches]
    pages = rng.permutation(total // page)
    raw = np.arange(n)
    slots = pages[: -(-n // page)][raw // page] * page + raw % page
    fresh = pages[-(-n // page):]
    table = torch.full((1, n + 64), -1, dtype=torch.int32, device=device)
    table[0, :n] = torch.from_numpy(slots.astype(np.int32)).to(device)
    birth = torch.from_numpy(slots.astype(np.int32)).to(device)
    rows = torch.zeros(1, dtype=torch.int64, device=device)
    if page == 1:
        inputs = tables.pack_compaction_inputs(layouts, device)
        out = tables.allocate_outputs(inputs, device, generated_total=None)
        taken = torch.from_numpy(fresh[: len(out.copy_src)].astype(np.int32)).to(device)
        tables.compact_rows(inputs, table, rows, taken, out, birth_slots=birth)
        status = out.status
    else:
        inputs = tables.pack_paged_inputs(layouts, page, device)
        out = tables.allocate_paged_outputs(inputs, device)
        taken = torch.from_numpy(fresh[: int(inputs.fresh_pages[0])].astype(np.int32)).to(device)
        tables.compact_pages(inputs, table, rows, taken, out, birth_slots=birth)
        status = None
    rope_table = rope.make_table("plain", d, n + 10, base=10000.0, dtype=torch.float32, device=device)
    pointers = [torch.tensor([c[i][j].data_ptr() for c in caches], dtype=torch.int64, device=device)
                for j in (0, 1) for i in (0, 1)]
    (kc, ks), (vc, vs) = caches[0]
    kv8.reposition_kv8_layers(*pointers, kc, vc, ks, vs, out.copy_src, out.copy_dst, out.copy_pairs, rope_table,
                              scale_block=block, status=status)
    src, dst, pairs = (t.cpu().numpy() for t in (out.copy_src, out.copy_dst, out.copy_pairs))
    assert len(src) > 100
    at = rope_table.cpu().numpy()
    for cache, held in zip(caches, before):
        for i, ((codes, scales), (c, s)) in enumerate(zip(cache, held)):
            moved, units = oracle.moved_rows(c, s, src, pairs, at, block, d, True, np.float32, i == 0)
            oracle.store(c, s, moved, dst, block, "e4m3", units=units)
            np.testing.assert_array_equal(values(codes), c)
            np.testing.assert_array_equal(f64(scales), s)
    # one token decodes over what was kept
    kept = int(layouts[0].keep_mask.sum())
    compacted = table[0, :n][layouts[0].keep_mask.to(device)]
    q = torch.randn((1, 4, d), device=device).to(torch.bfloat16)
    result = torch.empty_like(q, dtype=torch.float32)
    indptr = lambda x: torch.tensor([0, x], dtype=torch.int32, device=device)  # noqa: E731
    kv8.attention_kv8(q, kc, vc, ks, vs, indptr(1), indptr(kept), compacted.contiguous(), result, scale=0.125,
                      max_len=kept, max_new=1, scale_block=block)
    dense = [c * np.repeat(s, block, 0)[..., None] for c, s in before[0]]
    slots = compacted.cpu().numpy()
    y, size, spread = drafts.tree_attention(f64(q), *dense, [(0, slots, np.ones((1, kept), dtype=bool))], 0.125)
    assert (np.abs(f64(result) - y) <= kv8_tolerance(torch.bfloat16, torch.float32, kept, y, size, spread)).all()


def test_rows_and_scales_travel(device):
    """The handoff's row copy takes codes and, at a scale a token, scales as they are."""
    hk, d, n = 4, 64, 33
    source, target = (layer(device, 70 + i, 128, hk, d, "e4m3", 1) for i in range(2))
    src = torch.randperm(128, device=device)[:n].int()
    dst = torch.randperm(128, device=device)[:n].int()
    address = lambda t: torch.tensor([t.data_ptr()], dtype=torch.int64, device=device)  # noqa: E731
    for j, dtype in ((0, torch.uint8), (1, torch.float32)):
        (a, b), (x, y) = ([part[j].view(dtype).view(128, hk, -1) for part in cache] for cache in (source, target))
        transfer.copy_kv_rows(address(a), address(b), a, address(x), address(y), x, n, src_slots=src, dst_slots=dst)
        assert torch.equal(x[dst.long()], a[src.long()]) and torch.equal(y[dst.long()], b[src.long()])
