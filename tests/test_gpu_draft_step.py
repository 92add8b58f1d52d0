"""The step that verifies drafted tokens, its operators one behind the other as a
serving loop calls them: metadata, norms with the pool write, attention of a
full and of a sliding-window layer; eagerly, on another stream, in a captured
graph, and beside the operators it stands next to."""

import numpy as np
import pytest
import torch

from akv_amd import attention, context_attention, ops, page_table, qk_norm, rope
from oracle import drafts
from tests.drafts import HALF, attention_tolerance, f64, random_tree

pytestmark = pytest.mark.gpu
EPS, WINDOW = 1e-6, 24


class Step:
    """A batch of requests with registry rows over one layer's pool, and buffers
    of a fixed capacity for its drafted tokens."""

    def __init__(self, device, seed, old, new, *, page=1, q_heads=8, kv_heads=2, d=64, capacity=None, requests=None,
                 max_new=16, max_len=400):
        self.device, self.page, self.d, self.hq, self.hk = device, page, d, q_heads, kv_heads
        self.old, self.new = list(old), list(new)
        self.batch, self.capacity = requests or len(old), capacity or sum(new)
        self.max_len, self.max_new = max_len, max_new
        self.slots = 1024
        gen = torch.Generator().manual_seed(seed)
        make = lambda *shape: torch.randn(shape, generator=gen).to(torch.bfloat16).to(device)  # noqa: E731
        self.k, self.v = make(self.slots * page, kv_heads, d), make(self.slots * page, kv_heads, d)
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
        self.raw, self.pos = torch.zeros(4096, **i32), torch.zeros(4096, **i32)
        self.qo, self.kv = torch.zeros(self.batch + 1, **i32), torch.zeros(self.batch + 1, **i32)
        self.slot_map, self.positions = torch.zeros(self.capacity, **i64), torch.zeros(self.capacity, **i64)
        self.blocks = torch.zeros((self.batch, -(-max_len // page)), **i32)
        self.mask, self.near = torch.zeros((self.capacity, 1), **i64), torch.zeros((self.capacity, 1), **i64)
        self.starts = torch.zeros(self.capacity, **i32)
        self.q = torch.zeros((self.capacity, q_heads, d), dtype=torch.bfloat16, device=device)
        self.out, self.win = torch.zeros_like(self.q), torch.zeros_like(self.q)
        need = attention.tree_workspace_bytes(self.capacity, self.batch, q_heads, kv_heads, d, max_len, max_new)
        self.workspace = torch.empty(need, dtype=torch.uint8, device=device)
        self.set(seed, old, new)

    def set(self, seed, old, new):
        """Another batch in the same buffers (padded with empty requests)."""
        rng = np.random.default_rng(seed)
        self.old = list(old) + [0] * (self.batch - len(old))
        self.new = list(new) + [0] * (self.batch - len(new))
        ids = rng.permutation(self.slots)
        self.requests, at, kept_at = [], 0, 0
        table = np.full(tuple(self.table.shape), -1, dtype=np.int32)
        registry = np.zeros((self.batch, 6), dtype=np.int64)
        raw_all, pos_all = np.zeros(4096, np.int32), np.zeros(4096, np.int32)
        for b, (o, n) in enumerate(zip(self.old, self.new)):
            rank = np.arange(o + n)
            own = ids[at: at + -(-(o + n) // self.page)]
            at += len(own)
            slots = own[rank // self.page] * self.page + rank % self.page if o + n else rank
            columns, positions = rank, rank
            if o and b % 2 == 0:  # kept tokens, positions with gaps
                raw = np.sort(rng.choice(2 * o, o, replace=False))
                pos = np.sort(rng.choice(2 * o, o, replace=False))
                columns = np.concatenate((raw, raw[-1] + 1 + np.arange(n)))
                positions = np.concatenate((pos, pos[-1] + 1 + np.arange(n)))
                registry[b] = (self.raw.data_ptr() + 4 * kept_at, self.pos.data_ptr() + 4 * kept_at, raw[-1] + 1, o,
                               pos[-1] + 1, 0)
                raw_all[kept_at: kept_at + o], pos_all[kept_at: kept_at + o] = raw, pos
                kept_at += o
            table[b, columns] = slots
            self.requests.append((slots, positions))
        self.trees = [random_tree(rng, n) if n else [] for n in self.new]
        parents = np.zeros(self.capacity, np.int32)
        flat = np.concatenate([np.asarray(t, np.int32) for t in self.trees] + [np.zeros(0, np.int32)])
        parents[: len(flat)] = flat
        for to, a in ((self.table, table), (self.registry, registry), (self.raw, raw_all), (self.pos, pos_all),
                      (self.seq, np.add(self.old, self.new)), (self.fresh, self.new), (self.parents, parents)):
            to.copy_(torch.from_numpy(np.ascontiguousarray(a)).to(to.dtype))
        gen = torch.Generator().manual_seed(seed + 7)
        self.qkv.copy_(torch.randn(tuple(self.qkv.shape), generator=gen).to(torch.bfloat16))

    def run(self):
        hq, hk = self.hq, self.hk
        page_table.context_step_maps(
            self.registry, self.table, self.rows, self.seq, self.fresh, self.qo, self.kv, self.slot_map, self.positions,
            block_tables=self.blocks, page_size=self.page, parents=self.parents, tree_mask=self.mask, window=WINDOW,
            window_mask=self.near, window_starts=self.starts)
        q, k, v = self.qkv.split((hq, hk, hk), 1)
        qk_norm.qk_norm_rope(q, k, v, *self.weights, self.positions, self.rope, self.q, eps=EPS,
                             slot_map=self.slot_map, k_buffer=self.k, v_buffer=self.v)
        args = (self.q, self.k, self.v, self.qo, self.kv, self.blocks)
        common = dict(scale=self.d ** -0.5, max_new=self.max_new, page_size=self.page, sinks=self.sinks,
                      workspace=self.workspace)
        attention.tree_attention(*args, self.out, max_len=self.max_len, tree_mask=self.mask, **common)
        attention.tree_attention(*args, self.win, max_len=WINDOW + self.max_new + 1, tree_mask=self.near,
                                 key_starts=self.starts, **common)

    def check(self):
        want = drafts.step_maps(self.requests, self.new, page_size=self.page, pages=self.blocks.shape[1],
                                parents=self.trees, window=WINDOW, capacity=self.capacity)
        got = dict(qo_indptr=self.qo, kv_indptr=self.kv, slot_map=self.slot_map, positions=self.positions,
                   block_tables=self.blocks, tree_mask=self.mask, window_mask=self.near, window_starts=self.starts)
        for name, t in got.items():
            np.testing.assert_array_equal(t.cpu().numpy(), want[name], err_msg=name)
        total = int(want["qo_indptr"][-1])
        at = f64(self.rope)[want["positions"][:total]]
        heads = {"q": (slice(0, self.hq), self.q[:total]),
                 "k": (slice(self.hq, self.hq + self.hk), self.k[self.slot_map[:total]])}
        for i, (name, (of, have)) in enumerate(heads.items()):
            y, size = drafts.qk_norm_rope(f64(self.qkv[:total, of]), f64(self.weights[i]), EPS, at, self.d, True)
            tol = (self.d / 2 + 10) * 2.0 ** -24 * size + HALF[torch.bfloat16] * np.abs(y) * 1.001 + 1e-37
            assert (np.abs(f64(have) - y) <= tol).all(), name
        assert torch.equal(self.v[self.slot_map[:total]], self.qkv[:total, self.hq + self.hk:])
        for out, limit in ((self.out, None), (self.win, WINDOW)):
            requests, first = [], 0
            for (slots, _), o, n, tree in zip(self.requests, self.old, self.new, self.trees):
                seen = np.ones((n, o + n), dtype=bool)
                if limit is not None:
                    seen[:, :o] = np.arange(o)[None] >= want["window_starts"][first: first + n, None]
                seen[:, o:] = drafts.ancestors(tree, limit)
                requests.append((first, slots, seen))
                first += n
            y, size, spread = drafts.tree_attention(f64(self.q), f64(self.k), f64(self.v), requests, self.d ** -0.5,
                                                    f64(self.sinks))
            tol = attention_tolerance(torch.bfloat16, torch.bfloat16, self.max_len, y, size, spread, 0)
            assert (np.abs(f64(out) - y)[:total] <= tol[:total]).all(), limit


@pytest.mark.parametrize("page", [1, 16])
def test_step_in_order(device, page):
    s = Step(device, 1, [200, 0, 33, 90], [9, 4, 16, 1], page=page)
    s.run()
    s.check()
    s.set(2, [5, 300, 64], [16, 2, 7])
    s.run()
    s.check()


def test_padded_batch(device):
    """A batch in buffers made for a larger one: what lies behind its last token
    stays out of the pool and of the outputs."""
    s = Step(device, 3, [150, 40], [7, 5], capacity=40, requests=6)
    pool = s.k.clone()
    s.out.fill_(7)
    s.run()
    s.check()
    assert (s.out[12:] == 7).all()
    untouched = torch.ones(s.k.shape[0], dtype=torch.bool, device=device)
    untouched[s.slot_map[:12]] = False
    assert torch.equal(s.k[untouched], pool[untouched])


def test_other_streams_beside_each_other(device):
    """Two batches on two streams, each with its own workspace."""
    steps = [Step(device, 10 + i, [300, 120 + i], [16, 9]) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device) for _ in steps]
    for _ in range(4):
        for s, stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                s.run()
    torch.cuda.synchronize()
    for s in steps:
        s.check()


def test_captured_step_follows_its_inputs(device):
    """One captured step, replayed for batches of other lengths and trees, with
    eager work between the replays; two graphs of the same buffers."""
    s = Step(device, 20, [100, 60, 7], [8, 3, 16], capacity=48, requests=5)
    eager = Step(device, 20, [100, 60, 7], [8, 3, 16], capacity=48, requests=5)
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        s.run()  # what a first call sets up
    torch.cuda.current_stream(device).wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            s.run()
        graphs.append(graph)
    batches = [([100, 60, 7], [8, 3, 16]), ([350], [16]), ([0, 1, 2, 3, 4], [1, 2, 3, 4, 5]), ([30, 0, 200], [0, 16, 6])]
    for i, (old, new) in enumerate(batches * 2):
        print(f"captured draft step, replay {i}", flush=True)
        for t in (s, eager):
            t.set(40 + i, old, new)
        graphs[i % 2].replay()
        eager.k.copy_(s.k), eager.v.copy_(s.v)
        eager.run()
        torch.cuda.synchronize()
        s.check()
        total = sum(new)
        assert torch.equal(s.out[:total], eager.out[:total]) and torch.equal(s.win[:total], eager.win[:total])


def test_one_token_is_a_decode_step(device):
    """A tree of one token: decode attention over the same slots."""
    s = Step(device, 30, [300, 5, 129], [1, 1, 1])
    s.run()
    s.check()
    total = int(s.kv[-1])
    indices = torch.zeros(total, dtype=torch.int32, device=device)
    page_table.context_decode_indices(s.registry, s.table, s.rows, s.seq, s.kv, indices)
    outs = [torch.empty_like(s.q) for _ in range(2)]
    attention.decode_attention(s.q, s.k, s.v, s.kv, indices, outs[0], scale=0.125, max_len=400, sinks=s.sinks)
    attention.tree_attention(s.q, s.k, s.v, s.qo, s.kv, indices, outs[1], scale=0.125, max_len=400, max_new=1,
                             tree_mask=s.mask, sinks=s.sinks)
    requests = [(b, slots, np.ones((1, len(slots)), dtype=bool)) for b, (slots, _) in enumerate(s.requests)]
    y, size, spread = drafts.tree_attention(f64(s.q), f64(s.k), f64(s.v), requests, 0.125, f64(s.sinks))
    tol = attention_tolerance(torch.bfloat16, torch.bfloat16, 400, y, size, spread, 0)
    for out in outs + [s.out]:
        assert (np.abs(f64(out) - y) <= tol).all()


def test_a_chain_is_an_extend_forward(device):
    """Drafts without branches: extend attention over the same prefix."""
    s = Step(device, 31, [257, 31], [12, 5])
    s.trees = [list(range(-1, n - 1)) for n in s.new]
    s.parents.copy_(torch.tensor(sum(s.trees, []), dtype=torch.int32))
    s.run()
    s.check()
    prefix = torch.cat([torch.from_numpy(slots[:o].astype(np.int32)) for (slots, _), o in zip(s.requests, s.old)])
    kv = torch.tensor(np.concatenate(([0], np.cumsum(s.old))), dtype=torch.int32, device=device)
    out = torch.empty_like(s.q)
    at = s.slot_map
    context_attention.extend_attention_fwd(s.q, s.k[at], s.v[at], out, s.k, s.v, s.qo, kv, prefix.to(device), None, True,
                                           None, 12, sm_scale=0.125, sinks=s.sinks)
    # both are within their bound of the same 64-bit rows
    assert (out.float() - s.out.float()).abs().max() <= 2 * 2 ** -7 * s.v.abs().max().float()


def test_stored_keys_move_as_the_reposition_moves_them(device):
    """Keys normed at one position and repositioned to another are the keys
    normed there, up to the two roundings to bf16."""
    d, n = 64, 40
    s = Step(device, 32, [0], [n], capacity=n, max_new=n)
    s.run()
    src = s.slot_map.int()
    taken = set(src.tolist())
    dst = torch.tensor([i for i in range(s.slots) if i not in taken][:n], dtype=torch.int32, device=device)
    target = torch.randint(0, 2000, (n,), generator=torch.Generator().manual_seed(3)).to(device)
    pairs = torch.stack((s.positions, target), 1).int()
    ptr = lambda t: torch.tensor([t.data_ptr()], dtype=torch.int64, device=device)  # noqa: E731
    ops.reposition_kv_layers(ptr(s.k), ptr(s.v), s.k, s.v, src, dst, pairs, s.rope)
    k = s.qkv[:, s.hq: s.hq + s.hk]
    want, _ = drafts.qk_norm_rope(f64(k), f64(s.weights[1]), EPS, f64(s.rope)[target.cpu().numpy()], d, True)
    # the stored pair is off by at most half a step in each half; a rotation
    # carries both into each result, which is rounded again
    pair = np.abs(want) + np.abs(np.roll(want, d // 2, -1))
    tol = 2.0 ** -8 * 1.5 * pair + 2.0 ** -8 * np.abs(want) + 1e-5 * pair
    assert (np.abs(f64(s.k[dst.long()]) - want) <= tol).all()
    assert torch.equal(s.v[dst.long()], s.v[src.long()])


class CutStep(Step):
    """A step whose full layer is cut into pieces and merged: its bound is past
    what one workgroup takes, as a server's is, however short the requests are."""

    def __init__(self, *args, max_len=5000, **more):
        super().__init__(*args, max_len=max_len, **more)
        assert self.workspace.numel() > 16

    def check(self):
        # errors are counted by the keys that are there
        bound, self.max_len = self.max_len, max(np.add(self.old, self.new))
        super().check()
        self.max_len = bound


@pytest.mark.parametrize("d,q_heads,page", [(64, 8, 1), (64, 16, 16), (128, 8, 1)])
def test_cut_step_in_order(device, d, q_heads, page):
    s = CutStep(device, 41, [400, 0, 33, 290], [9, 4, 16, 1], page=page, d=d, q_heads=q_heads)
    s.run()
    s.check()
    s.set(42, [5, 700, 64], [16, 2, 7])
    s.run()
    s.check()


def test_cut_padded_batch(device):
    s = CutStep(device, 43, [500, 140], [7, 5], capacity=40, requests=6)
    pool = s.k.clone()
    s.out.fill_(7)
    s.run()
    s.check()
    assert (s.out[12:] == 7).all()
    untouched = torch.ones(s.k.shape[0], dtype=torch.bool, device=device)
    untouched[s.slot_map[:12]] = False
    assert torch.equal(s.k[untouched], pool[untouched])


def test_cut_steps_on_streams_beside_each_other(device):
    """Each stream with its own workspace: neither's pieces reach the other."""
    steps = [CutStep(device, 50 + i, [700, 120 + i], [16, 9]) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device) for _ in steps]
    for _ in range(20):
        for s, stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                s.run()
    torch.cuda.synchronize()
    for s in steps:
        s.check()


def test_cut_captured_steps_share_a_workspace(device):
    """Two graphs over one workspace, replayed in turn for batches that leave
    other pieces and owners in it, with eager work of the same between them."""
    s = CutStep(device, 60, [400, 60, 7], [8, 3, 16], capacity=48, requests=5)
    eager = CutStep(device, 60, [400, 60, 7], [8, 3, 16], capacity=48, requests=5)
    eager.workspace = s.workspace
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        s.run()
    torch.cuda.current_stream(device).wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            s.run()
        graphs.append(graph)
    batches = [([400, 60, 7], [8, 3, 16]), ([900], [16]), ([0, 1, 2, 3, 4], [1, 2, 3, 4, 5]), ([30, 0, 500], [0, 16, 6])]
    for i, (old, new) in enumerate(batches * 2):
        print(f"cut captured step, replay {i}", flush=True)
        for t in (s, eager):
            t.set(70 + i, old, new)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        s.check()
        eager.k.copy_(s.k), eager.v.copy_(s.v)
        eager.run()
        torch.cuda.synchronize()
        total = sum(new)
        assert torch.equal(s.out[:total], eager.out[:total]) and torch.equal(s.win[:total], eager.win[:total])
