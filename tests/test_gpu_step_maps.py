"""The metadata of a step's new tokens on the GPU against the oracle."""

import functools

import numpy as np
import pytest
import torch

from akv_amd import page_table
from oracle import drafts
from tests.drafts import random_tree

pytestmark = pytest.mark.gpu


class Batch:
    """Requests of ``old + new`` ranks; some with registry rows (kept tokens,
    positions with gaps or dense), some with side rows, some with holes."""

    def __init__(self, device, seed, old, new, *, kept, gaps=True, side=False, holes=0, page=1, extra_generated=0):
        rng = np.random.default_rng(seed)
        self.new, self.keep_alive = list(new), []
        B, width = len(old), 8
        plan = []
        for b, (o, n) in enumerate(zip(old, new)):
            is_kept = bool(kept[b]) and o > 0
            active = max(1, o - extra_generated) if is_kept else o
            raw = np.sort(rng.choice(4 * active + 3, active, replace=False)) if is_kept else np.arange(o)
            prompt = int(raw[-1]) + 1 + int(rng.integers(0, 3)) if is_kept else 0
            if is_kept:
                columns = np.concatenate((raw, prompt + np.arange(o + n - active)))
                pos = np.sort(rng.choice(3 * active + 5, active, replace=False)) if gaps else np.arange(active)
                nxt = int(pos[-1]) + 1 + int(rng.integers(0, 9))
                positions = np.concatenate((pos, nxt + np.arange(o + n - active)))
            else:
                columns = positions = np.arange(o + n)
                pos, nxt = None, 0
            plan.append((is_kept, raw, prompt, active, pos, nxt, columns, positions))
            width = max(width, int(columns[-1]) + 1 if len(columns) else 0)
        table = rng.integers(1, 1 << 20, (B + 2, width)).astype(np.int32) * page
        rows = rng.permutation(B + 2)[:B]
        registry = np.zeros((B + 2, 6), dtype=np.int64)
        self.requests = []
        for b, (is_kept, raw, prompt, active, pos, nxt, columns, positions) in enumerate(plan):
            r = rows[b]
            for _ in range(holes):
                table[r, rng.integers(0, width)] = -1
            if is_kept:
                arrays = [torch.from_numpy(np.asarray(x, dtype=np.int32)).to(device) for x in (raw, pos)]
                self.keep_alive += arrays
                registry[r] = (arrays[0].data_ptr(), arrays[1].data_ptr(), prompt, active, nxt, 0)
            row = table[r]
            if side and b % 2:
                own = torch.from_numpy(rng.integers(1, 1 << 20, width).astype(np.int32) * page).to(device)
                self.keep_alive.append(own)
                registry[r, 5] = own.data_ptr()
                row = own.cpu().numpy()
            self.requests.append((row[columns], positions))
        put = lambda a, t=np.int64: torch.from_numpy(np.asarray(a, dtype=t)).to(device)  # noqa: E731
        self.device, self.registry, self.table, self.rows = device, put(registry), put(table, np.int32), put(rows)
        self.seq, self.fresh = put([o + n for o, n in zip(old, new)]), put(new)
        self.trees = [random_tree(rng, n) if n else [] for n in new]


def _run(b, *, page=1, window=None, tree=True, words=None, capacity=None, pages=None, dtypes=(torch.int32,) * 3,
         masks=True, blocks=True):
    total, device = sum(b.new), b.device
    capacity = total if capacity is None else capacity
    words = words or max(1, -(-max(b.new + [1]) // 64))
    longest = max([len(s) for s, _ in b.requests] + [1])
    pages = -(-longest // page) + 2 if pages is None else pages
    indptr, slots, positions = dtypes
    full = lambda shape, dtype: torch.full(shape, 77, dtype=dtype, device=device)  # noqa: E731
    out = dict(qo_indptr=full((len(b.new) + 1,), indptr), kv_indptr=full((len(b.new) + 1,), indptr),
               slot_map=full((capacity,), slots), positions=full((capacity,), positions),
               block_tables=full((len(b.new), pages), torch.int32) if blocks else None,
               tree_mask=full((capacity, words), torch.int64) if masks else None,
               window_mask=full((capacity, words), torch.int64) if window is not None and masks else None,
               window_starts=full((capacity,), torch.int32) if window is not None else None)
    parents = None
    if tree:
        flat = np.concatenate([np.asarray(t, dtype=np.int32) for t in b.trees] + [np.zeros(capacity, np.int32)])
        parents = torch.from_numpy(flat[:capacity].copy()).to(device)
    page_table.context_step_maps(
        b.registry, b.table, b.rows, b.seq, b.fresh, out["qo_indptr"], out["kv_indptr"], out["slot_map"],
        out["positions"], block_tables=out["block_tables"], page_size=page, parents=parents,
        tree_mask=out["tree_mask"], window=window, window_mask=out["window_mask"], window_starts=out["window_starts"])
    want = drafts.step_maps(b.requests, b.new, page_size=page, pages=pages, parents=b.trees if tree else None,
                            words=words, window=window, capacity=capacity)
    for name, got in out.items():
        if got is not None:
            np.testing.assert_array_equal(got.cpu().numpy(), want[name], err_msg=name)


@pytest.mark.parametrize("window", [None, 0, 5, 128])
@pytest.mark.parametrize("page", [1, 16, 3])
def test_matches_oracle(device, page, window):
    print(f"step maps page {page} window {window}", flush=True)
    b = Batch(device, page, [300, 0, 1, 64, 900, 17], [4, 3, 1, 0, 33, 16], kept=[1, 0, 1, 1, 1, 0], page=page)
    for tree in (True, False):
        _run(b, page=page, window=window, tree=tree)


@pytest.mark.parametrize("gaps", [True, False])
def test_windows_over_positions(device, gaps):
    """First keys of windows of every width, over gaps and dense positions."""
    b = Batch(device, 5, [2000, 30, 5, 700], [60, 9, 40, 2], kept=[1, 1, 1, 1], gaps=gaps, extra_generated=6)
    for window in (0, 1, 2, 30, 100, 1500, 2 ** 31 - 1):
        print(f"step maps window {window} gaps {gaps}", flush=True)
        _run(b, window=window)


def test_large_trees_and_few_words(device):
    """More than a word of nodes, more nodes than words hold, and trees longer
    than what a workgroup stages."""
    b = Batch(device, 6, [50, 3], [130, 65], kept=[1, 0])
    _run(b, window=9)
    _run(b, window=9, words=1)
    _run(b, window=9, words=5)
    deep = Batch(device, 7, [20], [2500], kept=[1])
    _run(deep, window=100)
    _run(deep, window=100, tree=False)


def test_padding_types_and_capacity(device):
    b = Batch(device, 8, [40, 90, 7], [3, 1, 8], kept=[0, 1, 1], side=True, holes=5)
    for dtypes in ((torch.int32, torch.int64, torch.int64), (torch.int64, torch.int32, torch.int32)):
        _run(b, capacity=sum(b.new) + 700, dtypes=dtypes, window=20)
    b.rows, b.seq, b.fresh = b.rows.int(), b.seq.int(), b.fresh.int()
    _run(b, blocks=False, masks=False)
    _run(b, pages=2, page=16)  # a table narrower than the requests
    _run(b, pages=0)


def test_more_new_tokens_than_ranks(device):
    """new_lens is held to the length, and no further than the capacity."""
    b = Batch(device, 9, [0, 0], [5, 2], kept=[0, 0])
    b.fresh = torch.tensor([9, -3], device=device)
    b.new = [5, 0]
    b.trees = [random_tree(np.random.default_rng(1), 5), []]
    _run(b)
    out = [torch.full((3,), 7, dtype=torch.int32, device=device) for _ in range(2)]
    maps = torch.full((4,), 7, dtype=torch.int64, device=device)
    page_table.context_step_maps(b.registry, b.table, b.rows, b.seq, b.fresh, *out, maps[:3], maps[:3].clone())
    assert out[0].tolist() == [0, 5, 5] and maps[3] == 7


def test_prefill_chunks_and_many_requests(device):
    rng = np.random.default_rng(3)
    b = Batch(device, 10, [100, 0], [5000, 3000], kept=[1, 0])
    _run(b, tree=False, masks=False, window=100, page=16)
    old, new = rng.integers(0, 60, 700), rng.integers(0, 9, 700)
    many = Batch(device, 11, old.tolist(), new.tolist(), kept=rng.random(700) < 0.5)
    _run(many, window=12)


def test_empty_batch_and_closed_gate(device):
    empty = torch.zeros(0, dtype=torch.int64, device=device)
    qo, kv = (torch.full((1,), 7, dtype=torch.int32, device=device) for _ in range(2))
    slots, positions = (torch.full((5,), 7, dtype=torch.int64, device=device) for _ in range(2))
    b = Batch(device, 12, [9], [2], kept=[0])
    page_table.context_step_maps(b.registry, b.table, empty, empty, empty, qo, kv, slots, positions)
    assert qo.item() == 0 and kv.item() == 0 and (slots == -1).all() and (positions == 0).all()
    qo, kv = (torch.full((2,), 7, dtype=torch.int32, device=device) for _ in range(2))
    page_table.context_step_maps(b.registry, b.table, b.rows, b.seq, b.fresh, qo, kv, slots, positions,
                                 status=torch.tensor([2], dtype=torch.int32, device=device))
    assert (qo == 7).all() and (slots == -1).all()


@pytest.mark.parametrize("copies", [1, 17])
def test_long_requests_on_both_sides_of_the_batch_rule(device, copies):
    """Requests that take every workgroup a request may have (chains, which need
    no ancestors: positions ascend by one from the root's)."""
    for old, new, kept, window in (([230000] + [5] * (copies - 1), [70000] + [3] * (copies - 1), [1] + [0] * (copies - 1), 100),
                                   ([9000] * copies, [1200] * copies, [1] * copies, None)):
        print(f"step maps {copies} requests of {old[0]} + {new[0]}", flush=True)
        b = Batch(device, 20 + copies + len(kept), old, new, kept=kept, holes=3)
        total, longest = sum(new), max(len(s) for s, _ in b.requests)
        full = lambda *shape, t=torch.int32: torch.full(shape, 77, dtype=t, device=device)  # noqa: E731
        qo, kv, table = full(copies + 1), full(copies + 1), full(copies, longest + 2)
        slot_map, positions, starts = full(total, t=torch.int64), full(total, t=torch.int64), full(total)
        page_table.context_step_maps(b.registry, b.table, b.rows, b.seq, b.fresh, qo, kv, slot_map, positions,
                                     block_tables=table, window=window, window_starts=starts if window else None)
        want = dict(slots=[], positions=[], starts=[])
        for r, ((slots, pos), o, n) in enumerate(zip(b.requests, old, new)):
            row = np.full(longest + 2, -1)
            row[: len(slots)] = np.maximum(slots, -1)
            np.testing.assert_array_equal(table[r].cpu().numpy(), row)
            at = pos[o] + np.arange(n)
            want["slots"].append(slots[o:])
            want["positions"].append(at)
            want["starts"].append(np.searchsorted(pos[:o], at - (window or 0)))
        np.testing.assert_array_equal(qo.cpu().numpy(), np.concatenate(([0], np.cumsum(new))))
        np.testing.assert_array_equal(kv.cpu().numpy(), np.concatenate(([0], np.cumsum(np.add(old, new)))))
        np.testing.assert_array_equal(slot_map.cpu().numpy(), np.concatenate(want["slots"]))
        np.testing.assert_array_equal(positions.cpu().numpy(), np.concatenate(want["positions"]))
        if window:
            np.testing.assert_array_equal(starts.cpu().numpy(), np.concatenate(want["starts"]))


def test_side_rows_beside_a_table_without_columns(device):
    """Requests whose rows all lie elsewhere: the table need not hold anything."""
    b = Batch(device, 30, [0, 50, 0, 9], [0, 4, 0, 3], kept=[0, 1, 0, 0], side=True)
    b.table = b.table[:, :0].clone()
    assert b.table.data_ptr() == 0
    _run(b, window=20)


@pytest.mark.parametrize("gaps", [True, False])
@pytest.mark.parametrize("active", ["some", "all", "beyond"])
def test_chunks_that_begin_among_the_active_ranks(device, monkeypatch, active, gaps):
    """A prompt's next chunk: some or all of its ranks, or not even the last of
    them, are the registry's kept tokens, whose positions have gaps."""
    monkeypatch.setattr(drafts, "step_maps", functools.partial(drafts.step_maps, chunk=True))
    old, new = [300, 1, 90, 20, 5], [70, 300, 64, 20, 600]
    extra = {"some": 20, "all": 20, "beyond": 20}[active]
    if active == "all":
        new = [20] * 5
    b = Batch(device, 40, old, new, kept=[1, 1, 1, 0, 1], gaps=gaps, extra_generated=-extra)
    if active == "beyond":
        # the batch ends 5 ranks before the active ones do
        new = [15] * 5
        b.new = new
        b.requests = [(s[: o + 15], p[: o + 15]) for (s, p), o in zip(b.requests, old)]
        b.seq, b.fresh = (torch.tensor(x, device=device) for x in ([o + 15 for o in old], new))
        b.trees = [random_tree(np.random.default_rng(2), 15) for _ in old]
    for window in (None, 0, 1, 9, 100, 5000, 2 ** 31 - 1):
        for tree in (False, True):
            print(f"step maps chunk {active} window {window} tree {tree}", flush=True)
            _run(b, window=window, tree=tree, page=1)
    _run(b, window=9, tree=False, words=1)


@pytest.mark.parametrize("row", [-1, 10 ** 6, 2 ** 40])
def test_requests_without_ranks_may_name_any_row(device, row):
    """What a padded batch leaves in its last rows is not followed."""
    b = Batch(device, 50, [30, 0, 900, 0, 0], [4, 0, 9, 0, 0], kept=[1, 0, 1, 0, 0])
    b.rows[b.seq == 0] = row
    for window in (None, 20):
        _run(b, window=window, capacity=20)


def test_the_largest_batch(device):
    """65534 requests, most of them of one new token."""
    rng = np.random.default_rng(8)
    old, new = rng.integers(0, 5, 65534), np.minimum(rng.integers(0, 9, 65534), 2) // 2
    kept = rng.random(65534) < 0.001
    b = Batch(device, 60, old.tolist(), new.tolist(), kept=kept)
    _run(b, window=2, tree=False)
