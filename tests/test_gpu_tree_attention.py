"""Tree attention on the GPU against the 64-bit oracle, at the sizes, layouts
and masks where it can go wrong."""

import numpy as np
import pytest
import torch

from akv_amd import attention
from oracle import drafts
from tests.drafts import Cache, attention_tolerance, f64

pytestmark = pytest.mark.gpu


def _run(c, *, mask, starts=None, sinks=None, out_dtype=None, scale=None, max_len=None, max_new=None, out=None,
         k=None, v=None, workspace=None, indptr=torch.int32, q=None):
    scale = c.q.shape[2] ** -0.5 if scale is None else scale
    if out is None:
        out = torch.full(c.q.shape, 7.0, dtype=out_dtype or c.q.dtype, device=c.device)
    attention.tree_attention(
        c.q if q is None else q, c.k.to(c.device) if k is None else k, c.v.to(c.device) if v is None else v,
        c.qo.to(indptr), c.kv.to(indptr), c.indices, out, scale=scale, max_len=c.max_len if max_len is None else max_len,
        max_new=c.max_new if max_new is None else max_new, page_size=c.page, tree_mask=mask,
        key_starts=None if starts is None else torch.tensor(starts, dtype=torch.int32, device=c.device), sinks=sinks,
        workspace=workspace)
    return out


def _check(c, out, requests, *, sinks=None, scale=None):
    scale = c.q.shape[2] ** -0.5 if scale is None else scale
    want, size, spread = drafts.tree_attention(f64(c.q), f64(c.k), f64(c.v), requests, scale,
                                               None if sinks is None else f64(sinks))
    got = f64(out)
    tol = attention_tolerance(c.q.dtype, out.dtype, c.max_len, want, size, spread, np.abs(f64(c.v)).max(initial=0.0))
    here = slice(0, c.total)
    off = np.abs(got - want)[here] - tol[here]
    assert not np.isnan(got[here]).any()
    assert (off <= 0).all(), f"{(off > 0).sum()} values off, worst by {off.max():.3g}"
    assert (got[c.total:] == 7.0).all(), "rows behind the last token were written"


SHAPES = [
    # q heads, kv heads, head_dim, dtype, page, old, new
    (8, 1, 64, torch.bfloat16, 1, [0], [1]),
    (8, 1, 64, torch.bfloat16, 1, [1], [1]),
    (2, 2, 64, torch.bfloat16, 1, [63, 64, 65, 0, 255, 256, 257], [1, 2, 3, 4, 5, 16, 17]),
    (16, 2, 64, torch.bfloat16, 1, [700, 0, 40, 300], [8, 5, 0, 33]),
    (16, 2, 64, torch.bfloat16, 16, [700, 3, 40, 300], [8, 5, 0, 33]),
    (16, 2, 64, torch.float16, 5, [511, 513, 1], [64, 65, 70]),
    (14, 2, 64, torch.bfloat16, 1, [1000, 129], [9, 100]),
    (3, 1, 128, torch.bfloat16, 1, [130, 127, 128, 0], [7, 11, 1, 40]),
    (16, 4, 128, torch.float16, 16, [1500, 10], [8, 32]),
    (12, 1, 128, torch.bfloat16, 1, [31, 33], [65, 130]),
    (6, 2, 96, torch.bfloat16, 1, [200, 90], [6, 21]),
    (4, 2, 80, torch.float16, 3, [200, 90], [6, 21]),
    (5, 1, 40, torch.bfloat16, 1, [77], [19]),
    (2, 1, 8, torch.float16, 1, [77, 5], [3, 64]),
]


@pytest.mark.parametrize("kind", ["chain", "tree", "any"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_matches_oracle(device, shape, kind):
    hq, hk, d, dtype, page, old, new = SHAPES[shape]
    print(f"tree attention shape {shape} {SHAPES[shape]} {kind}", flush=True)
    c = Cache(device, 100 + shape, old, new, q_heads=hq, kv_heads=hk, head_dim=d, dtype=dtype, page=page,
              capacity=sum(new) + shape % 3)
    seen, mask = c.masks(kind)
    sinks = torch.randn(hq, generator=torch.Generator().manual_seed(shape)).to(device) if shape % 2 else None
    out = _run(c, mask=mask, sinks=sinks, out_dtype=torch.float32 if kind == "any" else None,
               indptr=torch.int64 if kind == "tree" else torch.int32)
    _check(c, out, c.visible(seen), sinks=sinks)


@pytest.mark.parametrize("d,page", [(64, 1), (64, 16), (128, 1), (96, 4)])
def test_first_keys_of_a_window(device, d, page):
    """Windows that begin anywhere, behind every key, and below zero."""
    old, new = [900, 40, 0, 500], [6, 12, 3, 20]
    c = Cache(device, 7 + d, old, new, q_heads=4, kv_heads=2, head_dim=d, dtype=torch.bfloat16, page=page)
    rng = np.random.default_rng(d)
    starts = np.concatenate([rng.integers(max(0, o - 130), o + 1, n) for o, n in zip(old, new)])
    starts[:3] = [old[0], 0, old[0] - 1]
    passed = starts.copy()
    passed[3], starts[3] = -50, 0
    passed[4], starts[4] = 5000, old[0]  # past the earlier keys: none of them
    for kind in ("tree", "any"):
        print(f"tree attention windows d={d} page={page} {kind}", flush=True)
        seen, mask = c.masks(kind)
        out = _run(c, mask=mask, starts=passed, max_len=160)
        _check(c, out, c.visible(seen, starts))


def test_narrow_window_of_a_long_request(device):
    """Only the window's keys count, wherever the chunks begin."""
    old, new = [5000, 3000], [16, 7]
    c = Cache(device, 5, old, new, q_heads=8, kv_heads=2, head_dim=64, dtype=torch.bfloat16)
    seen, mask = c.masks("tree")
    starts = np.concatenate([np.full(n, o - 128) for o, n in zip(old, new)]) + np.arange(23) % 9
    sinks = torch.linspace(-3, 3, 8, device=device)
    out = _run(c, mask=mask, starts=starts, sinks=sinks, max_len=128 + 17)
    _check(c, out, c.visible(seen, starts), sinks=sinks)


@pytest.mark.parametrize("d", [64, 128])
def test_long_requests_in_many_chunks(device, d):
    old, new = [6000, 1, 2500], [3, 9, 16]
    c = Cache(device, 11 + d, old, new, q_heads=8, kv_heads=2, head_dim=d, dtype=torch.bfloat16)
    seen, mask = c.masks("tree")
    out = _run(c, mask=mask, out_dtype=torch.float32)
    _check(c, out, c.visible(seen))


def test_bounds_only_size_the_launch(device):
    """Bounds below and far above what the batch holds give the same rows."""
    c = Cache(device, 21, [1200, 30, 700], [20, 3, 9], q_heads=8, kv_heads=2, head_dim=64, dtype=torch.bfloat16)
    seen, mask = c.masks("tree")
    for max_len, max_new in ((c.max_len, c.max_new), (1, 1), (0, 0), (100000, 400), (300, 64)):
        print(f"tree attention bounds {max_len} {max_new}", flush=True)
        _check(c, _run(c, mask=mask, max_len=max_len, max_new=max_new), c.visible(seen))


@pytest.mark.parametrize("page", [1, 16])
def test_holes_are_not_read(device, page):
    """Slots outside the pool, and lists shorter than the lengths say."""
    c = Cache(device, 31, [400, 90], [5, 9], q_heads=4, kv_heads=2, head_dim=64, dtype=torch.bfloat16, page=page,
              holes=6)
    seen, mask = c.masks("tree")
    _check(c, _run(c, mask=mask), c.visible(seen))
    # the last request's entries end early
    if page == 1:
        cut = 40
        c.indices = c.indices[: -1 - cut].contiguous()
        c.slots[1][-cut:] = -1
    else:
        keep = 3
        c.indices = c.indices[:, :keep].contiguous()
        for s in c.slots:
            s[keep * page:] = -1
    _check(c, _run(c, mask=mask), c.visible(seen))


@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (128, torch.float16), (96, torch.bfloat16)])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan"), "lowest"])
def test_what_a_token_does_not_see_cannot_reach_it(device, d, dtype, value):
    """Infinities, NaN and the type's lowest value in keys and values that are
    hidden from some tokens; those that see them are left out here."""
    value = torch.finfo(dtype).min if value == "lowest" else value
    old, new = [130, 70], [12, 40]
    c = Cache(device, 41 + d, old, new, q_heads=4, kv_heads=2, head_dim=d, dtype=dtype)
    seen, mask = c.masks("any")
    starts = np.concatenate([np.full(n, 20) + np.arange(n) % 7 for n in new])
    # a drafted token's rows, and earlier keys below some or all starts
    bad = {0: [3, 21, 23, 130 + 4, 130 + 7], 1: [0, 24, 70 + 2, 70 + 33]}
    for b, ranks in bad.items():
        for r in ranks:
            c.v[c.slots[b][r], :, (5 * r) % d] = value
            if r % 2:
                c.k[c.slots[b][r], :, (3 * r) % d] = value
    out = f64(_run(c, mask=mask, starts=starts))
    clean = Cache(device, 41 + d, old, new, q_heads=4, kv_heads=2, head_dim=d, dtype=dtype)
    requests = c.visible(seen, starts)
    want, size, spread = drafts.tree_attention(f64(c.q), f64(clean.k), f64(clean.v), requests, d ** -0.5)
    tol = attention_tolerance(dtype, dtype, c.max_len, want, size, spread, np.abs(f64(clean.v)).max())
    checked = 0
    for b, (first, _, keys) in enumerate(requests):
        for i in range(len(keys)):
            if not keys[i][bad[b]].any():
                checked += 1
                assert (np.abs(out[first + i] - want[first + i]) <= tol[first + i]).all(), (b, i)
    assert checked >= 4
    # a token that sees a NaN or infinite value (its key untouched) has it in that dim
    if value != torch.finfo(dtype).min:
        hit = 0
        for b, (first, _, keys) in enumerate(requests):
            for r in bad[b]:
                for i in np.flatnonzero(keys[:, r]):
                    if r % 2 == 0 and not any(keys[i][o] for o in bad[b] if o % 2 and o != r):
                        hit += 1
                        assert not np.isfinite(out[first + i, :, (5 * r) % d]).any(), (b, i, r)
        assert hit


def test_nan_queries_stay_in_their_rows(device):
    c = Cache(device, 51, [300], [9], q_heads=8, kv_heads=2, head_dim=64, dtype=torch.bfloat16)
    seen, mask = c.masks("tree")
    clean = f64(_run(c, mask=mask))
    c.q[4, 3] = float("nan")
    out = f64(_run(c, mask=mask))
    assert np.isnan(out[4, 3]).all()
    out[4, 3] = clean[4, 3]
    np.testing.assert_array_equal(out, clean)


@pytest.mark.parametrize("scores", ["rising", "falling", "far"])
def test_scores_far_apart(device, scores):
    """Maxima that keep moving, by little and by more than fp32's range."""
    c = Cache(device, 61, [900], [10], q_heads=4, kv_heads=1, head_dim=64, dtype=torch.bfloat16)
    ramp = torch.linspace(-1, 1, 910) if scores != "far" else torch.where(torch.arange(910) % 300 == 299, 40.0, -1.0)
    c.k[:] = 0.01 * c.k
    c.k[torch.from_numpy(c.slots[0]), 0, 0] = ((-ramp if scores == "falling" else ramp) * 30).to(torch.bfloat16)
    c.q[:] = 0.01 * c.q
    c.q[:, :, 0] = 2.0
    seen, mask = c.masks("tree")
    _check(c, _run(c, mask=mask, scale=1.0, out_dtype=torch.float32), c.visible(seen), scale=1.0)


def test_strides(device):
    """q, K, V and out as views: padded heads, a pool of interleaved K and V, a
    wider table."""
    c = Cache(device, 71, [200, 60], [7, 4], q_heads=4, kv_heads=2, head_dim=64, dtype=torch.bfloat16, page=16)
    q = torch.zeros((c.total, 4, 80), dtype=torch.bfloat16, device=device)[:, :, 8:72]
    q.copy_(c.q)
    both = torch.stack((c.k, c.v), 2).to(device)  # [slots, heads, 2, dim]
    store = torch.full((c.total, 6, 64), 7.0, dtype=torch.bfloat16, device=device)
    c.indices = torch.nn.functional.pad(c.indices, (0, 5), value=123456)[:, : c.indices.shape[1]]
    seen, mask = c.masks("tree")
    mask = torch.nn.functional.pad(mask, (0, 3), value=-1)[:, : mask.shape[1]]
    out = _run(c, mask=mask, q=q, k=both[:, :, 0], v=both[:, :, 1], out=store[:, 1:5])
    _check(c, out, c.visible(seen))
    assert (store[:, 0] == 7).all() and (store[:, 5] == 7).all()


def test_one_workspace_for_changing_batches(device):
    """Whatever an earlier call left in a workspace does not matter."""
    shape = dict(q_heads=8, kv_heads=2, head_dim=64, dtype=torch.bfloat16)
    batches = [Cache(device, 81, [900, 10], [12, 3], **shape), Cache(device, 82, [40], [2], **shape),
               Cache(device, 83, [300, 2000, 5], [1, 16, 4], **shape)]
    need = max(attention.tree_workspace_bytes(c.capacity, len(c.new), 8, 2, 64, c.max_len, c.max_new) for c in batches)
    ws = torch.full((need,), 255, dtype=torch.uint8, device=device)
    for c in batches:
        seen, mask = c.masks("tree")
        _check(c, _run(c, mask=mask, workspace=ws), c.visible(seen))


def test_gate_and_empty_batches(device):
    c = Cache(device, 91, [30], [4], q_heads=4, kv_heads=2, head_dim=64, dtype=torch.bfloat16)
    out = torch.full(c.q.shape, 7.0, dtype=torch.bfloat16, device=device)
    closed = torch.tensor([1], dtype=torch.int32, device=device)
    attention.tree_attention(c.q, c.k.to(device), c.v.to(device), c.qo, c.kv, c.indices, out, scale=0.125, max_len=34,
                             max_new=4, status=closed)
    assert (out == 7).all()
    none = Cache(device, 92, [30, 0], [0, 0], q_heads=4, kv_heads=2, head_dim=64, dtype=torch.bfloat16, capacity=3)
    out = _run(none, mask=None)
    assert (out == 7).all()
    assert attention.tree_attention(c.q[:0], c.k.to(device), c.v.to(device), c.qo[:1], c.kv[:1], c.indices, c.q[:0],
                                    scale=0.125, max_len=0, max_new=0).numel() == 0


def test_random_batches(device):
    for seed in range(24):
        rng = np.random.default_rng(1000 + seed)
        b = int(rng.integers(1, 7))
        hi = int(rng.choice([5, 70, 400, 1200]))
        old, new = rng.integers(0, hi, b), rng.integers(0, int(rng.choice([2, 12, 70])), b)
        new[0] = max(new[0], 1)
        hk = int(rng.choice([1, 2, 3]))
        hq = hk * int(rng.choice([1, 2, 5, 8]))
        d = int(rng.choice([16, 64, 64, 72, 128]))
        dtype = torch.bfloat16 if rng.random() < 0.6 else torch.float16
        page = int(rng.choice([1, 1, 2, 16, 64]))
        spread = float(rng.choice([1.0, 3.0]))
        print(f"tree attention random {seed}: {old.tolist()} {new.tolist()} {hq}/{hk}x{d} page {page} {dtype}",
              flush=True)
        c = Cache(device, seed, old.tolist(), new.tolist(), q_heads=hq, kv_heads=hk, head_dim=d, dtype=dtype,
                  page=page, holes=int(rng.integers(0, 3)), spread=spread, capacity=int(sum(new)) + int(rng.integers(0, 4)))
        seen, mask = c.masks(str(rng.choice(["chain", "tree", "any"])))
        starts = None
        if rng.random() < 0.4:
            starts = np.concatenate([rng.integers(0, o + 1, n) for o, n in zip(old, new)])
        full = None if starts is None else np.concatenate((starts, np.zeros(c.capacity - c.total, np.int64)))
        sinks = torch.randn(hq, generator=torch.Generator().manual_seed(seed)).to(device) if seed % 2 else None
        _check(c, _run(c, mask=mask, starts=full, sinks=sinks), c.visible(seen, starts), sinks=sinks)


@pytest.mark.parametrize("bound", [1, 5000])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_whole_and_shared_out(device, shape, bound):
    """Every shape as one workgroup per block of rows, and on the line."""
    hq, hk, d, dtype, page, old, new = SHAPES[shape]
    print(f"tree attention shape {shape} {SHAPES[shape]} bound {bound}", flush=True)
    c = Cache(device, 200 + shape, old, new, q_heads=hq, kv_heads=hk, head_dim=d, dtype=dtype, page=page, holes=2)
    seen, mask = c.masks("any")
    starts = np.concatenate([c.rng.integers(0, o + 1, n) for o, n in zip(old, new)])
    sinks = torch.randn(hq, generator=torch.Generator().manual_seed(shape)).to(device) if shape % 2 == 0 else None
    _check(c, _run(c, mask=mask, max_len=bound, max_new=max(1, c.max_new // 3)), c.visible(seen))
    _check(c, _run(c, mask=mask, starts=starts, sinks=sinks, max_len=bound), c.visible(seen, starts), sinks=sinks)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bound", [1, 5000])
def test_trees_of_many_words(device, d, bound):
    """More drafted tokens than the mask words kept at hand, and words that end
    before the tokens do."""
    old, new = [300, 1], [200, 333]
    c = Cache(device, 300 + d, old, new, q_heads=4, kv_heads=2, head_dim=d, dtype=torch.bfloat16)
    starts = np.concatenate([c.rng.integers(0, o + 1, n) for o, n in zip(old, new)])
    for kind in ("chain", "tree", "any"):
        print(f"tree attention large trees d={d} bound {bound} {kind}", flush=True)
        seen, mask = c.masks(kind)
        _check(c, _run(c, mask=mask, starts=starts, max_len=bound), c.visible(seen, starts))
        if mask is None:
            continue
        short = [s.copy() for s in seen]
        for s in short:
            s[:, 192:] = False
        _check(c, _run(c, mask=mask[:, :3], max_len=bound), c.visible(short))


@pytest.mark.parametrize("bound", [1, 900, 5000])
def test_many_requests(device, bound):
    """More requests than a wave has lanes, empty ones among them."""
    rng = np.random.default_rng(9)
    old = [int(rng.integers(0, 900)) if i % 3 else 0 for i in range(150)]
    new = [0 if i % 7 == 3 or 64 <= i < 130 else int(rng.integers(0, 6)) for i in range(150)]
    c = Cache(device, 400, old, new, q_heads=6, kv_heads=3, head_dim=64, dtype=torch.float16)
    seen, mask = c.masks("tree")
    _check(c, _run(c, mask=mask, max_len=bound), c.visible(seen))
    c = Cache(device, 401, old, [20 if i == 149 else 0 for i in range(150)], q_heads=24, kv_heads=1, head_dim=64,
              dtype=torch.bfloat16)  # a block of rows that only the last request has
    seen, mask = c.masks("tree")
    _check(c, _run(c, mask=mask, max_len=bound), c.visible(seen))


@pytest.mark.parametrize("page", [1, 16])
def test_slots_past_32_bits(device, page):
    """A layer whose rows lie 2 MiB apart: offsets beyond 4 GiB in bytes."""
    c = Cache(device, 500 + page, [2300], [5], q_heads=4, kv_heads=2, head_dim=64, dtype=torch.bfloat16, page=page)
    stride, n = 1 << 20, c.k.shape[0]
    store = torch.empty(n * stride, dtype=torch.bfloat16, device=device)
    k, v = (store.as_strided((n, 2, 64), (stride, 64, 1), at) for at in (0, 4096))
    k.copy_(c.k), v.copy_(c.v)
    seen, mask = c.masks("tree")
    _check(c, _run(c, mask=mask, k=k, v=v), c.visible(seen))


@pytest.mark.parametrize("d,out_dtype", [(64, torch.float32), (128, torch.bfloat16), (96, torch.float32)])
def test_unaligned_outputs(device, d, out_dtype):
    for old in ([300, 20], [3000, 20]):
        c = Cache(device, 600 + d, old, [7, 4], q_heads=4, kv_heads=2, head_dim=d, dtype=torch.bfloat16)
        store = torch.full((c.total, 4, d + 3), 7.0, dtype=out_dtype, device=device)
        seen, mask = c.masks("tree")
        out = _run(c, mask=mask, out=store[:, :, 1: d + 1])
        _check(c, out, c.visible(seen))
        assert (store[:, :, 0] == 7).all() and (store[:, :, d + 1:] == 7).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [2, 40])
def test_maxima_that_jump_behind_the_first_tiles(device, d, dtype, new):
    """Keys that every token sees, their scores above the first ones' by more
    than a weight of the storage type can hold, in some rows only."""
    c = Cache(device, 700 + d, [1400], [new], q_heads=4, kv_heads=1, head_dim=d, dtype=dtype)
    c.k[:] = 0.01 * c.k
    c.q[:] = 0.01 * c.q
    ranks = torch.from_numpy(c.slots[0])
    jump = torch.zeros(1400 + new)
    for at, by in ((100, 6.0), (300, 12.0), (301, 13.0), (700, 40.0), (1200, 41.0)):
        jump[at] = by
    c.k[ranks, 0, 0] = jump.to(dtype)
    c.q[::2, 1:3, 0] = 2.0
    seen, mask = c.masks("tree")
    for bound in (1, 5000):
        _check(c, _run(c, mask=mask, scale=1.0, out_dtype=torch.float32, max_len=bound), c.visible(seen), scale=1.0)


@pytest.mark.parametrize("bound", [1, 5000])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_odd_values_in_pieces(device, value, bound):
    """Infinities and NaN of one dim: in the rows that see the key, that dim is
    not finite and the others are right; the other rows are."""
    old, new = [2000, 300], [6, 30]
    c = Cache(device, 800, old, new, q_heads=4, kv_heads=2, head_dim=64, dtype=torch.bfloat16)
    seen, mask = c.masks("any")
    starts = np.concatenate([np.linspace(0, o, n).astype(np.int64) for o, n in zip(old, new)])
    clean = f64(c.v)
    bad = {0: [1, 130, 777, 1500, 2003], 1: [5, 290, 303]}
    for b, ranks in bad.items():
        for r in ranks:
            c.v[c.slots[b][r], :, r % 64] = value
    got = f64(_run(c, mask=mask, starts=starts, max_len=bound))
    requests = c.visible(seen, starts)
    want, size, spread = drafts.tree_attention(f64(c.q), f64(c.k), clean, requests, 0.125)
    tol = attention_tolerance(c.q.dtype, c.q.dtype, c.max_len, want, size, spread, 0)
    hit = np.zeros(want.shape, dtype=bool)
    for b, (first, _, keys) in enumerate(requests):
        for r in bad[b]:
            for i in np.flatnonzero(keys[:, r]):
                hit[first + i, :, r % 64] = True
    assert hit.any() and not np.isfinite(got[hit]).any()
    assert (np.abs(got - want)[~hit] <= tol[~hit]).all()


@pytest.mark.parametrize("fill", [0, 1, 170])
def test_any_workspace_contents(device, fill):
    c = Cache(device, 900, [2600, 0, 700], [7, 0, 12], q_heads=8, kv_heads=2, head_dim=64, dtype=torch.bfloat16,
              capacity=25)
    seen, mask = c.masks("tree")
    need = attention.tree_workspace_bytes(25, 3, 8, 2, 64, c.max_len, c.max_new)
    ws = torch.full((need,), fill, dtype=torch.uint8, device=device)
    first = _run(c, mask=mask, workspace=ws)
    _check(c, first, c.visible(seen))
    for _ in range(3):  # sums are in a fixed order
        assert torch.equal(_run(c, mask=mask, workspace=ws), first)


@pytest.mark.parametrize("bound", [1, 5000])
def test_large_values_under_rising_scores(device, bound):
    """bf16 values of 2^90 and below, weights of up to 2^31 against the first keys'."""
    c = Cache(device, 950, [1500], [5], q_heads=4, kv_heads=2, head_dim=64, dtype=torch.bfloat16)
    c.k[:] = 0.01 * c.k
    c.q[:] = 0.01 * c.q
    c.q[:, :, 0] = 2.0
    c.k[torch.from_numpy(c.slots[0]), :, 0] = torch.linspace(0, 10, 1505).to(torch.bfloat16)[:, None]
    c.v *= 2.0 ** 88
    seen, mask = c.masks("tree")
    out = _run(c, mask=mask, scale=1.0, out_dtype=torch.float32, max_len=bound)
    assert torch.isfinite(out).all()
    _check(c, out, c.visible(seen), scale=1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bound", [1, 9000])
def test_sums_that_stay_large(device, bound, dtype):
    """A few keys whose weights nearly fill the sum's range against the first
    ones', among thousands that are close to those."""
    c = Cache(device, 960, [6000], [5], q_heads=4, kv_heads=2, head_dim=64, dtype=dtype)
    c.k[:] = 0.01 * c.k
    c.q[:] = 0.01 * c.q
    c.q[:, :, 0] = 2.0
    level = torch.zeros(6005)
    level[64:] = 0.02 * torch.rand(6005 - 64, generator=torch.Generator().manual_seed(1))
    # log2 weights of 31.7 (beside the sum's limit), of 15.9 (beside fp16's)
    level[100:104] = (31.7 if dtype == torch.bfloat16 else 15.9) / 2 / np.log2(np.e)
    c.k[torch.from_numpy(c.slots[0]), :, 0] = level.to(dtype)[:, None]
    seen, mask = c.masks("tree")
    _check(c, _run(c, mask=mask, scale=1.0, out_dtype=torch.float32, max_len=bound), c.visible(seen), scale=1.0)


@pytest.mark.parametrize("bound", [1, 5000])
def test_a_stretch_of_a_larger_batch(device, bound):
    """Indptrs that begin past zero: the rows and entries before stay out of it."""
    c = Cache(device, 970, [700, 30], [6, 9], q_heads=8, kv_heads=2, head_dim=64, dtype=torch.bfloat16)
    seen, mask = c.masks("any")
    alone = _run(c, mask=mask, max_len=bound)
    _check(c, alone, c.visible(seen))
    pad = lambda t, n: torch.cat((torch.full((n, *t.shape[1:]), 5, dtype=t.dtype, device=device), t))  # noqa: E731
    q, out = pad(c.q, 3), torch.full((c.total + 3, 8, 64), 7.0, dtype=torch.bfloat16, device=device)
    attention.tree_attention(q, c.k.to(device), c.v.to(device), c.qo + 3, c.kv + 4, pad(c.indices, 4), out, scale=0.125,
                             max_len=bound, max_new=9, tree_mask=pad(mask, 3))
    assert (out[:3] == 7).all() and torch.equal(out[3:], alone)


def test_one_workspace_while_a_batch_drains(device):
    """Sized once for the full batch, which runs whole; its last requests are cut."""
    shape = dict(q_heads=16, kv_heads=4, head_dim=64, dtype=torch.bfloat16)
    need = attention.tree_workspace_bytes(4 * 40, 40, 16, 4, 64, 1000, 4)
    ws = torch.full((need,), 255, dtype=torch.uint8, device=device)
    for requests in (40, 32, 31, 3, 1):
        print(f"tree attention, {requests} requests of 40", flush=True)
        old = [(37 * i) % 130 + 800 * (i == 0) for i in range(requests)]
        c = Cache(device, 980 + requests, old, [4] * requests, **shape)
        seen, mask = c.masks("tree")
        _check(c, _run(c, mask=mask, workspace=ws, max_len=1000), c.visible(seen))


@pytest.mark.parametrize("d", [64, 128])
def test_largest_values_in_every_piece(device, d):
    """bf16 values of 2^94, in pieces that each begin with low scores and end with
    a weight of 2^31.9 against them in every wave: 512 pieces of 8 units (a piece's
    tiles of 128 / 64 keys, with 2 / 3 units before the first one).  All values of a
    dim are equal, so the result is that value whatever the weights: each wave's
    sums of weights and of weighted values add some 40 terms each, their joining
    512 and about 64 products, each off by 2^-24."""
    keys = 128 if d == 64 else 64
    ahead = 2 if d == 64 else 3
    tiles = 512 * 8 - ahead
    n_keys, n, heads = tiles * keys, 2, 4
    k = torch.zeros((n_keys, 1, d), dtype=torch.bfloat16, device=device)
    rank = torch.arange(n_keys, device=device)
    k[(rank // keys % 8 == 7 - ahead) & (rank % 32 == 9), 0, 0] = 11.0625  # 2 x 11.0625 x log2(e) = 31.92
    value = torch.tensor([2.0 ** 94, -2.0 ** 94, 1.0, 2.0 ** -90], device=device).repeat(d // 4).to(torch.bfloat16)
    v = value.expand(n_keys, 1, d).contiguous()
    q = torch.zeros((n, heads, d), dtype=torch.bfloat16, device=device)
    q[:, :, 0] = 2.0
    out = torch.empty((n, heads, d), dtype=torch.float32, device=device)
    indptr = lambda x: torch.tensor([0, x], dtype=torch.int32, device=device)  # noqa: E731
    for sinks in (None, torch.full((heads,), 2.0, device=device)):
        attention.tree_attention(q, k, v, indptr(n), indptr(n_keys), rank.int(), out, scale=1.0, max_len=n_keys,
                                 max_new=n, sinks=sinks)
        # (e^2 beside more than 512 weights of e^22)
        tol = 656 * 2.0 ** -24 + (0 if sinks is None else np.exp(2 - 22.125) / 512)
        worst = ((out - value.float()).abs() / value.float().abs()).max().item()
        assert worst <= tol, f"off by {worst:.3g} of the value, {tol:.3g} allowed"


@pytest.mark.parametrize("bound", [1, 5000])
def test_a_mask_without_words_shows_no_drafted_token(device, bound):
    c = Cache(device, 990, [700, 0, 40], [6, 3, 9], q_heads=8, kv_heads=2, head_dim=64, dtype=torch.bfloat16)
    none = [np.zeros((n, n), dtype=bool) for n in c.new]
    mask = torch.zeros((c.total, 0), dtype=torch.int64, device=device)
    _check(c, _run(c, mask=mask, max_len=bound), c.visible(none))
    # the words of a wider store, none of them taken
    store = torch.full((c.total, 2), -1, dtype=torch.int64, device=device)
    _check(c, _run(c, mask=store[:, :0], max_len=bound), c.visible(none))


@pytest.mark.parametrize("bound", [1, 5000])
@pytest.mark.parametrize("page", [1, 16])
@pytest.mark.parametrize("d", [64, 128, 40])
def test_pools_and_lists_of_nothing(device, bound, page, d):
    """A pool without slots, and a list or block table without entries: holes alone."""
    c = Cache(device, 995, [700, 3], [6, 9], q_heads=8, kv_heads=2, head_dim=d, dtype=torch.bfloat16, page=page)
    seen, mask = c.masks("tree")
    sinks = torch.zeros(8, device=device)
    for kind in ("pool", "list"):
        print(f"tree attention without a {kind}, bound {bound} page {page} d {d}", flush=True)
        k, v = c.k.to(device), c.v.to(device)
        indices = c.indices
        if kind == "pool":
            k, v = k[:0].clone(), v[:0].clone()
            assert k.data_ptr() == 0
        else:
            c.indices = indices[..., :0].contiguous()
            assert c.indices.data_ptr() == 0
        for s in (None, sinks):
            out = _run(c, mask=mask, k=k, v=v, sinks=s, max_len=bound)
            assert (out[: c.total] == 0).all()
        c.indices = indices


@pytest.mark.parametrize("d,heads", [(8, 64), (128, 2)])
def test_more_rows_than_one_launch_has_threads_for(device, d, heads):
    """Outputs made for 2^32 threads' worth of rows, of which the last 40 tokens'
    and the first ones' are the batch's: 16 (32) threads of the merge for each."""
    rows = (1 << 32) // (16 if d == 8 else 32)
    capacity = rows // heads + 100
    print(f"tree attention, capacity of {capacity} tokens, {heads} heads of {d}", flush=True)
    c = Cache(device, 1000 + d, [900, 1200], [7, 40], q_heads=heads, kv_heads=2, head_dim=d, dtype=torch.bfloat16)
    requests = c.visible(c.masks("chain")[0])
    q = torch.zeros(capacity, heads, d, dtype=torch.bfloat16, device=device)
    out = torch.full_like(q, 7.0)
    for first in (0, capacity - 47):
        q[first: first + 47] = c.q
        attention.tree_attention(q, c.k.to(device), c.v.to(device), c.qo + first, c.kv, c.indices, out,
                                 scale=d ** -0.5, max_len=5000, max_new=40)
        _check(c, out[first: first + 47], requests)
        out[first: first + 47] = 7.0
        assert (out[:100] == 7).all() and (out[-100:] == 7).all()


def test_more_row_blocks_than_one_launch_has_threads_for(device):
    """4096 short requests under a bound of a million new tokens each."""
    capacity, batch = 1 << 20, 4096
    rng = np.random.default_rng(4)
    old, new = rng.integers(0, 60, batch), rng.integers(0, 4, batch)
    old[-1], new[-1] = 100, 90
    c = Cache(device, 1010, old.tolist(), new.tolist(), q_heads=64, kv_heads=8, head_dim=8, dtype=torch.bfloat16)
    want = _run(c, mask=None)
    q = torch.zeros(capacity, 64, 8, dtype=torch.bfloat16, device=device)
    q[: c.total] = c.q
    out = torch.full_like(q, 7.0)
    attention.tree_attention(q, c.k.to(device), c.v.to(device), c.qo, c.kv, c.indices, out, scale=8 ** -0.5,
                             max_len=c.max_len, max_new=capacity)
    # (blocks of other sizes than under the tight bound: both within their bound of the same rows)
    seen = c.visible(c.masks("chain")[0])
    last = len(seen) - 1
    for b in (0, 1, batch // 2, last - 1, last):
        first, slots, keys = seen[b]
        here = slice(first, first + len(keys))
        y, size, spread = drafts.tree_attention(f64(c.q[here]), f64(c.k), f64(c.v), [(0, slots, keys)], 8 ** -0.5)
        tol = attention_tolerance(c.q.dtype, c.q.dtype, c.max_len, y, size, spread, 0)
        for got in (out, want):
            assert (np.abs(f64(got[here]) - y) <= tol).all(), b
    assert not (out[: c.total] == 7).all(-1).any() and (out[c.total:] == 7).all()


@pytest.mark.parametrize("bound", [1, 5000])
def test_the_largest_batch(device, bound):
    """65534 requests of one drafted token over one key, every 1000th without."""
    batch, d = 65534, 8
    gen = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(s, 1, d, generator=gen).to(torch.bfloat16).to(device) for s in (batch, 2 * batch, 2 * batch))
    lens = torch.full((batch,), 2)
    lens[::1000] = 1
    kv = torch.cat((torch.zeros(1, dtype=torch.int64), lens.cumsum(0)))
    slots = torch.randperm(2 * batch, generator=gen)
    qo = torch.arange(batch + 1, dtype=torch.int32, device=device)
    out = torch.empty(batch, 1, d, dtype=torch.float32, device=device)
    attention.tree_attention(q, k, v, qo, kv.int().to(device), slots.int().to(device), out, scale=0.5, max_len=bound,
                             max_new=1)
    own, before = slots[kv[1:] - 1].numpy(), slots[kv[:-1]].numpy()
    scores = 0.5 * np.stack([(f64(q) * f64(k)[at]).sum(-1)[:, 0] for at in (own, before)], -1)
    spread = 0.5 * np.stack([np.abs(f64(q) * f64(k)[at]).sum(-1)[:, 0] for at in (own, before)], -1).max(-1)[:, None]
    scores[::1000, 1] = -np.inf
    w = np.exp(scores - scores.max(-1, keepdims=True))
    w /= w.sum(-1, keepdims=True)
    want, size = (w[:, :1, None] * f(f64(v)[own]) + w[:, 1:, None] * f(f64(v)[before]) for f in (np.array, np.abs))
    tol = attention_tolerance(torch.bfloat16, torch.float32, 2, want, size, spread, 0)
    assert (np.abs(f64(out) - want) <= tol).all()
