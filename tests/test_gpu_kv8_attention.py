"""Attention over an 8-bit cache on the GPU against the 64-bit oracle, at the
sizes, layouts, scales and masks where it can go wrong."""

import numpy as np
import pytest
import torch

from akv_amd import attention, kv8
from oracle import drafts
from tests.drafts import f64
from tests.kv8 import FORMATS, Cache8, codes_of, kv8_tolerance

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _run(c, *, mask, starts=None, first=0, sinks=None, out_dtype=None, scale=None, max_len=None, max_new=None, out=None,
         workspace=None, indptr=torch.int32, q=None, parts=None, status=None):
    scale = c.q.shape[2] ** -0.5 if scale is None else scale
    if out is None:
        out = torch.full(c.q.shape, 7.0, dtype=out_dtype or c.q.dtype, device=c.device)
    (k, ks), (v, vs) = c.parts if parts is None else parts
    kv8.attention_kv8(
        c.q if q is None else q, k, v, ks, vs, c.qo.to(indptr), c.kv.to(indptr), c.indices, out, scale=scale,
        max_len=c.max_len if max_len is None else max_len, max_new=c.max_new if max_new is None else max_new,
        page_size=c.page, scale_block=c.block, tree_mask=mask,
        key_starts=None if starts is None else torch.tensor(starts, dtype=torch.int32, device=c.device),
        first_keys=first, sinks=sinks, workspace=workspace, status=status)
    return out


def _check(c, out, requests, *, sinks=None, scale=None, k=None, v=None, rows=None):
    scale = c.q.shape[2] ** -0.5 if scale is None else scale
    want, size, spread = drafts.tree_attention(f64(c.q), f64(c.k if k is None else k), f64(c.v if v is None else v),
                                               requests, scale, None if sinks is None else f64(sinks))
    got = f64(out)
    tol = kv8_tolerance(c.q.dtype, out.dtype, c.max_len, want, size, spread)
    here = np.arange(c.total) if rows is None else rows
    off = np.abs(got - want)[here] - tol[here]
    assert not np.isnan(got[here]).any()
    assert (off <= 0).all(), f"{(off > 0).sum()} values off, worst by {off.max():.3g}"
    assert (got[c.total:] == 7.0).all(), "rows behind the last token were written"


SHAPES = [
    # q heads, kv heads, head_dim, q dtype, format, page, block, old, new
    (8, 1, 64, BF16, "e4m3", 1, 1, [0], [1]),
    (8, 1, 64, BF16, "e5m2", 1, 1, [1], [1]),
    (2, 2, 64, BF16, "e4m3", 1, 1, [63, 64, 65, 0, 255, 256, 257, 511, 512, 513], [1, 2, 3, 4, 5, 16, 17, 1, 1, 1]),
    (16, 2, 64, BF16, "e4m3", 1, 16, [700, 0, 40, 300], [8, 5, 0, 33]),
    (16, 2, 64, F16, "e5m2", 16, 16, [700, 3, 40, 300], [8, 5, 0, 33]),
    (16, 2, 64, F16, "e4m3", 5, 2, [511, 513, 1], [64, 65, 70]),
    (14, 2, 64, BF16, "e5m2", 1, 64, [1000, 129], [9, 100]),
    (3, 1, 128, BF16, "e4m3", 1, 1, [130, 127, 128, 0, 129], [7, 11, 1, 40, 1]),
    (16, 4, 128, F16, "e4m3", 16, 16, [1500, 10], [8, 32]),
    (12, 1, 128, BF16, "e5m2", 64, 64, [31, 33], [65, 130]),
    (6, 2, 96, BF16, "e4m3", 16, 4, [200, 90], [6, 21]),
    (4, 2, 80, F16, "e5m2", 3, 1, [200, 90], [6, 21]),
    (5, 1, 48, BF16, "e4m3", 1, 8, [77], [19]),
    (2, 1, 16, F16, "e4m3", 1, 1, [77, 5], [3, 64]),
]


def _cache(device, seed, shape, **more):
    hq, hk, d, dtype, form, page, block, old, new = shape
    return Cache8(device, seed, old, new, q_heads=hq, kv_heads=hk, head_dim=d, dtype=dtype, form=form, page=page,
                  block=block, **more)


@pytest.mark.parametrize("kind", ["chain", "tree", "any"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_matches_oracle(device, shape, kind):
    """As one workgroup per block of rows, and shared out; rows without a key among them."""
    print(f"kv8 attention shape {shape} {SHAPES[shape]} {kind}", flush=True)
    hq, new = SHAPES[shape][0], SHAPES[shape][-1]
    c = _cache(device, 100 + shape, SHAPES[shape], capacity=sum(new) + shape % 3)
    seen, mask = c.masks(kind)
    sinks = torch.randn(hq, generator=torch.Generator().manual_seed(shape)).to(device) if shape % 2 else None
    for bound in (None, 1, 5000):
        out = _run(c, mask=mask, sinks=sinks, out_dtype=F32 if kind == "any" else None, max_len=bound,
                   indptr=torch.int64 if kind == "tree" else torch.int32, max_new=max(1, c.max_new // 3) if bound else None)
        _check(c, out, c.visible(seen), sinks=sinks)


@pytest.mark.parametrize("first", [0, 1, 4, 33, 300, 2000])
@pytest.mark.parametrize("d,page", [(64, 1), (64, 16), (128, 16), (96, 4)])
def test_windows_with_first_keys(device, d, page, first):
    """Windows that begin anywhere, behind every key and below zero, with first
    keys that end before, inside and behind them."""
    old, new = [900, 40, 0, 500], [6, 12, 3, 20]
    c = Cache8(device, 7 + d, old, new, q_heads=4, kv_heads=2, head_dim=d, dtype=BF16, page=page, block=4 if page > 1 else 1)
    rng = np.random.default_rng(d)
    starts = np.concatenate([rng.integers(max(0, o - 130), o + 1, n) for o, n in zip(old, new)])
    starts[:3] = [old[0], 0 if first == 1 else old[0] - 60, old[0] - 1]
    passed = starts.copy()
    passed[3], starts[3] = -50, 0
    passed[4], starts[4] = 5000, old[0]  # past the earlier keys: none of them but the first ones
    for kind in ("tree", "any", "chain"):
        for bound in (160 + first, 5000):
            print(f"kv8 windows d={d} page={page} first={first} {kind} {bound}", flush=True)
            seen, mask = c.masks(kind)
            out = _run(c, mask=mask, starts=passed, first=first, max_len=bound)
            _check(c, out, c.visible(seen, starts, first))


@pytest.mark.parametrize("first", [0, 4, 40])
@pytest.mark.parametrize("block", [1, 16])
def test_narrow_windows_of_long_requests(device, first, block):
    """What no token sees is not read: codes and scales there are NaN."""
    old, new = [5000, 3000], [4, 9]
    c = Cache8(device, 61, old, new, q_heads=8, kv_heads=2, head_dim=64, dtype=BF16, page=16, block=block)
    starts = np.concatenate([o - 128 + np.arange(n) for o, n in zip(old, new)])
    k, v = c.k.clone(), c.v.clone()
    for slots, o in zip(c.slots, old):
        hidden = slots[first: o - 128]
        whole = [s for s in np.unique(hidden // block) if np.isin(np.arange(s * block, (s + 1) * block), hidden).all()]
        for codes, scales in c.parts:
            codes.view(torch.uint8)[hidden] = 0x7f
            scales[whole] = float("nan")
    seen, mask = c.masks("tree")
    out = _run(c, mask=mask, starts=starts, first=first, max_len=first + 128 + 9 + 1)
    _check(c, out, c.visible(seen, starts, first), k=k, v=v)


@pytest.mark.parametrize("d,dtype", [(64, BF16), (128, BF16), (64, F16)])
def test_long_requests_in_many_pieces(device, d, dtype):
    c = Cache8(device, 11 + d, [6000, 1, 2500], [3, 9, 16], q_heads=8, kv_heads=2, head_dim=d, dtype=dtype)
    seen, mask = c.masks("tree")
    _check(c, _run(c, mask=mask, out_dtype=F32), c.visible(seen))


@pytest.mark.parametrize("d,new", [(64, 300), (128, 170)])
def test_chunks_of_a_prompt(device, d, new):
    """Chains of many tokens: blocks of rows end with their last token's key."""
    c = Cache8(device, 13, [700, 0, 5], [new, new // 2, 2 * new], q_heads=8, kv_heads=2, head_dim=d, dtype=BF16, page=16,
               block=16)
    seen, mask = c.masks("chain")
    for bound in (1, 5000):
        _check(c, _run(c, mask=mask, max_len=bound), c.visible(seen))


def test_bounds_only_size_the_launch(device):
    c = Cache8(device, 21, [1200, 30, 700], [20, 3, 9], q_heads=8, kv_heads=2, head_dim=64, dtype=BF16)
    seen, mask = c.masks("tree")
    for max_len, max_new in ((c.max_len, c.max_new), (1, 1), (0, 0), (100000, 400), (300, 64)):
        print(f"kv8 attention bounds {max_len} {max_new}", flush=True)
        _check(c, _run(c, mask=mask, max_len=max_len, max_new=max_new), c.visible(seen))


@pytest.mark.parametrize("page", [1, 16])
def test_holes_are_not_read(device, page):
    """Slots outside the pool, lists shorter than the lengths say; slot 0, whose
    codes and scale stand in for a hole's, holds NaN."""
    c = Cache8(device, 31, [400, 90], [5, 9], q_heads=4, kv_heads=2, head_dim=64, dtype=BF16, page=page, holes=6)
    used = np.concatenate(c.slots)
    if not (used == 0).any():
        for codes, scales in c.parts:
            codes.view(torch.uint8)[0] = 0x7f
            scales[0] = float("nan")
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
    for bound in (1, 5000):
        _check(c, _run(c, mask=mask, max_len=bound), c.visible(seen))


@pytest.mark.parametrize("form,code", [("e4m3", 0x7f), ("e4m3", 0xff), ("e5m2", 0x7c), ("e5m2", 0xfc), ("e5m2", 0x7d),
                                       ("e4m3", 0xfe)])
@pytest.mark.parametrize("d,dtype,bound", [(64, BF16, 1), (128, F16, 5000), (96, BF16, 1), (64, F16, 5000)])
def test_what_a_token_does_not_see_cannot_reach_it(device, d, dtype, bound, form, code):
    """NaN and infinite codes (and the lowest value) in keys and values hidden from
    some tokens: the others' rows are right; in the rows that see a value, that dim is not
    finite and the others are right."""
    old, new = [2000, 300], [12, 40]
    make = lambda: Cache8(device, 41 + d, old, new, q_heads=4, kv_heads=2, head_dim=d, dtype=dtype, form=form)  # noqa: E731
    c, clean = make(), make()
    seen, mask = c.masks("any")
    starts = np.concatenate([np.linspace(0, o, n).astype(np.int64) for o, n in zip(old, new)])
    bad = {0: [1, 130, 777, 1500, 2003], 1: [5, 290, 303]}
    keys_too = {(0, 777), (1, 5)}
    finite = code == 0xfe
    for b, ranks in bad.items():
        for r in ranks:
            slot = int(c.slots[b][r])
            c.parts[1][0].view(torch.uint8)[slot, :, r % d] = code
            if (b, r) in keys_too:
                c.parts[0][0].view(torch.uint8)[slot, :, (3 * r) % d] = code
    if finite:
        c.refresh()
        _check(c, _run(c, mask=mask, starts=starts, max_len=bound), c.visible(seen, starts))
        return
    got = f64(_run(c, mask=mask, starts=starts, max_len=bound))
    requests = c.visible(seen, starts)
    want, size, spread = drafts.tree_attention(f64(c.q), f64(clean.k), f64(clean.v), requests, d ** -0.5)
    tol = kv8_tolerance(dtype, dtype, c.max_len, want, size, spread)
    hit, unknown = np.zeros(want.shape, dtype=bool), np.zeros(want.shape[:1], dtype=bool)
    for b, (first, _, keys) in enumerate(requests):
        for r in bad[b]:
            for i in np.flatnonzero(keys[:, r]):
                hit[first + i, :, r % d] = True
                unknown[first + i] |= (b, r) in keys_too  # (its scores are not finite: nor is the row, or it is 0)
    ok = ~hit & ~unknown[:, None, None]
    assert hit.any() and unknown.any() and ok.any()
    assert not np.isfinite(got[hit & ~unknown[:, None, None]]).any()
    assert (np.abs(got - want)[ok] <= tol[ok]).all()


def test_nan_queries_stay_in_their_rows(device):
    for old in (300, 3000):
        c = Cache8(device, 51, [old], [9], q_heads=8, kv_heads=2, head_dim=64, dtype=BF16)
        seen, mask = c.masks("tree")
        clean = f64(_run(c, mask=mask))
        c.q[4, 3] = float("nan")
        out = f64(_run(c, mask=mask))
        assert np.isnan(out[4, 3]).all()
        out[4, 3] = clean[4, 3]
        np.testing.assert_array_equal(out, clean)


def _level(c, values):
    """Keys of small codes but for dim 0, which has these values (held exactly:
    the scales become 1); queries 2 in dim 0."""
    for codes, scales in c.parts[:1]:
        codes.copy_((codes.float() / 4096).to(codes.dtype))
        scales.fill_(1.0)
        codes[torch.from_numpy(c.slots[0]).to(c.device), :, 0] = values[:, None].to(codes.dtype).to(c.device)
    c.refresh()
    c.q[:] = 0.01 * c.q
    c.q[:, :, 0] = 2.0


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("scores", ["rising", "falling", "far"])
def test_scores_far_apart(device, scores, dtype):
    """Maxima that keep moving, by little and by more than fp32's range."""
    c = Cache8(device, 61, [900], [10], q_heads=4, kv_heads=1, head_dim=64, dtype=dtype)
    ramp = torch.linspace(-30, 30, 910) if scores != "far" else torch.where(torch.arange(910) % 300 == 299, 240.0, -30.0)
    _level(c, -ramp if scores == "falling" else ramp)
    seen, mask = c.masks("tree")
    for bound in (1, 5000):
        _check(c, _run(c, mask=mask, scale=1.0, out_dtype=F32, max_len=bound), c.visible(seen), scale=1.0)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [2, 40])
def test_maxima_that_jump_behind_the_first_tiles(device, d, dtype, new):
    """Scores above the first ones' by more than a weight can hold, in some rows only."""
    c = Cache8(device, 700 + d, [1400], [new], q_heads=4, kv_heads=1, head_dim=d, dtype=dtype)
    jump = torch.zeros(1400 + new)
    for at, by in ((100, 6.0), (300, 12.0), (301, 13.0), (700, 40.0), (1200, 44.0)):
        jump[at] = by
    _level(c, jump)
    c.q[1::2, :, 0] = 0.0
    c.q[:, 0, 0] = 0.0
    seen, mask = c.masks("tree")
    for bound in (1, 5000):
        _check(c, _run(c, mask=mask, scale=1.0, out_dtype=F32, max_len=bound), c.visible(seen), scale=1.0)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bound", [1, 9000])
def test_sums_that_stay_large(device, bound, dtype):
    """A few keys whose weights nearly fill the sum's range against the first
    ones', among thousands that are close to those."""
    c = Cache8(device, 960, [6000], [5], q_heads=4, kv_heads=2, head_dim=64, dtype=dtype)
    level = torch.zeros(6005)
    level[64:] = 0.02 * torch.rand(6005 - 64, generator=torch.Generator().manual_seed(1))
    level[100:104] = 10.0  # log2 weights of 28.9: 2^30 in a sum, a quarter of which a lane may hold
    _level(c, level)
    seen, mask = c.masks("tree")
    _check(c, _run(c, mask=mask, scale=1.0, out_dtype=F32, max_len=bound), c.visible(seen), scale=1.0)


@pytest.mark.parametrize("bound", [1, 5000])
@pytest.mark.parametrize("power", [88, -90])
def test_scales_of_any_size(device, bound, power):
    """V values around 2^88 and 2^-90 under rising scores, K scales of 2^-60 with
    codes of K = 1 under a large score scale, and negative scales."""
    c = Cache8(device, 950, [1500], [5], q_heads=4, kv_heads=2, head_dim=64, dtype=BF16)
    _level(c, torch.linspace(0, 10, 1505))
    c.parts[1][1].mul_(2.0 ** power)
    c.parts[1][1][::2] *= -1
    c.parts[0][1].mul_(2.0 ** -20)
    c.refresh()
    seen, mask = c.masks("tree")
    out = _run(c, mask=mask, scale=2.0 ** 20, out_dtype=F32, max_len=bound)
    assert torch.isfinite(out).all()
    _check(c, out, c.visible(seen), scale=2.0 ** 20)


def test_fp16_queries_and_tiny_values(device):
    """Values far below fp16's smallest one, in f32 outputs."""
    c = Cache8(device, 955, [700], [9], q_heads=8, kv_heads=2, head_dim=64, dtype=F16)
    c.parts[1][1].mul_(2.0 ** -60)
    c.refresh()
    seen, mask = c.masks("tree")
    _check(c, _run(c, mask=mask, out_dtype=F32), c.visible(seen))


@pytest.mark.parametrize("block", [1, 16])
def test_strides(device, block):
    """q, K, V, scales and out as views: padded heads, a pool of interleaved K and
    V, scales side by side and with the heads outside, a wider table."""
    c = Cache8(device, 71, [200, 60], [7, 4], q_heads=4, kv_heads=2, head_dim=64, dtype=BF16, page=16, block=block)
    q = torch.zeros((c.total, 4, 80), dtype=BF16, device=device)[:, :, 8:72]
    q.copy_(c.q)
    both = torch.stack([p[0].view(torch.uint8) for p in c.parts], 2).view(c.parts[0][0].dtype)  # [slots, heads, 2, dim]
    pair = torch.stack([p[1] for p in c.parts], -1)
    outer = [p[1].T.contiguous().T for p in c.parts]
    store = torch.full((c.total, 6, 64), 7.0, dtype=BF16, device=device)
    c.indices = torch.nn.functional.pad(c.indices, (0, 5), value=123456)[:, : c.indices.shape[1]]
    seen, mask = c.masks("tree")
    mask = torch.nn.functional.pad(mask, (0, 3), value=-1)[:, : mask.shape[1]]
    plain = _run(c, mask=mask)
    _check(c, plain, c.visible(seen))
    for scales in ([pair[..., 0], pair[..., 1]], outer):
        parts = [[both[:, :, i], scales[i]] for i in (0, 1)]
        out = _run(c, mask=mask, q=q, parts=parts, out=store[:, 1:5])
        assert torch.equal(out, plain)
        assert (store[:, 0] == 7).all() and (store[:, 5] == 7).all()


@pytest.mark.parametrize("d,out_dtype", [(64, F32), (128, BF16), (96, F32)])
def test_unaligned_outputs(device, d, out_dtype):
    for old in ([300, 20], [3000, 20]):
        c = Cache8(device, 600 + d, old, [7, 4], q_heads=4, kv_heads=2, head_dim=d, dtype=BF16)
        store = torch.full((c.total, 4, d + 3), 7.0, dtype=out_dtype, device=device)
        seen, mask = c.masks("tree")
        _check(c, _run(c, mask=mask, out=store[:, :, 1: d + 1]), c.visible(seen))
        assert (store[:, :, 0] == 7).all() and (store[:, :, d + 1:] == 7).all()


def test_gate_and_empty_batches(device):
    for old in ([30], [3000]):
        c = Cache8(device, 91, old, [4], q_heads=4, kv_heads=2, head_dim=64, dtype=BF16)
        closed = torch.tensor([1], dtype=torch.int32, device=device)
        assert (_run(c, mask=None, status=closed) == 7).all()
        seen, _ = c.masks("chain")
        _check(c, _run(c, mask=None, status=closed * 4), c.visible(seen))
    none = Cache8(device, 92, [30, 0], [0, 0], q_heads=4, kv_heads=2, head_dim=64, dtype=BF16, capacity=3)
    for bound in (1, 5000):
        assert (_run(none, mask=None, max_len=bound) == 7).all()
    empty = _run(c, mask=None, q=c.q[:0], out=c.q[:0])
    assert empty.numel() == 0


@pytest.mark.parametrize("seed", range(30))
def test_random_batches(device, seed):
    rng = np.random.default_rng(1000 + seed)
    b = int(rng.integers(1, 7))
    hi = int(rng.choice([5, 70, 400, 1200]))
    old, new = rng.integers(0, hi, b), rng.integers(0, int(rng.choice([2, 12, 70])), b)
    new[0] = max(new[0], 1)
    hk = int(rng.choice([1, 2, 3]))
    hq = hk * int(rng.choice([1, 2, 5, 8]))
    d = int(rng.choice([16, 64, 64, 80, 112, 128]))
    dtype = BF16 if rng.random() < 0.6 else F16
    page, block = int(rng.choice([1, 1, 2, 16, 64])), int(rng.choice([1, 2, 16, 64]))
    form, first = str(rng.choice(list(FORMATS))), int(rng.choice([0, 0, 3, 50]))
    print(f"kv8 attention random {seed}: {old.tolist()} {new.tolist()} {hq}/{hk}x{d} page {page} block {block} {dtype} "
          f"{form} first {first}", flush=True)
    c = Cache8(device, seed, old.tolist(), new.tolist(), q_heads=hq, kv_heads=hk, head_dim=d, dtype=dtype, form=form,
               page=page, block=block, holes=int(rng.integers(0, 3)), capacity=int(sum(new)) + int(rng.integers(0, 4)))
    seen, mask = c.masks(str(rng.choice(["chain", "tree", "any"])))
    starts = None
    if rng.random() < 0.5:
        starts = np.concatenate([rng.integers(0, o + 1, n) for o, n in zip(old, new)])
    full = None if starts is None else np.concatenate((starts, np.zeros(c.capacity - c.total, np.int64)))
    sinks = torch.randn(hq, generator=torch.Generator().manual_seed(seed)).to(device) if seed % 2 else None
    for bound in (1, 5000):
        _check(c, _run(c, mask=mask, starts=full, first=first, sinks=sinks, max_len=bound), c.visible(seen, starts, first),
               sinks=sinks)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bound", [1, 5000])
def test_trees_of_many_words(device, d, bound):
    """More new tokens than the mask words kept at hand, and words that end before
    the tokens do."""
    old, new = [300, 1], [200, 333]
    c = Cache8(device, 300 + d, old, new, q_heads=4, kv_heads=2, head_dim=d, dtype=BF16)
    starts = np.concatenate([c.rng.integers(0, o + 1, n) for o, n in zip(old, new)])
    for kind in ("chain", "tree", "any"):
        print(f"kv8 attention large trees d={d} bound {bound} {kind}", flush=True)
        seen, mask = c.masks(kind)
        _check(c, _run(c, mask=mask, starts=starts, first=7, max_len=bound), c.visible(seen, starts, 7))
        if mask is None:
            continue
        short = [s.copy() for s in seen]
        for s in short:
            s[:, 192:] = False
        _check(c, _run(c, mask=mask[:, :3], max_len=bound), c.visible(short))


@pytest.mark.parametrize("bound", [1, 5000])
def test_a_mask_without_words_shows_no_new_token(device, bound):
    c = Cache8(device, 990, [700, 0, 40], [6, 3, 9], q_heads=8, kv_heads=2, head_dim=64, dtype=BF16)
    none = [np.zeros((n, n), dtype=bool) for n in c.new]
    mask = torch.zeros((c.total, 0), dtype=torch.int64, device=device)
    _check(c, _run(c, mask=mask, max_len=bound), c.visible(none))
    store = torch.full((c.total, 2), -1, dtype=torch.int64, device=device)
    _check(c, _run(c, mask=store[:, :0], max_len=bound), c.visible(none))


@pytest.mark.parametrize("bound", [1, 900, 5000])
def test_many_requests(device, bound):
    """More requests than a wave has lanes, empty ones among them."""
    rng = np.random.default_rng(9)
    old = [int(rng.integers(0, 900)) if i % 3 else 0 for i in range(150)]
    new = [0 if i % 7 == 3 or 64 <= i < 130 else int(rng.integers(0, 6)) for i in range(150)]
    c = Cache8(device, 400, old, new, q_heads=6, kv_heads=3, head_dim=64, dtype=F16)
    seen, mask = c.masks("tree")
    _check(c, _run(c, mask=mask, max_len=bound), c.visible(seen))
    c = Cache8(device, 401, old, [20 if i == 149 else 0 for i in range(150)], q_heads=24, kv_heads=1, head_dim=64,
               dtype=BF16)  # a block of rows that only the last request has
    seen, mask = c.masks("tree")
    _check(c, _run(c, mask=mask, max_len=bound), c.visible(seen))


@pytest.mark.parametrize("page", [1, 16])
def test_slots_past_32_bits(device, page):
    """A layer whose rows lie 2 MiB apart, and its scales 2 MiB: offsets beyond 4 GiB."""
    c = Cache8(device, 500 + page, [2300], [5], q_heads=4, kv_heads=2, head_dim=64, dtype=BF16, page=page)
    stride, n = 1 << 21, c.k.shape[0]
    store = torch.empty(n * stride, dtype=torch.uint8, device=device)
    scales = torch.empty(n << 19, dtype=F32, device=device)
    parts = []
    for i, (codes, s) in enumerate(c.parts):
        far = store.as_strided((n, 2, 64), (stride, 64, 1), 4096 * i)
        far.copy_(codes.view(torch.uint8))
        far_s = scales.as_strided((n, 2), (1 << 19, 1), 64 * i)
        far_s.copy_(s)
        parts.append([far.view(codes.dtype), far_s])
    seen, mask = c.masks("tree")
    _check(c, _run(c, mask=mask, parts=parts), c.visible(seen))


def test_one_workspace_for_changing_batches(device):
    """Whatever an earlier call left in a workspace does not matter, and one sized
    for the full batch serves it while it drains; sums are in a fixed order."""
    shape = dict(q_heads=16, kv_heads=4, head_dim=64, dtype=BF16)
    need = kv8.attention_kv8_workspace_bytes(4 * 40, 40, 16, 4, 64, 1500, 4)
    ws = torch.full((need,), 255, dtype=torch.uint8, device=device)
    for requests in (40, 32, 31, 3, 1):
        print(f"kv8 attention, {requests} requests of 40", flush=True)
        old = [(37 * i) % 130 + 1100 * (i == 0) for i in range(requests)]
        c = Cache8(device, 980 + requests, old, [4] * requests, **shape)
        seen, mask = c.masks("tree")
        first = _run(c, mask=mask, workspace=ws, max_len=1500)
        _check(c, first, c.visible(seen))
        for fill in (0, 170):
            ws.fill_(fill)
            assert torch.equal(_run(c, mask=mask, workspace=ws, max_len=1500), first)


@pytest.mark.parametrize("bound", [1, 5000])
def test_a_stretch_of_a_larger_batch(device, bound):
    """Indptrs that begin past zero: the rows and entries before stay out of it."""
    c = Cache8(device, 970, [700, 30], [6, 9], q_heads=8, kv_heads=2, head_dim=64, dtype=BF16)
    seen, mask = c.masks("any")
    alone = _run(c, mask=mask, max_len=bound)
    _check(c, alone, c.visible(seen))
    pad = lambda t, n: torch.cat((torch.full((n, *t.shape[1:]), 5, dtype=t.dtype, device=device), t))  # noqa: E731
    q, out = pad(c.q, 3), torch.full((c.total + 3, 8, 64), 7.0, dtype=BF16, device=device)
    (k, ks), (v, vs) = c.parts
    kv8.attention_kv8(q, k, v, ks, vs, c.qo + 3, c.kv + 4, pad(c.indices, 4), out, scale=0.125, max_len=bound, max_new=9,
                      tree_mask=pad(mask, 3))
    assert (out[:3] == 7).all() and torch.equal(out[3:], alone)


@pytest.mark.parametrize("bound", [1, 5000])
@pytest.mark.parametrize("page", [1, 16])
def test_pools_and_lists_of_nothing(device, bound, page):
    """A pool without slots, and a list or block table without entries: holes alone."""
    c = Cache8(device, 995, [700, 3], [6, 9], q_heads=8, kv_heads=2, head_dim=64, dtype=BF16, page=page)
    seen, mask = c.masks("tree")
    sinks = torch.zeros(8, device=device)
    for kind in ("pool", "list"):
        parts, indices = None, c.indices
        if kind == "pool":
            parts = [[t[:0].clone() for t in p] for p in c.parts]
        else:
            c.indices = indices[..., :0].contiguous()
        for s in (None, sinks):
            out = _run(c, mask=mask, parts=parts, sinks=s, max_len=bound)
            assert (out[: c.total] == 0).all()
        c.indices = indices


@pytest.mark.parametrize("bound", [1, 5000])
def test_the_largest_batch(device, bound):
    """65534 requests of one token over two keys, every 1000th over its own alone."""
    batch, d = 65534, 16
    gen = torch.Generator().manual_seed(1)
    q = torch.randn(batch, 1, d, generator=gen).to(BF16).to(device)
    k, v = (codes_of(gen, (2 * batch, 1, d), "e4m3").to(device) for _ in range(2))
    ks, vs = (0.02 * torch.rand(2 * batch, 1, generator=gen).to(device) for _ in range(2))
    lens = torch.full((batch,), 2)
    lens[::1000] = 1
    kv = torch.cat((torch.zeros(1, dtype=torch.int64), lens.cumsum(0)))
    slots = torch.randperm(2 * batch, generator=gen)
    out = torch.empty(batch, 1, d, dtype=F32, device=device)
    kv8.attention_kv8(q, k, v, ks, vs, torch.arange(batch + 1, dtype=torch.int32, device=device), kv.int().to(device),
                      slots.int().to(device), out, scale=0.25, max_len=bound, max_new=1)
    own, before = slots[kv[1:] - 1].numpy(), slots[kv[:-1]].numpy()
    kf, vf = (f64(t.float()) * f64(s)[..., None] for t, s in ((k, ks), (v, vs)))
    scores = 0.25 * np.stack([(f64(q) * kf[at]).sum(-1)[:, 0] for at in (own, before)], -1)
    spread = 0.25 * np.stack([np.abs(f64(q) * kf[at]).sum(-1)[:, 0] for at in (own, before)], -1).max(-1)[:, None]
    scores[::1000, 1] = -np.inf
    w = np.exp(scores - scores.max(-1, keepdims=True))
    w /= w.sum(-1, keepdims=True)
    want, size = (w[:, :1, None] * f(vf[own]) + w[:, 1:, None] * f(vf[before]) for f in (np.array, np.abs))
    assert (np.abs(f64(out) - want) <= kv8_tolerance(BF16, F32, 2, want, size, spread)).all()


def test_is_tree_attention_of_the_same_values(device):
    """Codes at scales of a power of two are bf16 values: both caches give one
    result, but for where each rounds its weights."""
    c = Cache8(device, 77, [900, 20], [6, 9], q_heads=8, kv_heads=2, head_dim=64, dtype=BF16, page=16, block=16)
    for _, scales in c.parts:
        scales.copy_(torch.exp2(torch.round(torch.log2(scales))))
    c.refresh()
    seen, mask = c.masks("tree")
    k, v = c.k.to(BF16), c.v.to(BF16)
    assert torch.equal(k.double(), c.k) and torch.equal(v.double(), c.v)
    other = torch.empty_like(c.q, dtype=F32)
    attention.tree_attention(c.q, k, v, c.qo, c.kv, c.indices, other, scale=0.125, max_len=c.max_len, max_new=c.max_new,
                             page_size=16, tree_mask=mask)
    out = _run(c, mask=mask, out_dtype=F32)
    _check(c, out, c.visible(seen))
    want, size, spread = drafts.tree_attention(f64(c.q), f64(c.k), f64(c.v), c.visible(seen), 0.125)
    tol = kv8_tolerance(BF16, F32, c.max_len, want, size, spread) + 2.0 ** -8 * (size + np.abs(want)) * 1.01
    assert (np.abs(f64(out) - f64(other)) <= tol).all()


# ---------------------------------------------------------------------------
# Two heads to a workgroup: cut batches of 64 dims and an even number of KV heads,
# by their bounds larger than the last-level cache

LARGE = 10 ** 7

PAIRS = [
    # q heads, kv heads, head_dim, q dtype, format, page, block, old, new, bound on the new tokens
    (8, 8, 64, BF16, "e4m3", 1, 1, [1700, 3], [1, 1], 1),
    (14, 2, 64, BF16, "e5m2", 1, 1, [900, 0, 77], [1, 5, 9], 9),       # groups of 7: blocks end inside no token
    (60, 4, 64, F16, "e4m3", 16, 16, [400, 1600], [2, 3], 2),          # groups of 15, a request past its bound
    (64, 2, 64, BF16, "e4m3", 1, 4, [700, 31], [1, 4], 1),             # groups of 32: a token to a block
    (82, 2, 64, BF16, "e4m3", 16, 1, [500, 90], [1, 3], 1),            # 41: rows of a half-filled block
    (10, 2, 48, F16, "e5m2", 5, 2, [300, 0, 1100], [20, 33, 40], 6),   # seven blocks of rows
    (6, 6, 16, BF16, "e4m3", 1, 8, [640, 20], [65, 2], 32),
    (4, 2, 64, F16, "e4m3", 64, 64, [257, 511], [64, 128], 64),
]


@pytest.mark.parametrize("kind", ["chain", "tree", "any"])
@pytest.mark.parametrize("case", range(len(PAIRS)))
def test_pairs_of_heads(device, case, kind):
    *shape, most = PAIRS[case]
    print(f"kv8 attention pairs {PAIRS[case]} {kind}", flush=True)
    c = _cache(device, 1100 + case, shape, capacity=sum(shape[-1]) + case % 2, holes=case % 3)
    seen, mask = c.masks(kind)
    sinks = torch.randn(shape[0], generator=torch.Generator().manual_seed(case)).to(device) if case % 2 else None
    for most_new in (most, c.max_new):
        out = _run(c, mask=mask, sinks=sinks, max_len=LARGE, max_new=most_new, out_dtype=F32 if kind == "any" else None)
        _check(c, out, c.visible(seen), sinks=sinks)
    starts = np.concatenate([c.rng.integers(0, o + 1, n) for o, n in zip(shape[-2], shape[-1])])
    full = np.concatenate((starts, np.zeros(c.capacity - c.total, np.int64)))
    _check(c, _run(c, mask=mask, starts=full, first=5, max_len=LARGE), c.visible(seen, starts, 5))


@pytest.mark.parametrize("form", list(FORMATS))
def test_what_one_head_of_a_pair_holds_stays_its_own(device, form):
    """NaN codes and scales of one head, in keys that are seen, make its rows NaN and no others."""
    c = Cache8(device, 1200, [900, 40], [3, 5], q_heads=12, kv_heads=4, head_dim=64, dtype=BF16, form=form, block=4, page=16)
    seen, mask = c.masks("tree")
    plain = _run(c, mask=mask, max_len=LARGE)
    for head in range(4):
        parts = [[codes.clone(), scales.clone()] for codes, scales in c.parts]
        parts[1][0].view(torch.uint8)[:, head] = 0x7f
        parts[0][1][:, head] = float("nan")
        out = _run(c, mask=mask, parts=parts, max_len=LARGE)
        others = [h for h in range(12) if h // 3 != head]
        assert torch.equal(out[: c.total, others], plain[: c.total, others])
        assert torch.isnan(out[: c.total, 3 * head: 3 * head + 3].float()).all()


@pytest.mark.parametrize("block", [1, 16])
def test_strides_of_pairs(device, block):
    """K and V interleaved head by head, padded heads, scales with the heads outside."""
    c = Cache8(device, 1210, [2000, 60], [7, 4], q_heads=8, kv_heads=4, head_dim=64, dtype=BF16, page=16, block=block)
    both = torch.stack([p[0].view(torch.uint8) for p in c.parts], 2).view(c.parts[0][0].dtype)
    wide = torch.zeros((*c.parts[0][0].shape[:2], 112), dtype=torch.uint8, device=device)
    wide[..., 16:80] = c.parts[0][0].view(torch.uint8)
    outer = [p[1].T.contiguous().T for p in c.parts]
    beside = torch.stack([p[1] for p in c.parts], -1)
    seen, mask = c.masks("tree")
    plain = _run(c, mask=mask, max_len=LARGE)
    _check(c, plain, c.visible(seen))
    for parts in ([[both[:, :, i], outer[i]] for i in (0, 1)],
                  [[wide[..., 16:80].view(both.dtype), beside[..., 0]], [c.parts[1][0], beside[..., 1]]]):
        assert torch.equal(_run(c, mask=mask, parts=parts, max_len=LARGE), plain)


@pytest.mark.parametrize("bound", [5000, LARGE])
@pytest.mark.parametrize("hk,d", [(4, 64), (3, 64), (2, 128)])
def test_cut_batches_are_the_same_every_time(device, hk, d, bound):
    """Whatever an earlier call left in the workspace; with more blocks of rows and
    requests than a wave has lanes, and in a draining batch."""
    need = kv8.attention_kv8_workspace_bytes(70 * 9 + 300, 70, 4 * hk, hk, d, bound, 300)
    ws = torch.full((need,), 255, dtype=torch.uint8, device=device)
    for requests, long in ((70, 300), (40, 300), (9, 9), (1, 2)):
        print(f"kv8 attention, {requests} requests cut, {hk} heads of {d}", flush=True)
        old = [(37 * i) % 130 + 1100 * (i == 0) for i in range(requests)]
        new = [1 + i % 9 for i in range(requests)]
        new[-1] = long
        c = Cache8(device, 1220 + requests, old, new, q_heads=4 * hk, kv_heads=hk, head_dim=d, dtype=BF16)
        seen, mask = c.masks("chain")
        first = _run(c, mask=mask, workspace=ws, max_len=bound)
        _check(c, first, c.visible(seen))
        for fill in (0, 170):
            ws.fill_(fill)
            assert torch.equal(_run(c, mask=mask, workspace=ws, max_len=bound), first)
