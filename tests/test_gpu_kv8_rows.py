"""Rows into an 8-bit cache on the GPU, bit for bit against the oracle in fp32."""

import numpy as np
import pytest
import torch

from akv_amd import kv8, rope
from oracle import kv8 as oracle
from tests.drafts import HALF, f64
from tests.kv8 import FORMATS, LARGEST, layer, paged_slots, same, values

pytestmark = pytest.mark.gpu


def _want(cache, rows, slots, block, form, live=None, units=(1.0, 1.0)):
    """What the oracle leaves of [[k codes, k scales], [v codes, v scales]]."""
    out = []
    for (codes, scales), x, unit in zip(cache, rows, units):
        w, s = values(codes), f64(scales).copy()
        oracle.store(w, s, x, slots, block, form, live, unit)
        out.append((w, s))
    return out


def _f32(t):
    return t.detach().cpu().float().numpy()


def _append(device, seed, slots, total, *, hq, hk, d, rotary, neox=True, dtype=torch.bfloat16, form="e4m3", block=1,
            index=torch.int64, positions=None, spread=1.0, table_dtype=torch.float32, change=None, cache=None,
            q_in_place=False, rows=None):
    """One call against the oracle; returns the cache."""
    slots = np.asarray(slots)
    n, gen = len(slots), torch.Generator().manual_seed(seed)
    if rows is None:
        rows = (spread * torch.randn((n, hq + 2 * hk, d), generator=gen)).to(dtype)
    rows = rows.to(device)
    if cache is None:
        cache = layer(device, seed + 1, total, hk, d, form, block)
    if change is not None:
        rows, cache = change(rows, cache)
    q, k, v = rows.split((hq, hk, hk), 1)
    rope_args, table, q_out = {}, None, None
    if positions is None:
        positions = np.random.default_rng(seed).integers(0, 600, n)
    if rotary:
        table = rope.make_table("plain", rotary, 600, base=10000.0, dtype=table_dtype, device=device)
        rope_args = dict(positions=torch.from_numpy(np.asarray(positions)).to(index).to(device), cos_sin_cache=table,
                         rotary_dim=rotary, is_neox_style=neox)
        if hq:
            q_out = q if q_in_place else torch.full((n, hq, d), 7.0, dtype=dtype, device=device)
            rope_args.update(q=q, q_out=q_out)
    at = None if table is None else _f32(table)
    x = [oracle.rows_at(_f32(t), positions, at, rotary, neox, np.float32) for t in ((q, k) if rotary else (k,))]
    if not rotary:
        x = [None, *x]
    want = _want(cache, (x[1], _f32(v)), slots, block, form)
    kv8.append_kv8(k, v, torch.from_numpy(slots).to(index).to(device), cache[0][0], cache[1][0], cache[0][1],
                   cache[1][1], scale_block=block, **rope_args)
    for got, w in zip(cache, want):
        same(got, w)
    if q_out is not None:
        np.testing.assert_array_equal(f64(q_out), f64(torch.from_numpy(x[0]).to(dtype)))
    return cache


SHAPES = [
    # q heads, kv heads, head_dim, rotary, block, page, per request [from, to)
    (64, 8, 64, 64, 16, 16, [(4101, 4102)]),
    (2, 1, 16, 16, 1, 1, [(0, 1)]),
    (4, 2, 64, 64, 1, 1, [(0, 3), (7, 9), (100, 150)]),
    (6, 3, 64, 32, 2, 16, [(0, 37), (3, 4), (5, 8), (15, 16), (16, 17), (31, 33)]),
    (8, 8, 64, 64, 16, 16, [(0, 16), (1, 16), (15, 49), (7, 8), (5, 70)]),
    (5, 5, 128, 64, 4, 16, [(0, 333), (2, 3), (17, 18), (6, 30)]),
    (32, 8, 128, 128, 16, 16, [(0, 40), (9, 10), (8, 9), (7, 31), (30, 31)]),
    (7, 7, 80, 80, 8, 16, [(0, 19), (12, 15), (3, 9)]),
    (3, 1, 96, 48, 32, 32, [(0, 70), (31, 65), (16, 20), (33, 34)]),
    (2, 2, 64, 64, 64, 64, [(0, 130), (63, 65), (1, 64), (17, 20)]),
    (4, 4, 128, 128, 64, 64, [(0, 129), (40, 64), (7, 8)]),
    (2, 1, 112, 112, 1, 16, [(3, 40)]),
    (3, 3, 64, 20, 4, 16, [(0, 21), (6, 7), (2, 12)]),
    (2, 1, 48, 10, 1, 1, [(0, 9)]),
    (0, 4, 64, 64, 16, 16, [(3, 30)]),
    (0, 8, 128, 0, 16, 16, [(5, 100), (0, 3)]),
    (0, 3, 32, 0, 1, 1, [(0, 11)]),
]


@pytest.mark.parametrize("dtype,form", [(torch.bfloat16, "e4m3"), (torch.float16, "e5m2"), (torch.float32, "e4m3"),
                                        (torch.bfloat16, "e5m2")])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_append_is_the_oracles(device, shape, dtype, form):
    hq, hk, d, rotary, block, page, lengths = SHAPES[shape]
    for neox in (True, False):
        for spread in (1.0, 0.02):  # blocks that grow, and blocks that hold
            print(f"append {SHAPES[shape]} {dtype} {form} neox {neox} x {spread}", flush=True)
            slots, total = paged_slots(np.random.default_rng(shape), lengths, page)
            _append(device, shape, np.concatenate(slots), total, hq=hq, hk=hk, d=d, rotary=rotary, neox=neox, dtype=dtype,
                    form=form, block=block, spread=spread)


@pytest.mark.parametrize("d,block,tokens", [(64, 16, 5000), (128, 16, 2600), (64, 4, 9000), (128, 64, 3000),
                                            (64, 1, 4500)])
def test_many_tokens(device, d, block, tokens):
    """Several entries of the list to a wave, q rows one wave per token."""
    lengths = [(5, 5 + tokens // 3), (0, tokens // 2), (37, 38)] + [(i, i + 1) for i in range(60)]
    slots, total = paged_slots(np.random.default_rng(d), lengths, 64)
    _append(device, d + block, np.concatenate(slots), total, hq=5, hk=4, d=d, rotary=d // 2, block=block)


@pytest.mark.parametrize("rotary", [64, 20])
@pytest.mark.parametrize("block", [1, 16])
def test_entries_without_a_slot_or_position(device, rotary, block):
    """Padding among and behind the tokens takes nothing; a position outside the
    table gives NaN rows, which do not enter the scales."""
    slots, total = paged_slots(np.random.default_rng(1), [(0, 20), (3, 25), (40, 41)], 16)
    slots = np.concatenate((slots[0], [-1, total, -(2 ** 30)], slots[1], [-1] * 5, slots[2], [2 ** 31 - 1, -1]))
    positions = np.random.default_rng(2).integers(0, 600, len(slots))
    positions[[0, 9, 30]] = [-1, 600, 2 ** 31 - 1]
    for index in (torch.int32, torch.int64):
        cache = _append(device, 5, slots, total, hq=3, hk=2, d=64, rotary=rotary, block=block, positions=positions,
                        index=index)
        assert torch.isnan(cache[0][0][slots[0]].float()).all() and torch.isfinite(cache[1][0].float()).all()


@pytest.mark.parametrize("form", ["e4m3", "e5m2"])
@pytest.mark.parametrize("rotary", [0, 64])
def test_extreme_rows(device, form, rotary):
    """Zeros, the largest and smallest fp32 values, infinities and NaN, in fresh
    blocks and behind rows whose scale is tiny, huge, or no positive number."""
    slots, total = paged_slots(np.random.default_rng(3), [(0, 9), (2, 6), (5, 12), (0, 30), (1, 3)], 4)
    slots = np.concatenate(slots)
    n, hk, d = len(slots), 3, 64
    gen = torch.Generator().manual_seed(1)
    rows = torch.randn((n, 2 * hk, d), generator=gen)
    rows *= torch.exp2(torch.randint(-120, 110, (n, 2 * hk, 1), generator=gen).float())
    rows[::5] = 0
    rows[3, 0, 7], rows[3, 4, 9] = float("inf"), float("-inf")
    rows[11, 1, 0], rows[11, 5, 63] = float("nan"), float("nan")
    rows[12] = float("inf")
    rows[14, 0] = LARGEST[form]  # on the border of a power of two
    rows[14, 1] = float(np.nextafter(np.float32(LARGEST[form]), np.float32(np.inf)))

    def change(rows, cache):
        for i, (_, scales) in enumerate(cache):
            odd = torch.tensor([0.0, -1.0, float("nan"), float("inf"), 2.0 ** -120, 2.0 ** -149, 2.0 ** 100, 0.3])
            scales.view(-1)[i::3] = odd.repeat(1 + scales.numel())[: len(scales.view(-1)[i::3])].to(scales.device)
        return rows, cache

    with np.errstate(all="ignore"):
        _append(device, 3, slots, total, hq=0, hk=hk, d=d, rotary=rotary, dtype=torch.float32, form=form, block=4,
                rows=rows, change=change)


@pytest.mark.parametrize("offset", [0, 3, 8])
@pytest.mark.parametrize("block", [1, 16])
def test_strided_and_unaligned(device, offset, block):
    """Padded projections, K and V side by side in one pool, scales with the heads
    outside; at offset 3 nothing is aligned."""
    slots, total = paged_slots(np.random.default_rng(7), [(3, 40), (0, 7)], 16)
    slots, hk, d = np.concatenate(slots), 3, 64

    def change(rows, cache):
        wide = torch.zeros((rows.shape[0], rows.shape[1], d + 16), dtype=rows.dtype, device=device)
        wide[:, :, offset: offset + d] = rows
        both = torch.empty((total, hk, 2, d + 16), dtype=cache[0][0].dtype, device=device)
        flat = torch.empty((2, hk, -(-total // block) + 5), device=device)
        out = []
        for i, (codes, scales) in enumerate(cache):
            view = both[:, :, i, offset: offset + d]
            view.view(torch.uint8).copy_(codes.view(torch.uint8))
            s = flat[i].T[: len(scales)]
            s.copy_(scales)
            out.append([view, s])
        return wide[:, :, offset: offset + d], out

    _append(device, 11, slots, total, hq=4, hk=hk, d=d, rotary=64, block=block, dtype=torch.float16, change=change)


@pytest.mark.parametrize("rotary", [64, 20])
@pytest.mark.parametrize("n", [7, 2100])
def test_q_in_place_and_narrow_tables(device, rotary, n):
    slots, total = paged_slots(np.random.default_rng(8), [(0, n)], 16)
    _append(device, 12, slots[0], total, hq=9, hk=2, d=64, rotary=rotary, block=16, q_in_place=True,
            table_dtype=torch.bfloat16 if rotary == 64 else torch.float16, index=torch.int32)


def test_what_is_not_written_stays(device):
    """Rows above the last of a block, other blocks, other scales."""
    cache = layer(device, 1, 64, 2, 64, "e4m3", 16)
    before = [[t.clone() for t in part] for part in cache]
    _append(device, 13, [19, 20], 64, hq=0, hk=2, d=64, rotary=64, block=16, cache=cache, spread=50.0)
    for (codes, scales), (c0, s0) in zip(cache, before):
        kept = [i for i in range(64) if not 16 <= i <= 20]
        assert torch.equal(codes.view(torch.uint8)[kept], c0.view(torch.uint8)[kept])
        assert torch.equal(scales[[0, 2, 3]], s0[[0, 2, 3]]) and (scales[1] > s0[1]).all()


def test_no_tokens_and_pools_of_nothing(device):
    cache = layer(device, 1, 16, 2, 64, "e4m3", 1)
    _append(device, 14, np.zeros(0, dtype=np.int64), 16, hq=2, hk=2, d=64, rotary=64, cache=cache)
    empty = [[t[:0] for t in part] for part in cache]
    # every slot is outside: q is rotated all the same
    _append(device, 15, np.arange(5), 0, hq=2, hk=2, d=64, rotary=64, cache=empty)


def test_slots_past_32_bits(device):
    """Codes that lie beyond 4 GiB of their buffer."""
    hk, d, slots = 8, 128, (1 << 22) + 64
    pools = [torch.zeros((slots, hk, d), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.zeros((slots // 16, hk), device=device) for _ in range(2)]
    k, v = (torch.randn((40, hk, d), device=device, dtype=torch.bfloat16) for _ in range(2))
    far = torch.arange(40, device=device) + slots - 40
    kv8.append_kv8(k, v, far, *pools, *scales, scale_block=16)
    near = [torch.zeros((48, hk, d), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2)]
    near_scales = [torch.zeros((3, hk), device=device) for _ in range(2)]
    kv8.append_kv8(k, v, torch.arange(8, 48, device=device), *near, *near_scales, scale_block=16)
    for p, s, q, t in zip(pools, scales, near, near_scales):
        assert torch.equal(p.view(torch.uint8)[-40:], q.view(torch.uint8)[-40:]) and torch.equal(s[-3:], t)
        assert not p.view(torch.uint8)[:-40].any() and not s[:-3].any()
    # and moved from there to slots of the lower half
    src = far.int()[8:24].contiguous()
    dst, pairs = torch.arange(32, 48, dtype=torch.int32, device=device), torch.full((16, 2), 5, dtype=torch.int32, device=device)
    table = rope.make_table("plain", d, 10, base=10000.0, dtype=torch.float32, device=device)
    pointers = [torch.tensor([t.data_ptr()], dtype=torch.int64, device=device) for t in (*pools, *scales)]
    kv8.reposition_kv8_layers(*pointers, *pools, *scales, src, dst, pairs, table, scale_block=16)
    for p, s in zip(pools, scales):
        a, b = values(p[dst.long()]) * f64(s[2])[:, None], values(p[src.long()]) * f64(s[src.long() // 16])[..., None]
        np.testing.assert_array_equal(a, b)  # (powers of two: nothing is rounded that is not tiny)


# ---------------------------------------------------------------------------
# Reposition


def _move(device, seed, src, dst, pairs, slots, *, layers=3, heads=2, d=64, rotary=64, neox=True, form="e4m3", block=1,
          skip=False, status=None, pad=0, table_dtype=torch.float32, untouched=False):
    src, dst, pairs = (np.asarray(t) for t in (src, dst, pairs))
    caches = [layer(device, seed + i, slots, heads, d, form, block) for i in range(layers)]
    if pad:  # layers that begin at odd addresses
        for cache in caches:
            for part in cache:
                raw = torch.zeros(part[0].numel() + pad, dtype=torch.uint8, device=device)[pad:]
                raw.copy_(part[0].view(torch.uint8).flatten())
                part[0] = raw.view(part[0].dtype).view(part[0].shape)
    table = rope.make_table("plain", rotary, 600, base=10000.0, dtype=table_dtype, device=device)
    usable = (src >= int(skip)) & (src < slots)
    at = np.where(usable, src, 0)
    to = np.where((dst >= int(skip)) & (dst < slots), dst, -1)
    want = []
    for cache in caches:
        rows = [oracle.moved_rows(values(c), f64(s), at, pairs, _f32(table), block, rotary, neox, np.float32, i == 0)
                for i, (c, s) in enumerate(cache)]
        rows, units = zip(*rows)
        want.append([(values(c), f64(s)) for c, s in cache] if untouched
                    else _want(cache, rows, to, block, form, usable, units))
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to(device)  # noqa: E731
    pointers = [torch.tensor([c[i][j].data_ptr() for c in caches], dtype=torch.int64, device=device)
                for j in (0, 1) for i in (0, 1)]
    kv8.reposition_kv8_layers(*pointers, caches[0][0][0], caches[0][1][0], caches[0][0][1], caches[0][1][1], dev(src),
                              dev(dst), dev(pairs), table, scale_block=block, is_neox_style=neox, rotary_dim=rotary,
                              skip_unmapped=skip, status=status)
    for cache, w in zip(caches, want):
        for got, one in zip(cache, w):
            same(got, one)
    return caches


MOVES = [
    # heads, head_dim, rotary, block, page, layers, per request kept [from, to)
    (8, 64, 64, 1, 1, 3, [(10, 90), (5, 30)]),
    (2, 64, 64, 1, 1, 1, [(3, 4)]),
    (8, 64, 64, 16, 16, 5, [(0, 100), (32, 50)]),
    (5, 128, 128, 16, 16, 4, [(16, 49), (0, 1)]),
    (3, 128, 64, 4, 16, 2, [(0, 37)]),
    (1, 80, 80, 8, 16, 9, [(0, 21)]),
    (2, 96, 48, 64, 64, 2, [(0, 130), (64, 80)]),
    (4, 64, 64, 32, 32, 3, [(32, 99)]),
    (2, 128, 128, 64, 64, 2, [(0, 65)]),
    (2, 64, 20, 4, 16, 2, [(0, 19)]),
    (1, 16, 16, 2, 16, 6, [(0, 5)]),
]


@pytest.mark.parametrize("form", ["e4m3", "e5m2"])
@pytest.mark.parametrize("case", range(len(MOVES)))
def test_reposition_is_the_oracles(device, case, form):
    heads, d, rotary, block, page, layers, lengths = MOVES[case]
    for neox in (True, False):
        print(f"move {MOVES[case]} {form} neox {neox}", flush=True)
        rng = np.random.default_rng(case)
        slots, total = paged_slots(rng, [(0, 200)] + lengths, page)
        dst = np.concatenate(slots[1:])
        src = rng.permutation(slots[0])[: len(dst)]
        pairs = rng.integers(0, 600, (len(dst), 2))
        pairs[::4, 1] = pairs[::4, 0]
        _move(device, 20 + case, src, dst, pairs, total, layers=layers, heads=heads, d=d, rotary=rotary, neox=neox,
              form=form, block=block)


@pytest.mark.parametrize("block,tokens", [(1, 3000), (16, 6000), (4, 5000)])
def test_reposition_of_many_tokens(device, block, tokens):
    rng = np.random.default_rng(block)
    slots, total = paged_slots(rng, [(0, tokens)] + [(0, tokens // 9)] * 9, 16)
    dst = np.concatenate(slots[1:])
    src = rng.permutation(slots[0])[: len(dst)]
    _move(device, 40, src, dst, rng.integers(0, 600, (len(dst), 2)), total, layers=13, heads=4, block=block)


@pytest.mark.parametrize("skip", [True, False])
@pytest.mark.parametrize("block", [1, 4])
def test_reposition_passes_over_what_has_no_slot(device, skip, block):
    """Sources and destinations outside the pool, slot 0 with and without
    skip_unmapped, positions outside the table."""
    src = np.array([1, 2, 3, -1, 5, 0, 7, 8, 9, 40, 11, 12])
    dst = np.array([16, 17, 18, 19, 20, 24, 25, -1, 28, 29, 30, 60])
    pairs = np.stack((np.arange(12) * 3, np.arange(12)), 1)
    pairs[1], pairs[2], pairs[6] = [-4, 7], [3, 600], [-9, -9]
    caches = _move(device, 50, src, dst, pairs, 40, skip=skip, block=block)
    assert torch.isnan(caches[0][0][0][17].float()).all() and torch.isfinite(caches[0][0][0][25].float()).all()


@pytest.mark.parametrize("form", ["e4m3", "e5m2"])
def test_values_that_only_move_keep_code_and_scale(device, form):
    """A scale for each token: V rows always, K rows at their position."""
    src, dst = np.arange(30), np.arange(30, 60)
    pairs = np.stack((np.arange(30), np.arange(30)), 1)
    caches = [layer(device, 9, 64, 2, 64, form, 1)]
    for codes, _ in caches[0]:  # every row's largest code is one that its scale was chosen for
        codes.view(torch.uint8)[:, :, 5] = 0x7e if form == "e4m3" else 0x7b
    pointers = [torch.tensor([caches[0][i][j].data_ptr()], dtype=torch.int64, device=device) for j in (0, 1) for i in (0, 1)]
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to(device)  # noqa: E731
    table = rope.make_table("plain", 64, 600, base=10000.0, dtype=torch.float32, device=device)
    (k, ks), (v, vs) = caches[0]
    kv8.reposition_kv8_layers(*pointers, k, v, ks, vs, dev(src), dev(dst), dev(pairs), table)
    for codes, scales in caches[0]:
        assert torch.equal(codes.view(torch.uint8)[30:60], codes.view(torch.uint8)[:30])
        assert torch.equal(scales[30:60], scales[:30])


@pytest.mark.parametrize("pad", [1, 4, 8])
@pytest.mark.parametrize("rotary", [64, 20])
def test_reposition_of_layers_at_any_address(device, pad, rotary):
    slots, total = paged_slots(np.random.default_rng(pad), [(0, 64), (0, 40)], 16)
    pairs = np.random.default_rng(1).integers(0, 600, (40, 2))
    _move(device, 60, slots[0][:40], slots[1], pairs, total, block=16, pad=pad, rotary=rotary)


@pytest.mark.parametrize("table_dtype", [torch.float16, torch.bfloat16])
def test_reposition_with_narrow_tables(device, table_dtype):
    _move(device, 61, np.arange(20), np.arange(20, 40), np.stack((np.arange(20) + 300, np.arange(20)), 1), 40,
          table_dtype=table_dtype)


def test_reposition_behind_a_gate(device):
    word = torch.tensor([1], dtype=torch.int32, device=device)
    args = (device, 62, np.arange(8), np.arange(8, 16), np.stack((np.arange(8) + 9, np.arange(8)), 1), 16)
    _move(*args, status=word, untouched=True)
    word.fill_(4)
    _move(*args, status=word)


@pytest.mark.parametrize("form,block", [("e4m3", 1), ("e4m3", 16), ("e5m2", 16)])
def test_moved_rows_are_those_appended_there(device, form, block):
    """Rows appended at p and moved to p' are the rows appended at p', but for
    two roundings to 8 bits: half a step each, of the row's value and, where a
    pair's other value is larger, of that one."""
    n, hk, d = 48, 2, 64
    gen = torch.Generator().manual_seed(4)
    k, v = (torch.randn((n, hk, d), generator=gen).to(torch.bfloat16).to(device) for _ in range(2))
    table = rope.make_table("plain", d, 600, base=10000.0, dtype=torch.float32, device=device)
    cache = layer(device, 5, 3 * 48, hk, d, form, block)
    (kc, ks), (vc, vs) = cache
    old, new = torch.arange(n, device=device) + 400, torch.arange(n, device=device) + 7
    at = lambda i: torch.arange(48 * i, 48 * i + n, device=device)  # noqa: E731
    kv8.append_kv8(k, v, at(0), kc, vc, ks, vs, scale_block=block, positions=old, cos_sin_cache=table)
    kv8.append_kv8(k, v, at(1), kc, vc, ks, vs, scale_block=block, positions=new, cos_sin_cache=table)
    pointers = [torch.tensor([t.data_ptr()], dtype=torch.int64, device=device) for t in (kc, vc, ks, vs)]
    kv8.reposition_kv8_layers(*pointers, kc, vc, ks, vs, at(0).int(), at(2).int(),
                              torch.stack((old, new), 1).int().contiguous(), table, scale_block=block)
    value = lambda c, s, i: values(c[at(i)]) * f64(s)[at(i).cpu().numpy() // block][..., None]  # noqa: E731
    moved, there = value(kc, ks, 2), value(kc, ks, 1)
    half = d // 2
    pair = np.hypot(there[..., :half], there[..., half:])
    pair = np.concatenate((pair, pair), -1)
    half_step = {"e4m3": 2.0 ** -4, "e5m2": 2.0 ** -3}[form]
    # three roundings: at p, at p', and after the move; tiny values by half the smallest step of a scale
    smallest = f64(ks).max() * {"e4m3": 2.0 ** -10, "e5m2": 2.0 ** -17}[form]
    assert (np.abs(moved - there) <= 3 * half_step * 1.5 * pair + 6 * smallest).all()
    np.testing.assert_allclose(value(vc, vs, 2), value(vc, vs, 0), atol=2 * f64(vs).max() * (2.0 ** -10 if form == "e4m3" else 2.0 ** -17))


# ---------------------------------------------------------------------------
# Rotations of an odd number of eights


HALF_CHUNKS = [
    # head_dim, rotary, block
    (80, 40, 16), (80, 40, 1), (64, 24, 4), (64, 56, 1), (128, 8, 64), (16, 8, 16), (112, 56, 32), (128, 120, 1), (48, 24, 64),
]


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("case", range(len(HALF_CHUNKS)))
def test_rotations_that_end_inside_a_chunk(device, case, neox):
    """Infinities and NaN behind the rotation touch no value of it, and q may be q_out."""
    d, rotary, block = HALF_CHUNKS[case]
    slots, total = paged_slots(np.random.default_rng(case), [(0, 90), (3, 20), (7, 8)], 64)
    slots = np.concatenate(slots)
    rows = torch.randn((len(slots), 4, d), generator=torch.Generator().manual_seed(case))
    rows[3, 0, rotary], rows[9, 1, d - 1], rows[17, 2, rotary:] = float("inf"), float("nan"), float("-inf")
    for dtype, form in ((torch.bfloat16, "e4m3"), (torch.float32, "e5m2"), (torch.float16, "e4m3")):
        print(f"append {HALF_CHUNKS[case]} {dtype} neox {neox}", flush=True)
        with np.errstate(all="ignore"):
            _append(device, case, slots, total, hq=0, hk=2, d=d, rotary=rotary, neox=neox, dtype=dtype, form=form,
                    block=block, rows=rows.to(dtype))
        _append(device, case, slots, total, hq=3, hk=2, d=d, rotary=rotary, neox=neox, dtype=dtype, form=form, block=block,
                q_in_place=True, table_dtype=torch.bfloat16 if case % 2 else torch.float32)
    print(f"move {HALF_CHUNKS[case]} neox {neox}", flush=True)
    fresh, total = paged_slots(np.random.default_rng(case), [(0, 100), (0, 65), (0, 9)], 64)
    src, dst = fresh[0][:74], np.concatenate(fresh[1:])
    pairs = np.random.default_rng(case).integers(0, 600, (74, 2))
    pairs[::5, 1] = pairs[::5, 0]
    _move(device, 70 + case, src, dst, pairs, total, layers=2, heads=3, d=d, rotary=rotary, neox=neox, block=block)
    pairs[7, 0] = 600  # a position outside the table: the other form of the kernel
    _move(device, 70 + case, src, dst, pairs, total, layers=2, heads=3, d=d, rotary=rotary, neox=neox, block=block, pad=3)


# ---------------------------------------------------------------------------
# Streams and graphs


def test_captured_calls_follow_their_inputs(device):
    """A captured append and move, replayed over changing rows with eager work
    between, against eager calls on a copy."""
    n, hk, d, block = 33, 2, 64, 16
    gen = torch.Generator().manual_seed(6)
    table = rope.make_table("plain", d, 600, base=10000.0, dtype=torch.float32, device=device)
    k, v = (torch.zeros((n, hk, d), dtype=torch.bfloat16, device=device) for _ in range(2))
    q, q_out = (torch.zeros((n, 4, d), dtype=torch.bfloat16, device=device) for _ in range(2))
    slots, positions = torch.arange(5, 5 + n, device=device), torch.arange(n, device=device)
    src, dst = slots[:20].int().contiguous(), torch.arange(48, 68, dtype=torch.int32, device=device)
    pairs = torch.stack((torch.arange(20), torch.arange(20) + 100), 1).int().to(device)

    def step(cache, q_out):
        (kc, ks), (vc, vs) = cache
        kv8.append_kv8(k, v, slots, kc, vc, ks, vs, scale_block=block, positions=positions, cos_sin_cache=table, q=q,
                       q_out=q_out)
        kv8.reposition_kv8_layers(*pointers[id(cache)], kc, vc, ks, vs, src, dst, pairs, table, scale_block=block)

    caches = [layer(device, 7, 96, hk, d, "e4m3", block) for _ in range(2)]
    pointers = {id(c): [torch.tensor([c[i][j].data_ptr()], dtype=torch.int64, device=device) for j in (0, 1) for i in (0, 1)]
                for c in caches}
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        step(caches[0], q_out)
    eager_out = torch.empty_like(q_out)
    for i in range(4):
        for t in (q, k, v):
            t.copy_((torch.randn(t.shape, generator=gen) * 3.0 ** i).to(t.dtype))
        if i == 2:
            torch.cuda.synchronize()
        graph.replay()
        step(caches[1], eager_out)
        torch.cuda.synchronize()
        assert torch.equal(q_out, eager_out)
        for one, two in zip(*caches):
            assert torch.equal(one[0].view(torch.uint8), two[0].view(torch.uint8)) and torch.equal(one[1], two[1])


def test_two_streams_beside_each_other(device):
    """Different rows of one cache, on two streams at once."""
    n, hk, d = 64, 2, 64
    cache = layer(device, 8, 2 * n, hk, d, "e4m3", 16)
    (kc, ks), (vc, vs) = cache
    rows = [torch.randn((n, 2 * hk, d), device=device, dtype=torch.bfloat16) for _ in range(2)]
    want = _want(cache, [np.concatenate([_f32(r[:, :hk]) for r in rows]), np.concatenate([_f32(r[:, hk:]) for r in rows])],
                 np.arange(2 * n), 16, "e4m3")
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            kv8.append_kv8(rows[i][:, :hk], rows[i][:, hk:], torch.arange(n, device=device) + n * i, kc, vc, ks, vs,
                           scale_block=16)
    torch.cuda.synchronize()
    for got, w in zip(cache, want):
        same(got, w)


def test_formats_are_torchs():
    assert set(FORMATS.values()) == {torch.float8_e4m3fn, torch.float8_e5m2}
    assert HALF[torch.bfloat16] == torch.finfo(torch.bfloat16).eps / 2
