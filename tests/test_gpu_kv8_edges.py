"""Rows of an 8-bit cache where a call has little to write or tiny units: destinations
without a source, blocks whose scale lies at the end of fp32's range."""

import numpy as np
import pytest
import torch

from akv_amd import kv8, rope
from oracle import kv8 as oracle
from tests.drafts import f64
from tests.kv8 import LARGEST, layer, same, values
from tests.test_gpu_kv8_rows import _move, _want

pytestmark = pytest.mark.gpu


def _pointers(caches):
    """The Reposition's tables of addresses: K, V, their scales."""
    return [torch.tensor([c[i][j].data_ptr() for c in caches], dtype=torch.int64, device=caches[0][0][0].device)
            for j in (0, 1) for i in (0, 1)]


def _i32(x, device):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to(device)


@pytest.mark.parametrize("rotary", [64, 20])
@pytest.mark.parametrize("skip,source", [(False, -1), (False, 320), (True, 0), (True, -1)])
@pytest.mark.parametrize("block", [1, 4, 16, 64])
def test_destinations_without_a_source_keep_codes_and_scale(device, block, skip, source, rotary):
    """Whole blocks, a block's first slots, slots behind rows: what they hold is the
    values that they held, in every layer, beside a row that does move."""
    dst, moved = np.concatenate((np.arange(64, 131), [197, 198, 256])), 256
    src = np.full(len(dst), source)
    src[-1] = 7
    pairs = np.stack((np.arange(len(dst)) + 9, np.arange(len(dst))), 1)
    caches = [layer(device, 80 + i, 320, 2, 64, "e4m3", block) for i in range(3)]
    before = [[[t.clone() for t in part] for part in cache] for cache in caches]
    table = rope.make_table("plain", rotary, 600, base=10000.0, dtype=torch.float32, device=device)
    (k, ks), (v, vs) = caches[0]
    kv8.reposition_kv8_layers(*_pointers(caches), k, v, ks, vs, _i32(src, device), _i32(dst, device), _i32(pairs, device),
                              table, scale_block=block, rotary_dim=rotary, skip_unmapped=skip)
    slots = np.delete(np.arange(320), moved)
    blocks = np.delete(np.arange(320 // block), moved // block)
    for cache, held in zip(caches, before):
        for (codes, scales), (c0, s0) in zip(cache, held):
            codes, c0 = codes.view(torch.uint8), c0.view(torch.uint8)
            assert not torch.equal(codes[moved], c0[moved])
            assert torch.equal(codes[slots], c0[slots]) and torch.equal(scales[blocks], s0[blocks])


@pytest.mark.parametrize("form", ["e4m3", "e5m2"])
@pytest.mark.parametrize("scale", [2.0 ** -149, 3 * 2.0 ** -149, 2.0 ** -130, 2.0 ** -127, 2.0 ** -126, 2.0 ** -101])
def test_rows_behind_the_smallest_scales(device, form, scale):
    """Rows that a block's tiny scale holds, zeros among them, are their codes in its
    units, appended or moved there."""
    hk, d, block = 2, 64, 4
    units = torch.arange(-8, 8).repeat(4).float()  # whole numbers up to 8 are codes
    rows = torch.stack((units, torch.zeros(d), units.flip(0)))[:, None].expand(3, hk, d)
    cache = layer(device, 90, 16, hk, d, form, block)
    for codes, scales in cache:
        scales[1:] = scale
        codes[12:15] = rows.to(device).to(codes.dtype)  # (the source of the move)
    (kc, ks), (vc, vs) = cache
    held = [t.view(torch.uint8)[:5].clone() for t in (kc, vc)]
    x = (rows.double() * scale).float().to(device)
    assert torch.equal(x.double().cpu(), rows.double() * scale)
    table = rope.make_table("plain", d, 10, base=10000.0, dtype=torch.float32, device=device)
    kv8.append_kv8(x, x, torch.arange(5, 8, device=device), kc, vc, ks, vs, scale_block=block)
    kv8.reposition_kv8_layers(*_pointers([cache]), kc, vc, ks, vs, _i32([12, 13, 14], device), _i32([9, 10, 11], device),
                              _i32([[3, 3]] * 3, device), table, scale_block=block)
    for (codes, scales), before in zip(cache, held):
        assert (scales[1:] == scale).all()
        assert torch.equal(codes.view(torch.uint8)[:5], before)
        for at in (5, 9):
            np.testing.assert_array_equal(values(codes[at: at + 3]), rows.double().numpy())


@pytest.mark.parametrize("form", ["e4m3", "e5m2"])
@pytest.mark.parametrize("block", [1, 4, 16, 64])
@pytest.mark.parametrize("d,rotary", [(64, 64), (128, 128), (80, 40), (64, 20)])
def test_a_table_at_any_address(device, d, rotary, block, form):
    """Rows of a table an odd number of elements apart, from an odd one on: the same
    codes and scales, bit for bit, whatever its type."""
    dst = np.concatenate((np.arange(128, 195), [256]))
    pairs = np.random.default_rng(block).integers(0, 600, (len(dst), 2))
    pairs[::7, 1] = pairs[::7, 0]
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        table = rope.make_table("plain", rotary, 600, base=10000.0, dtype=dtype, device=device)
        wide = torch.full((600, rotary + 9), 7.0, dtype=dtype, device=device)
        wide[:, 3: 3 + rotary] = table
        found = []
        for one in (table, wide[:, 3: 3 + rotary]):
            caches = [layer(device, 95 + i, 320, 3, d, form, block) for i in range(2)]
            (k, ks), (v, vs) = caches[0]
            kv8.reposition_kv8_layers(*_pointers(caches), k, v, ks, vs, _i32(np.arange(len(dst)), device),
                                      _i32(dst, device), _i32(pairs, device), one, scale_block=block, rotary_dim=rotary)
            found.append([(codes.view(torch.uint8), scales) for cache in caches for codes, scales in cache])
        for (c0, s0), (c1, s1) in zip(*found):
            assert torch.equal(c0, c1) and torch.equal(s0, s1)


@pytest.mark.parametrize("form", ["e4m3", "e5m2"])
def test_appended_values_that_only_move_are_the_same(device, form):
    """A scale for each token; among the rows some whose largest value was rounded down
    to what half their scale holds."""
    n, hk, d, most = 40, 2, 64, LARGEST[form]
    gen = torch.Generator().manual_seed(9)
    rows = torch.randn((n, 2 * hk, d), generator=gen) * torch.exp2(torch.randint(-20, 20, (n, 2 * hk, 1), generator=gen).float())
    rows[::3] *= most / 2 * 1.005 / rows[::3].abs().amax(-1, keepdim=True)
    cache = layer(device, 91, 2 * n, hk, d, form, 1)
    (kc, ks), (vc, vs) = cache
    rows = rows.to(device)
    kv8.append_kv8(rows[:, :hk], rows[:, hk:], torch.arange(n, device=device), kc, vc, ks, vs)
    held = [values(c[:n]) * f64(s[:n])[..., None] for c, s in cache]
    table = rope.make_table("plain", d, 50, base=10000.0, dtype=torch.float32, device=device)
    at = torch.arange(n, dtype=torch.int32, device=device)
    kv8.reposition_kv8_layers(*_pointers([cache]), kc, vc, ks, vs, at, at + n, torch.stack((at, at), 1), table)
    for (c, s), want in zip(cache, held):
        assert torch.equal(s[n::3], s[:n:3] / 2)
        np.testing.assert_array_equal(values(c[n:]) * f64(s[n:])[..., None], want)


@pytest.mark.parametrize("form", ["e4m3", "e5m2"])
@pytest.mark.parametrize("heads,d,rotary,block", [(3, 64, 64, 2), (2, 64, 64, 4), (5, 128, 128, 16), (1, 80, 40, 16),
                                                  (2, 64, 20, 8), (2, 96, 96, 32), (4, 128, 64, 64)])
def test_reposition_behind_rows(device, heads, d, rotary, block, form):
    """Runs that begin inside a block, whose scale grows for some heads and holds for
    others; one that fills its block, one of a single row, one that goes on into a fresh block."""
    first, last = 64 * 3 + 1, 64 * 5 + block + block // 2 + 1
    dst = np.concatenate((np.arange(first, 64 * 3 + block), [64 * 4 + block - 1], np.arange(64 * 5 + 1, last)))
    rng = np.random.default_rng(block)
    src = rng.permutation(64 * 3)[: len(dst)]
    pairs = rng.integers(0, 600, (len(dst), 2))
    pairs[::3, 1] = pairs[::3, 0]
    for neox in (True, False):
        print(f"move behind rows {heads} {d} {rotary} {block} {form} neox {neox}", flush=True)
        _move(device, 100 + block, src, dst, pairs, 64 * 7, heads=heads, d=d, rotary=rotary, neox=neox, form=form, block=block)


@pytest.mark.parametrize("form", ["e4m3", "e5m2"])
@pytest.mark.parametrize("rotary", [64, 20])
@pytest.mark.parametrize("block", [1, 4, 16])
def test_sources_under_scales_that_are_no_numbers(device, block, rotary, form):
    """NaN and infinite scales, codes of zero and others under them, to fresh blocks and behind
    rows: NaN (or infinite) codes, and the scale of the rows that are finite."""
    cache = layer(device, 97, 192, 2, 64, form, block)
    for codes, scales in cache:
        scales[: 32 // block] = float("nan")
        scales[32 // block: 64 // block] = float("inf")
        codes.view(torch.uint8)[:48:2] = 0
    dst = np.concatenate((np.arange(128, 128 + 2 * block), np.arange(160 + (block > 1), 160 + max(block, 2))))
    src = np.concatenate((np.arange(16, 16 + block), np.arange(47, 47 + len(dst) - block)))
    pairs = np.stack((np.arange(len(dst)) + 9, np.arange(len(dst))), 1)
    table = rope.make_table("plain", rotary, 600, base=10000.0, dtype=torch.float32, device=device)
    with np.errstate(all="ignore"):
        rows, units = zip(*(oracle.moved_rows(values(c), f64(s), src, pairs, table.cpu().numpy(), block, rotary, True,
                                              np.float32, i == 0) for i, (c, s) in enumerate(cache)))
        want = _want(cache, rows, dst, block, form, None, units)
    (k, ks), (v, vs) = cache
    kv8.reposition_kv8_layers(*_pointers([cache]), k, v, ks, vs, _i32(src, device), _i32(dst, device),
                              _i32(pairs, device), table, scale_block=block, rotary_dim=rotary)
    for got, w in zip(cache, want):
        same(got, w)
