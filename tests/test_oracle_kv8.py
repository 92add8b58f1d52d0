"""The 8-bit cache's oracle against torch's 8-bit types and against itself."""

import numpy as np
import pytest
import torch

from akv_amd import rope
from oracle import kv8 as oracle
from tests.kv8 import FORMATS, LARGEST, paged_slots, values


@pytest.mark.parametrize("form", ["e4m3", "e5m2"])
def test_rounding_is_torchs(form):
    codes = torch.arange(256, dtype=torch.uint8).view(FORMATS[form])
    table = np.unique(values(codes)[np.isfinite(values(codes))])
    assert table.max() == LARGEST[form] == oracle.LARGEST[form]
    between = (table[1:] + table[:-1]) / 2
    x = np.concatenate((table, between, np.nextafter(between.astype(np.float32), np.float32(np.inf)),
                        np.nextafter(between.astype(np.float32), np.float32(-np.inf)), [0.0, np.nan]))
    x = x.astype(np.float32)
    want = torch.from_numpy(x).to(FORMATS[form])
    np.testing.assert_array_equal(oracle.rounded(x, form), values(want))
    special = oracle.rounded([np.inf, -np.inf], form)
    assert np.isnan(special).all() if form == "e4m3" else (special == [np.inf, -np.inf]).all()


@pytest.mark.parametrize("form", ["e4m3", "e5m2"])
def test_scales_are_the_least_that_hold(form):
    rng = np.random.default_rng(1)
    top = np.concatenate((np.exp(rng.uniform(-60, 60, 400)), LARGEST[form] * 2.0 ** np.arange(-90, 40),
                          np.nextafter(LARGEST[form] * 2.0 ** np.arange(-90, 40), np.inf))).astype(np.float32)
    top = np.concatenate((top, np.nextafter(top, np.float32(np.inf)), np.nextafter(top, np.float32(0))))
    s = oracle.fitting(top, form)
    assert (np.frexp(s)[0] == 0.5).all()
    assert (top <= LARGEST[form] * s).all()
    assert ((top > LARGEST[form] * s / 2) | (s == oracle.LEAST_SCALE)).all()
    assert (oracle.fitting(np.array([0.0, 1e-38]), form) == oracle.LEAST_SCALE).all()
    before = np.exp(rng.uniform(-30, 30, len(top))).astype(np.float32).astype(np.float64)
    after = oracle.grown(top, before, form)
    ratio = after / before
    assert (np.frexp(ratio)[0] == 0.5).all() and (ratio >= 1).all()
    assert (top <= LARGEST[form] * after * (1 + 2.0 ** -23)).all()
    assert (top[ratio > 1] > LARGEST[form] * after[ratio > 1] / 2 * (1 - 2.0 ** -23)).all()
    for odd in (0.0, -1.0, np.nan, np.inf):
        assert oracle.grown(np.array([3.0]), np.array([odd]), form) == oracle.fitting(3.0, form)


def test_runs():
    assert oracle.runs([3, 4, 5, 8, 9, -1, 10, 12, 12, 40], 4, 16) == [(0, 1), (1, 2), (3, 2), (6, 1), (7, 1), (8, 1)]
    assert oracle.runs([0, 1, 2], 1, 3) == [(0, 1), (1, 1), (2, 1)]


@pytest.mark.parametrize("form", ["e4m3", "e5m2"])
@pytest.mark.parametrize("block", [1, 4, 16])
def test_together_or_one_by_one(form, block):
    """The scales are the same; codes differ where a growing scale took them
    below the smallest normal one, by a step there."""
    rng = np.random.default_rng(block)
    slots, total = paged_slots(rng, [(0, 33), (5, 20)], 16)
    slots = np.concatenate(slots)
    rows = rng.standard_normal((len(slots), 2, 16)) * np.exp(rng.uniform(-3, 3, (len(slots), 1, 1)))
    caches = []
    for step in (len(slots), 1):
        codes, scales = np.ones((total, 2, 16)), np.full((total // block, 2), 2.0 ** -7)
        for t in range(0, len(slots), step):
            oracle.store(codes, scales, rows[t: t + step], slots[t: t + step], block, form)
        caches.append((codes, scales))
    np.testing.assert_array_equal(caches[0][1], caches[1][1])
    normal = 2.0 ** oracle.SMALLEST[form]
    step = normal * 2.0 ** -oracle.DIGITS[form]
    off = np.abs(caches[0][0] - caches[1][0])
    assert (off[np.abs(caches[0][0]) > normal] == 0).all() and off.max() <= 2 * step


@pytest.mark.parametrize("form", ["e4m3", "e5m2"])
@pytest.mark.parametrize("neox", [True, False])
def test_fp32_rows_are_the_64_bit_rows(form, neox):
    """Rotated rows: two products and a sum, 2^-24 each of the magnitudes they
    add, and for moved ones the factors' six operations more."""
    rng = np.random.default_rng(3)
    table = rope.make_table("plain", 32, 900, base=10000.0, dtype=torch.float32, device="cpu").numpy()
    x, positions = rng.standard_normal((40, 2, 48)).astype(np.float32), rng.integers(-2, 902, 40)
    got, want = (oracle.rows_at(x, positions, table, 32, neox, real) for real in (np.float32, np.float64))
    size = np.abs(x).max()
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    assert np.nanmax(np.abs(got - want)) <= 3 * 2.0 ** -24 * 2 * size
    assert np.isnan(want[(positions < 0) | (positions >= 900)]).all()
    codes = oracle.rounded(rng.standard_normal((64, 2, 48)) * 50, form)
    scales = np.exp2(rng.integers(-9, -5, (16, 2)).astype(np.float64))
    src, pairs = rng.permutation(64)[:30], rng.integers(0, 900, (30, 2))
    pairs[::5, 1] = pairs[::5, 0]
    got, want = (np.multiply(*oracle.moved_rows(codes, scales, src, pairs, table, 4, 32, neox, real, True))
                 for real in (np.float32, np.float64))
    size = np.abs(want).max()
    assert np.abs(got - want).max() <= 10 * 2.0 ** -24 * 2 * size
    # the definition: the old position undone, the new one done
    half = 16
    one = np.arange(half) if neox else 2 * np.arange(half)
    two = one + half if neox else one + 1
    phase = table[:, :half].astype(np.float64) + 1j * table[:, half:]
    raw = codes[src] * scales[src // 4][..., None]
    z = (raw[..., one] + 1j * raw[..., two]) * (phase[pairs[:, 1]] / phase[pairs[:, 0]])[:, None]
    moved = pairs[:, 0] != pairs[:, 1]
    np.testing.assert_allclose(want[moved][..., one], z[moved].real, atol=1e-12)
    np.testing.assert_allclose(want[moved][..., two], z[moved].imag, atol=1e-12)
    np.testing.assert_array_equal(want[~moved], raw[~moved])


@pytest.mark.parametrize("form", ["e4m3", "e5m2"])
@pytest.mark.parametrize("block", [1, 4])
def test_runs_without_a_live_row_leave_the_block(form, block):
    """A slot behind rows, a block's first ones, a whole block; of one with a live row the others' codes stay."""
    rng = np.random.default_rng(block)
    codes, scales = oracle.rounded(rng.standard_normal((24, 2, 16)) * 40, form), np.full((24 // block, 2), 0.25)
    slots = np.array([5, 8, 9, 12, 13, 14, 15, 16, 17])
    live = np.array([0, 0, 0, 0, 0, 0, 0, 0, 1], dtype=bool)
    before = codes.copy(), scales.copy()
    oracle.store(codes, scales, np.full((9, 2, 16), 3.0), slots, block, form, live)
    at = 17 // block
    np.testing.assert_array_equal(np.delete(codes, 17, 0), np.delete(before[0], 17, 0))
    np.testing.assert_array_equal(np.delete(scales, at, 0), np.delete(before[1], at, 0))
    np.testing.assert_array_equal(codes[17] * scales[at][:, None], np.full((2, 16), 3.0))


@pytest.mark.parametrize("form", ["e4m3", "e5m2"])
@pytest.mark.parametrize("real", [np.float32, np.float64])
def test_rows_behind_the_smallest_scales(form, real):
    """Multiples of a scale that holds them are those codes, also where 1 / scale is past fp32's range."""
    units = np.array([0.0, 1.0, -7.0, 8.0]).repeat(4)[None, None]
    for scale in (2.0 ** -149, 3 * 2.0 ** -149, 2.0 ** -130, 2.0 ** -126):
        for unit in (1.0, scale):
            codes, scales = np.zeros((4, 1, 16)), np.full((1, 1), scale)
            oracle.store(codes, scales, (units * (scale / unit)).astype(real), [2], 4, form, units=unit)
            np.testing.assert_array_equal(codes[2:3], units)
            assert scales[0, 0] == scale


@pytest.mark.parametrize("slots", [[4, 6], [4, -1, 5], [5, 4], [0, 4, 1]])
def test_lists_that_come_to_a_block_twice(slots):
    """What such a call leaves is undefined: the oracle says so, and no test compares with it."""
    rows = np.ones((len(slots), 1, 16))
    with pytest.raises(ValueError):
        oracle.store(np.zeros((8, 1, 16)), np.ones((2, 1)), rows, np.array(slots), 4, "e4m3")
    oracle.store(np.zeros((8, 1, 16)), np.ones((8, 1)), rows, np.array(slots), 1, "e4m3")
