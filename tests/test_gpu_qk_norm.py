"""Norms, rotation and pool write on the GPU against the 64-bit oracle."""

import numpy as np
import pytest
import torch

from akv_amd import qk_norm, rope
from oracle import drafts
from tests.drafts import HALF, f64

pytestmark = pytest.mark.gpu


def _tolerance(dtype, d, want, size):
    """fp32: the mean of d squares is off by at most d 2^-24 of itself, its root
    by half that; the root, the division, the two products and the rotation's
    three operations by 2^-24 each of the magnitudes they add; then one rounding
    (fp16 results below its normal range: half its smallest step)."""
    tol = (d / 2 + 10) * 2.0 ** -24 * size + HALF[dtype] * np.abs(want) * 1.001
    return tol + (2.0 ** -25 if dtype == torch.float16 else 0) + 1e-37


def _case(device, seed, n, hq, hk, d, dtype, *, weights=True, weight_dtype=None, table_dtype=torch.float32, rotary=None,
          scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    rotary = rotary or d
    make = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    qkv = (make(n, hq + 2 * hk, d) * scale).to(dtype).to(device)
    w = [(1 + 0.3 * make(d)).to(weight_dtype or dtype).to(device) if weights else None for _ in range(2)]
    table = rope.make_table("plain", rotary, 500, base=10000.0, dtype=table_dtype, device=device)
    slots = n + 5
    return dict(qkv=qkv, q=qkv[:, :hq], k=qkv[:, hq: hq + hk], v=qkv[:, hq + hk:], w=w, table=table, rotary=rotary,
                positions=torch.randint(0, 500, (n,), generator=gen).to(device),
                slots=torch.randperm(slots, generator=gen)[:n].to(device),
                pool=[torch.full((slots, hk, d), 7.0, dtype=dtype, device=device) for _ in range(2)])


def _want(c, x, w, neox, eps):
    pos = c["positions"].cpu().numpy().astype(np.int64)
    rows = f64(c["table"])
    known = (pos >= 0) & (pos < len(rows))
    at = np.where(known[:, None], rows[np.where(known, pos, 0)], np.nan)
    return drafts.qk_norm_rope(f64(x), None if w is None else f64(w), eps, at, c["rotary"], neox)


def _check(c, q_out, k_out, *, neox=True, eps=1e-6, pool=True, k=None, q=None):
    d, dtype = c["q"].shape[2], c["q"].dtype
    for x, w, got in ((c["q"] if q is None else q, c["w"][0], q_out), (c["k"] if k is None else k, c["w"][1], k_out)):
        if got is None:
            continue
        want, size = _want(c, x, w, neox, eps)
        have = f64(got)
        np.testing.assert_array_equal(np.isnan(have), np.isnan(want))
        off = np.abs(have - want) - _tolerance(dtype, d, want, size)
        assert (np.nan_to_num(off, nan=0.0) <= 0).all(), f"worst off by {np.nanmax(off):.3g}"
    if pool:
        want, size = _want(c, c["k"] if k is None else k, c["w"][1], neox, eps)
        kp, vp = f64(c["pool"][0]), f64(c["pool"][1])
        slots = c["slots"].cpu().numpy().astype(np.int64)
        stored = np.ones(len(kp), dtype=bool)
        for t, s in enumerate(slots):
            if not 0 <= s < len(kp):
                continue
            np.testing.assert_array_equal(vp[s], f64(c["v"][t]))
            if np.isnan(want[t]).any():
                assert (kp[s] == 7).all()
            else:
                assert (np.abs(kp[s] - want[t]) <= _tolerance(dtype, d, want[t], size[t])).all()
            stored[s] = False
        assert (kp[stored] == 7).all() and (vp[stored] == 7).all(), "rows of other slots were written"


def _run(c, *, neox=True, eps=1e-6, k_out=None, q_out=None, pool=True):
    q_out = torch.empty_like(c["q"]) if q_out is None else q_out
    extra = dict(slot_map=c["slots"], k_buffer=c["pool"][0], v_buffer=c["pool"][1]) if pool else {}
    got = qk_norm.qk_norm_rope(c["q"], c["k"], c["v"] if pool else None, c["w"][0], c["w"][1], c["positions"], c["table"],
                               q_out, eps=eps, k_out=k_out, rotary_dim=c["rotary"], is_neox_style=neox, **extra)
    assert got is q_out
    return q_out


SHAPES = [
    # tokens, q heads, kv heads, head_dim, rotary
    (1, 64, 8, 64, 64), (1, 1, 1, 16, 16), (3, 4, 2, 128, 64), (67, 32, 8, 128, 128), (130, 7, 1, 80, 80),
    (33, 6, 3, 96, 48), (5, 3, 1, 256, 32), (4, 2, 2, 512, 512), (9, 5, 2, 64, 20), (11, 3, 1, 40, 10),
    (2, 2, 1, 7, 4), (17, 9, 4, 48, 16), (5, 1, 1, 32, 32), (4097, 8, 2, 64, 64),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_matches_oracle(device, shape, dtype):
    n, hq, hk, d, rotary = SHAPES[shape]
    for neox in (True, False):
        print(f"qk norm {SHAPES[shape]} {dtype} neox {neox}", flush=True)
        c = _case(device, shape, n, hq, hk, d, dtype, rotary=rotary)
        k_out = torch.empty_like(c["k"]) if neox else None
        _check(c, _run(c, neox=neox, k_out=k_out), k_out, neox=neox)


@pytest.mark.parametrize("d", [64, 72])
@pytest.mark.parametrize("weight_dtype,table_dtype", [(torch.float32, torch.bfloat16), (torch.float16, torch.float16),
                                                      (torch.bfloat16, torch.float32), (None, torch.float32)])
def test_weight_and_table_types(device, d, weight_dtype, table_dtype):
    c = _case(device, 3, 21, 4, 2, d, torch.bfloat16, weights=weight_dtype is not None, weight_dtype=weight_dtype,
              table_dtype=table_dtype)
    _check(c, _run(c), None)


@pytest.mark.parametrize("d", [64, 72])
def test_in_place_and_without_a_pool(device, d):
    c = _case(device, 4, 19, 6, 2, d, torch.bfloat16)
    q, k, v = c["q"].clone(), c["k"].clone(), c["v"].clone()
    _run(c, q_out=c["q"], k_out=c["k"], pool=False)
    _check(c, c["q"], c["k"], pool=False, q=q, k=k)
    assert torch.equal(v, c["v"])
    one = _case(device, 5, 19, 6, 2, d, torch.bfloat16)
    qk_norm.qk_norm_rope(one["q"], one["k"], None, one["w"][0], None, one["positions"].int(), one["table"], one["q"],
                         k_out=one["k"], eps=0.5)


@pytest.mark.parametrize("d", [64, 72])
def test_slots_and_positions_outside(device, d):
    """No slot: no pool row; no table row: NaN, and no K pool row."""
    c = _case(device, 6, 40, 4, 2, d, torch.bfloat16)
    c["slots"][[0, 7, 8]] = torch.tensor([-1, len(c["pool"][0]), -(2 ** 40)], device=device)
    c["positions"][[3, 7, 11]] = torch.tensor([-1, 500, 2 ** 40], device=device)
    k_out = torch.empty_like(c["k"])
    _check(c, _run(c, k_out=k_out), k_out)
    assert torch.isnan(k_out[3]).all()


@pytest.mark.parametrize("offset", [0, 4])
def test_strided_and_unaligned(device, offset):
    """Padded projections, pools of interleaved K and V, and rows that are not
    16-byte aligned."""
    n, hq, hk, d = 23, 4, 2, 64
    c = _case(device, 8, n, hq, hk, d, torch.float16)
    wide = torch.zeros((n, hq + 2 * hk, d + 16), dtype=torch.float16, device=device)
    wide[:, :, offset: offset + d] = c["qkv"]
    c["q"], c["k"], c["v"] = wide[:, :, offset: offset + d].split((hq, hk, hk), 1)
    both = torch.full((n + 5, hk, 2, d), 7.0, dtype=torch.float16, device=device)
    c["pool"] = [both[:, :, 0], both[:, :, 1]]
    out = torch.full((n, hq, d + 8), 7.0, dtype=torch.float16, device=device)
    _check(c, _run(c, q_out=out[:, :, :d], eps=1e-5), None, eps=1e-5)
    assert (out[:, :, d:] == 7).all()


def test_extreme_rows(device):
    """A row of zeros stays zero, large and tiny rows keep their norm, NaN and
    infinities stay in their rows."""
    c = _case(device, 9, 8, 2, 1, 64, torch.bfloat16)
    c["q"][0] = 0
    c["q"][1] *= 1e15
    c["q"][2] *= 1e-18  # mean(x^2) under eps
    c["q"][3, 0, 5] = float("nan")
    c["q"][4, 1, 9] = float("inf")
    out = f64(_run(c, eps=1e-6, pool=False, k_out=torch.empty_like(c["k"])))
    assert (out[0] == 0).all() and np.isnan(out[3, 0]).all() and np.isnan(out[4, 1, 9])
    assert np.isfinite(out[[0, 1, 2, 5, 6, 7]]).all() and np.isfinite(out[3, 1]).all() and np.isfinite(out[4, 0]).all()
    rows = f64(c["table"])[c["positions"].cpu().numpy()]
    want, size = drafts.qk_norm_rope(f64(c["q"])[:3], f64(c["w"][0]), 1e-6, rows[:3], 64, True)
    assert (np.abs(out[:3] - want) <= _tolerance(torch.bfloat16, 64, want, size)).all()


def test_no_tokens_and_int32_vectors(device):
    c = _case(device, 10, 12, 4, 2, 64, torch.bfloat16)
    c["positions"], c["slots"] = c["positions"].int(), c["slots"].int()
    _check(c, _run(c), None)
    empty = _case(device, 10, 0, 4, 2, 64, torch.bfloat16)
    _run(empty)
    assert (empty["pool"][0] == 7).all()


@pytest.mark.parametrize("n", [2047, 2048, 2053])
@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (128, torch.float16), (80, torch.float32)])
def test_around_the_split_of_a_token(device, n, d, dtype):
    """Token counts on both sides of the rule that gives a token to one wave."""
    print(f"qk norm {n} tokens of {d} {dtype}", flush=True)
    c = _case(device, n + d, n, 9, 4, d, dtype)
    q_out, k_out = torch.empty_like(c["q"]), torch.empty_like(c["k"])
    qk_norm.qk_norm_rope(c["q"], c["k"], c["v"], *c["w"], c["positions"], c["table"], q_out, k_out=k_out,
                         slot_map=c["slots"], k_buffer=c["pool"][0], v_buffer=c["pool"][1])
    _check(c, q_out, k_out)


@pytest.mark.parametrize("d", [64, 40])
def test_a_pool_without_slots(device, d):
    """Every token's slot is outside it: the call is the one without a pool."""
    gen = torch.Generator().manual_seed(d)
    q, k, v = (torch.randn(7, h, d, generator=gen).to(torch.bfloat16).to(device) for h in (4, 2, 2))
    table = torch.randn(9, d, generator=gen).to(device)
    positions, slots = torch.arange(7, device=device), torch.arange(7, device=device)
    pools = [torch.empty(0, 2, d, dtype=torch.bfloat16, device=device) for _ in range(2)]
    assert pools[0].data_ptr() == 0
    outs = [(torch.empty_like(q), torch.empty_like(k)) for _ in range(3)]
    qk_norm.qk_norm_rope(q, k, None, None, None, positions, table, outs[0][0], k_out=outs[0][1])
    pool = dict(slot_map=slots, k_buffer=pools[0], v_buffer=pools[1])
    qk_norm.qk_norm_rope(q, k, v, None, None, positions, table, outs[1][0], k_out=outs[1][1], **pool)
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    qk_norm.qk_norm_rope(q, k, v, None, None, positions, table, outs[2][0], **pool)
    assert torch.equal(outs[0][0], outs[2][0])


@pytest.mark.parametrize("hq,hk,d,n,vector", [(60, 2, 2, 1_100_001, False), (1, 1, 16, 67_200_003, True)])
def test_more_tokens_than_one_launch_has_threads_for(device, hq, hk, d, n, vector):
    """A wave per row (any widths) or per token: 2^26 of them have 2^32 threads.
    The tokens at both ends and around every 2^20th are those of small calls."""
    print(f"norms of {n} tokens, {hq} + {hk} heads of {d}", flush=True)
    gen = torch.Generator(device=device).manual_seed(n)
    q = torch.randn(n, hq, d, generator=gen, device=device, dtype=torch.bfloat16)
    k = q[:, -hk:]
    table = torch.randn(50, d, generator=gen, device=device)
    positions = torch.randint(0, 50, (n,), generator=gen, device=device, dtype=torch.int32)
    outs = [torch.full_like(q, 7), torch.full_like(q[:, :hk], 7)]
    qk_norm.qk_norm_rope(q, k, None, None, None, positions, table, outs[0], k_out=outs[1])
    at = torch.arange(0, n, 1 << 20, device=device)[:, None] + torch.arange(-4, 5, device=device)
    at = torch.cat((at.flatten(), torch.arange(n - 9, n, device=device)))
    at = at[(at >= 0) & (at < n)]
    want = [torch.empty_like(t[at]) for t in outs]
    qk_norm.qk_norm_rope(q[at], k[at], None, None, None, positions[at], table, want[0], k_out=want[1])
    for got, w in zip(outs, want):
        assert torch.equal(got[at], w)
        assert not (got == 7).all(-1).any()


def test_stretches_of_tokens_with_a_pool(device):
    """The same with slots and a pool that holds some of the tokens."""
    n, d, slots = 1_500_000, 2, 1000
    gen = torch.Generator(device=device).manual_seed(5)
    x = torch.randn(n, 50, d, generator=gen, device=device, dtype=torch.bfloat16)
    q, k, v = x.split((46, 2, 2), 1)
    table = torch.randn(50, d, generator=gen, device=device)
    positions = torch.randint(0, 50, (n,), generator=gen, device=device)
    taken = torch.arange(slots, device=device) * 1499 + 700
    slot_map = torch.full((n,), -1, dtype=torch.int64, device=device)
    slot_map[taken] = torch.randperm(slots, generator=gen, device=device)
    pools = [torch.zeros(slots, 2, d, dtype=torch.bfloat16, device=device) for _ in range(2)]
    out = torch.empty(n, 46, d, dtype=torch.bfloat16, device=device)
    qk_norm.qk_norm_rope(q, k, v, None, None, positions, table, out, slot_map=slot_map, k_buffer=pools[0],
                         v_buffer=pools[1])
    at = taken.clone()
    few, k_few = torch.empty(slots, 46, d, dtype=torch.bfloat16, device=device), torch.empty_like(pools[0])
    qk_norm.qk_norm_rope(q[at], k[at], None, None, None, positions[at], table, few, k_out=k_few)
    assert torch.equal(out[at], few)
    assert torch.equal(pools[0][slot_map[at]], k_few) and torch.equal(pools[1][slot_map[at]], v[at])
