"""A KV cache held in 8 bits, restated on the CPU: formats, scales, stores.

No counterpart in the reference, whose Reposition takes unquantized KV only
(``akv/system/sglang/kernels/ops/attention/context_reposition.py:149-152``): this
module is the extension's specification.  It is pinned by torch's own 8-bit
types (``tests/test_oracle_kv8.py``: every code's value, rounding of values at
and beside every tie) and by properties (the least power of two that holds a
block, rows stored one by one or together).  ``real`` is the type that rows are
computed in: float64 for the definition, float32 with every operation rounded
for what the kernels compute.
"""

import numpy as np

LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
DIGITS = {"e4m3": 3, "e5m2": 2}          # of a code's fraction
SMALLEST = {"e4m3": -6, "e5m2": -14}     # exponent of the smallest normal code
LEAST_SCALE = 2.0 ** -100


def rounded(x, form):
    """To the nearest value of the format, ties to even; infinities and NaN as
    the format has them."""
    x = np.asarray(x, dtype=np.float64)
    with np.errstate(invalid="ignore"):
        exponent = np.frexp(np.where(np.isfinite(x), x, 0.0))[1] - 1
        step = np.exp2(np.maximum(exponent, SMALLEST[form]).astype(np.float64) - DIGITS[form])
        out = np.round(x / step) * step
    assert not (np.abs(out[np.isfinite(x)]) > LARGEST[form]).any()
    out = np.where(np.isfinite(x), out, x)
    return np.where(np.isinf(out), np.nan, out) if form == "e4m3" else out


def fitting(top, form):
    """The smallest power of two s >= 2^-100 with top <= F s."""
    digits, exponent = np.frexp(np.asarray(top, dtype=np.float64) / LARGEST[form])
    s = np.ldexp(1.0, exponent - (digits == 0.5))
    return np.where(top > 0, np.maximum(s, LEAST_SCALE), LEAST_SCALE)


def grown(top, before, form):
    """A block's scale when values up to ``top`` join those that ``before`` scales."""
    out = np.empty(len(before))
    for i, (t, s) in enumerate(zip(np.asarray(top, dtype=np.float64), np.asarray(before, dtype=np.float64))):
        if not 0 < s < np.inf:
            out[i] = fitting(t, form)
        elif t <= np.float32(np.float32(LARGEST[form]) * np.float32(s)):
            out[i] = s
        elif s < LEAST_SCALE:
            out[i] = fitting(t, form)
        else:
            while t > np.float32(np.float32(LARGEST[form]) * np.float32(s)):
                s *= 2
            out[i] = s
    return out


def turned(x, cos, sin, rotary_dim, neox):
    """Rows ``[N, heads, D]`` with their pairs (a, b) -> (a cos - b sin, b cos + a
    sin); cos / sin ``[N, rotary_dim / 2]`` in x's type."""
    half = rotary_dim // 2
    one = np.arange(half) if neox else 2 * np.arange(half)
    two = one + half if neox else one + 1
    out, a, b = x.copy(), x[..., one], x[..., two]
    c, s = cos[:, None], sin[:, None]
    out[..., one], out[..., two] = a * c - b * s, b * c + a * s
    return out


def rows_at(x, positions, table, rotary_dim, neox, real):
    """K (or q) rows rotated by the table's rows; NaN for positions outside it."""
    x = np.asarray(x, dtype=real)
    if table is None:
        return x
    positions = np.asarray(positions, dtype=np.int64)
    known = (positions >= 0) & (positions < len(table))
    row = np.asarray(table, dtype=real)[np.where(known, positions, 0)]
    out = turned(x, row[:, : rotary_dim // 2], row[:, rotary_dim // 2:], rotary_dim, neox)
    out[~known] = np.nan
    return out


def runs(slots, block, total):
    """(first entry, entries) of the runs of a list: slots of one block, ascending by 1."""
    out, t = [], 0
    while t < len(slots):
        n = 1
        if 0 <= slots[t] < total:
            while t + n < len(slots) and slots[t + n] == slots[t] + n and slots[t + n] % block and slots[t + n] < total:
                n += 1
            out.append((t, n))
        t += n
    return out


def store(codes, scales, rows, slots, block, form, live=None, units=1.0):
    """Rows ``[N, heads, D]`` in units ``[N, heads, 1]`` into ``codes`` ``[slots,
    heads, D]`` (the codes' values) and ``scales`` ``[blocks, heads]``, in place.
    ``live``: rows that are written (a run without any leaves its block's scale as it is)."""
    rows, real = np.asarray(rows), np.asarray(rows).dtype.type
    units = np.broadcast_to(np.asarray(units, dtype=real), (*rows.shape[:2], 1))
    begun = set()
    for t, n in runs(slots, block, len(codes)):
        at, first = slots[t] // block, slots[t] % block
        if at in begun:
            raise ValueError("a block's rows follow one another in a call")
        begun.add(at)
        here = np.arange(t, t + n)
        if live is not None:
            here = here[np.asarray(live)[t: t + n]]
            if not len(here):
                continue
        x, unit = rows[here], units[here]
        with np.errstate(over="ignore", invalid="ignore"):
            y = x * unit
        top = np.where(np.isfinite(y), np.abs(y), 0).max((0, 2), initial=0)
        before = scales[at].copy()
        after = grown(top, before, form) if first else fitting(top, form)
        scales[at] = after
        if first:
            lower = slice(at * block, at * block + first)
            with np.errstate(over="ignore", invalid="ignore"):
                ratio = np.where((before > 0) & (before < np.inf), before / after, 0.0).astype(real)
            changed = after != before
            codes[lower] = np.where(changed[None, :, None], rounded(codes[lower] * ratio[None, :, None], form), codes[lower])
        with np.errstate(over="ignore", invalid="ignore"):
            lift = np.where(after < 2.0 ** -126, 2.0 ** 24, 1.0).astype(real)  # (1 / s has no fp32 value)
            by = unit * (real(1) / (after.astype(real) * lift))[None, :, None]
            by = np.where((by == np.inf) & (unit < np.inf), np.finfo(real).max, by)  # (a row of zeros)
            codes[np.asarray(slots)[here]] = rounded(x * lift[None, :, None] * by, form)


def moved_rows(codes, scales, src, pairs, table, block, rotary_dim, neox, real, rotates):
    """The values of slots ``src``, K's turned from pairs[:, 0] to pairs[:, 1], and
    the units they are in, their scales."""
    x, unit = codes[src].astype(real), scales[np.asarray(src) // block].astype(real)[..., None]
    if not rotates:
        return x, unit
    half, pairs = rotary_dim // 2, np.asarray(pairs, dtype=np.int64)
    known = ((pairs >= 0) & (pairs < len(table))).all(1)
    old, new = (np.asarray(table, dtype=real)[np.where(known, pairs[:, i], 0)] for i in (0, 1))
    co, so, cn, sn = old[:, :half], old[:, half:], new[:, :half], new[:, half:]
    norm = co * co + so * so
    out = turned(x, (cn * co + sn * so) / norm, (sn * co - cn * so) / norm, rotary_dim, neox)
    out[~known] = np.nan
    same = pairs[:, 0] == pairs[:, 1]
    out[same] = x[same]
    return out, unit
