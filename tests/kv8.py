"""Seeded 8-bit caches for the tests, and what the oracle makes of them."""

import numpy as np
import torch

from tests.drafts import HALF, Cache, f64

FORMATS = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}


def codes_of(gen, shape, form, spread=0.2):
    """Codes of normal values: ``spread`` of the largest one."""
    F = LARGEST[form]
    return (F * spread * torch.randn(shape, generator=gen)).clamp(-F, F).to(FORMATS[form])


def values(codes):
    """float64 values of 8-bit codes."""
    return codes.detach().cpu().float().double().numpy()


class Cache8(Cache):
    """``tests.drafts.Cache`` whose K/V are held in 8 bits, at scales that are no
    powers of two; ``k`` / ``v`` are their values."""

    def __init__(self, device, seed, old, new, *, form="e4m3", block=1, **shape):
        super().__init__(device, seed, old, new, **shape)
        gen = torch.Generator().manual_seed(seed + 1)
        n, hk, d = self.k.shape
        self.form, self.block, self.parts = form, block, []
        for name in ("k", "v"):
            codes = codes_of(gen, (n, hk, d), form)
            scales = (0.5 + torch.rand((-(-n // block), hk), generator=gen)) * 5 / LARGEST[form]
            self.parts.append([codes.to(device), scales.to(device)])
        self.refresh()

    def refresh(self):
        """k and v from the codes and scales as they are."""
        at = torch.arange(len(self.parts[0][0]), device=self.device) // self.block
        self.k, self.v = (codes.float().double() * scales.double()[at][..., None] for codes, scales in self.parts)

    def visible(self, seen, starts=None, first=0):
        out = super().visible(seen, starts)
        for (_, _, keys), o in zip(out, self.old):
            keys[:, : min(first, o)] = True
        return out


def kv8_tolerance(dtype, out_dtype, keys, want, size, spread):
    """How far a row may be off.  A weight's exponent carries the fp32 errors of
    a product of up to 128 terms, of its two scalings and exp2: 2^-24 (128 + 5)
    spread + 2^-22 relative, in the sum as in the products; errors d_j move o by
    at most max|d_j| (sum w|v| + |o|).  A weight times its V scale is rounded to
    bf16, off by 2^-8 (fp16 queries: to two bf16 values, 2^-16), in the products
    alone: 2^-8 sum w|v|.  fp32 sums over the keys add keys 2^-23 sum w|v|."""
    delta = 133 * 2.0 ** -24 * spread[..., None] + 2.0 ** -22
    weight = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -16
    tol = delta * (size + np.abs(want)) + (weight + 2.0 ** -22 + keys * 2.0 ** -23) * size + HALF[out_dtype] * np.abs(want)
    return tol * 1.01 + (2.0 ** -25 if out_dtype == torch.float16 else 0) + 1e-30


def layer(device, seed, slots, heads, d, form, block):
    """[codes, scales] of K and of V, powers of two as the writers leave them."""
    gen = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        scales = torch.exp2(torch.randint(-9, -5, (-(-slots // block), heads), generator=gen).float())
        out.append([codes_of(gen, (slots, heads, d), form).to(device), scales.to(device)])
    return out


def same(got, want):
    """Codes and scales against the oracle's values, NaN for NaN."""
    (codes, scales), (w_codes, w_scales) = got, want
    np.testing.assert_array_equal(f64(scales), w_scales)
    np.testing.assert_array_equal(values(codes), w_codes)


def paged_slots(rng, lengths, page, extra=3):
    """Random pages of requests whose keys' numbers [from, to) are asked for: the
    slots of each, and the slots there are."""
    pages = [-(-to // page) for _, to in lengths]
    ids = rng.permutation(sum(pages) + extra)
    out, at = [], 0
    for (lo, to), n in zip(lengths, pages):
        rank = np.arange(lo, to)
        out.append(ids[at: at + n][rank // page] * page + rank % page)
        at += n
    return out, (sum(pages) + extra) * page
