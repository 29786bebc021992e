"""Caches of 4-bit numbers on top of paged_ref.py: the quantiser in 64 bits, the pages' layout,
and a Setup whose keys and values are what such a cache holds.  Test infrastructure."""
from __future__ import annotations

import numpy as np

from paged_ref import F16, Device, Setup

Q4_0 = 2
ORDER = [0, 2, 4, 6, 1, 3, 5, 7]  # channels of a word from its lowest four bits up


def quantise(x):
    """n (0..15) [..., hd] and d [..., hd / 32] of numbers x [..., hd], block by block, in 64 bits."""
    x = np.asarray(x, np.float64)
    n, d = np.empty(x.shape, np.uint8), np.empty(x.shape[:-1] + (x.shape[-1] // 32,))
    for b in range(d.shape[-1]):
        y = x[..., 32 * b:32 * b + 32]
        bad = ~np.isfinite(y).all(-1)
        y = np.where(bad[..., None], 0.0, y)
        low, high = y.min(-1), y.max(-1)
        size = np.where(-low >= high, -low, high) / 8.0
        with np.errstate(divide="ignore"):
            step = np.exp2(np.maximum(np.frexp(size)[1] - 8.0, -24.0))
        scale = np.minimum(np.rint(size / step) * step, 8160.0) * np.where(-low >= high, 1.0, -1.0)
        with np.errstate(divide="ignore", invalid="ignore"):
            q = np.clip(np.floor(y / scale[..., None] + 8.5), 0, 15)
        n[..., 32 * b:32 * b + 32] = np.where(scale[..., None] == 0, 8, q)
        d[..., b] = np.where(bad, np.nan, scale)
    return n, d


def values(n, d):
    """What numbers n and scales d (fp16) stand for: the product rounded to fp16."""
    with np.errstate(invalid="ignore", over="ignore"):
        return (np.repeat(d.astype(np.float64), 32, -1) * (n.astype(np.float64) - 8)).astype(np.float16)


def pack(n, d):
    """Pages [pages, kv_heads, bytes] from n [pages, kv_heads, page, hd] and d [pages, kv_heads, page, hd / 32]."""
    pages, heads, page, hd = n.shape
    bits = n.reshape(pages, heads, page, hd // 8, 8)[..., ORDER].reshape(pages, heads, page, hd // 2, 2)
    numbers = (bits[..., 0] | bits[..., 1] << 4).reshape(pages, heads, -1)
    with np.errstate(invalid="ignore"):
        scales = np.ascontiguousarray(d.astype(np.float16).swapaxes(-1, -2)).view(np.uint8).reshape(pages, heads, -1)
    return np.concatenate((numbers, scales), -1)


def unpack(b, page, hd):
    """n and d (fp16) of pages `b`."""
    split = page * hd // 2
    x = b[..., :split].reshape(*b.shape[:2], page, hd // 2)
    n = np.stack((x & 15, x >> 4), -1).reshape(*b.shape[:2], page, hd // 8, 8)[..., np.argsort(ORDER)]
    d = np.ascontiguousarray(b[..., split:]).view(np.float16).reshape(*b.shape[:2], hd // 32, page)
    return n.reshape(*b.shape[:2], page, hd), d.swapaxes(-1, -2)


class SetupQ4(Setup):
    """A Setup whose cache holds 4-bit numbers: k and v are their values (fp16), kn, kd, vn, vd what
    is stored; where no sequence owns a slot the scales are NaN and infinite."""

    def __init__(self, heads, kv_heads, hd, page, q, kv, **kw):
        super().__init__(F16, heads, kv_heads, hd, page, q, kv, **kw)
        for name in "kv":
            x = getattr(self, name)
            junk = ~np.isfinite(x.astype(np.float32)).all(-1)
            n, d = quantise(np.where(junk[..., None], 0, x))
            d[junk] = self.rng.choice([np.nan, np.inf, -np.inf], d[junk].shape)
            n[junk] = self.rng.integers(0, 16, n[junk].shape)
            self.put(name, n, d)

    def put(self, name, n, d):
        setattr(self, name + "n", n)
        setattr(self, name + "d", d.astype(np.float16))
        setattr(self, name, values(n, d.astype(np.float16)))
        if name == "k":
            lo, hi = self.bounds[:, :, 0], self.bounds[:, :, 1]
            for s in range(self.seqs):
                for i in range(-(-self.kv[s] // self.page)):
                    p, m = self.table[s, i], min(self.page, self.kv[s] - i * self.page)
                    lo[p], hi[p] = self.k[p, :, :m].min(1), self.k[p, :, :m].max(1)

    def scale_values(self, name, f):
        """All scales times f."""
        self.put(name, getattr(self, name + "n"), getattr(self, name + "d").astype(np.float64) * f)


class DeviceQ4(Device):
    def __init__(self, lib, torch, s):
        super().__init__(lib, torch, s)
        self.cache.type = Q4_0
        self.upload()

    def upload(self):
        s = self.s
        self.k, self.v = (self.torch.from_numpy(pack(getattr(s, x + "n"), getattr(s, x + "d"))).cuda() for x in "kv")
        self.cache.k, self.cache.v = self.k.data_ptr(), self.v.data_ptr()

    def read(self):
        s = self.s
        self.k_out, self.v_out = (self.torch.full((s.tokens, s.kv_heads, s.hd), 777.0, device="cuda") for _ in "kv")
        self.lib.kv_read_dev(self.cache, self.batch, self.k_out.data_ptr(), self.v_out.data_ptr(), self.stream())
        return self.k_out, self.v_out

    def held(self):
        """The Setup's numbers, scales and values as the device's pages hold them now."""
        for name in "kv":
            n, d = unpack(getattr(self, name).cpu().numpy(), self.s.page, self.s.hd)
            setattr(self.s, name + "n", n)
            setattr(self.s, name + "d", d)
            setattr(self.s, name, values(n, d))
        return self.s
