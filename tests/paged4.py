"""A paged K/V cache held in 4 bits on both sides: the packing in numpy, and Paged over the values that the packed rows stand for (each
of them an f16, so that the definition in 64 bits is that of an f16 cache)."""
import importlib

import numpy as np

from paged import Paged

SHIFT = np.array([[4 * i, 16 + 4 * i] for i in range(4)], np.uint32)


def scale_of(blocks):
    """f16 scales of f32 numbers [..., 32]: -1/8 of the first one of the largest size, to eight significant bits."""
    finite = np.isfinite(blocks).all(-1)
    safe = np.where(finite[..., None], blocks, 0).astype(np.float32)
    at = np.abs(safe).argmax(-1)[..., None]
    d = np.clip(np.take_along_axis(safe, at, -1)[..., 0] * np.float32(-0.125), np.float32(-8160), np.float32(8160))
    u = d.view(np.uint32).astype(np.uint64)
    d = ((u + 0x7fff + ((u >> 16) & 1)) & 0xffff0000).astype(np.uint32).view(np.float32)
    return np.where(finite, d, np.nan).astype(np.float16)


def pack(x):
    """codes [..., d / 8] words and scales [..., d / 32] of f32 rows [..., d]."""
    b = np.ascontiguousarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    s = scale_of(b)
    d = s.astype(np.float64)[..., None]
    with np.errstate(all="ignore"):
        c = np.where((d != 0) & np.isfinite(d), np.rint(b.astype(np.float64) / np.where(d != 0, d, 1)), 0)
    c = np.clip(np.where(np.isfinite(c), c, 0) + 8, 0, 15).astype(np.uint32).reshape(*b.shape[:-1], 4, 4, 2)
    return (c << SHIFT).sum((-1, -2), dtype=np.uint32).reshape(*x.shape[:-1], -1), s


def unpack(words, scales):
    """The values as f16, which they are exactly."""
    c = ((words[..., None, None] >> SHIFT) & 15).astype(np.float64).reshape(*scales.shape, 32) - 8
    with np.errstate(all="ignore"):
        v = (c * scales.astype(np.float64)[..., None]).reshape(*scales.shape[:-1], -1)
        h = v.astype(np.float16)
    assert np.array_equal(h.astype(np.float64)[~np.isnan(v)], v[~np.isnan(v)])
    return h


def to_buffer(values_or_rows):
    """K or V [blocks, layers, heads, places, d] (or anything to be packed to them) as the header lays it out."""
    words, scales = pack(values_or_rows.astype(np.float32))
    return np.concatenate([words.reshape(-1).view(np.uint8), np.ascontiguousarray(np.swapaxes(scales, -1, -2)).reshape(-1).view(np.uint8)])


def split_buffer(raw, shape):
    """(words, scales) [..., d / 8], [..., d / 32] of a buffer."""
    blocks, layers, heads, places, d = shape
    n = blocks * layers * heads * places * d // 2
    words = raw[:n].copy().view(np.uint32).reshape(*shape[:-1], d // 8)
    scales = raw[n:].copy().view(np.float16).reshape(blocks, layers, heads, d // 32, places)
    return words, np.ascontiguousarray(np.swapaxes(scales, -1, -2))


class Paged4(Paged):
    """Paged of f16 values that 4-bit rows stand for, on the device as those rows."""

    def __init__(self, rng, n_layer, n_head_kv, head_dim, kv_block, lens, **kw):
        super().__init__(rng, True, n_layer, n_head_kv, head_dim, kv_block, lens, **kw)
        self.settle()

    def settle(self):
        """K and V as what their packed rows stand for.  Packed again they are the same rows, whose largest element is -8 d, unless d is so
        small that an f16 has fewer than eight bits for it."""
        self.k, self.v = (unpack(*pack(x.astype(np.float32))) for x in (self.k, self.v))

    def up(self, *args, **kw):
        pkg = importlib.import_module("llama-rust_amd")
        super().up(*args, **kw)
        self.dk, self.dv = (self.hip.DeviceBuffer.from_numpy(to_buffer(x)) for x in (self.k, self.v))
        self.settle()  # what was packed just now
        self.cache = pkg.KvCache(pkg.Q4_0, self.n_layer, self.hkv, self.d, self.kvb, self.n_blocks, self.dk.ptr, self.dv.ptr, self.dw.ptr if self.dw else 0)
        assert self.dk.nbytes == pkg.q4_0_bytes(self.n_layer, self.hkv, self.d, self.kvb, self.n_blocks)
        return self

    def packed(self):
        """(words, scales) of K and of V as the device has them."""
        return [split_buffer(x.to_numpy(np.uint8), self.k.shape) for x in (self.dk, self.dv)]

    def down(self):
        (kw, ks), (vw, vs) = self.packed()
        return unpack(kw, ks), unpack(vw, vs), self.dw.to_numpy(np.float32).reshape(self.w.shape) if self.dw else None
