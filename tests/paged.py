"""A paged K/V cache on both sides: numpy arrays with the definition of the operators in 64 bits, device buffers with the calls."""
import importlib

import numpy as np

NOWHERE = 0xffffffff


class Paged:
    """Blocks in a random order, every sequence with its own; slots that no sequence holds are filled with `garbage`."""

    def __init__(self, rng, f16, n_layer, n_head_kv, head_dim, kv_block, lens, room=0, weights=False, garbage=np.nan, spare=2, extra_blocks=0):
        self.rng, self.f16, self.n_layer, self.hkv, self.d, self.kvb = rng, f16, n_layer, n_head_kv, head_dim, kv_block
        self.lens = np.array(lens, np.uint32)
        pages = [-(-(int(n) + room) // kv_block) for n in lens]
        self.stride = max(max(pages), 1) + 1
        self.n_blocks = sum(pages) + spare + extra_blocks
        ids = rng.permutation(self.n_blocks)
        self.tables = np.full((len(lens), self.stride), NOWHERE, np.uint32)
        at = 0
        for b, n in enumerate(pages):
            self.tables[b, :n] = ids[at:at + n]
            at += n
        self.free = ids[at:]
        shape = (self.n_blocks, n_layer, n_head_kv, kv_block, head_dim)
        dt = np.float16 if f16 else np.float32
        self.k, self.v = (np.full(shape, garbage, dt) for _ in range(2))
        self.w = np.full(shape[:-1], garbage, np.float32) if weights else None
        for b, n in enumerate(lens):
            for t in range(int(n)):
                self.k[self.at(b, t)] = rng.normal(0, 1, (n_layer, n_head_kv, head_dim)).astype(dt)
                self.v[self.at(b, t)] = rng.normal(0, 1, (n_layer, n_head_kv, head_dim)).astype(dt)
                if weights:
                    self.w[self.at(b, t)] = rng.exponential(1, (n_layer, n_head_kv)).astype(np.float32)

    def at(self, b, t):
        return self.tables[b, t // self.kvb], slice(None), slice(None), t % self.kvb

    def there(self, b, t):
        return t // self.kvb < self.stride and self.tables[b, t // self.kvb] < self.n_blocks

    def up(self, starts=None, max_new=1, max_len=None, n_tokens=None):
        pkg, hip = importlib.import_module("llama-rust_amd"), importlib.import_module("llama-rust_amd.hiprt")
        self.hip = hip
        buf = hip.DeviceBuffer.from_numpy
        self.dk, self.dv, self.dt, self.dl = buf(self.k), buf(self.v), buf(self.tables), buf(self.lens)
        self.dw = buf(self.w) if self.w is not None else None
        self.ds = buf(np.array(starts, np.uint32)) if starts is not None else None
        self.cache = pkg.KvCache(pkg.F16 if self.f16 else pkg.F32, self.n_layer, self.hkv, self.d, self.kvb, self.n_blocks, self.dk.ptr, self.dv.ptr,
                                 self.dw.ptr if self.dw else 0)
        n = n_tokens if n_tokens is not None else int(starts[-1]) if starts is not None else len(self.lens)
        most = max_len if max_len is not None else int(min(self.lens.max(), self.stride * self.kvb)) if len(self.lens) else 0
        self.seqs = pkg.KvSeqs(len(self.lens), self.dt.ptr, self.stride, self.dl.ptr, most, self.ds.ptr if self.ds else 0, n, max_new)
        return self

    def down(self):
        dt = np.float16 if self.f16 else np.float32
        k, v = (x.to_numpy(dt).reshape(self.k.shape) for x in (self.dk, self.dv))
        return k, v, self.dw.to_numpy(np.float32).reshape(self.w.shape) if self.dw else None

    # ---- the definition
    def attend(self, layer, q, scale, starts=None, window=0, sinks=0):
        """(out, tolerance, [per sequence and kv head: summed probabilities, tolerance]) in 64 bits; q [tokens, heads, d]."""
        starts = np.arange(len(self.lens) + 1) if starts is None else np.asarray(starts)
        out, tol = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
        heads, group = q.shape[1], q.shape[1] // self.hkv
        sums = {}
        for b in range(len(self.lens)):
            n, length = int(starts[b + 1] - starts[b]), int(self.lens[b])
            pos = [t for t in range(length) if self.there(b, t)]
            for h in range(self.hkv):
                k = np.array([self.k[self.tables[b, t // self.kvb], layer, h, t % self.kvb] for t in pos], np.float64).reshape(len(pos), self.d)
                v = np.array([self.v[self.tables[b, t // self.kvb], layer, h, t % self.kvb] for t in pos], np.float64).reshape(len(pos), self.d)
                ws, wt = np.zeros(len(pos)), np.zeros(len(pos))
                for i in range(n):
                    p, t = length - n + i, np.array(pos, np.int64)
                    sees = (t <= p) & ((t > p - window) | (t < sinks) if window else True)
                    for g in range(group):
                        row, head = int(starts[b]) + i, h * group + g
                        qr = q[row, head].astype(np.float64)
                        if p < 0 or not sees.any():
                            out[row, head], tol[row, head] = 0, 0
                            continue
                        with np.errstate(all="ignore"):
                            s = (k[sees] @ qr) * scale
                            e = np.exp(s - s.max()) if s.max() != -np.inf else np.zeros(len(s))
                            pr = e / e.sum() if e.sum() != 0 else e
                            out[row, head] = pr @ v[sees]
                            # f32 sums of d products, of a probability's and an output's terms; q and the probabilities in two f16 parts
                            # (2^-22 each); one part in 2^23 for every rounding of a sum, twice the half step it is
                            size = (np.abs(k[sees]) @ np.abs(qr)).max() * abs(scale)
                            rel = (2 * (self.d + 24) * size + int(sees.sum()) + 80) * 2.0 ** -23
                            tol[row, head] = rel * (pr @ np.abs(v[sees])) + 1e-37
                            ws[sees] += pr
                            wt[sees] += (rel + n * group * 2.0 ** -23) * pr + 2.0 ** -120
                if n:
                    sums[b, h] = (pos, ws, wt)
        return out, tol, sums

    def weigh(self, layer, sums, decay):
        """(weights, tolerance) of the whole plane after a call."""
        w, tol = self.w.astype(np.float64), np.zeros(self.w.shape)
        for (b, h), (pos, ws, wt) in sums.items():
            for t, x, y in zip(pos, ws, wt):
                i = self.tables[b, t // self.kvb], layer, h, t % self.kvb
                old = 0.0 if decay == 0 else float(np.float32(decay)) * w[i]
                w[i], tol[i] = old + x, y + 2 * 2.0 ** -24 * abs(old + x)
        return w, tol

    def evict(self, layers, keep, first, recent, dst=None):
        """New lengths; K, V and w as they are afterwards."""
        k, v, w = self.k.copy(), self.v.copy(), self.w.copy()
        new = np.minimum(self.lens, keep).astype(np.uint32)
        tables = self.tables if dst is None else dst
        for b, length in enumerate(self.lens.astype(int)):
            if dst is None and length <= keep:
                continue
            for la in layers:
                for h in range(self.hkv):
                    stays = list(range(length))
                    if length > keep:
                        mid = list(range(first, length - recent))

                        def order(t):
                            if not self.there(b, t):
                                return (2, 0.0, t)
                            x = self.w[self.tables[b, t // self.kvb], la, h, t % self.kvb]
                            return (0, 0.0, t) if np.isnan(x) else (1, -float(x), t)
                        mid = sorted(mid, key=order)[:keep - first - recent]
                        stays = sorted(list(range(first)) + mid + list(range(length - recent, length)))
                    for i, t in enumerate(stays):
                        if not self.there(b, t) or tables[b, i // self.kvb] >= self.n_blocks:
                            continue
                        to, fr = (tables[b, i // self.kvb], la, h, i % self.kvb), (self.tables[b, t // self.kvb], la, h, t % self.kvb)
                        k[to], v[to], w[to] = self.k[fr], self.v[fr], self.w[fr]
        return new, k, v, w


def same_bits(a, b):
    """Equal, NaN in the same places."""
    return np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(a[~np.isnan(a)], b[~np.isnan(b)])
