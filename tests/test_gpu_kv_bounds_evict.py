"""Bounds after an eviction: what moved makes those that were there wrong; formed anew over every position, the choice by them is the definition's."""
import importlib

import numpy as np
import pytest

from paged import same_bits
from test_gpu_attn_select import KINDS, bounds_of, cache_of, definition

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu(pkg):
    g = pkg.HipGemv(0)
    yield g
    g.close()


@pytest.fixture(scope="module")
def hip():
    return importlib.import_module("llama-rust_amd.hiprt")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("d,block", [(64, 16), (96, 7)])
def test_bounds_are_formed_anew(gpu, hip, pkg, kind, in_place, d, block):
    """An eviction to 90 positions, then one call of every position as a new token, its starts a running sum of the new lengths."""
    rng = np.random.default_rng(d)
    layers, hkv, keep = 2, 2, 90
    c = cache_of(kind, rng, layers, hkv, d, block, [200, 90, 0, 131], weights=True, extra_blocks=4 * (keep // block + 1)).up()
    n = len(c.lens)
    before = bounds_of(c, kind)
    db = hip.DeviceBuffer.from_numpy(before)
    pages = -(-keep // block)
    dst = None if in_place else c.free[:n * pages].reshape(n, pages).astype(np.uint32)
    new, k, v, w = c.evict(range(layers), keep, 2, 9, dst)
    dd = None if in_place else hip.DeviceBuffer.from_numpy(dst)
    gpu.kv_evict_device(c.cache, c.seqs, 0, layers, keep, 2, 9, dd.ptr if dd else 0, pages, c.dl.ptr)
    if not in_place:
        c.tables, c.stride = dst, pages
        c.dt = dd
    c.lens, c.k, c.v, c.w = new, k, v, w
    want = bounds_of(c, kind)
    held = [(c.tables[b, j], slice(None), slice(None)) for b in range(n) for j in range(-(-int(new[b]) // block))]
    assert any(not same_bits(want[i], before[i]) for i in held)  # those that were there are wrong
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
    ds = hip.DeviceBuffer.from_numpy(starts)
    every = pkg.KvSeqs(n, c.dt.ptr, c.stride, c.dl.ptr, keep, ds.ptr, n * keep, keep)
    for layer in range(layers):
        gpu.kv_bounds_device(c.cache, every, layer, db.ptr)
    hip.device_synchronize()
    assert np.array_equal(c.dl.to_numpy(np.uint32), new)
    got = db.to_numpy(want.dtype).reshape(want.shape)
    assert all(same_bits(got[i], want[i]) for i in held)
    q = rng.normal(0, 1, (n, 6, d)).astype(np.float32)
    scale, most = np.float32(d ** -0.5), 4
    wc, ws, tol = definition(c, kind, want, 1, q, float(scale), list(range(n + 1)), most, 1, 1)
    dq, do, dc = hip.DeviceBuffer.from_numpy(q), hip.DeviceBuffer(q.nbytes), hip.DeviceBuffer(n * hkv * most * 4)
    seqs = pkg.KvSeqs(n, c.dt.ptr, c.stride, c.dl.ptr, keep)
    gpu.attn_select_device(c.cache, seqs, 1, 6, db.ptr, most, 1, 1, dq.ptr, do.ptr, scale, chosen_ptr=dc.ptr)
    hip.device_synchronize()
    assert np.array_equal(dc.to_numpy(np.uint32).reshape(wc.shape), wc)
    assert np.all(np.abs(do.to_numpy(np.float32).reshape(q.shape) - ws) <= tol + 1e-7 * np.abs(ws))
