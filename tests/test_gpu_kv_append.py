"""Rows turned by their positions on the way into the paged cache (lnh_kv_append_device) and the angles' table on the GPU: a turned number is
that of 64 bits, rounded to f32 once, so that every bit is known."""
import importlib

import numpy as np
import pytest

from paged import NOWHERE, Paged, same_bits
from paged4 import Paged4, pack, unpack

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu(pkg):
    g = pkg.HipGemv(0)
    yield g
    g.close()


@pytest.fixture(scope="module")
def hip():
    return importlib.import_module("llama-rust_amd.hiprt")


def turned(x, angles, n_rot, halves):
    """Rows x [rows, heads, d] by angles [rows, n_rot / 2, 2]."""
    y = x.astype(np.float64)
    h = n_rot // 2
    a, b = (slice(0, h), slice(h, n_rot)) if halves else (slice(0, n_rot, 2), slice(1, n_rot, 2))
    c, s = (angles[:, None, :, i].astype(np.float64) for i in (0, 1))
    first, second = y[..., a].copy(), y[..., b].copy()
    y[..., a], y[..., b] = first * c - second * s, first * s + second * c
    return y.astype(np.float32)


def cache_of(kind, rng, layers, hkv, d, block, lens, **kw):
    return Paged4(rng, layers, hkv, d, block, lens, **kw) if kind == "q4_0" else Paged(rng, kind == "f16", layers, hkv, d, block, lens, **kw)


def held(kind, rows):
    """What the cache makes of f32 rows."""
    if kind == "q4_0":
        return unpack(*pack(rows))
    with np.errstate(over="ignore"):
        return rows.astype(np.float16) if kind == "f16" else rows


CASES = [(32, 8, 128, 128, 16), (1, 1, 32, 32, 7), (14, 2, 64, 20, 16), (6, 2, 96, 44, 20), (3, 1, 256, 254, 1), (0, 3, 64, 64, 32), (5, 4, 160, 2, 16), (40, 1, 64, 0, 16)]


@pytest.mark.parametrize("kind", ["f32", "f16", "q4_0"])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("heads,hkv,d,n_rot,block", CASES)
@pytest.mark.parametrize("in_place", [False, True])
def test_rows_are_turned(gpu, hip, pkg, kind, halves, heads, hkv, d, n_rot, block, in_place):
    """Layouts, parts of a head, pairs of either kind; rows apart, rows of nobody, a block that is not there, positions of their own and beyond the
    table, weights of new positions."""
    rng = np.random.default_rng(d + n_rot)
    starts, lens = [0, 9, 9, 12, 50], [30, 4, 2, 61]
    c = cache_of(kind, rng, 2, hkv, d, block, lens, weights=True)
    c.tables[3, 30 // block] = NOWHERE
    c.up(starts, max_new=38)
    before = c.down()
    rows, pairs, n_pos = 52, max(n_rot // 2, 1), 40
    qs, os, ks, vs = heads * d + 8, heads * d + (8 if in_place else 12), hkv * d + 4, hkv * d
    q, k, v = (rng.normal(0, 1, (rows, n)).astype(np.float32) for n in (qs, ks, vs))
    angles = rng.normal(0, 1, (n_pos, pairs + 3, 2)).astype(np.float32)
    positions = rng.integers(0, n_pos + 5, rows).astype(np.uint32)
    given = halves or in_place  # positions of their own or the places
    dq, dk, dv, da, dp = (hip.DeviceBuffer.from_numpy(x) for x in (q, k, v, angles, positions))
    out = q.copy() if in_place else np.full((rows, os), 4.5, np.float32)
    do = dq if in_place else hip.DeviceBuffer.from_numpy(out)
    rope = pkg.Rope(da.ptr, pairs + 3, n_pos, n_rot, halves=halves, positions_ptr=dp.ptr if given else 0)
    gpu.kv_append_device(c.cache, c.seqs, 1, rope, heads, dq.ptr if heads else 0, do.ptr if heads else 0, dk.ptr, dv.ptr, q_stride=qs, q_out_stride=os,
                         k_stride=ks, v_stride=vs)
    hip.device_synchronize()
    got_q = do.to_numpy(np.float32).reshape(rows, os)
    want_q, (want_k, want_v, want_w) = out.copy(), before
    for b in range(4):
        n = starts[b + 1] - starts[b]
        for i in range(n):
            row, t = starts[b] + i, lens[b] - n + i
            if t < 0:
                continue
            at = angles[None, min(int(positions[row]) if given else t, n_pos - 1), :n_rot // 2]
            want_q[row, :heads * d] = turned(q[row, :heads * d].reshape(1, heads, d), at, n_rot, halves).ravel()
            if not c.there(b, t):
                continue
            to = (c.tables[b, t // block], 1, slice(None), t % block)
            want_k[to] = held(kind, turned(k[row, :hkv * d].reshape(1, hkv, d), at, n_rot, halves)[0])
            want_v[to] = held(kind, v[row].reshape(hkv, d))
            want_w[to] = 0
    assert np.array_equal(got_q, want_q)
    assert all(same_bits(x, y) for x, y in zip(c.down(), (want_k, want_v, want_w)))


@pytest.mark.parametrize("n_rot,base,scale,n,divided", [(128, 500000.0, 1.0, 3, False), (64, 10000.0, 0.25, 70001, True), (2, 10.0, 1.0, 1, False), (250, 1.0, 1e3, 900, True)])
def test_angles(gpu, hip, n_rot, base, scale, n, divided):
    """Against 80 bits; pieces behind a position's pairs stay as they were."""
    rng = np.random.default_rng(n)
    pairs = n_rot // 2
    divisors = rng.uniform(1, 8, pairs).astype(np.float32)
    to, dd = hip.DeviceBuffer.from_numpy(np.full((n, pairs + 1, 2), 9, np.float32)), hip.DeviceBuffer.from_numpy(divisors)
    gpu.rope_table_device(n_rot, base, n, to.ptr, angle_stride=pairs + 1, scale=scale, divisors_ptr=dd.ptr if divided else 0)
    hip.device_synchronize()
    got = to.to_numpy(np.float32).reshape(n, pairs + 1, 2)
    assert np.all(got[:, pairs] == 9)
    i = np.arange(pairs, dtype=np.longdouble)
    angle = np.arange(n, dtype=np.longdouble)[:, None] * np.longdouble(scale) * np.longdouble(base) ** (-i / pairs)
    if divided:
        angle = angle / divisors.astype(np.longdouble)
    # half a step of an f32 below one, and of the angle what its factors are off by: an exponent of up to 20 in 53 bits, three roundings more
    tol = 2.0 ** -25 + angle * 2.0 ** -47
    for j, f in enumerate((np.cos, np.sin)):
        assert np.all(np.abs(got[:, :pairs, j] - f(angle)) <= tol)


@pytest.mark.parametrize("kind", ["f32", "q4_0"])
def test_a_prompt_then_tokens_one_by_one(gpu, hip, pkg, kind):
    """Angles made, rows appended and attended to as a session does: the prompt's rows once in one call, once token by token; the cache is the same,
    bit for bit, and the outputs are those of the definition."""
    rng = np.random.default_rng(5)
    d, heads, hkv, n = 64, 6, 2, 50
    q, k, v = (rng.normal(0, 1, (n, m, d)).astype(np.float32) for m in (heads, hkv, hkv))
    da = hip.DeviceBuffer(64 * d // 2 * 8)
    gpu.rope_table_device(d, 10000.0, 64, da.ptr)
    rope = pkg.Rope(da.ptr, d // 2, 64, d)
    angles = da.to_numpy(np.float32).reshape(64, d // 2, 2)[:n]
    caches, outs = [], []
    for one_by_one in (False, True):
        c = cache_of(kind, np.random.default_rng(1), 1, hkv, d, 16, [0], room=64, garbage=0.0)
        c.up([0, n] if not one_by_one else None, max_new=n if not one_by_one else 1, max_len=64)
        out = np.zeros((n, heads, d), np.float32)
        for i in range(n if one_by_one else 1):
            rows = slice(i, i + 1) if one_by_one else slice(0, n)
            c.dl.upload(np.array([i + 1 if one_by_one else n], np.uint32))
            dq, dk, dv = (hip.DeviceBuffer.from_numpy(x[rows]) for x in (q, k, v))
            do = hip.DeviceBuffer(out[rows].nbytes)
            gpu.kv_append_device(c.cache, c.seqs, 0, rope, heads, dq.ptr, dq.ptr, dk.ptr, dv.ptr)
            gpu.attn_device(c.cache, c.seqs, 0, heads, dq.ptr, do.ptr, 0.125)
            hip.device_synchronize()
            out[rows] = do.to_numpy(np.float32).reshape(out[rows].shape)
        caches.append(c)
        outs.append(out)
    assert all(same_bits(x, y) for x, y in zip(caches[0].down()[:2], caches[1].down()[:2]))
    c = caches[0]
    c.k, c.v, _ = c.down()
    c.lens = np.array([n], np.uint32)
    want, tol, _ = c.attend(0, turned(q, angles, d, False), 0.125, [0, n])
    for out in outs:
        assert np.all(np.abs(out - want) <= tol + 1e-7 * np.abs(want))


def test_refusals_touch_nothing(gpu, hip, pkg):
    rng = np.random.default_rng(0)
    c = Paged4(rng, 1, 2, 64, 16, [30], weights=True, garbage=0.0).up()
    rows = hip.DeviceBuffer.from_numpy(np.ones(4096, np.float32))
    out = hip.DeviceBuffer.from_numpy(np.full(4096, 5, np.float32))
    before = c.down()

    def append(rope=None, heads=4, q=rows.ptr, to=out.ptr, k=rows.ptr, **kw):
        gpu.kv_append_device(c.cache, c.seqs, kw.pop("layer", 0), rope, heads, q, to, k, rows.ptr, **kw)

    for match, call in (("no such layer", lambda: append(layer=1)), ("even in number", lambda: append(pkg.Rope(rows.ptr, 32, 8, 63))),
                        ("within the head", lambda: append(pkg.Rope(rows.ptr, 64, 8, 66))), ("buffer pointer is null", lambda: append(pkg.Rope(0, 32, 8, 64))),
                        ("of no position", lambda: append(pkg.Rope(rows.ptr, 32, 0, 64))), ("fewer than its pairs", lambda: append(pkg.Rope(rows.ptr, 31, 8, 64))),
                        ("8-byte aligned", lambda: append(pkg.Rope(rows.ptr + 4, 32, 8, 64))), ("have one stride", lambda: append(to=rows.ptr, q_out_stride=260)),
                        ("buffer pointer is null", lambda: append(k=0)), ("16-byte aligned", lambda: append(q=rows.ptr + 8)),
                        ("less than the row", lambda: append(k_stride=124)),
                        ("less than the row", lambda: gpu.kv_load_device(c.cache, c.seqs, 0, out.ptr, out.ptr, k_stride=64)),
                        ("buffer pointer is null", lambda: gpu.kv_load_device(c.cache, c.seqs, 0, out.ptr, 0)),
                        ("positive and finite", lambda: gpu.rope_table_device(64, 0.0, 4, out.ptr)),
                        ("even in number", lambda: gpu.rope_table_device(7, 1e4, 4, out.ptr)),
                        ("buffer pointer is null", lambda: gpu.rope_table_device(64, 1e4, 4, 0))):
        with pytest.raises(pkg.NativeHipError, match=match) as e:
            call()
        assert e.value.code == pkg.ERR_INVALID
    c.cache.head_dim = 40
    with pytest.raises(pkg.NativeHipError, match="multiples of 32") as e:
        append()
    assert e.value.code == pkg.ERR_UNSUPPORTED
    c.cache.head_dim = 64
    hip.device_synchronize()
    assert np.all(out.to_numpy(np.float32) == 5) and all(same_bits(x, y) for x, y in zip(c.down(), before))
    # nothing to do
    none = pkg.KvSeqs(0, 0, 2, 0, 0, n_tokens=0)
    gpu.kv_append_device(c.cache, none, 0, None, 4, 0, 0, 0, 0)
    gpu.kv_load_device(c.cache, none, 0, 0, 0)
    gpu.rope_table_device(64, 1e4, 0, 0)


def test_a_captured_append_on_a_stream_of_its_own(gpu, hip, pkg):
    """Replayed with other rows, lengths and positions, between other work; two graphs of one executor."""
    rng = np.random.default_rng(3)
    stream = hip.Stream()
    c = Paged(rng, False, 1, 2, 64, 16, [0, 0], room=80, garbage=0.0)
    starts = [0, 3, 5]
    c.up(starts, max_new=3, max_len=80)
    angles = rng.normal(0, 1, (30, 32, 2)).astype(np.float32)
    da, dp = hip.DeviceBuffer.from_numpy(angles), hip.DeviceBuffer(5 * 4)
    q, k, v = (hip.DeviceBuffer(5 * n * 64 * 4) for n in (4, 2, 2))
    out, back = hip.DeviceBuffer(5 * 4 * 64 * 4), [hip.DeviceBuffer(5 * 2 * 64 * 4) for _ in range(2)]
    rope = pkg.Rope(da.ptr, 32, 30, 64, halves=True, positions_ptr=dp.ptr)
    graphs = [hip.Graph(stream, lambda s: gpu.kv_append_device(c.cache, c.seqs, 0, rope, 4, q.ptr, out.ptr, k.ptr, v.ptr, stream=s.ptr)),
              hip.Graph(stream, lambda s: gpu.kv_load_device(c.cache, c.seqs, 0, back[0].ptr, back[1].ptr, stream=s.ptr))]
    for turn in range(5):
        rows = [rng.normal(0, 1, (5, n, 64)).astype(np.float32) for n in (4, 2, 2)]
        pos = rng.integers(0, 30, 5).astype(np.uint32)
        for b, x in zip((q, k, v, dp), rows + [pos]):
            b.upload(x)
        c.dl.upload(np.array([3 + 7 * turn, 2 + 11 * turn], np.uint32))
        for g in graphs:
            g.launch()
        stream.synchronize()
        assert np.array_equal(out.to_numpy(np.float32).reshape(5, 4, 64), turned(rows[0], angles[pos], 64, True))
        assert np.array_equal(back[0].to_numpy(np.float32).reshape(5, 2, 64), turned(rows[1], angles[pos], 64, True))
        assert np.array_equal(back[1].to_numpy(np.float32).reshape(5, 2, 64), rows[2])
    for g in graphs:
        g.destroy()
    stream.destroy()
