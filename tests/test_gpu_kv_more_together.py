"""4-bit caches, rotated appends and chosen blocks as programs use them together: several executors and graphs, batches larger than a launch takes at a time,
blocks that sequences share, calls that no launch holds."""
import importlib

import numpy as np
import pytest

from paged import Paged, same_bits
from paged4 import Paged4
from test_gpu_attn_select import bounds_of, cache_of, definition
from test_gpu_kv_4bit import attend, check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu(pkg):
    g = pkg.HipGemv(0)
    yield g
    g.close()


@pytest.fixture(scope="module")
def hip():
    return importlib.import_module("llama-rust_amd.hiprt")


def test_executors_and_streams_at_the_same_time(hip, pkg):
    """Two programs' steps in turn without a wait between them: each has its own workspace, the outcome is a step's alone."""
    rng = np.random.default_rng(0)
    sides = []
    for kind, lens in (("q4_0", [900, 40]), ("f16", [700, 300])):
        gpu, stream = pkg.HipGemv(0), hip.Stream()
        c = cache_of(kind, rng, 1, 2, 64, 16, lens, room=20, garbage=0.0)
        c.up()
        q = [hip.DeviceBuffer.from_numpy(rng.normal(0, 1, (2, 8, 64)).astype(np.float32)) for _ in range(6)]
        k, v = (hip.DeviceBuffer.from_numpy(rng.normal(0, 1, (2, 2, 64)).astype(np.float32)) for _ in range(2))
        outs = [[hip.DeviceBuffer(2 * 8 * 64 * 4) for _ in range(2)] for _ in q]
        bounds = hip.DeviceBuffer.from_numpy(bounds_of(c, kind))

        def step(i, gpu=gpu, stream=stream, c=c, q=q, k=k, v=v, outs=outs, bounds=bounds):
            gpu.kv_append_device(c.cache, c.seqs, 0, None, 0, 0, 0, k.ptr, v.ptr, stream=stream.ptr)
            gpu.kv_bounds_device(c.cache, c.seqs, 0, bounds.ptr, stream=stream.ptr)
            gpu.attn_device(c.cache, c.seqs, 0, 8, q[i].ptr, outs[i][0].ptr, 0.125, stream=stream.ptr)
            gpu.attn_select_device(c.cache, c.seqs, 0, 8, bounds.ptr, 5, 1, 1, q[i].ptr, outs[i][1].ptr, 0.125, stream=stream.ptr)

        sides.append((gpu, stream, step, outs))
    alone = []
    for gpu, stream, step, outs in sides:
        for i in range(6):
            step(i)
            stream.synchronize()
        alone.append([[o.to_numpy(np.uint32) for o in pair] for pair in outs])
        for pair in outs:
            for o in pair:
                o.upload(np.zeros(2 * 8 * 64, np.float32))
    for i in range(6):
        for _, _, step, _ in sides:
            step(i)
    hip.device_synchronize()
    for (gpu, stream, _, outs), want in zip(sides, alone):
        for pair, pair_want in zip(outs, want):
            assert all(np.array_equal(o.to_numpy(np.uint32), x) for o, x in zip(pair, pair_want))
        assert np.any(want[0][0]) and np.any(want[0][1])
        stream.destroy()
        gpu.close()


def test_two_graphs_of_one_workspace(gpu, hip):
    """A long call in shares and one over chosen blocks captured apart, replayed in turn with eager calls of the same executor between."""
    rng = np.random.default_rng(1)
    stream = hip.Stream()
    c = cache_of("q4_0", rng, 1, 2, 128, 16, [3000, 700]).up()
    db = hip.DeviceBuffer.from_numpy(bounds_of(c, "q4_0"))
    q = hip.DeviceBuffer(2 * 8 * 128 * 4)
    outs = [hip.DeviceBuffer(2 * 8 * 128 * 4) for _ in range(4)]
    scale = np.float32(128 ** -0.5)
    calls = [lambda s, out: gpu.attn_device(c.cache, c.seqs, 0, 8, q.ptr, out.ptr, scale, stream=s.ptr),
             lambda s, out: gpu.attn_select_device(c.cache, c.seqs, 0, 8, db.ptr, 20, 1, 2, q.ptr, out.ptr, scale, stream=s.ptr)]
    q.upload(np.zeros(2 * 8 * 128, np.float32))
    for call in calls:
        call(stream, outs[0])
    stream.synchronize()
    graphs = [hip.Graph(stream, lambda s, i=i: calls[i](s, outs[i])) for i in range(2)]
    for turn in range(4):
        q.upload(rng.normal(0, 1, (2, 8, 128)).astype(np.float32))
        for i in ((0, 1), (1, 0))[turn % 2]:
            graphs[i].launch()
            calls[1 - i](stream, outs[3 - i])
        stream.synchronize()
        assert np.array_equal(outs[0].to_numpy(np.uint32), outs[2].to_numpy(np.uint32))
        assert np.array_equal(outs[1].to_numpy(np.uint32), outs[3].to_numpy(np.uint32))
        assert not np.array_equal(outs[0].to_numpy(np.uint32), outs[1].to_numpy(np.uint32))
    for g in graphs:
        g.destroy()
    stream.destroy()


@pytest.mark.parametrize("d,block", [(64, 16), (128, 20), (96, 7)])
@pytest.mark.parametrize("new,most", [(1, 40), (4, 40), (1, 700), (4, 700)])
def test_more_sequences_than_go_at_once(gpu, d, block, new, most):
    """300 sequences in two launches, short ones alone and long ones among them; eight query heads a key-value head: one tile of rows, two."""
    rng = np.random.default_rng(most + new)
    lens = [int(x) for x in rng.integers(0, 40, 300)]
    lens[7], lens[290] = most, most - 3
    starts = list(range(0, 300 * new + 1, new))
    c = Paged4(rng, 1, 1, d, block, lens).up(starts if new > 1 else None, max_new=new)
    q = rng.normal(0, 1, (300 * new, 8, d)).astype(np.float32)
    scale = np.float32(d ** -0.5)
    want, tol, _ = c.attend(0, q, float(scale), starts)
    check(attend(gpu, c, 0, q, scale), want, tol + 1e-7 * np.abs(want))


@pytest.mark.parametrize("kind", ["f32", "f16", "q4_0"])
@pytest.mark.parametrize("seqs,hkv,heads,d,new,most", [(277, 8, 8, 32, 1, 20), (131, 8, 16, 64, 1, 20), (67, 8, 64, 32, 3, 14), (277, 8, 8, 160, 1, 9), (300, 8, 8, 32, 1, 300)])
def test_several_sequences_a_workgroup(gpu, kind, seqs, hkv, heads, d, new, most):
    """Short sequences by the hundred, each some wavefronts of a workgroup, the last workgroup's not all there; some hold nothing, have places that are not there,
    rows whose scores are computed again; the weights of a few query heads a key-value head from the scores that are kept."""
    rng = np.random.default_rng(seqs + d)
    lens = [int(x) for x in rng.integers(0, 15 if most == 300 else most, seqs)]
    lens[5], lens[seqs - 2] = most, most - 1
    weights = new == 1
    c = (Paged4(rng, 1, hkv, d, 8, lens, weights=weights) if kind == "q4_0" else Paged(rng, kind == "f16", 1, hkv, d, 8, lens, weights=weights))
    c.tables[6, 0] = c.n_blocks
    starts = list(range(0, seqs * new + 1, new))
    c.up(starts if new > 1 else None, max_new=new)
    q = rng.normal(0, 1, (seqs * new, heads, d)).astype(np.float32)
    q[::11] *= np.float32(1e6)
    scale = np.float32(d ** -0.5)
    want, tol, sums = c.attend(0, q, float(scale), starts)
    got = attend(gpu, c, 0, q, scale)
    check(got, want, tol + 1e-7 * np.abs(want))
    assert np.array_equal(attend(gpu, c, 0, q, scale), got)
    if weights:
        assert np.array_equal(attend(gpu, c, 0, q, scale, weights=True, decay=0.5), got)
        w, w_tol = c.weigh(0, sums, 0.5)
        after = c.down()[2]
        held = ~np.isnan(w)
        assert same_bits(after[~held], c.w[~held])
        off = np.abs(after[held] - w[held])
        assert np.all(off <= w_tol[held]), np.max(off - w_tol[held])


@pytest.mark.parametrize("new", [1, 24])
def test_rows_of_nobody_and_blocks_of_several(gpu, hip, pkg, new):
    """A prefix that two sequences share, a block that stands twice in one table, rows before the first sequence and behind the last."""
    rng = np.random.default_rng(new)
    block = 16
    c = Paged4(rng, 1, 2, 64, block, [150, 130, 200])
    c.tables[1, :4] = c.tables[0, :4]
    c.tables[2, 5] = c.tables[2, 2]
    starts = [3, 3 + new, 3 + 2 * new, 3 + 3 * new]
    n = 3 + 3 * new + 5
    c.up(starts, max_new=new, n_tokens=n)
    q = rng.normal(0, 1, (n, 6, 64)).astype(np.float32)
    want, tol, _ = c.attend(0, q, 0.125, starts)
    got = attend(gpu, c, 0, q, 0.125)
    held = slice(3, 3 + 3 * new)
    assert np.all(got[:3] == 7.25) and np.all(got[held.stop:] == 7.25)
    check(got[held], want[held], (tol + 1e-7 * np.abs(want))[held])
    bounds = bounds_of(c, "q4_0")
    wc, ws, tol = definition(c, "q4_0", bounds, 0, q, 0.125, starts, 5, 1, 1)
    dq, db = hip.DeviceBuffer.from_numpy(q), hip.DeviceBuffer.from_numpy(bounds)
    do, dc = hip.DeviceBuffer.from_numpy(np.full(q.shape, 7.25, np.float32)), hip.DeviceBuffer.from_numpy(np.full((n, 2, 5), 0xabcd, np.uint32))
    gpu.attn_select_device(c.cache, c.seqs, 0, 6, db.ptr, 5, 1, 1, dq.ptr, do.ptr, 0.125, chosen_ptr=dc.ptr)
    hip.device_synchronize()
    got = do.to_numpy(np.float32).reshape(q.shape)
    assert np.array_equal(dc.to_numpy(np.uint32).reshape(n, 2, 5), wc)
    assert np.all(got[:3] == 7.25) and np.all(got[held.stop:] == 7.25)
    assert np.all(np.abs(got - ws)[held] <= (tol + 1e-7 * np.abs(ws))[held])
    # appended and read back: only the sequences' rows
    k, v, back_k, back_v = (hip.DeviceBuffer.from_numpy(x) for x in [rng.normal(0, 1, (n, 2, 64)).astype(np.float32) for _ in range(2)] +
                            [np.full((n, 2, 64), 3, np.float32) for _ in range(2)])
    out = hip.DeviceBuffer.from_numpy(np.full(q.shape, 7.25, np.float32))
    gpu.kv_append_device(c.cache, c.seqs, 0, None, 6, dq.ptr, out.ptr, k.ptr, v.ptr)
    gpu.kv_load_device(c.cache, c.seqs, 0, back_k.ptr, back_v.ptr)
    hip.device_synchronize()
    out = out.to_numpy(np.float32).reshape(q.shape)
    assert np.array_equal(out[held], q[held]) and np.all(out[:3] == 7.25) and np.all(out[held.stop:] == 7.25)
    for x in (back_k, back_v):
        x = x.to_numpy(np.float32).reshape(n, 2, 64)
        assert np.all(x[:3] == 3) and np.all(x[held.stop:] == 3) and np.all(np.any(x[held] != 3, axis=(1, 2)))


def test_bounds_and_choice_in_a_cache_of_more_than_four_gigabytes(gpu, hip, pkg):
    """The last blocks of a cache of 5 GB of keys, which nothing else is written to; its bounds lie beyond 4 GB as well."""
    d, block, heads = 256, 2, 4
    n_blocks = 5 * (1 << 30) // (heads * block * d * 2)
    k = hip.DeviceBuffer(n_blocks * heads * block * d * 2)
    db = hip.DeviceBuffer(n_blocks * heads * 2 * d * 2)
    assert db.nbytes > 1 << 32
    rng = np.random.default_rng(1)
    pages = 30
    table = np.array([[n_blocks - 1 - j for j in range(pages)]], np.uint32)
    dt, dl, ds = (hip.DeviceBuffer.from_numpy(np.array(x, np.uint32)) for x in (table, [59], [0, 59]))
    rows = rng.normal(0, 1, (59, heads, d)).astype(np.float16).astype(np.float32)
    dk = hip.DeviceBuffer.from_numpy(rows)
    cache = pkg.KvCache(pkg.F16, 1, heads, d, block, n_blocks, k.ptr, k.ptr)  # values are the keys: written twice, the same
    whole = pkg.KvSeqs(1, dt.ptr, pages, dl.ptr, 59, ds.ptr, 59, 59)
    gpu.kv_append_device(cache, whole, 0, None, 0, 0, 0, dk.ptr, dk.ptr)
    gpu.kv_bounds_device(cache, whole, 0, db.ptr)
    q = rng.normal(0, 1, (1, heads, d)).astype(np.float32)
    dq, do, dc = hip.DeviceBuffer.from_numpy(q), hip.DeviceBuffer(q.nbytes), hip.DeviceBuffer(heads * 8 * 4)
    gpu.attn_select_device(cache, pkg.KvSeqs(1, dt.ptr, pages, dl.ptr, 59), 0, heads, db.ptr, 8, 1, 2, dq.ptr, do.ptr, 1 / 16, chosen_ptr=dc.ptr)
    hip.device_synchronize()
    got, chosen = do.to_numpy(np.float32).reshape(heads, d), dc.to_numpy(np.uint32).reshape(heads, 8)
    x = rows.astype(np.float64)
    for h in range(heads):
        qr = q[0, h].astype(np.float64)
        blocks = [x[2 * j:2 * j + 2, h] for j in range(pages)]
        score = [np.float32((np.where(qr > 0, b.max(0), b.min(0)) * qr).sum()) for b in blocks]
        kept = sorted([0, 28, 29] + sorted(range(1, 28), key=lambda j: (-score[j], j))[:5])
        assert list(chosen[h]) == kept
        kv = np.concatenate([blocks[j] for j in kept])
        s = kv @ qr / 16
        p = np.exp(s - s.max())
        p /= p.sum()
        size = (np.abs(kv) @ np.abs(qr)).max() / 16
        tol = (2 * (d + 24) * size + len(kv) + 80) * 2.0 ** -23 * (p @ np.abs(kv))  # as in paged.py
        assert np.all(np.abs(got[h] - p @ kv) <= tol)
    for b in (k, db):
        b.free()


def test_calls_that_no_launch_holds(gpu, hip, pkg):
    """Refused on the host, before anything is looked at."""
    rng = np.random.default_rng(0)
    rows = hip.DeviceBuffer.from_numpy(np.ones(4096, np.float32))
    n = 6 << 20
    for kind in ("f32", "f16", "q4_0"):
        c = cache_of(kind, rng, 1, 2, 64, 16, [30]).up()
        before = c.down()
        many = pkg.KvSeqs(n, c.dt.ptr, c.stride, c.dl.ptr, 30)
        for call in (lambda: gpu.kv_append_device(c.cache, many, 0, None, 4, rows.ptr, rows.ptr, rows.ptr, rows.ptr),
                     lambda: gpu.kv_store_device(c.cache, many, 0, rows.ptr, rows.ptr), lambda: gpu.kv_load_device(c.cache, many, 0, rows.ptr, rows.ptr),
                     lambda: gpu.kv_bounds_device(c.cache, many, 0, rows.ptr),
                     lambda: gpu.attn_select_device(c.cache, many, 0, 4, rows.ptr, 2, 0, 1, rows.ptr, rows.ptr + 4096, 0.125)):
            with pytest.raises(pkg.NativeHipError, match="larger than one launch") as e:
                call()
            assert e.value.code == pkg.ERR_INVALID
        hip.device_synchronize()
        assert np.all(rows.to_numpy(np.float32) == 1) and all(same_bits(x, y) for x, y in zip(c.down()[:2], before[:2]))
