"""A K/V cache held in 4 bits on the GPU: rows packed bit for bit as numpy packs them, read back, and everything over such a cache -
attention, weights, eviction - against the definition in 64 bits over the values that the rows stand for (tests/paged4.py)."""
import importlib

import numpy as np
import pytest

from paged import NOWHERE, same_bits
from paged4 import Paged4, pack, to_buffer, unpack

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu(pkg):
    g = pkg.HipGemv(0)
    yield g
    g.close()


@pytest.fixture(scope="module")
def hip():
    return importlib.import_module("llama-rust_amd.hiprt")


def attend(gpu, c, layer, q, scale, out=None, stream=0, **kw):
    """The call, synchronised; out keeps what it held in rows the call leaves alone."""
    dq = c.hip.DeviceBuffer.from_numpy(q.astype(np.float32))
    start = np.full(q.shape, 7.25, np.float32) if out is None else out
    do = c.hip.DeviceBuffer.from_numpy(start)
    gpu.attn_device(c.cache, c.seqs, layer, kw.pop("heads", q.shape[-2]), dq.ptr, do.ptr, scale, stream=stream, **kw)
    c.hip.device_synchronize()
    return do.to_numpy(np.float32).reshape(start.shape)


def check(got, want, tol, what=""):
    assert np.all(np.isfinite(got)), what
    off = np.abs(got.astype(np.float64) - want)
    worst = np.unravel_index(np.argmax(off - tol), off.shape)
    assert np.all(off <= tol), (what, worst, got[worst], want[worst], tol[worst])


def hard_rows(rng, n, d):
    """Rows where packing can go wrong: zeros, equal largest ones of both signs, exact ties, sizes from f32's least to beyond f16, what is not
    finite."""
    x = rng.normal(0, 1, (n, d)).astype(np.float32)
    x[0] = 0
    x[1, ::2] = -0.0
    x[2, :32] = np.where(np.arange(32) % 2, 1.5, -1.5)  # the first of the largest: -1.5
    x[3, :32] = np.where(np.arange(32) % 2, -1.5, 1.5)
    x[4] = (np.arange(d) % 32 - 16) * 0.5  # d = 1 from the first element of size 8, every other one a tie
    x[5] = (np.arange(d) % 17 - 8) * np.float32(2.0 ** -20)
    x[6] *= np.float32(1e-30)
    x[7] *= np.float32(1e-7)
    x[8] *= np.float32(3e5)
    x[9] *= np.float32(1e38)
    x[10, 5] = np.inf
    x[11, d - 1] = np.nan
    x[12, 3] = -np.inf
    x[13] = np.nextafter(np.float32(0.5), np.float32(rng.integers(0, 2)), dtype=np.float32) * (np.arange(d) % 16)
    x[14] = np.ldexp(np.float32(1), rng.integers(-149, 16, d)).astype(np.float32)
    x[15, :32] = np.float32(8160 * 8) * np.linspace(-1, 1, 32, dtype=np.float32)
    return x


@pytest.mark.parametrize("d,hkv,block", [(32, 3, 16), (64, 2, 7), (96, 1, 1), (128, 8, 16), (160, 2, 20), (256, 1, 64)])
@pytest.mark.parametrize("starts,lens", [(None, [16, 0, 33, 5] * 6), ([0, 24, 24, 41, 42], [30, 9, 17, 80])])
def test_rows_are_packed_bit_for_bit(gpu, hip, pkg, d, hkv, block, starts, lens):
    """kv_store and kv_append without a rotation leave what numpy packs, in their rows alone; kv_load gives what it stands for."""
    rng = np.random.default_rng(d + block)
    n = starts[-1] if starts else len(lens)
    news = np.diff(starts) if starts else np.ones(n, int)
    starts_or = starts or list(range(n + 1))
    k = np.concatenate([hard_rows(rng, 24, d)[rng.permutation(24)] for _ in range(hkv)] * 2)[:n * hkv].reshape(n, hkv, d)
    v = k[::-1, :, ::-1].copy()
    for way in ("store", "append"):
        c = Paged4(rng, 2, hkv, d, block, lens, weights=True).up(starts, max_new=int(max(news)))
        before = c.packed()
        dk, dv = hip.DeviceBuffer.from_numpy(k), hip.DeviceBuffer.from_numpy(v)
        if way == "store":
            gpu.kv_store_device(c.cache, c.seqs, 1, dk.ptr, dv.ptr)
        else:
            gpu.kv_append_device(c.cache, c.seqs, 1, None, 0, 0, 0, dk.ptr, dv.ptr)
        hip.device_synchronize()
        w = c.dw.to_numpy(np.float32).reshape(c.w.shape)
        want = [[x.copy() for x in pair] for pair in before]
        want_w, back = c.w.copy(), [np.zeros_like(k) for _ in range(2)]
        for b in range(len(lens)):
            for i in range(int(news[b])):
                t, row = int(lens[b]) - int(news[b]) + i, starts_or[b] + i
                if t < 0:
                    continue
                at = (c.tables[b, t // block], 1, slice(None), t % block)
                for which, rows in enumerate((k, v)):
                    words, scales = pack(rows[row])
                    want[which][0][at], want[which][1][at] = words, scales
                    back[which][row] = unpack(words, scales)
                if way == "append":
                    want_w[at] = 0
        assert same_bits(w, want_w)
        for (gw, gs), (ww, ws) in zip(c.packed(), want):
            assert np.array_equal(np.isnan(gs), np.isnan(ws)) and np.array_equal(gs[~np.isnan(gs)], ws[~np.isnan(ws)])
            told = np.repeat(~np.isnan(gs), 4, -1)  # codes under a scale of NaN say nothing
            assert np.array_equal(gw[told], ww[told])
        lk, lv = (hip.DeviceBuffer.from_numpy(np.full((n + 1, hkv * d + 4), 3.5, np.float32)) for _ in range(2))
        gpu.kv_load_device(c.cache, c.seqs, 1, lk.ptr, lv.ptr, k_stride=hkv * d + 4, v_stride=hkv * d + 4)
        hip.device_synchronize()
        for got, rows in ((lk, back[0]), (lv, back[1])):
            got = got.to_numpy(np.float32).reshape(n + 1, -1)
            assert np.all(got[n] == 3.5) and np.all(got[:, hkv * d:] == 3.5)
            assert same_bits(got[:n, :hkv * d], rows.reshape(n, -1))


@pytest.mark.parametrize("kind", ["f32", "f16", "q4_0"])
def test_load_of_what_is_not_there(gpu, hip, pkg, kind):
    """A block that no table names and tokens below position 0 give zeros; the other types' rows come as they are."""
    from paged import Paged
    rng = np.random.default_rng(4)
    args = (2, 2, 64, 16, [40, 2, 20])
    c = Paged4(rng, *args) if kind == "q4_0" else Paged(rng, kind == "f16", *args)
    c.tables[0, 1], c.tables[2, 0] = NOWHERE, c.n_blocks
    starts = [0, 40, 45, 50]
    c.up(starts, max_new=40)
    out = [hip.DeviceBuffer.from_numpy(np.full((50, 2, 64), 9, np.float32)) for _ in range(2)]
    gpu.kv_load_device(c.cache, c.seqs, 0, out[0].ptr, out[1].ptr)
    hip.device_synchronize()
    for got, held in zip(out, (c.k, c.v)):
        got = got.to_numpy(np.float32).reshape(50, 2, 64)
        for b, (n, length) in enumerate(zip(np.diff(starts), c.lens)):
            for i in range(n):
                t = int(length) - int(n) + i
                want = held[c.tables[b, t // 16], 0, :, t % 16].astype(np.float32) if t >= 0 and c.there(b, t) else np.zeros((2, 64), np.float32)
                assert np.array_equal(got[starts[b] + i], want), (b, i)


LAYOUTS = [(1, 1, 32), (4, 4, 128), (8, 2, 128), (14, 2, 64), (32, 4, 96), (16, 1, 256), (12, 4, 192), (71, 1, 64), (34, 2, 160), (6, 2, 224)]


@pytest.mark.parametrize("heads,hkv,d", LAYOUTS)
@pytest.mark.parametrize("block", [16, 20])
def test_one_token_a_sequence(gpu, heads, hkv, d, block):
    """Lengths around the tiles' and blocks' ends, a sequence that holds nothing."""
    rng = np.random.default_rng(d + heads)
    c = Paged4(rng, 2, hkv, d, block, [1, 0, 15, 16, 17, 33, 64, 130, 300]).up()
    q = rng.normal(0, 1, (9, heads, d)).astype(np.float32)
    want, tol, _ = c.attend(1, q, d ** -0.5)
    got = attend(gpu, c, 1, q, np.float32(d ** -0.5))
    check(got, want, tol + 1e-7 * np.abs(want))
    assert np.all(got[1] == 0)


@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("block", [32, 12, 6])
@pytest.mark.parametrize("group", [3, 8, 9, 20])
def test_heads_blocks_and_groups(gpu, d, block, group):
    """Every way that rows are read, up to eight rows a head, more than eight, more than sixteen; shares of several tiles of every wavefront, blocks
    that are not there and a window with first tokens among them."""
    rng = np.random.default_rng(d + block)
    c = Paged4(rng, 1, 1, d, block, [700, 45])
    c.tables[0, 9] = NOWHERE
    c.up()
    q = rng.normal(0, 1, (2, group, d)).astype(np.float32)
    scale = np.float32(d ** -0.5)
    for window, sinks in ((0, 0), (90, 5)):
        want, tol, _ = c.attend(0, q, float(scale), window=window, sinks=sinks)
        check(attend(gpu, c, 0, q, scale, window=window, sinks=sinks), want, tol)


@pytest.mark.parametrize("block", [1, 3, 8, 48, 256])
def test_blocks_of_any_size(gpu, block):
    rng = np.random.default_rng(block)
    c = Paged4(rng, 3, 2, 64, block, [5, 257, 100]).up()
    q = rng.normal(0, 1, (3, 4, 64)).astype(np.float32)
    want, tol, _ = c.attend(2, q, 0.125)
    check(attend(gpu, c, 2, q, 0.125), want, tol)


@pytest.mark.parametrize("d,block", [(64, 32), (128, 20)])
def test_long_sequences_are_shared_and_joined(gpu, d, block):
    """Many shares beside few; large scores in one place, so that a row's maximum rises late."""
    rng = np.random.default_rng(3)
    c = Paged4(rng, 1, 2, d, block, [5000, 40, 2999])
    c.k[c.at(0, 4000)] *= 20
    c.k[c.at(2, 3)] *= 20
    c.settle()
    c.up()
    q = rng.normal(0, 1, (3, 8, d)).astype(np.float32)
    want, tol, _ = c.attend(0, q, d ** -0.5)
    # An element of the heavy position's V is zero as often as not, so that a row's value may be the light ones' alone.  A probability is held in
    # two f16 parts at 2^8 times its size, the heaviest at least at 2^8: the second part's half step of 2^-25 is 2^-33 of the heaviest, for
    # each position.
    light = c.lens[:, None, None] * 2.0 ** -33 * float(np.nanmax(np.abs(c.v.astype(np.float64))))
    check(attend(gpu, c, 0, q, np.float32(d ** -0.5)), want, tol + 1e-7 * np.abs(want) + light)


RAGGED = [([0, 1, 4, 4, 21, 22], [1, 3, 9, 17, 60]), ([0, 40, 41, 105, 105, 170], [40, 90, 64, 5, 200])]


@pytest.mark.parametrize("starts,lens", RAGGED)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (7, 3), (40, 4), (1000, 4), (30, 50)])
@pytest.mark.parametrize("d,block", [(64, 16), (96, 5)])
def test_several_tokens_a_sequence(gpu, starts, lens, window, sinks, d, block):
    rng = np.random.default_rng(window + sinks)
    c = Paged4(rng, 2, 2, d, block, lens).up(starts, max_new=int(np.diff(starts).max()))
    q = rng.normal(0, 1, (starts[-1], 6, d)).astype(np.float32)
    want, tol, _ = c.attend(0, q, d ** -0.5, starts, window, sinks)
    check(attend(gpu, c, 0, q, np.float32(d ** -0.5), window=window, sinks=sinks), want, tol + 1e-7 * np.abs(want))


@pytest.mark.parametrize("heads,hkv,d,block", [(4, 4, 128, 16), (8, 1, 256, 20), (10, 2, 96, 16), (40, 2, 32, 7), (9, 1, 192, 64), (4, 2, 160, 1)])
def test_prompts_in_other_layouts(gpu, heads, hkv, d, block):
    rng = np.random.default_rng(d)
    starts = [0, 33, 34, 120]
    c = Paged4(rng, 1, hkv, d, block, [33, 50, 150]).up(starts, max_new=86)
    q = rng.normal(0, 1, (120, heads, d)).astype(np.float32)
    for window, sinks in ((0, 0), (20, 4)):
        want, tol, _ = c.attend(0, q, d ** -0.5, starts, window, sinks)
        check(attend(gpu, c, 0, q, np.float32(d ** -0.5), window=window, sinks=sinks), want, tol + 1e-7 * np.abs(want))


def test_a_long_prompt_chunk(gpu):
    """Rows for 128 a workgroup, shares of a block's steps."""
    rng = np.random.default_rng(12)
    c = Paged4(rng, 1, 1, 128, 16, [900]).up([0, 260], max_new=260)
    q = rng.normal(0, 1, (260, 4, 128)).astype(np.float32)
    want, tol, _ = c.attend(0, q, 128 ** -0.5, [0, 260])
    check(attend(gpu, c, 0, q, np.float32(128 ** -0.5)), want, tol + 1e-7 * np.abs(want))


@pytest.mark.parametrize("new", [1, 40])
def test_what_no_row_sees_reaches_none(gpu, new):
    """Rows of NaN scales behind a window's back and in places of nobody; a row that sees one is NaN."""
    rng = np.random.default_rng(5)
    lens, starts = [100, 90], [0, new, 2 * new]
    c = Paged4(rng, 1, 2, 64, 16, lens)
    for t in range(4, 30):
        c.k[c.at(0, t)] = np.nan
        c.v[c.at(0, t)] = np.nan
    c.v[c.at(1, 60 if new == 40 else 89)][..., 0:3] = np.nan
    c.settle()
    c.up(starts, max_new=new)
    q = rng.normal(0, 1, (2 * new, 4, 64)).astype(np.float32)
    want, tol, _ = c.attend(0, q, 0.125, starts, 30, 4)
    got = attend(gpu, c, 0, q, 0.125, window=30, sinks=4)
    check(got[:new], want[:new], tol[:new])
    assert np.array_equal(np.isnan(got[new:]), np.isnan(want[new:]))
    assert np.isnan(got[new:]).any()
    fine = ~np.isnan(want[new:])
    assert np.all(np.abs(got[new:][fine] - want[new:][fine]) <= tol[new:][fine])


@pytest.mark.parametrize("size", [2.0 ** -22, 2.0 ** -13, 3e4, 1e9])
@pytest.mark.parametrize("new", [1, 33])
def test_values_of_any_size(gpu, size, new):
    """Scales and values down to f16's least, which the matrix cores have to keep, and up to the largest that a row can hold."""
    rng = np.random.default_rng(7)
    c = Paged4(rng, 1, 1, 64, 16, [70])
    c.v = (c.v.astype(np.float32) * np.float32(size)).astype(np.float16) if size < 1e4 else c.v
    c.k = (c.k.astype(np.float32) * np.float32(min(size, 1.0))).astype(np.float16)
    c.settle()
    if size > 1e4:
        c.v = unpack(*pack(rng.normal(0, 1, c.v.shape).astype(np.float32) * np.float32(size)))
    c.up([0, new], max_new=new)
    q = (rng.normal(0, 1, (new, 2, 64)) / min(size, 1.0)).astype(np.float32)
    want, tol, _ = c.attend(0, q, 0.125, [0, new])
    got = attend(gpu, c, 0, q, 0.125)
    assert np.abs(want).max() > 0
    check(got, want, tol)


def test_blocks_that_are_not_there(gpu):
    rng = np.random.default_rng(9)
    for block in (16, 7):
        c = Paged4(rng, 2, 2, 64, block, [70, 16, 120])
        c.tables[0, 1], c.tables[1, 0], c.tables[2, 3] = c.n_blocks, NOWHERE, 0x80000000
        for starts in (None, [0, 40, 50, 120]):
            c.up(starts, max_new=70 if starts else 1)
            q = rng.normal(0, 1, (120 if starts else 3, 4, 64)).astype(np.float32)
            want, tol, _ = c.attend(1, q, 0.125, starts)
            check(attend(gpu, c, 1, q, 0.125), want, tol)


@pytest.mark.parametrize("decay", [0.0, 0.5])
@pytest.mark.parametrize("starts,lens,window,sinks", [(None, [1, 0, 31, 64, 700], 0, 0), ([0, 40, 41, 105, 105, 170], [40, 90, 64, 5, 200], 0, 0),
                                                       ([0, 3, 60], [90, 57], 25, 4)])
@pytest.mark.parametrize("d", [64, 96])
def test_weights_are_summed(gpu, decay, starts, lens, window, sinks, d):
    rng = np.random.default_rng(len(lens))
    news = np.diff(starts) if starts else [1]
    c = Paged4(rng, 2, 2, d, 16, lens, weights=True).up(starts, max_new=int(max(news)))
    q = rng.normal(0, 1, (starts[-1] if starts else len(lens), 6, d)).astype(np.float32)
    scale = np.float32(d ** -0.5)
    want, tol, sums = c.attend(1, q, float(scale), starts, window, sinks)
    check(attend(gpu, c, 1, q, scale, window=window, sinks=sinks, weights=True, decay=decay), want, tol)
    w, w_tol = c.weigh(1, sums, decay)
    after = c.down()[2]
    held = ~np.isnan(w)
    assert same_bits(after[~held], c.w[~held])
    off = np.abs(after[held] - w[held])
    assert np.all(off <= w_tol[held]), np.max(off - w_tol[held])


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("d,hkv,block,keep,first,recent", [(64, 2, 16, 20, 2, 5), (32, 3, 7, 33, 0, 0), (160, 1, 20, 50, 4, 46), (128, 2, 16, 0, 0, 0)])
def test_eviction(gpu, hip, in_place, d, hkv, block, keep, first, recent):
    """Codes and scales move together, bit for bit."""
    rng = np.random.default_rng(keep + d)
    c = Paged4(rng, 3, hkv, d, block, [60, 3, 0, 300, 20], weights=True, extra_blocks=80)
    c.w[:, :, :, ::3] = 0.5  # ties
    c.up()
    dst = None
    if not in_place:
        dst = np.full((5, 24), NOWHERE, np.uint32)
        at = 0
        for b, n in enumerate(c.lens):
            pages = -(-min(int(n), keep) // block)
            dst[b, :pages] = c.free[at:at + pages]
            at += pages
    dd = hip.DeviceBuffer.from_numpy(dst) if dst is not None else None
    new = hip.DeviceBuffer.from_numpy(np.zeros(5, np.uint32))
    gpu.kv_evict_device(c.cache, c.seqs, 1, 2, keep, first, recent, dd.ptr if dd else 0, 24 if dd else 0, new.ptr)
    hip.device_synchronize()
    lens, k, v, w = c.evict([1, 2], keep, first, recent, dst)
    gk, gv, gw = c.down()
    assert np.array_equal(new.to_numpy(np.uint32), lens)
    assert same_bits(gk, k) and same_bits(gv, v) and same_bits(gw, w)


def test_eviction_in_place_in_strips(gpu, hip):
    """More rows than a strip holds, in slices and whole."""
    rng = np.random.default_rng(10)
    for d, hkv, layers in ((128, 1, 1), (32, 4, 2)):
        c = Paged4(rng, layers, hkv, d, 64, [5000], weights=True).up()
        new = hip.DeviceBuffer.from_numpy(np.zeros(1, np.uint32))
        gpu.kv_evict_device(c.cache, c.seqs, 0, layers, 3500, 4, 100, 0, 0, new.ptr)
        hip.device_synchronize()
        _, k, v, w = c.evict(range(layers), 3500, 4, 100)
        assert all(same_bits(x, y) for x, y in zip(c.down(), (k, v, w)))


@pytest.mark.parametrize("new", [1, 40])
def test_a_captured_step_follows_its_arrays(gpu, hip, new):
    """Append, attention and load of a step captured once, replayed with other rows, lengths and tables between other work."""
    rng = np.random.default_rng(new)
    stream = hip.Stream()
    lens = [130, 77]
    starts = [0, new, 2 * new]
    c = Paged4(rng, 1, 2, 128, 16, lens, room=200).up(starts, max_new=new, max_len=300)
    q = hip.DeviceBuffer(2 * new * 8 * 128 * 4)
    k, v, out = (hip.DeviceBuffer(2 * new * n * 128 * 4) for n in (2, 2, 8))
    scale = np.float32(128 ** -0.5)

    def step(s):
        gpu.kv_append_device(c.cache, c.seqs, 0, None, 0, 0, 0, k.ptr, v.ptr, stream=s.ptr)
        gpu.attn_device(c.cache, c.seqs, 0, 8, q.ptr, out.ptr, scale, stream=s.ptr)

    for b in (q, k, v):
        b.upload(np.zeros(b.nbytes // 4, np.float32))
    step(stream)
    stream.synchronize()
    for buf, x in zip((c.dk, c.dv), (c.k, c.v)):  # as before that step
        buf.upload(to_buffer(x))
    graph = hip.Graph(stream, step)
    for turn in range(4):
        rows = [rng.normal(0, 1, (2 * new, n, 128)).astype(np.float32) for n in (8, 2, 2)]
        for b, x in zip((q, k, v), rows):
            b.upload(x)
        c.lens = np.array([130 + turn * new, 77 + turn * new], np.uint32)
        c.dl.upload(c.lens)
        if turn == 2:  # blocks change places
            c.tables[0, :2] = c.tables[0, 1::-1]
            c.dt.upload(c.tables)
        graph.launch()
        stream.synchronize()
        for b in range(2):
            for i in range(new):
                at = (c.tables[b, (int(c.lens[b]) - new + i) // 16], 0, slice(None), (int(c.lens[b]) - new + i) % 16)
                c.k[at], c.v[at] = unpack(*pack(rows[1][starts[b] + i])), unpack(*pack(rows[2][starts[b] + i]))
        want, tol, _ = c.attend(0, rows[0], float(scale), starts)
        got = out.to_numpy(np.float32).reshape(2 * new, 8, 128)
        check(got, want, tol + 1e-7 * np.abs(want), turn)
        assert np.array_equal(attend(gpu, c, 0, rows[0], scale), got)
    gk, gv, _ = c.down()
    assert same_bits(gk, c.k) and same_bits(gv, c.v)
    graph.destroy()
    stream.destroy()


def test_a_cache_of_more_than_four_gigabytes(gpu, hip, pkg):
    """Offsets of codes and scales beyond 32 bits: the last blocks of a cache of 9 GB an array's codes, which nothing else is written to."""
    d, block, heads = 256, 64, 4
    n_blocks = 9 * (1 << 30) // (heads * block * d // 2)
    nbytes = pkg.q4_0_bytes(1, heads, d, block, n_blocks)
    k, v = hip.DeviceBuffer(nbytes), hip.DeviceBuffer(nbytes)
    rng = np.random.default_rng(1)
    table = np.array([[n_blocks - 1, 0, n_blocks - 2]], np.uint32)
    n = 150
    dt, dl, ds = (hip.DeviceBuffer.from_numpy(np.array(x, np.uint32)) for x in (table, [n], [0, n]))
    rows = [rng.normal(0, 1, (n, heads, d)).astype(np.float32) for _ in range(2)]
    dk, dv = (hip.DeviceBuffer.from_numpy(x) for x in rows)
    cache = pkg.KvCache(pkg.Q4_0, 1, heads, d, block, n_blocks, k.ptr, v.ptr)
    seqs = pkg.KvSeqs(1, dt.ptr, 3, dl.ptr, n, ds.ptr, n, n)
    gpu.kv_store_device(cache, seqs, 0, dk.ptr, dv.ptr)
    back = [hip.DeviceBuffer(x.nbytes) for x in rows]
    gpu.kv_load_device(cache, seqs, 0, back[0].ptr, back[1].ptr)
    q = rng.normal(0, 1, (n, 2 * heads, d)).astype(np.float32)
    outs = []
    held = [unpack(*pack(x)).astype(np.float64) for x in rows]
    for few in (False, True):
        dq, do = hip.DeviceBuffer.from_numpy(q), hip.DeviceBuffer(q.nbytes)
        one = pkg.KvSeqs(1, dt.ptr, 3, dl.ptr, n) if few else seqs
        gpu.attn_device(cache, one, 0, 2 * heads, dq.ptr, do.ptr, 1 / 16)
        hip.device_synchronize()
        outs.append(do.to_numpy(np.float32).reshape(q.shape))
    for x, got in zip(held, back):
        assert np.array_equal(got.to_numpy(np.float32).reshape(x.shape), x.astype(np.float32))
    for got, row, seen in ((outs[0], n - 1, n), (outs[1], 0, n), (outs[0], 70, 71)):
        for h in range(2 * heads):
            qr = q[row, h].astype(np.float64)
            s = held[0][:seen, h // 2] @ qr / 16
            p = np.exp(s - s.max())
            p /= p.sum()
            size = (np.abs(held[0][:seen, h // 2]) @ np.abs(qr)).max() / 16
            tol = (2 * (d + 24) * size + seen + 80) * 2.0 ** -23 * (p @ np.abs(held[1][:seen, h // 2]))  # as in paged.py
            assert np.all(np.abs(got[row, h] - p @ held[1][:seen, h // 2]) <= tol)
    for b in (k, v):
        b.free()
