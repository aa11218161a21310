"""Operators over the paged K/V cache on the GPU against their definition in 64 bits (tests/paged.py): types, head layouts,
lengths from none to thousands, windows, tables that name no block, infinities where nobody looks, graphs, streams."""
import importlib

import numpy as np
import pytest

from paged import NOWHERE, Paged, same_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu(pkg):
    g = pkg.HipGemv(0)
    yield g
    g.close()


@pytest.fixture(scope="module")
def hip():
    return importlib.import_module("llama-rust_amd.hiprt")


def attend(gpu, c, layer, q, scale, out=None, q_stride=None, out_stride=None, stream=0, **kw):
    """The call, synchronised; out keeps what it held in rows the call leaves alone."""
    hip = c.hip
    dq = hip.DeviceBuffer.from_numpy(q.astype(np.float32))
    start = np.full(q.shape, 7.25, np.float32) if out is None else out
    do = hip.DeviceBuffer.from_numpy(start)
    gpu.attn_device(c.cache, c.seqs, layer, kw.pop("heads", q.shape[-2]), dq.ptr, do.ptr, scale, q_stride=q_stride, out_stride=out_stride, stream=stream, **kw)
    hip.device_synchronize()
    return do.to_numpy(np.float32).reshape(start.shape)


def check(got, want, tol, what=""):
    assert np.all(np.isfinite(got)), what
    off = np.abs(got.astype(np.float64) - want)
    worst = np.unravel_index(np.argmax(off - tol), off.shape)
    assert np.all(off <= tol), (what, worst, got[worst], want[worst], tol[worst])


LAYOUTS = [(1, 1, 64), (4, 4, 128), (8, 2, 128), (14, 2, 64), (32, 4, 80), (6, 2, 40), (3, 1, 8), (16, 1, 256), (12, 4, 192), (71, 1, 64), (34, 2, 136)]


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("heads,hkv,d", LAYOUTS)
def test_one_token_a_sequence(gpu, f16, heads, hkv, d):
    """Lengths around the tiles' and blocks' ends, a sequence that holds nothing, blocks of sixteen."""
    rng = np.random.default_rng(d + heads)
    c = Paged(rng, f16, 2, hkv, d, 16, [1, 0, 15, 16, 17, 33, 64, 130, 300]).up()
    q = rng.normal(0, 1, (9, heads, d)).astype(np.float32)
    want, tol, _ = c.attend(1, q, d ** -0.5)
    got = attend(gpu, c, 1, q, np.float32(d ** -0.5))
    check(got, want, tol + 1e-7 * np.abs(want))
    assert np.all(got[1] == 0)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("block", [1, 3, 16, 20, 48, 256])
def test_blocks_of_any_size(gpu, f16, block):
    rng = np.random.default_rng(block)
    c = Paged(rng, f16, 3, 2, 64, block, [5, 257, 100]).up()
    q = rng.normal(0, 1, (3, 4, 64)).astype(np.float32)
    want, tol, _ = c.attend(2, q, 0.125)
    check(attend(gpu, c, 2, q, 0.125), want, tol)


@pytest.mark.parametrize("f16", [False, True])
def test_long_sequences_are_shared_and_joined(gpu, f16):
    """Lengths that are cut into many shares, beside one that leaves most shares empty; large scores in one place, so that a row's
    maximum rises late."""
    rng = np.random.default_rng(3)
    c = Paged(rng, f16, 1, 2, 64, 32, [5000, 40, 2999])
    c.k[c.at(0, 4000)] *= 20
    c.k[c.at(2, 3)] *= 20
    c.up()
    q = rng.normal(0, 1, (3, 8, 64)).astype(np.float32)
    want, tol, _ = c.attend(0, q, 0.125)
    check(attend(gpu, c, 0, q, 0.125), want, tol)


RAGGED = [([0, 1, 4, 4, 21, 22], [1, 3, 9, 17, 60]), ([0, 40, 41, 105, 105, 170], [40, 90, 64, 5, 200])]


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("starts,lens", RAGGED)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (7, 0), (7, 3), (40, 4), (1000, 4), (30, 50)])
def test_several_tokens_a_sequence(gpu, f16, starts, lens, window, sinks):
    """Prompts and remainders of any length, one of them without new tokens; causal, in a window, with first tokens."""
    rng = np.random.default_rng(window + sinks)
    c = Paged(rng, f16, 2, 2, 64, 16, lens).up(starts, max_new=int(np.diff(starts).max()))
    q = rng.normal(0, 1, (starts[-1], 6, 64)).astype(np.float32)
    want, tol, _ = c.attend(0, q, 0.125, starts, window, sinks)
    check(attend(gpu, c, 0, q, 0.125, window=window, sinks=sinks), want, tol)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("heads,hkv,d,block", [(4, 4, 128, 16), (8, 1, 256, 20), (10, 2, 96, 16), (40, 2, 40, 7), (9, 1, 192, 64)])
def test_prompts_in_other_layouts(gpu, f16, heads, hkv, d, block):
    rng = np.random.default_rng(d)
    starts = [0, 33, 34, 120]
    c = Paged(rng, f16, 1, hkv, d, block, [33, 50, 150]).up(starts, max_new=86)
    q = rng.normal(0, 1, (120, heads, d)).astype(np.float32)
    for window, sinks in ((0, 0), (20, 4)):
        want, tol, _ = c.attend(0, q, d ** -0.5, starts, window, sinks)
        check(attend(gpu, c, 0, q, np.float32(d ** -0.5), window=window, sinks=sinks), want, tol + 1e-7 * np.abs(want))


@pytest.mark.parametrize("f16", [False, True])
def test_rows_apart_and_rows_of_nobody(gpu, f16):
    """Strides wider than a row; rows before the first sequence and behind the last stay as they were."""
    rng = np.random.default_rng(11)
    starts = [2, 3, 8]
    c = Paged(rng, f16, 1, 2, 64, 16, [30, 44]).up(starts, max_new=5, n_tokens=11)
    q = np.full((11, 300), np.nan, np.float32)
    q[:, :256] = rng.normal(0, 1, (11, 256))
    out = rng.normal(0, 1, (11, 272)).astype(np.float32)
    got = attend(gpu, c, 0, q, 0.125, out=out.copy(), q_stride=300, out_stride=272, heads=4)
    want, tol, _ = c.attend(0, q[:, :256].reshape(11, 4, 64), 0.125, starts)
    check(got[2:8, :256].reshape(6, 4, 64), want[2:8], tol[2:8])
    assert np.array_equal(got[:2], out[:2]) and np.array_equal(got[8:], out[8:]) and np.array_equal(got[:, 256:], out[:, 256:])


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_no_row_sees_reaches_none(gpu, f16, bad):
    """Infinities and NaN behind the length, before the window, in a later token of the same call."""
    rng = np.random.default_rng(5)
    starts = [0, 20, 21]
    c = Paged(rng, f16, 1, 2, 64, 16, [50, 90], garbage=bad)
    for x in (c.k, c.v):
        x[c.at(0, 41)] = bad  # token 11 of the first sequence
        x[c.at(1, 20)] = bad  # outside the second one's window
    c.up(starts, max_new=20)
    q = rng.normal(0, 1, (21, 4, 64)).astype(np.float32)
    got = attend(gpu, c, 0, q, 0.125, window=30, sinks=4)
    want, tol, _ = c.attend(0, q, 0.125, starts, 30, 4)
    check(got[:11], want[:11], tol[:11])
    check(got[20:], want[20:], tol[20:])


@pytest.mark.parametrize("f16", [False, True])
def test_infinities_that_are_seen(gpu, f16):
    """As the definition has them: a score of -infinity counts nothing, all of them leave zeros, an infinite value passes, +infinity and NaN
    in a score are NaN."""
    rng = np.random.default_rng(6)
    c = Paged(rng, f16, 1, 1, 64, 16, [40] * 5)
    q = np.abs(rng.normal(0, 1, (5, 2, 64))).astype(np.float32) + 0.1
    c.k[c.at(0, 7)] = -np.inf
    for t in range(40):
        c.k[c.at(1, t)] = -np.inf
    c.v[c.at(2, 30)] = np.inf
    c.k[c.at(3, 9)] = np.inf
    c.k[c.at(4, 9)] = np.nan
    c.up()
    got = attend(gpu, c, 0, q, 0.125)
    want, tol, _ = c.attend(0, q, 0.125)
    check(got[0], want[0], tol[0])
    assert np.all(got[1] == 0)
    assert np.all(got[2] == np.inf)
    assert np.all(np.isnan(got[3])) and np.all(np.isnan(got[4]))


@pytest.mark.parametrize("f16", [False, True])
def test_scores_of_any_size(gpu, f16):
    """Queries far above and below one: the softmax picks one position, or weighs all alike."""
    rng = np.random.default_rng(8)
    c = Paged(rng, f16, 1, 1, 64, 16, [200] * 6).up()
    q = rng.normal(0, 1, (6, 4, 64)).astype(np.float32) * np.array([1e-38, 1e-30, 1e-3, 30, 1e5, 1e20], np.float32)[:, None, None]
    want, tol, _ = c.attend(0, q, 0.125)
    got = attend(gpu, c, 0, q, 0.125)
    check(got[:4], want[:4], tol[:4])
    assert np.all(np.isfinite(got))


@pytest.mark.parametrize("f16", [False, True])
def test_blocks_that_are_not_there(gpu, f16):
    """Entries of a table that name no block are as if their positions were not; a length beyond max_len and row starts out of order stay in
    bounds."""
    rng = np.random.default_rng(9)
    c = Paged(rng, f16, 2, 2, 64, 16, [70, 16, 120])
    c.tables[0, 1] = c.n_blocks
    c.tables[1, 0] = NOWHERE
    c.tables[2, 3] = 0x80000000
    c.up()
    q = rng.normal(0, 1, (3, 4, 64)).astype(np.float32)
    want, tol, _ = c.attend(1, q, 0.125)
    got = attend(gpu, c, 1, q, 0.125)
    check(got, want, tol)
    assert np.all(got[1] == 0)
    c.lens = np.array([70, 16, 100], np.uint32)
    c.dl.upload(np.array([70, 16, 1 << 30], np.uint32))
    c.seqs.max_len = 100
    want, tol, _ = c.attend(1, q, 0.125)
    check(attend(gpu, c, 1, q, 0.125), want, tol)
    c.up([0, 3, 1, 90], max_new=2, n_tokens=3, max_len=100)
    got = attend(gpu, c, 1, q, 0.125)
    assert np.all(np.isfinite(got))


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("decay", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("starts,lens,window,sinks", [(None, [1, 0, 31, 64, 700], 0, 0), ([0, 40, 41, 105, 105, 170], [40, 90, 64, 5, 200], 0, 0),
                                                       ([0, 3, 60], [90, 57], 25, 4)])
def test_weights_are_summed(gpu, f16, decay, starts, lens, window, sinks):
    rng = np.random.default_rng(len(lens))
    news = np.diff(starts) if starts else [1]
    c = Paged(rng, f16, 2, 2, 64, 16, lens, weights=True).up(starts, max_new=int(max(news)))
    q = rng.normal(0, 1, (starts[-1] if starts else len(lens), 6, 64)).astype(np.float32)
    want, tol, sums = c.attend(1, q, 0.125, starts, window, sinks)
    got = attend(gpu, c, 1, q, 0.125, window=window, sinks=sinks, weights=True, decay=decay)
    check(got, want, tol)
    w, w_tol = c.weigh(1, sums, decay)
    after = c.down()[2]
    held = ~np.isnan(w)
    assert same_bits(after[~held], c.w[~held])
    off = np.abs(after[held] - w[held])
    assert np.all(off <= w_tol[held]), np.max(off - w_tol[held])


def test_weights_do_not_change_the_output(gpu):
    rng = np.random.default_rng(2)
    for starts in (None, [0, 30, 70]):
        c = Paged(rng, True, 1, 2, 64, 16, [300, 500], weights=True).up(starts, max_new=40 if starts else 1)
        q = rng.normal(0, 1, (70 if starts else 2, 8, 64)).astype(np.float32)
        assert np.array_equal(attend(gpu, c, 0, q, 0.125), attend(gpu, c, 0, q, 0.125, weights=True))


@pytest.mark.parametrize("f16", [False, True])
def test_store(gpu, hip, f16):
    """Rows of several sequences with strides of their own, into blocks that exist; nothing else is touched."""
    rng = np.random.default_rng(4)
    starts = [1, 4, 4, 30, 31, 33]
    lens = [5, 9, 40, 1, 1]  # the last has more new tokens than positions
    c = Paged(rng, f16, 2, 3, 40, 7, lens, garbage=-1.0)
    c.tables[2, 3] = c.n_blocks + 5
    c.up(starts, max_new=26, n_tokens=35, max_len=40)
    k, v = rng.normal(0, 1, (35, 124)).astype(np.float32), rng.normal(0, 1, (35, 160)).astype(np.float32)
    k[5, :4] = [1e-9, 65519.0, 65520.0, -1e9]
    k[6, 0], k[6, 1] = np.inf, np.nan
    dk, dv = hip.DeviceBuffer.from_numpy(k), hip.DeviceBuffer.from_numpy(v)
    gpu.kv_store_device(c.cache, c.seqs, 1, dk.ptr, dv.ptr, k_stride=124, v_stride=160)
    hip.device_synchronize()
    want_k, want_v = c.k.copy(), c.v.copy()
    with np.errstate(over="ignore"):
        for b, (n0, n1) in enumerate(zip(starts, starts[1:])):
            for i in range(n1 - n0):
                t = lens[b] - (n1 - n0) + i
                if t < 0 or not c.there(b, t):
                    continue
                want_k[c.tables[b, t // 7], 1, :, t % 7] = k[n0 + i, :120].reshape(3, 40).astype(want_k.dtype)
                want_v[c.tables[b, t // 7], 1, :, t % 7] = v[n0 + i, :120].reshape(3, 40).astype(want_v.dtype)
    got_k, got_v, _ = c.down()
    assert same_bits(got_k, want_k) and same_bits(got_v, want_v)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("keep,first,recent", [(40, 4, 8), (40, 0, 0), (40, 20, 20), (1, 0, 0), (1, 0, 1), (0, 0, 0), (129, 4, 100), (5000, 4, 4)])
def test_eviction(gpu, hip, f16, in_place, keep, first, recent):
    """Lengths below, at and above the budget; ties, zeros of both signs, infinities and NaN among the weights; a block missing."""
    rng = np.random.default_rng(keep + first)
    lens = [1, 0, 39, 40, 41, 128, 300, 3000]
    c = Paged(rng, f16, 3, 2, 40, 16, lens, weights=True, garbage=-3.0, extra_blocks=sum(-(-min(n, keep) // 16) for n in lens))
    for t in range(0, 300, 3):
        c.w[c.at(6, t)] = np.float32(0.5)
    for t, x in ((10, np.nan), (11, np.inf), (12, -0.0), (13, 0.0), (14, -1.0), (15, -np.inf), (16, np.float32(1e-42))):
        c.w[c.at(5, t)] = x
    c.w[c.at(7, 0)] = 0
    for t in range(500, 2500):
        c.w[c.at(7, t)] = np.float32(rng.integers(0, 3))
    c.tables[6, 5] = NOWHERE
    dst, at = None, 0
    if not in_place:
        stride = max(1, -(-min(keep, 3000) // 16))
        dst = np.full((len(lens), stride), NOWHERE, np.uint32)
        for b, n in enumerate(lens):
            pages = -(-min(n, keep) // 16)
            dst[b, :pages] = c.free[at:at + pages]
            at += pages
    c.up()
    dd = hip.DeviceBuffer.from_numpy(dst) if dst is not None else None
    new = c.dl if in_place else hip.DeviceBuffer(4 * len(lens))
    gpu.kv_evict_device(c.cache, c.seqs, 1, 2, keep, first, recent, dd.ptr if dd else 0, dst.shape[1] if dd else 0, new.ptr)
    hip.device_synchronize()
    want_len, k, v, w = c.evict([1, 2], keep, first, recent, dst)
    got_k, got_v, got_w = c.down()
    assert np.array_equal(new.to_numpy(np.uint32), want_len)
    if in_place:  # what lies behind the new lengths may be anything that was there
        for b, n in enumerate(want_len.astype(int)):
            for t in range(n):
                if c.there(b, t):
                    at = c.at(b, t)
                    assert same_bits(got_k[at], k[at]) and same_bits(got_v[at], v[at]) and same_bits(got_w[at], w[at]), (b, t)
        assert same_bits(got_k[:, 0], c.k[:, 0]) and same_bits(got_w[c.free], c.w[c.free])
    assert same_bits(got_k, k) and same_bits(got_v, v) and same_bits(got_w, w)


def test_a_cache_of_more_than_four_gigabytes(gpu, hip, pkg):
    """Rows whose offset does not fit 32 bits, in elements or bytes."""
    rng = np.random.default_rng(1)
    d, block, n_blocks = 256, 64, 300000  # 4.9e9 elements
    size = n_blocks * block * d * 2
    dk, dv, dw = hip.DeviceBuffer(size), hip.DeviceBuffer(size), hip.DeviceBuffer(n_blocks * block * 4)
    table = np.array([[299999, 3, 280001, 270000]], np.uint32)
    dt, dl = hip.DeviceBuffer.from_numpy(table), hip.DeviceBuffer.from_numpy(np.array([180], np.uint32))
    cache = pkg.KvCache(pkg.F16, 1, 1, d, block, n_blocks, dk.ptr, dv.ptr, dw.ptr)
    starts = hip.DeviceBuffer.from_numpy(np.array([0, 180], np.uint32))
    seqs = pkg.KvSeqs(1, dt.ptr, 4, dl.ptr, 180, starts.ptr, 180, 180)
    k, v, q = (rng.normal(0, 1, (180, d)).astype(np.float32) for _ in range(3))
    bk, bv, bq = (hip.DeviceBuffer.from_numpy(x) for x in (k, v, q))
    gpu.kv_store_device(cache, seqs, 0, bk.ptr, bv.ptr)
    out = hip.DeviceBuffer(180 * d * 4)
    gpu.attn_device(cache, seqs, 0, 1, bq.ptr, out.ptr, 0.0625, weights=True, decay=0.0)
    hip.device_synchronize()
    k16, v16 = k.astype(np.float16).astype(np.float64), v.astype(np.float16).astype(np.float64)
    s = np.where(np.tri(180, dtype=bool), (q.astype(np.float64) @ k16.T) * 0.0625, -np.inf)
    p = np.exp(s - s.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    size = (np.abs(q) @ np.abs(k16).T).max() * 0.0625
    rel = (2 * (d + 24) * size + 260) * 2.0 ** -23
    check(out.to_numpy(np.float32).reshape(180, d), p @ v16, rel * (p @ np.abs(v16)))
    new = hip.DeviceBuffer(4)
    gpu.kv_evict_device(cache, seqs, 0, 1, 60, 4, 16, 0, 0, new.ptr)
    one = pkg.KvSeqs(1, dt.ptr, 4, new.ptr, 60)
    gpu.attn_device(cache, one, 0, 1, bq.ptr, out.ptr, 0.0625)
    hip.device_synchronize()
    assert new.to_numpy(np.uint32)[0] == 60
    w = p.sum(0)
    order = np.argsort(-w[4:164], kind="stable")
    assert w[4 + order[39]] - w[4 + order[40]] > 1e-4 * w[4 + order[39]]  # the weights' own error decides nothing here
    stays = np.concatenate([np.arange(4), np.sort(4 + order[:40]), np.arange(164, 180)])
    s = (q[:1].astype(np.float64) @ k16[stays].T) * 0.0625
    p = np.exp(s - s.max())
    p /= p.sum()
    check(out.to_numpy(np.float32)[:d][None], p @ v16[stays], rel * (p @ np.abs(v16[stays])))


def test_a_decode_loop_with_an_eviction(gpu, hip):
    """Prompt, tokens one at a time, a cut, tokens again: store, attention with weights and eviction as a program chains them, on a stream of
    its own, against the definition step by step."""
    rng = np.random.default_rng(12)
    lens0 = [20, 1, 33]
    c = Paged(rng, True, 1, 2, 64, 16, lens0, room=40, weights=True, garbage=0.0)
    stream = hip.Stream()

    def step(news, lens):
        starts = np.concatenate([[0], np.cumsum(news)])
        n, q = int(starts[-1]), rng.normal(0, 1, (int(starts[-1]), 4, 64)).astype(np.float32)
        k, v = (rng.normal(0, 1, (n, 2, 64)).astype(np.float32) for _ in range(2))
        c.lens = np.array(lens, np.uint32)
        c.up(starts, max_new=int(max(news)), max_len=int(max(lens)))
        bk, bv = hip.DeviceBuffer.from_numpy(k), hip.DeviceBuffer.from_numpy(v)
        hip.device_synchronize()
        gpu.kv_store_device(c.cache, c.seqs, 0, bk.ptr, bv.ptr, stream=stream.ptr)
        for b in range(len(lens)):
            for i in range(news[b]):
                at = c.at(b, lens[b] - news[b] + i)
                row = starts[b] + i
                c.k[at[0], 0, :, at[3]], c.v[at[0], 0, :, at[3]] = k[row].astype(np.float16), v[row].astype(np.float16)
        got = attend(gpu, c, 0, q, 0.125, stream=stream.ptr, weights=True, decay=1.0)
        want, tol, sums = c.attend(0, q, 0.125, starts)
        check(got, want, tol)
        w, w_tol = c.weigh(0, sums, 1.0)
        got_k, got_v, got_w = c.down()
        assert same_bits(got_k, c.k) and same_bits(got_v, c.v)
        assert np.all(np.abs(got_w - w) <= w_tol)
        c.w = got_w  # what later steps add to, and the cut goes by

    step(lens0, lens0)
    lens = list(lens0)
    for _ in range(6):
        lens = [n + 1 for n in lens]
        step([1, 1, 1], lens)
    c.up(max_len=max(lens))
    hip.device_synchronize()
    gpu.kv_evict_device(c.cache, c.seqs, 0, 1, 16, 2, 5, 0, 0, c.dl.ptr, stream=stream.ptr)
    stream.synchronize()
    new, c.k, c.v, c.w = c.evict([0], 16, 2, 5)
    assert np.array_equal(c.dl.to_numpy(np.uint32), new)
    assert all(same_bits(x, y) for x, y in zip(c.down(), (c.k, c.v, c.w)))
    lens = [int(n) for n in new]
    for _ in range(3):
        lens = [n + 1 for n in lens]
        step([1, 1, 1], lens)
    stream.destroy()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("new", [1, 24])
def test_a_captured_step_follows_its_arrays(gpu, hip, f16, new):
    """Store, attention with weights and eviction in one graph, replayed with other lengths, tables and values; every replay equals the
    eager calls bit for bit."""
    rng = np.random.default_rng(21)
    starts = [0, new, 2 * new] if new > 1 else None
    c = Paged(rng, f16, 1, 2, 64, 16, [640, 500], room=16, weights=True, garbage=0.0)
    c.up(starts, max_new=new, max_len=656)
    bk, bv, bq, bo, bn = (hip.DeviceBuffer(2 * new * n * 4) for n in (128, 128, 256, 256, 1))
    stream = hip.Stream()

    def enqueue(s):
        gpu.kv_store_device(c.cache, c.seqs, 0, bk.ptr, bv.ptr, stream=s.ptr)
        gpu.attn_device(c.cache, c.seqs, 0, 4, bq.ptr, bo.ptr, 0.125, weights=True, decay=0.5, stream=s.ptr)
        gpu.kv_evict_device(c.cache, c.seqs, 0, 1, 300, 4, 32, 0, 0, bn.ptr, stream=s.ptr)

    def fill():
        c.dk.upload(c.k), c.dv.upload(c.v), c.dw.upload(c.w)

    enqueue(stream)  # sizes the workspace
    stream.synchronize()
    graph = hip.Graph(stream, enqueue)
    for lens in ([640, 500], [33, 656], [new, 301], [650, 40]):
        order = rng.permutation(2)
        tables = c.tables[order]
        rows = [rng.normal(0, 1, 2 * new * n).astype(np.float32) for n in (128, 128, 256)]
        got = []
        for run in (enqueue, lambda s: graph.launch(), enqueue, lambda s: graph.launch()):
            fill()
            c.dt.upload(tables), c.dl.upload(np.array(lens, np.uint32))
            for b, x in zip((bk, bv, bq), rows):
                b.upload(x)
            hip.device_synchronize()
            run(stream)
            stream.synchronize()
            got.append([bo.to_numpy(np.float32), bn.to_numpy(np.uint32, 2)] + list(c.down()))
        for other in got[1:]:
            assert all(np.array_equal(x.view(np.uint8), y.view(np.uint8)) for x, y in zip(got[0], other)), lens
        assert got[0][1].tolist() == [min(n, 300) for n in lens]
    graph.destroy()
    stream.destroy()


def test_growing_inside_a_capture_is_refused(pkg, hip):
    g = pkg.HipGemv(0)
    rng = np.random.default_rng(0)
    c = Paged(rng, False, 1, 1, 64, 16, [2000], weights=True, garbage=0.0).up()
    q, o = hip.DeviceBuffer(256), hip.DeviceBuffer(256)
    stream = hip.Stream()
    hip.device_synchronize()
    with pytest.raises(pkg.NativeHipError, match="while the stream is being captured: run the largest call once before capturing"):
        hip.Graph(stream, lambda s: g.attn_device(c.cache, c.seqs, 0, 1, q.ptr, o.ptr, 0.125, weights=True, stream=s.ptr))
    g.attn_device(c.cache, c.seqs, 0, 1, q.ptr, o.ptr, 0.125, weights=True, stream=stream.ptr)  # the executor is as usable as before
    stream.synchronize()
    stream.destroy()
    g.close()


def test_refusals_name_their_reason_and_touch_nothing(gpu, hip, pkg):
    rng = np.random.default_rng(0)
    c = Paged(rng, True, 2, 2, 64, 16, [30], weights=True, garbage=0.0).up()
    b = hip.DeviceBuffer.from_numpy(np.full(1024, 5, np.float32))
    o = hip.DeviceBuffer.from_numpy(np.full(1024, 5, np.float32))

    def attn(layer=0, heads=4, q=b.ptr, out=o.ptr, **kw):
        gpu.attn_device(c.cache, c.seqs, layer, heads, q, out, 0.125, **kw)

    for match, call in (("no such layer", lambda: attn(layer=2)), ("multiple of the key-value heads", lambda: attn(heads=3)),
                        ("buffer pointer is null", lambda: attn(q=0)), ("16-byte aligned", lambda: attn(out=o.ptr + 4)),
                        ("less than the row", lambda: attn(q_stride=252)), ("multiples of four", lambda: attn(out_stride=259)),
                        ("must not be the input", lambda: attn(out=b.ptr)), ("sinks without one", lambda: attn(sinks=4)),
                        ("scale and decay", lambda: attn(weights=True, decay=float("nan"))),
                        ("exceed those to keep", lambda: gpu.kv_evict_device(c.cache, c.seqs, 0, 1, 5, 3, 3, 0, 0, o.ptr)),
                        ("no such layers", lambda: gpu.kv_evict_device(c.cache, c.seqs, 1, 2, 5, 3, 2, 0, 0, o.ptr)),
                        ("do not hold what is kept", lambda: gpu.kv_evict_device(c.cache, c.seqs, 0, 1, 17, 3, 2, b.ptr, 1, o.ptr)),
                        ("no such layer", lambda: gpu.kv_store_device(c.cache, c.seqs, 2, b.ptr, b.ptr))):
        with pytest.raises(pkg.NativeHipError, match=match) as e:
            call()
        assert e.value.code == pkg.ERR_INVALID
    c.cache.ggml_type = pkg.Q8_0
    with pytest.raises(pkg.NativeHipError, match="f32 or f16") as e:
        attn()
    assert e.value.code == pkg.ERR_UNSUPPORTED
    hip.device_synchronize()
    assert np.all(o.to_numpy(np.float32) == 5)
    assert all(same_bits(x, y) for x, y in zip(c.down(), (c.k, c.v, c.w)))


def test_nothing_to_do_is_done(gpu, hip, pkg):
    """No sequence, no token, no position: the calls succeed."""
    rng = np.random.default_rng(0)
    c = Paged(rng, False, 1, 1, 64, 16, [30], weights=True, garbage=0.0).up()
    none = pkg.KvSeqs(0, 0, 2, 0, 0, n_tokens=0)
    gpu.kv_store_device(c.cache, none, 0, 0, 0)
    gpu.attn_device(c.cache, none, 0, 1, 0, 0, 0.125)
    gpu.kv_evict_device(c.cache, none, 0, 1, 5, 0, 0, 0, 0, 0)
    c.dl.upload(np.array([0], np.uint32))
    c.seqs.max_len = 0
    out = attend(gpu, c, 0, np.ones((1, 2, 64), np.float32), 0.125, weights=True)
    assert np.all(out == 0)
    assert all(same_bits(x, y) for x, y in zip(c.down(), (c.k, c.v, c.w)))


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("block", [16, 7])
def test_more_sequences_and_heads_than_compute_units(gpu, f16, block):
    """Sequences of any length among 300, whose units alone are more than one round; every fifth holds nothing, every seventh is long."""
    rng = np.random.default_rng(block)
    lens = [0 if i % 5 == 4 else int(rng.integers(200, 400)) if i % 7 == 3 else int(rng.integers(1, 30)) for i in range(300)]
    c = Paged(rng, f16, 1, 1, 16, block, lens, weights=True).up()
    q = rng.normal(0, 1, (300, 2, 16)).astype(np.float32)
    want, tol, sums = c.attend(0, q, 0.25)
    check(attend(gpu, c, 0, q, 0.25, weights=True), want, tol)
    w, w_tol = c.weigh(0, sums, 1.0)
    after = c.down()[2]
    held = ~np.isnan(w)
    assert same_bits(after[~held], c.w[~held]) and np.all(np.abs(after[held] - w[held]) <= w_tol[held])


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("heads,hkv,d,new,lens,window,sinks", [
    (20, 1, 64, 1, [1500, 3, 900], 0, 0),      # two tiles of rows of one token
    (4, 2, 128, 13, [1300, 13, 400], 0, 0),    # 26 rows a key-value head
    (4, 2, 128, 13, [1300, 13, 400], 300, 20),
    (8, 2, 64, 80, [1100, 80], 0, 0),          # blocks of rows that share their steps
    (8, 2, 64, 80, [1100, 80], 500, 3),
    (4, 1, 200, 40, [700, 41], 0, 0),
    (2, 1, 128, 300, [900, 310], 0, 0),        # several blocks of rows, the last of them short
    (2, 1, 128, 300, [900, 310], 128, 64),
])
def test_rows_and_positions_are_cut(gpu, f16, heads, hkv, d, new, lens, window, sinks):
    """Between the smallest and the largest variants, with the weights: tokens of several sequences behind long histories."""
    rng = np.random.default_rng(new + d)
    starts = [new * i for i in range(len(lens) + 1)]
    c = Paged(rng, f16, 1, hkv, d, 16, lens, weights=True).up(starts, max_new=new)
    q = rng.normal(0, 1, (starts[-1], heads, d)).astype(np.float32)
    want, tol, sums = c.attend(0, q, d ** -0.5, starts, window, sinks)
    check(attend(gpu, c, 0, q, np.float32(d ** -0.5), window=window, sinks=sinks, weights=True, decay=0.75), want, tol + 1e-7 * np.abs(want))
    w, w_tol = c.weigh(0, sums, 0.75)
    after = c.down()[2]
    held = ~np.isnan(w)
    assert same_bits(after[~held], c.w[~held])
    off = np.abs(after[held] - w[held])
    assert np.all(off <= w_tol[held] + 2e-7 * w[held]), np.max(off - w_tol[held])


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_weights_of_many_rows_beside_what_is_not_finite(gpu, f16, bad):
    """A key that is infinite or NaN at a late position: the tokens before it and their sums do not know of it."""
    rng = np.random.default_rng(31)
    c = Paged(rng, f16, 1, 1, 64, 16, [200], weights=True)
    c.w[:] = 0
    c.k[c.tables[0, 150 // 16], 0, 0, 150 % 16, 3] = bad
    c.up([0, 150], max_new=150)
    q = rng.normal(0, 1, (150, 1, 64)).astype(np.float32)
    q[:, 0, 3] = np.abs(q[:, 0, 3]) + 0.5
    got = attend(gpu, c, 0, q, 0.125, weights=True)
    after = c.down()[2]
    # tokens stand at 50 ..: those before 150 are as without the position, those from it see it
    clean = Paged(np.random.default_rng(31), f16, 1, 1, 64, 16, [200], weights=True)
    want, tol, _ = clean.attend(0, q, 0.125, [0, 150])
    check(got[:100], want[:100], tol[:100])
    if bad == -np.inf:  # a score of minus infinity is a position without weight
        assert np.all(np.isfinite(got)) and np.all(np.isfinite(after))
        assert after[c.tables[0, 9], 0, 0, 6] == 0
        assert abs(after.sum() - 150) < 1e-3
    else:
        assert np.all(np.isnan(got[100:]))
        seen = [after[c.tables[0, t // 16], 0, 0, t % 16] for t in range(200)]
        assert np.all(np.isnan(seen[:151]))  # a row of NaN gives every position it sees one


@pytest.mark.parametrize("in_place", [False, True])
def test_eviction_of_a_middle_beyond_one_block_of_keys(gpu, hip, in_place):
    """40000 positions, most weights equal to another's: the earliest of the equal ones stay."""
    rng = np.random.default_rng(6)
    lens, keep = [40000, 16500, 17000], 16400
    c = Paged(rng, True, 1, 1, 8, 64, lens, garbage=0, weights=True, extra_blocks=3 * 257)
    c.w[:] = rng.integers(0, 50, c.w.shape).astype(np.float32)
    for t in range(0, 40000, 3):
        c.w[c.at(0, t)] = np.float32(rng.exponential(30))
    c.up()
    dst = c.free[:3 * 257].reshape(3, 257).astype(np.uint32)
    dd, new = hip.DeviceBuffer.from_numpy(dst), hip.DeviceBuffer(12)
    gpu.kv_evict_device(c.cache, c.seqs, 0, 1, keep, 4, 100, 0 if in_place else dd.ptr, 0 if in_place else 257, new.ptr)
    hip.device_synchronize()
    want_len, k, v, w = c.evict([0], keep, 4, 100, None if in_place else dst)
    assert new.to_numpy(np.uint32).tolist() == want_len.tolist()
    for got, want in zip(c.down(), (k, v, w)):
        assert same_bits(got, want)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("d,hkv,layers", [(8, 1, 1), (40, 3, 2), (104, 1, 1), (128, 2, 1), (256, 1, 1)])
def test_eviction_in_place_in_strips(gpu, hip, f16, d, hkv, layers):
    """Rows of any size move forward past the end of a strip of rows; nothing to move at the front, everything behind it."""
    rng = np.random.default_rng(d)
    lens = [2600, 1100]
    c = Paged(rng, f16, layers, hkv, d, 16, lens, garbage=-2.0, weights=True).up()
    gpu.kv_evict_device(c.cache, c.seqs, 0, layers, 2100, 0, 0, 0, 0, c.dl.ptr)
    hip.device_synchronize()
    want_len, k, v, w = c.evict(range(layers), 2100, 0, 0)
    assert c.dl.to_numpy(np.uint32).tolist() == want_len.tolist()
    for got, want in zip(c.down(), (k, v, w)):
        assert same_bits(got, want)


def test_two_executors_at_once(pkg, hip):
    """Calls on streams of two executors, each with its own workspace, none waited for: the results of each alone."""
    rng = np.random.default_rng(17)
    made = []
    for f16, heads, lens in ((True, 8, [3000, 20, 700]), (False, 4, [100, 2500])):
        g, stream = pkg.HipGemv(0), hip.Stream()
        c = Paged(rng, f16, 1, 2, 64, 16, lens, weights=True, garbage=0).up()
        q = rng.normal(0, 1, (len(lens), heads, 64)).astype(np.float32)
        dq, outs = hip.DeviceBuffer.from_numpy(q), [hip.DeviceBuffer(q.nbytes) for _ in range(21)]
        made.append((g, stream, c, heads, dq, outs))
    hip.device_synchronize()

    def run(i, k):
        g, stream, c, heads, dq, outs = made[i]
        g.attn_device(c.cache, c.seqs, 0, heads, dq.ptr, outs[k].ptr, 0.125, weights=True, decay=0.5, stream=stream.ptr)

    for i in range(2):
        run(i, 20)
        hip.device_synchronize()
    for k in range(20):
        for i in range(2):
            run(i, k)
    hip.device_synchronize()
    for g, stream, c, heads, dq, outs in made:
        want = outs[20].to_numpy(np.float32)
        assert np.all(np.isfinite(want))
        for o in outs[:20]:
            assert np.array_equal(o.to_numpy(np.float32), want)
        stream.destroy()
        g.close()


def test_calls_larger_than_a_launch_are_refused(gpu, hip, pkg):
    """Sizes whose products pass 32 and 64 bits: refused by their numbers, with nothing launched."""
    rng = np.random.default_rng(0)
    c = Paged(rng, True, 1, 1, 64, 16, [20, 20], weights=True, garbage=0).up([0, 1, 2])
    q, out = hip.DeviceBuffer(1 << 16), hip.DeviceBuffer(1 << 16)
    out.fill_byte(0x11)
    hip.device_synchronize()
    for n_seqs, n_tokens, max_new, heads in ((1 << 23, 1 << 20, 1, 1), ((1 << 31) - 4096, 64, 64, 1), ((1 << 31) - 4096, (1 << 31) - 4096, (1 << 31) // 65536 - 1, 65536),
                                             (1, (1 << 31) - 4096, (1 << 31) - 4096, 1)):
        seqs = pkg.KvSeqs(n_seqs, c.dt.ptr, c.stride, c.dl.ptr, 20, c.ds.ptr, n_tokens, max_new)
        for weights in (False, True):
            with pytest.raises(pkg.NativeHipError, match="larger than one launch"):
                gpu.attn_device(c.cache, seqs, 0, heads, q.ptr, out.ptr, 0.125, weights=weights)
    many = pkg.KvSeqs(1 << 23, c.dt.ptr, c.stride, c.dl.ptr, 20, c.ds.ptr, 64, 1)
    with pytest.raises(pkg.NativeHipError, match="larger than one launch"):
        gpu.kv_store_device(c.cache, many, 0, q.ptr, q.ptr)
    with pytest.raises(pkg.NativeHipError, match="larger than one launch"):
        gpu.kv_evict_device(c.cache, many, 0, 1, 4, 0, 0, 0, 0, c.dl.ptr)
    hip.device_synchronize()
    assert np.all(out.to_numpy(np.uint8) == 0x11) and np.array_equal(c.dl.to_numpy(np.uint32), c.lens)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("heads,hkv,d,block,window,sinks", [(4, 4, 128, 16, 0, 0), (8, 1, 256, 20, 0, 0), (10, 2, 96, 16, 40, 2), (40, 2, 40, 7, 0, 0), (9, 1, 192, 64, 33, 0),
                                                            (2, 1, 8, 3, 0, 0), (6, 3, 136, 16, 0, 0)])
def test_weights_and_long_shares_in_other_layouts(gpu, f16, heads, hkv, d, block, window, sinks):
    """A prompt, a remainder behind a long history (many shares) and one token beside them, with the weights."""
    rng = np.random.default_rng(d + block)
    starts, lens = [0, 70, 75, 76], [90, 1500, 33]
    c = Paged(rng, f16, 1, hkv, d, block, lens, weights=True).up(starts, max_new=70)
    q = rng.normal(0, 1, (76, heads, d)).astype(np.float32)
    want, tol, sums = c.attend(0, q, d ** -0.5, starts, window, sinks)
    check(attend(gpu, c, 0, q, np.float32(d ** -0.5), window=window, sinks=sinks, weights=True, decay=1.0), want, tol + 1e-7 * np.abs(want))
    w, w_tol = c.weigh(0, sums, 1.0)
    after = c.down()[2]
    held = ~np.isnan(w)
    assert same_bits(after[~held], c.w[~held])
    off = np.abs(after[held] - w[held])
    assert np.all(off <= w_tol[held] + 2e-7 * w[held]), np.max(off - w_tol[held])


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("tokens", [1, 5, 16, 40])
def test_few_tokens_behind_a_long_history(gpu, f16, tokens):
    """Of one sequence: as many shares as the chip holds, joined side by side."""
    rng = np.random.default_rng(tokens)
    c = Paged(rng, f16, 1, 1, 128, 16, [9000]).up([0, tokens], max_new=tokens)
    q = rng.normal(0, 1, (tokens, 4, 128)).astype(np.float32)
    want, tol, _ = c.attend(0, q, 128 ** -0.5, [0, tokens])
    check(attend(gpu, c, 0, q, np.float32(128 ** -0.5)), want, tol + 1e-7 * np.abs(want))


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("n", [20, 33, 64])
def test_one_long_sequence_among_short_ones(gpu, f16, n):
    """Units that nearly fill, just pass and far pass the compute units, one of them with most of the positions."""
    rng = np.random.default_rng(n)
    lens = [40 + i for i in range(n)]
    lens[n // 2], lens[1] = 6000, 1
    c = Paged(rng, f16, 1, 8, 16, 16, lens, weights=True).up()
    q = rng.normal(0, 1, (n, 8, 16)).astype(np.float32)
    want, tol, sums = c.attend(0, q, 0.25)
    check(attend(gpu, c, 0, q, 0.25, weights=True), want, tol)
    w, w_tol = c.weigh(0, sums, 1.0)
    after = c.down()[2]
    held = ~np.isnan(w)
    assert np.all(np.abs(after[held] - w[held]) <= w_tol[held])


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("new", [1, 40])
def test_sequences_that_share_blocks(gpu, hip, f16, new):
    """A common beginning in the same blocks: attention reads them for both, and an eviction into other blocks takes from them twice."""
    rng = np.random.default_rng(41 + new)
    c = Paged(rng, f16, 1, 2, 64, 16, [320, 200], weights=True, extra_blocks=2 * 8)
    c.tables[1, :10] = c.tables[0, :10]  # 160 positions
    starts = [0, new, 2 * new]
    c.up(starts if new > 1 else None, max_new=new)
    q = rng.normal(0, 1, (2 * new, 4, 64)).astype(np.float32)
    want, tol, _ = c.attend(0, q, 0.125, starts)
    check(attend(gpu, c, 0, q, 0.125), want, tol)
    dst = c.free[:16].reshape(2, 8).astype(np.uint32)
    dd, out = hip.DeviceBuffer.from_numpy(dst), hip.DeviceBuffer(8)
    gpu.kv_evict_device(c.cache, c.seqs, 0, 1, 128, 4, 16, dd.ptr, 8, out.ptr)
    hip.device_synchronize()
    want_len, k, v, w = c.evict([0], 128, 4, 16, dst)
    assert out.to_numpy(np.uint32).tolist() == want_len.tolist()
    for got, want in zip(c.down(), (k, v, w)):
        assert same_bits(got, want)


@pytest.mark.parametrize("f16", [False, True])
def test_a_captured_call_follows_its_row_starts(gpu, hip, f16):
    """Many rows, with weights, replayed with other starts and lengths: rows of nobody stay as they are, the others equal the eager call."""
    rng = np.random.default_rng(51)
    c = Paged(rng, f16, 1, 2, 64, 16, [640, 500, 90], weights=True, garbage=0.0).up([0, 24, 48, 72], max_new=40, n_tokens=80, max_len=640)
    q, stream = hip.DeviceBuffer.from_numpy(rng.normal(0, 1, (80, 8, 64)).astype(np.float32)), hip.Stream()
    out = hip.DeviceBuffer(80 * 8 * 64 * 4)
    hip.device_synchronize()

    def enqueue(s):
        gpu.attn_device(c.cache, c.seqs, 0, 8, q.ptr, out.ptr, 0.125, weights=True, decay=0.5, stream=s.ptr)

    enqueue(stream)
    stream.synchronize()
    graph = hip.Graph(stream, enqueue)
    for starts, lens in (([0, 24, 48, 72], [640, 500, 90]), ([3, 3, 43, 44], [640, 77, 90]), ([0, 40, 80, 80], [40, 499, 1]), ([10, 10, 10, 10], [1, 1, 1]), ([79, 80, 80, 80], [600, 0, 0])):
        got = []
        for run in (enqueue, lambda s: graph.launch(), enqueue, lambda s: graph.launch()):
            c.ds.upload(np.array(starts, np.uint32)), c.dl.upload(np.array(lens, np.uint32)), c.dw.upload(c.w)
            out.fill_byte(0x22)
            hip.device_synchronize()
            run(stream)
            stream.synchronize()
            got.append((out.to_numpy(np.uint32).reshape(80, -1), c.down()[2].view(np.uint32)))
        for o, w in got[1:]:
            assert np.array_equal(o, got[0][0]) and np.array_equal(w, got[0][1]), starts
        mine = np.zeros(80, bool)
        mine[starts[0]:starts[-1]] = True
        assert np.all(got[0][0][~mine] == 0x22222222) and np.all(np.any(got[0][0][mine] != 0x22222222, axis=1))
    graph.destroy()
    stream.destroy()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("d,block", [(40, 16), (80, 7), (96, 16), (136, 16), (64, 16)])
@pytest.mark.parametrize("new", [1, 3])
def test_weights_of_few_rows_beside_keys_of_minus_infinity(gpu, f16, d, block, new):
    """A key whose first element is -infinity against positive queries scores -infinity: it counts nothing and gets weight 0, the
    others what the softmax without it gives them - also where the head ends inside a lane's piece and the first one is read instead."""
    rng = np.random.default_rng(d + new)
    heads, n, out_of = 4, 50, (3, 20, 44)
    c = Paged(rng, f16, 1, 1, d, block, [n, n], weights=True, garbage=0.0)
    for t in out_of:
        c.k[c.tables[0, t // block], 0, 0, t % block, 0] = -np.inf
    c.up([0, new, 2 * new] if new > 1 else None, max_new=new)
    q = rng.normal(0, 1, (2 * new, heads, d)).astype(np.float32)
    q[:, :, 0] = np.abs(q[:, :, 0]) + 0.5
    got = attend(gpu, c, 0, q, np.float32(d ** -0.5), weights=True, decay=0.5)
    after = c.down()[2]
    for b in range(2):
        k, v = (np.array([x[c.tables[b, t // block], 0, 0, t % block] for t in range(n)], np.float64) for x in (c.k, c.v))
        want, tol = np.zeros(n), np.zeros(n)
        for i in range(new):
            seen = np.array([t for t in range(n - new + i + 1) if b == 1 or t not in out_of])
            for h in range(heads):
                qr = q[b * new + i, h].astype(np.float64)
                s = k[seen] @ qr * float(np.float32(d ** -0.5))
                p = np.exp(s - s.max())
                p /= p.sum()
                # as Paged.attend and Paged.weigh have them
                rel = (2 * (d + 24) * (np.abs(k[seen]) @ np.abs(qr)).max() * d ** -0.5 + len(seen) + 80) * 2.0 ** -23
                assert np.all(np.abs(got[b * new + i, h] - p @ v[seen]) <= rel * (p @ np.abs(v[seen])) + 1e-37), (b, i, h)
                want[seen] += p
                tol[seen] += (rel + new * heads * 2.0 ** -23) * p + 2.0 ** -120
        for t in range(n):
            at = c.tables[b, t // block], 0, 0, t % block
            total = 0.5 * float(c.w[at]) + want[t]
            assert abs(after[at] - total) <= tol[t] + 2 * 2.0 ** -24 * total, (b, t, after[at], total)


@pytest.mark.parametrize("heads,d,new,lens", [(4, 64, 1, [200, 4, 3000]), (2, 40, 1, [77, 1]), (4, 128, 20, [300, 25]), (8, 64, 40, [1200, 41]), (2, 200, 30, [100, 30])])
def test_values_whose_sum_passes_f32(gpu, heads, d, new, lens):
    """Values near the largest f32: their weighted sum before it is divided is beyond it, their mean is not."""
    rng = np.random.default_rng(d + new)
    starts = [new * i for i in range(len(lens) + 1)]
    c = Paged(rng, False, 1, 1, d, 16, lens, weights=True)
    held = ~np.isnan(c.v)
    c.v[held] = (np.clip(c.v[held].astype(np.float64) * 4e37 + 2e38, -3.2e38, 3.2e38)).astype(np.float32)
    c.up(starts if new > 1 else None, max_new=new)
    q = rng.normal(0, 1, (starts[-1], heads, d)).astype(np.float32)
    want, tol, sums = c.attend(0, q, d ** -0.5, starts)
    got = attend(gpu, c, 0, q, np.float32(d ** -0.5), weights=True, decay=1.0)
    check(got, want, tol + 1e-7 * np.abs(want))
    w, w_tol = c.weigh(0, sums, 1.0)
    after = c.down()[2]
    held = ~np.isnan(w)
    assert np.all(np.abs(after[held] - w[held]) <= w_tol[held] + 2e-7 * w[held])


@pytest.mark.parametrize("d", [64, 40, 200])
@pytest.mark.parametrize("new,lens", [(1, [300, 9, 2000]), (30, [400, 30, 77])])
def test_products_beyond_f32_whose_scores_are_not(gpu, d, new, lens):
    """q k over an f32 cache passes the largest f32 for about every other position, scale q k is a few units: no score is lost to an
    infinity of either sign before the scale comes to it."""
    rng = np.random.default_rng(d + new)
    starts = [new * i for i in range(len(lens) + 1)]
    c = Paged(rng, False, 1, 1, d, 16, lens, weights=True)
    c.k *= np.float32(6e17)
    c.up(starts if new > 1 else None, max_new=new)
    q = rng.normal(0, 1, (starts[-1], 4, d)).astype(np.float32) * np.float32(1e20)
    scale = np.float32(1.2e-38)
    assert np.mean(np.abs(q[:, 0].astype(np.float64) @ c.k[c.at(0, 0)][0, 0].astype(np.float64)) > 3.4e38) > 0.2
    want, tol, sums = c.attend(0, q, float(scale), starts)
    check(attend(gpu, c, 0, q, scale, weights=True, decay=0.5), want, tol)
    w, w_tol = c.weigh(0, sums, 0.5)
    after = c.down()[2]
    held = ~np.isnan(w)
    assert np.all(np.abs(after[held] - w[held]) <= w_tol[held])


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("new", [1, 40])
def test_one_position_has_all_the_weight_whatever_its_score(gpu, f16, new):
    """A softmax over one position is 1 where its score is a finite f32, however far it lies below zero and however the factors of the
    score are distributed."""
    q0, k0, scale = (2.0 ** 125, -2.0 ** -24, 2.0 ** 17) if f16 else (1e20, -1e20, 1.2e-38)
    rng = np.random.default_rng(new)
    c = Paged(rng, f16, 1, 1, 64, 16, [new], weights=True)
    for t in range(new):
        c.k[c.at(0, t)] = k0
    c.up([0, new] if new > 1 else None, max_new=new)
    q = np.full((new, 4, 64), q0, np.float32)
    out = attend(gpu, c, 0, q, np.float32(scale), window=1)
    for t in range(new):
        v = c.v[c.tables[0, t // 16], 0, 0, t % 16].astype(np.float64)
        assert np.all(np.abs(out[t] - v) <= 2.0 ** -20 * np.abs(v)), t


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("size", [1e6, 3e8, 1e12, 1e30])
@pytest.mark.parametrize("new,lens", [(1, [300, 1]), (8, [90, 2000]), (40, [64, 300, 40])])
def test_rows_of_scores_far_from_zero(gpu, f16, size, new, lens):
    """Scores that f32 holds in steps of more than one: where the largest leads by many steps the row is that position's value, anywhere it is
    one between the values."""
    rng = np.random.default_rng(new)
    starts = [new * i for i in range(len(lens) + 1)]
    c = Paged(rng, f16, 1, 1, 64, 16, lens).up(starts if new > 1 else None, max_new=new)
    q = rng.normal(0, 1, (starts[-1], 4, 64)).astype(np.float32) * np.float32(size)
    got = attend(gpu, c, 0, q, 0.125).astype(np.float64)
    led = 0
    for b, n in enumerate(lens):
        k, v = (np.array([x[c.at(b, t)][0, 0] for t in range(n)], np.float64) for x in (c.k, c.v))
        for i in range(new):
            for h in range(4):
                row, here = starts[b] + i, n - new + i + 1
                assert np.all(np.isfinite(got[row, h])) and np.all(np.abs(got[row, h]) <= np.abs(v[:here]).max(axis=0) * (1 + 2.0 ** -20)), (b, i, h)
                s = k[:here] @ q[row, h].astype(np.float64) * 0.125
                first = int(np.argmax(s))
                # an f32 score of 64 products, q in 22 bits, is off by less than 100 parts in 2^22 of their sizes' sum; 30 units more leave
                # nothing to the others
                off = 100 * 2.0 ** -22 * (np.abs(k[:here]) @ np.abs(q[row, h].astype(np.float64))).max() * 0.125
                if here == 1 or np.sort(s)[-2] < s[first] - 2 * off - 30:
                    led += 1
                    assert np.all(np.abs(got[row, h] - v[first]) <= 2.0 ** -20 * np.abs(v[first]).max()), (b, i, h)
    assert led >= starts[-1] * 4 // 3


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("size", [1.0, 1e3, 1e5, 1e12, 1e30])
@pytest.mark.parametrize("heads,new,lens", [(4, 1, [300, 1]), (4, 8, [90, 500]), (4, 40, [64, 300, 40]), (2, 300, [310])])
def test_a_row_s_weights_sum_to_one(gpu, f16, size, heads, new, lens):
    """Whatever the scores' size, what a row gives is one in all: the weights are formed by the numbers that its softmax was.  Equal
    positions share alike."""
    rng = np.random.default_rng(new)
    starts = [new * i for i in range(len(lens) + 1)]
    c = Paged(rng, f16, 1, 1, 64, 16, lens, weights=True)
    for b, n in enumerate(lens):
        for t in range(n):
            c.k[c.at(b, t)] = c.k[c.at(b, t % 7)]
    c.up(starts if new > 1 else None, max_new=new)
    q = rng.normal(0, 1, (starts[-1], heads, 64)).astype(np.float32) * np.float32(size)
    attend(gpu, c, 0, q, 0.125, weights=True, decay=0.0)
    after = c.down()[2].astype(np.float64)
    for b, n in enumerate(lens):
        w = np.array([after[c.at(b, t)][0, 0] for t in range(n)])
        # an exponent of a probability that counts is below 32, rounded to 2^-20 at the most, twice; sums of n numbers and their quotient
        rel = 2 * np.log(2) * 2.0 ** -20 + (n + 80) * 2.0 ** -23
        assert abs(w.sum() - new * heads) <= rel * new * heads, (b, w.sum())
        for t in range(7, n - new):  # seen by every token, like the equal one before
            assert abs(w[t] - w[t % 7]) <= 2 * rel * w[t % 7] + 2.0 ** -100, (b, t)


def test_an_error_of_the_caller_s_is_not_the_call_s(gpu, hip):
    """A failed HIP call of the program before, which it has not looked at, does not make the operators fail."""
    rng = np.random.default_rng(3)
    c = Paged(rng, False, 1, 1, 64, 16, [50, 20], weights=True, garbage=0.0).up()
    q = rng.normal(0, 1, (2, 2, 64)).astype(np.float32)
    want, tol, _ = c.attend(0, q, 0.125)
    dq, out, new = hip.DeviceBuffer.from_numpy(q), hip.DeviceBuffer(q.nbytes), hip.DeviceBuffer(8)
    kv = hip.DeviceBuffer.from_numpy(np.ones(128, np.float32))
    for fails in (lambda: hip.rt().hipSetDevice(1000), lambda: hip.rt().hipMemcpy(None, None, 16, hip.H2D)):
        for call in (lambda: gpu.attn_device(c.cache, c.seqs, 0, 2, dq.ptr, out.ptr, 0.125, weights=True),
                     lambda: gpu.kv_evict_device(c.cache, c.seqs, 0, 1, 60, 0, 0, 0, 0, new.ptr),
                     lambda: gpu.kv_store_device(c.cache, c.seqs, 0, kv.ptr, kv.ptr)):
            c.dk.upload(c.k), c.dv.upload(c.v)
            hip.device_synchronize()
            assert fails() != 0
            call()
            hip.device_synchronize()
    check(out.to_numpy(np.float32).reshape(q.shape), want, tol)
    assert new.to_numpy(np.uint32).tolist() == [50, 20]


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("new", [1, 3])
def test_sequences_in_several_parts(gpu, hip, f16, new):
    """More sequences than a launch of few rows looks at, with rows of nobody before, behind and, by their starts, between; weights; captured and
    replayed with other lengths."""
    rng = np.random.default_rng(60 + new)
    n, heads = 601, 4
    lens = [int(rng.integers(new, 40)) if i % 50 else 700 for i in range(n)]
    lens[7] = lens[300] = lens[600] = 0
    starts = [5 + new * i for i in range(n + 1)] if new > 1 else None
    c = Paged(rng, f16, 1, 2, 16, 16, lens, weights=True, garbage=0.0).up(starts, max_new=new, n_tokens=n * new + 9 if starts else n)
    rows = n * new + 9 if starts else n
    q = rng.normal(0, 1, (rows, heads, 16)).astype(np.float32)
    want, tol, sums = c.attend(0, q, 0.25, starts)
    got = attend(gpu, c, 0, q, 0.25, weights=True, decay=0.5)
    mine = slice(5, 5 + n * new) if starts else slice(0, n)
    check(got[mine], want[mine], tol[mine])
    if starts:
        assert np.all(got[:5] == 7.25) and np.all(got[5 + n * new:] == 7.25)
    w, w_tol = c.weigh(0, sums, 0.5)
    after = c.down()[2]
    assert np.all(np.abs(after - w) <= w_tol)
    dq, out, stream = hip.DeviceBuffer.from_numpy(q), hip.DeviceBuffer(q.nbytes), hip.Stream()
    hip.device_synchronize()
    graph = hip.Graph(stream, lambda s: gpu.attn_device(c.cache, c.seqs, 0, heads, dq.ptr, out.ptr, 0.25, weights=True, decay=0.0, stream=s.ptr))
    for change in (lens, [min(x, 3 + i % 30) for i, x in enumerate(lens)], lens):
        c.lens = np.array(change, np.uint32)
        c.dl.upload(c.lens)
        hip.device_synchronize()
        eager = attend(gpu, c, 0, q, 0.25, weights=True, decay=0.0)
        eager_w = c.down()[2]
        out.fill_byte(0)
        graph.launch()
        stream.synchronize()
        assert np.array_equal(out.to_numpy(np.float32).reshape(q.shape)[mine], eager[mine]) and np.array_equal(c.down()[2], eager_w)
    graph.destroy()
    stream.destroy()


@pytest.mark.parametrize("new", [1, 20])
def test_sequences_in_parts_by_their_workspace(pkg, hip, new):
    """Bounds far beyond the lengths: weights and what an eviction looks up would take more than a GiB for all sequences together."""
    rng = np.random.default_rng(70 + new)
    n, far = 300, 65536  # table entries of 16 positions
    lens = [int(rng.integers(new, 60)) for i in range(n)]
    starts = [new * i for i in range(n + 1)]
    c = Paged(rng, True, 1, 1, 8, 16, lens, weights=True, garbage=0.0, extra_blocks=4 * n)
    tables = np.full((n, far), NOWHERE, np.uint32)
    tables[:, :c.stride] = c.tables
    c.tables, c.stride = tables, far
    c.up(starts if new > 1 else None, max_new=new, max_len=far * 16)
    g = pkg.HipGemv(0)
    q = rng.normal(0, 1, (n * new, 2, 8)).astype(np.float32)
    want, tol, sums = c.attend(0, q, 0.25, starts)
    check(attend(g, c, 0, q, 0.25, weights=True, decay=1.0), want, tol)
    w, w_tol = c.weigh(0, sums, 1.0)
    after = c.down()[2]
    assert np.all(np.abs(after - w) <= w_tol)
    c.w = after
    dst = np.full((n, far), NOWHERE, np.uint32)
    dst[:, :4] = c.free[:4 * n].reshape(n, 4)
    dd, out = hip.DeviceBuffer.from_numpy(dst), hip.DeviceBuffer(4 * n)
    g.kv_evict_device(c.cache, c.seqs, 0, 1, far * 16, 0, 0, dd.ptr, far, out.ptr)
    hip.device_synchronize()
    want_len, k, v, w = c.evict([0], far * 16, 0, 0, dst)
    assert out.to_numpy(np.uint32).tolist() == want_len.tolist()
    for got, expect in zip(c.down(), (k, v, w)):
        assert same_bits(got, expect)
    g.close()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("most,news,lens", [(2, [5, 1, 2], [9, 4, 30]), (3, [5, 9, 0], [200, 9, 40]), (40, [45, 70, 3], [45, 300, 60])])
def test_new_tokens_beyond_their_bound_are_left_out(gpu, hip, f16, most, news, lens):
    """A sequence with more new tokens than max_new: the first max_new of them are stored and attend from where they stand, the others' rows,
    places and weights stay as they are; so do tokens behind n_tokens."""
    rng = np.random.default_rng(most)
    starts = np.concatenate([[0], np.cumsum(news)]).astype(int)
    rows = int(starts[-1])
    c = Paged(rng, f16, 1, 2, 64, 16, lens, weights=True, garbage=0.0).up(starts, max_new=most)
    dt = c.k.dtype
    k, v = (rng.normal(0, 1, (rows, 2, 64)).astype(np.float32) for _ in range(2))
    dk, dv = hip.DeviceBuffer.from_numpy(k), hip.DeviceBuffer.from_numpy(v)
    gpu.kv_store_device(c.cache, c.seqs, 0, dk.ptr, dv.ptr)
    taken = np.zeros(rows, bool)
    for b, n in enumerate(news):
        for i in range(min(n, most)):
            taken[starts[b] + i] = True
            at = c.at(b, lens[b] - n + i)
            c.k[at[0], 0, :, at[3]], c.v[at[0], 0, :, at[3]] = k[starts[b] + i].astype(dt), v[starts[b] + i].astype(dt)
    q = rng.normal(0, 1, (rows, 8, 64)).astype(np.float32)
    got = attend(gpu, c, 0, q, 0.125, weights=True, decay=0.5)
    got_k, got_v, after = c.down()
    assert same_bits(got_k, c.k) and same_bits(got_v, c.v)
    want, tol, _ = c.attend(0, q, 0.125, starts)
    check(got[taken], want[taken], tol[taken])
    assert np.all(got[~taken] == 7.25)
    # the taken rows' weights: of the sequences without the others' rows, at the positions that they stand at
    total = 0.5 * c.w.astype(np.float64)
    for b, n in enumerate(news):
        if n == 0:
            continue
        cut = Paged.__new__(Paged)
        cut.__dict__.update(c.__dict__)
        cut.lens = np.array([lens[b] - n + min(n, most)], np.uint32)
        cut.tables = c.tables[b:b + 1]
        _, _, sums = cut.attend(0, q[starts[b]:starts[b] + min(n, most)], 0.125, [0, min(n, most)])
        for (_, h), (pos, ws, wt) in sums.items():
            for t, x, y in zip(pos, ws, wt):
                i = c.tables[b, t // 16], 0, h, t % 16
                total[i] += x
                assert abs(after[i] - total[i]) <= y + 2 * 2.0 ** -24 * total[i], (b, h, t)
        for t in range(lens[b] - n + min(n, most), lens[b]):  # positions of tokens that were left out: seen by none
            i = c.tables[b, t // 16], 0, slice(None), t % 16
            assert np.all(after[i] == (0.5 * c.w[i]).astype(np.float32))
    # n_tokens cuts the last sequence's rows, which then are the positions' last ones
    less = rows - 1
    c.seqs.n_tokens = less
    short = [int(min(s, less)) for s in starts]
    want, tol, _ = c.attend(0, q[:less], 0.125, short)
    got = attend(gpu, c, 0, q, 0.125)
    mine = np.zeros(rows, bool)
    for b in range(len(news)):
        mine[short[b]:short[b] + min(short[b + 1] - short[b], most)] = True
    check(got[mine], want[mine[:less]], tol[mine[:less]])
    assert np.all(got[~mine] == 7.25)


@pytest.mark.parametrize("f16", [False, True])
def test_a_padded_batch(gpu, f16):
    """Sequences that are only there to fill a fixed size: no positions, no rows, tables that name nothing."""
    rng = np.random.default_rng(81)
    for new, starts in ((1, None), (30, [0, 30, 30, 60, 60, 60])):
        lens = [50, 0, 75, 0, 0]
        c = Paged(rng, f16, 1, 2, 64, 16, lens, weights=True, garbage=0.0)
        c.tables[[1, 3, 4]] = NOWHERE
        c.up(starts, max_new=new)
        q = rng.normal(0, 1, (5 if starts is None else 60, 4, 64)).astype(np.float32)
        want, tol, sums = c.attend(0, q, 0.125, starts)
        got = attend(gpu, c, 0, q, 0.125, weights=True)
        check(got, want, tol)
        w, w_tol = c.weigh(0, sums, 1.0)
        assert np.all(np.abs(c.down()[2] - w) <= w_tol)
