"""Bounds of a block's keys and attention over the blocks that they promise most of, on the GPU: bounds and choices number by number, outputs against the
definition in 64 bits."""
import importlib

import numpy as np
import pytest

from paged import NOWHERE, Paged, same_bits
from paged4 import Paged4

pytestmark = pytest.mark.gpu
KINDS = ["f32", "f16", "q4_0"]


@pytest.fixture(scope="module")
def gpu(pkg):
    g = pkg.HipGemv(0)
    yield g
    g.close()


@pytest.fixture(scope="module")
def hip():
    return importlib.import_module("llama-rust_amd.hiprt")


def cache_of(kind, rng, layers, hkv, d, block, lens, **kw):
    c = Paged4(rng, layers, hkv, d, block, lens, **kw) if kind == "q4_0" else Paged(rng, kind == "f16", layers, hkv, d, block, lens, **kw)
    for b, n in enumerate(lens):  # keys of a block about a centre of its own
        for j in range(-(-n // block)):
            c.k[c.tables[b, j]] = (c.k[c.tables[b, j]].astype(np.float32) * np.float32(0.5) + rng.normal(0, 1, (layers, hkv, 1, d))).astype(c.k.dtype)
    if kind == "q4_0":
        c.settle()
    return c


def bounds_of(c, kind):
    """[blocks, layers, heads, 2, d] of what the sequences have in every block, garbage elsewhere."""
    out = np.full((c.n_blocks, c.n_layer, c.hkv, 2, c.d), 77, np.float32 if kind == "f32" else np.float16)
    for b, n in enumerate(c.lens.astype(int)):
        for j in range(-(-n // c.kvb)):
            if c.there(b, j * c.kvb):
                x = c.k[c.tables[b, j], :, :, :n - j * c.kvb]
                out[c.tables[b, j]] = np.stack([x.min(-2), x.max(-2)], -2)  # NaN where one is
    return out


def definition(c, kind, bounds, layer, q, scale, starts, most, first, recent):
    """(chosen, out, tolerance); -1 (0xffffffff) behind the last chosen, NaN for rows of nobody."""
    rows, heads, d = q.shape
    group = heads // c.hkv
    chosen = np.full((rows, c.hkv, most), 0xabcd, np.uint32)
    out, tol = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
    for b, length in enumerate(c.lens.astype(int)):
        n = starts[b + 1] - starts[b]
        for h in range(c.hkv):
            for i in range(n):
                p, row = length - n + i, starts[b] + i
                blocks = p // c.kvb + 1 if p >= 0 else 0
                kept = list(range(blocks))
                if blocks > most:
                    score = []
                    for j in range(first, blocks - recent):
                        if not c.there(b, j * c.kvb):
                            score.append((2, 0.0, j))
                            continue
                        lo, hi = bounds[c.tables[b, j], layer, h].astype(np.float64)
                        qr = q[row, h * group:(h + 1) * group].astype(np.float64)
                        with np.errstate(all="ignore"):
                            s = np.float32((np.where(qr > 0, hi, lo) * qr).sum(-1).max())
                        score.append((0, 0.0, j) if np.isnan(s) else (1, -float(s), j))
                    kept = sorted(kept[:first] + [x[2] for x in sorted(score)[:most - first - recent]] + kept[blocks - recent:])
                chosen[row, h] = NOWHERE
                chosen[row, h, :len(kept)] = kept
                pos = [t for j in kept for t in range(j * c.kvb, (j + 1) * c.kvb) if t <= p and c.there(b, t)]
                k, v = (np.array([x[c.tables[b, t // c.kvb], layer, h, t % c.kvb] for t in pos], np.float64).reshape(len(pos), d) for x in (c.k, c.v))
                for g in range(group):
                    qr, at = q[row, h * group + g].astype(np.float64), (row, h * group + g)
                    if not pos:
                        out[at], tol[at] = 0, 0
                        continue
                    with np.errstate(all="ignore"):
                        s = (k @ qr) * scale
                        e = np.exp(s - s.max())
                        pr = e / e.sum()
                        out[at] = pr @ v
                        size = (np.abs(k) @ np.abs(qr)).max() * scale
                        tol[at] = (2 * (d + 24) * size + len(pos) + 80) * 2.0 ** -23 * (pr @ np.abs(v)) + 1e-37  # as in paged.py
    return chosen, out, tol


def select(gpu, hip, c, bounds, layer, q, scale, most, first, recent, want_chosen=True, out=None, stream=0, **kw):
    dq, db = hip.DeviceBuffer.from_numpy(q), hip.DeviceBuffer.from_numpy(bounds)
    do = hip.DeviceBuffer.from_numpy(np.full(q.shape, 7.25, np.float32) if out is None else out)
    dc = hip.DeviceBuffer.from_numpy(np.full((q.shape[0], c.hkv, most), 0xabcd, np.uint32))
    gpu.attn_select_device(c.cache, c.seqs, layer, kw.pop("heads", q.shape[-2]), db.ptr, most, first, recent, dq.ptr, do.ptr, np.float32(scale),
                           chosen_ptr=dc.ptr if want_chosen else 0, stream=stream, **kw)
    hip.device_synchronize()
    return dc.to_numpy(np.uint32).reshape(q.shape[0], c.hkv, most), do.to_numpy(np.float32).reshape(q.shape if out is None else out.shape)


def check(gpu, hip, c, kind, layer, q, most, first, recent, starts=None, bounds=None):
    starts_or = starts or list(range(len(c.lens) + 1))
    bounds = bounds_of(c, kind) if bounds is None else bounds
    scale = c.d ** -0.5
    want_chosen, want, tol = definition(c, kind, bounds, layer, q, scale, starts_or, most, first, recent)
    chosen, out = select(gpu, hip, c, bounds, layer, q, scale, most, first, recent)
    assert np.array_equal(chosen, want_chosen)
    nobody = np.isnan(want)
    assert np.all(out[nobody] == 7.25)
    assert np.all(np.abs(out - want)[~nobody] <= (tol + 1e-7 * np.abs(want))[~nobody])
    assert np.array_equal(select(gpu, hip, c, bounds, layer, q, scale, most, first, recent, want_chosen=False)[1], out)
    return out


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d,hkv,block", [(64, 2, 16), (128, 3, 20), (256, 1, 64), (32, 8, 1), (96, 2, 7), (160, 1, 130)])
@pytest.mark.parametrize("starts,lens", [(None, [1, 0, 16, 33, 70]), ([0, 1, 40, 41, 45, 120], [1, 90, 16, 2, 75])])
def test_bounds(gpu, hip, kind, d, hkv, block, starts, lens):
    """Of the blocks that hold new tokens, and of those alone; a NaN, infinities, a block that is not there, a sequence of more tokens than places."""
    rng = np.random.default_rng(d)
    c = cache_of(kind, rng, 2, hkv, d, block, lens)
    c.k[c.at(4, 70 - 1 if starts is None else 50)][:, 0, 3] = np.nan
    if kind != "q4_0":
        c.k[c.at(3, 1)][:, 0, 5], c.k[c.at(3, 0)][:, 0, 6] = np.inf, -np.inf
    if kind == "q4_0":
        c.settle()
    c.tables[2, 0] = c.n_blocks
    c.up(starts, max_new=int(np.diff(starts).max()) if starts else 1)
    want = bounds_of(c, kind)
    start = rng.normal(0, 1, want.shape).astype(want.dtype)
    touched = np.zeros(c.n_blocks, bool)
    for b, n in enumerate(lens):
        new = 1 if starts is None else starts[b + 1] - starts[b]
        for t in range(max(0, n - new), n):
            if c.there(b, t):
                touched[c.tables[b, t // block]] = True
    db = hip.DeviceBuffer.from_numpy(start)
    gpu.kv_bounds_device(c.cache, c.seqs, 1, db.ptr)
    hip.device_synchronize()
    got = db.to_numpy(want.dtype).reshape(want.shape)
    assert same_bits(got[touched, 1], want[touched, 1])
    got[touched, 1] = start[touched, 1]
    assert np.array_equal(got, start)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,hkv,d,block,most,first,recent", [(8, 2, 64, 16, 5, 1, 2), (3, 3, 128, 8, 9, 0, 1), (14, 2, 64, 20, 4, 0, 3), (5, 1, 96, 7, 12, 2, 4),
                                                                 (4, 4, 32, 1, 40, 4, 8), (8, 1, 256, 32, 3, 0, 1), (40, 1, 64, 16, 4, 1, 1)])
def test_one_token_a_sequence(gpu, hip, kind, heads, hkv, d, block, most, first, recent):
    """Sequences of fewer blocks than are read, of as many, of more; one that holds nothing."""
    rng = np.random.default_rng(d + block)
    c = cache_of(kind, rng, 2, hkv, d, block, [1, 0, most * block, most * block + 1, 300, 530, 7]).up()
    q = rng.normal(0, 1, (7, heads, d)).astype(np.float32)
    out = check(gpu, hip, c, kind, 1, q, most, first, recent)
    assert np.all(out[1] == 0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("block", [16, 12])
def test_several_tokens_a_sequence(gpu, hip, kind, block):
    """Every token chooses for itself, those in the middle of a prompt too; rows of nobody, tokens beyond max_new and below position 0."""
    rng = np.random.default_rng(block)
    starts = [3, 3, 43, 44, 60]
    c = cache_of(kind, rng, 1, 2, 64, block, [20, 200, 90, 10])
    c.up(starts, max_new=40, n_tokens=64)
    q = rng.normal(0, 1, (64, 6, 64)).astype(np.float32)
    check(gpu, hip, c, kind, 0, q, 5, 1, 2, starts)
    # a bound that leaves tokens out: theirs stay as they were
    c.seqs.max_new = 30
    bounds = bounds_of(c, kind)
    chosen, out = select(gpu, hip, c, bounds, 0, q, 0.125, 5, 1, 2)
    want_chosen, want, tol = definition(c, kind, bounds, 0, q, 0.125, starts, 5, 1, 2)
    left_out = np.isnan(want)[:, 0, 0]
    left_out[33:43] = True
    assert np.all(out[left_out] == 7.25) and np.all(chosen[left_out] == 0xabcd)
    assert np.array_equal(chosen[~left_out], want_chosen[~left_out])
    assert np.all(np.abs(out - want)[~left_out] <= (tol + 1e-7 * np.abs(want))[~left_out])


@pytest.mark.parametrize("kind", KINDS)
def test_rows_apart(gpu, hip, kind):
    rng = np.random.default_rng(2)
    c = cache_of(kind, rng, 1, 2, 64, 16, [150, 80]).up()
    bounds = bounds_of(c, kind)
    wide = rng.normal(0, 1, (2, 4 * 64 + 12)).astype(np.float32)
    q = wide[:, :256].reshape(2, 4, 64).copy()
    _, want, tol = definition(c, kind, bounds, 0, q, 0.125, [0, 1, 2], 3, 1, 1)
    _, out = select(gpu, hip, c, bounds, 0, wide, 0.125, 3, 1, 1, out=np.full((2, 260), 3, np.float32), heads=4, q_stride=268, out_stride=260, want_chosen=False)
    assert np.all(out[:, 256:] == 3)
    assert np.all(np.abs(out[:, :256].reshape(q.shape) - want) <= tol + 1e-7 * np.abs(want))


@pytest.mark.parametrize("kind", KINDS)
def test_ties_and_what_is_not_a_number(gpu, hip, kind):
    """Equal scores go to the lower block; NaN in a block's bounds comes first, a block that is not there last; infinite bounds; q of zeros."""
    rng = np.random.default_rng(4)
    c = cache_of(kind, rng, 1, 1, 64, 8, [200, 200, 200, 200]).up()
    bounds = bounds_of(c, kind)
    t = c.tables
    bounds[t[0, 5]] = bounds[t[0, 9]] = bounds[t[0, 17]] = bounds[t[0, 2]]
    bounds[t[0, 12]] = -bounds[t[0, 2]]
    bounds[t[1, 7], 0, 0, 0, 1] = np.nan
    bounds[t[1, 11], 0, 0, 1, 9] = np.nan
    bounds[t[1, 13], 0, 0, 1, 2] = np.inf
    bounds[t[1, 14], 0, 0, 0, 2] = -np.inf
    bounds[t[1, 15], 0, 0, :, 4] = -np.inf
    c.tables[2, 3:20] = np.where(np.arange(17) % 2, NOWHERE, c.tables[2, 3:20])
    c.dt.upload(c.tables)
    q = rng.normal(0, 1, (4, 2, 64)).astype(np.float32)
    q[1, :, :10] = np.abs(q[1, :, :10])
    q[1, :, 1] *= -1
    q[3] = 0
    for most in (2, 3, 5, 12, 24):
        check(gpu, hip, c, kind, 0, q, most, 1, 1, bounds=bounds)


@pytest.mark.parametrize("most,first,recent", [(1, 0, 1), (4, 2, 2), (200, 1, 1), (1 << 20, 3, 5)])
def test_lists_of_any_length(gpu, hip, most, first, recent):
    """Nothing to choose between first and last ones, and all that there is: then it is attention over everything."""
    rng = np.random.default_rng(most % 97)
    c = cache_of("f16", rng, 1, 2, 64, 16, [700, 90]).up()
    q = rng.normal(0, 1, (2, 4, 64)).astype(np.float32)
    if most <= 200:
        check(gpu, hip, c, "f16", 0, q, most, first, recent)
        return
    want, tol, _ = c.attend(0, q, 0.125)
    dq, db, do = (hip.DeviceBuffer.from_numpy(x) for x in (q, bounds_of(c, "f16"), np.zeros_like(q)))
    gpu.attn_select_device(c.cache, c.seqs, 0, 4, db.ptr, most, first, recent, dq.ptr, do.ptr, 0.125)
    hip.device_synchronize()
    assert np.all(np.abs(do.to_numpy(np.float32).reshape(q.shape) - want) <= tol)


def test_many_blocks_and_rows(gpu, hip):
    """Thousands of blocks of one position, scores in several rounds of a workgroup; more rows than sequences go at once."""
    rng = np.random.default_rng(8)
    c = cache_of("f16", rng, 1, 1, 32, 1, [9000]).up()
    q = rng.normal(0, 1, (1, 2, 32)).astype(np.float32)
    check(gpu, hip, c, "f16", 0, q, 700, 3, 20)
    starts = [0, 280, 300]
    c = cache_of("f16", rng, 1, 1, 32, 4, [330, 60]).up(starts, max_new=280)
    q = rng.normal(0, 1, (300, 2, 32)).astype(np.float32)
    check(gpu, hip, c, "f16", 0, q, 9, 1, 2, starts)


def test_what_lies_in_other_places_reaches_none(gpu, hip):
    """NaN in blocks that are not chosen, behind the token, and in places of nobody."""
    rng = np.random.default_rng(6)
    for kind in KINDS:
        c = cache_of(kind, rng, 1, 2, 64, 16, [300]).up()
        bounds = bounds_of(c, kind)
        q = rng.normal(0, 1, (1, 4, 64)).astype(np.float32)
        chosen, out = select(gpu, hip, c, bounds, 0, q, 0.125, 4, 0, 1)
        for j in range(19):
            for h in range(2):
                if j not in chosen[0, h]:
                    c.k[c.tables[0, j], 0, h] = np.nan
                    c.v[c.tables[0, j], 0, h] = np.nan
        c.up()
        assert np.array_equal(select(gpu, hip, c, bounds, 0, q, 0.125, 4, 0, 1)[1], out)


def test_more_scores_than_the_workspace_holds_at_a_time(gpu, hip, pkg):
    """Rows in parts: the table's length, not the tokens', sizes the lists."""
    rng = np.random.default_rng(9)
    starts = [0, 60, 70]
    c = cache_of("f16", rng, 1, 2, 32, 1, [150, 40])
    c.up(starts, max_new=60)
    pages = 4 << 20
    table = np.full((2, pages), NOWHERE, np.uint32)
    table[:, :c.stride] = c.tables
    dt = hip.DeviceBuffer.from_numpy(table)
    bounds = bounds_of(c, "f16")
    q = rng.normal(0, 1, (70, 4, 32)).astype(np.float32)
    want_chosen, want, tol = definition(c, "f16", bounds, 0, q, 32 ** -0.5, starts, 20, 1, 2)
    c.seqs = pkg.KvSeqs(2, dt.ptr, pages, c.dl.ptr, pages, c.ds.ptr, 70, 60)  # 2 heads of 2^22 words a row: 31 rows a GiB
    chosen, out = select(gpu, hip, c, bounds, 0, q, 32 ** -0.5, 20, 1, 2)
    assert np.array_equal(chosen, want_chosen)
    assert np.all(np.abs(out - want) <= tol + 1e-7 * np.abs(want))


@pytest.mark.parametrize("kind", ["f16", "q4_0"])
def test_a_captured_step_follows_its_arrays(gpu, hip, pkg, kind):
    """Append, bounds and attention over chosen blocks in one graph, replayed as a sequence grows across a block's end, between other work."""
    rng = np.random.default_rng(1)
    stream = hip.Stream()
    c = cache_of(kind, rng, 1, 2, 64, 16, [110, 60], room=100, garbage=0.0)
    c.up(max_len=160)
    bounds = bounds_of(c, kind)
    db = hip.DeviceBuffer.from_numpy(bounds)
    q, k, v = (hip.DeviceBuffer(2 * n * 64 * 4) for n in (4, 2, 2))
    out, chosen = hip.DeviceBuffer(2 * 4 * 64 * 4), hip.DeviceBuffer(2 * 2 * 4 * 4)

    def step(s):
        gpu.kv_append_device(c.cache, c.seqs, 0, None, 0, 0, 0, k.ptr, v.ptr, stream=s.ptr)
        gpu.kv_bounds_device(c.cache, c.seqs, 0, db.ptr, stream=s.ptr)
        gpu.attn_select_device(c.cache, c.seqs, 0, 4, db.ptr, 4, 1, 1, q.ptr, out.ptr, 0.125, chosen_ptr=chosen.ptr, stream=s.ptr)

    zeros = [np.zeros(b.nbytes // 4, np.float32) for b in (q, k, v)]
    for b, x in zip((q, k, v), zeros):
        b.upload(x)
    c.dl.upload(np.array([111, 61], np.uint32))
    step(stream)
    stream.synchronize()
    graph = hip.Graph(stream, step)
    for turn in range(5):
        rows = [rng.normal(0, 1, (2, n, 64)).astype(np.float32) for n in (4, 2, 2)]
        for b, x in zip((q, k, v), rows):
            b.upload(x)
        c.lens = np.array([111 + turn, 61 + turn], np.uint32)
        c.dl.upload(c.lens)
        graph.launch()
        stream.synchronize()
        c.k, c.v, _ = c.down()
        want_bounds = bounds_of(c, kind)
        got_bounds = db.to_numpy(bounds.dtype).reshape(bounds.shape)
        used = np.unique(np.concatenate([c.tables[b, :-(-int(n) // 16)] for b, n in enumerate(c.lens)]))
        assert np.array_equal(got_bounds[used], want_bounds[used])
        want_chosen, want, tol = definition(c, kind, want_bounds, 0, rows[0], 0.125, [0, 1, 2], 4, 1, 1)
        assert np.array_equal(chosen.to_numpy(np.uint32).reshape(2, 2, 4), want_chosen)
        got = out.to_numpy(np.float32).reshape(2, 4, 64)
        assert np.all(np.abs(got - want) <= tol + 1e-7 * np.abs(want))
        assert np.array_equal(select(gpu, hip, c, want_bounds, 0, rows[0], 0.125, 4, 1, 1)[1], got)
    graph.destroy()
    stream.destroy()


def test_refusals_touch_nothing(gpu, hip, pkg):
    rng = np.random.default_rng(0)
    c = Paged(rng, True, 1, 2, 64, 16, [30]).up()
    rows = hip.DeviceBuffer.from_numpy(np.ones(4096, np.float32))
    out = hip.DeviceBuffer.from_numpy(np.full(4096, 5, np.float32))

    def call(bounds=rows.ptr, most=4, first=1, recent=2, heads=4, q=rows.ptr, to=out.ptr, layer=0, **kw):
        gpu.attn_select_device(c.cache, c.seqs, layer, heads, bounds, most, first, recent, q, to, kw.pop("scale", 0.125), **kw)

    for match, f in (("at least one", lambda: call(recent=0)), ("together exceed", lambda: call(first=3)), ("together exceed", lambda: call(first=(1 << 64) - 1)),
                     ("together exceed", lambda: call(most=0, first=0, recent=1)), ("exceed 31 bits of positions", lambda: call(most=1 << 28)),
                     ("buffer pointer is null", lambda: call(bounds=0)), ("16-byte aligned", lambda: call(bounds=rows.ptr + 8)),
                     ("must be 4-byte aligned", lambda: call(chosen_ptr=out.ptr + 2)), ("multiple of the key-value heads", lambda: call(heads=3)),
                     ("no such layer", lambda: call(layer=1)), ("must not be the input", lambda: call(to=rows.ptr)), ("scale must be positive", lambda: call(scale=0.0)),
                     ("no such layer", lambda: gpu.kv_bounds_device(c.cache, c.seqs, 1, out.ptr)),
                     ("buffer pointer is null", lambda: gpu.kv_bounds_device(c.cache, c.seqs, 0, 0)),
                     ("16-byte aligned", lambda: gpu.kv_bounds_device(c.cache, c.seqs, 0, out.ptr + 4))):
        with pytest.raises(pkg.NativeHipError, match=match) as e:
            f()
        assert e.value.code == pkg.ERR_INVALID, match
    hip.device_synchronize()
    assert np.all(out.to_numpy(np.float32) == 5)
    none = pkg.KvSeqs(0, 0, 2, 0, 0, n_tokens=0)
    gpu.kv_bounds_device(c.cache, none, 0, 0)
    gpu.attn_select_device(c.cache, none, 0, 4, 0, 4, 1, 2, 0, 0, 0.125)


@pytest.mark.parametrize("kind,heads,hkv,d,block", [("f16", 2, 2, 8, 16), ("q4_0", 33, 1, 64, 20)])
def test_more_rows_than_a_launch_has_workgroups(gpu, hip, pkg, kind, heads, hkv, d, block):
    """A prompt's rows in parts by the heads that they have (the check reads a few of them), its last token chosen for as if it were alone."""
    rng = np.random.default_rng(12)
    c = cache_of(kind, rng, 1, hkv, d, block, [3 * block])
    n = (0x3fffff // hkv + 700) if heads == hkv else 300
    c.up([0, n], max_new=n)  # all but the last 3 * block tokens are below position 0
    q = np.zeros((n, heads, d), np.float32)
    tail = rng.normal(0, 1, (3 * block, heads, d)).astype(np.float32)
    q[n - 3 * block:] = tail
    bounds = bounds_of(c, kind)
    scale = d ** -0.5
    want_chosen, want, tol = definition(c, kind, bounds, 0, tail, scale, [0, 3 * block], 2, 0, 1)
    chosen, out = select(gpu, hip, c, bounds, 0, q, scale, 2, 0, 1)
    assert np.array_equal(chosen[n - 3 * block:], want_chosen)
    assert np.all(np.abs(out[n - 3 * block:] - want) <= tol + 1e-7 * np.abs(want))
    assert np.all(out[:n - 3 * block] == 0)
