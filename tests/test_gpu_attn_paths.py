"""Attention over the paged cache by every kernel that a call may take (attn_path_cases.py says which, and a host test holds it): units in shares over caches of
any type, sequences in parts, lists of chosen blocks whole, in shares and of many rows - against the definition in 64 bits."""
import importlib

import numpy as np
import pytest

from attn_path_cases import KINDS, LISTS_MANY, LISTS_SHARED, LISTS_WHOLE, PARTS, SHARED
from paged import NOWHERE, Paged, same_bits
from paged4 import Paged4
from test_gpu_attn_select import bounds_of, cache_of
from test_gpu_attn_select import check as check_chosen
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


def name_of(c):
    return "-".join([KINDS[c["type"]], "d%d" % c["dim"], "b%d" % c["block"], "%dx%d" % (c["heads_kv"], c["heads"] // c["heads_kv"]), "n%d" % c.get("new", 1)])


def paged(c, rng, lens, **kw):
    args = (1, c["heads_kv"], c["dim"], c["block"], lens)
    return Paged4(rng, *args, **kw) if KINDS[c["type"]] == "q4_0" else Paged(rng, KINDS[c["type"]] == "f16", *args, **kw)


def beside(want, tol, lens, rows_of, v):
    """What is allowed beside tol, which knows roundings relative to the terms: over f16 and 4-bit caches a probability is held in two f16 parts at 2^8
    times its size, the heaviest at least at 2^8; the second part's half step of 2^-25 is 2^-33 of the heaviest, for each position."""
    light = np.repeat(lens.astype(np.float64), rows_of)[:, None, None] * 2.0 ** -33 * float(np.nanmax(np.abs(v.astype(np.float64))))
    return tol + 1e-7 * np.abs(want) + light


def check_weights(c, sums, decay):
    w, w_tol = c.weigh(0, sums, decay)
    after = c.down()[2]
    held = ~np.isnan(w)
    assert same_bits(after[~held], c.w[~held])
    off = np.abs(after[held] - w[held])
    assert np.all(off <= w_tol[held]), np.max(off - w_tol[held])


@pytest.mark.parametrize("case", SHARED, ids=name_of)
def test_shares(gpu, case):
    """Blocks that are not there at the start, within a share and at the end of one; all positions, a window with first tokens; weights."""
    rng = np.random.default_rng(case["dim"] + case["block"] + case["group"])
    new, seqs, lens = case["new"], case["seqs"], case["lens"]
    c = paged(case, rng, lens, weights=True)
    pages = -(-lens[0] // case["block"])
    c.tables[0, [0, pages // 3, pages - 3]] = NOWHERE, c.n_blocks, NOWHERE
    starts = list(range(0, seqs * new + 1, new))
    c.up(starts if new > 1 else None, max_new=new)
    q = (rng.normal(0, 1, (seqs * new, case["heads"], case["dim"])) * 1.5).astype(np.float32)
    scale = np.float32(case["dim"] ** -0.5)
    for window, sinks in ((2500, 40), (0, 0)):
        want, tol, sums = c.attend(0, q, float(scale), starts, window, sinks)
        got = attend(gpu, c, 0, q, scale, window=window, sinks=sinks)
        check(got, want, beside(want, tol, c.lens, new, c.v))
    assert same_bits(c.down()[2], c.w)
    assert np.array_equal(attend(gpu, c, 0, q, scale, weights=True, decay=0.5), got)
    check_weights(c, sums, 0.5)


@pytest.mark.parametrize("case", PARTS, ids=name_of)
def test_parts(gpu, hip, case):
    """A few long sequences among hundreds of short ones, in the first part, at its end and in the last; weights; captured, and replayed with other lengths and
    between eager calls."""
    rng = np.random.default_rng(case["dim"] + case["seqs"])
    new, n, most = case["new"], case["seqs"], case["len"]
    lens = [int(x) for x in rng.integers(0, 40, n)]
    lens[3], lens[n // 2 - 1], lens[n // 2], lens[n - 2], lens[5] = most, most // 3, most // 2, most - 7, 0
    c = paged(case, rng, lens, weights=True, garbage=0.0)
    c.tables[3, 4] = NOWHERE
    starts = list(range(0, n * new + 1, new))
    c.up(starts if new > 1 else None, max_new=new)
    q = rng.normal(0, 1, (n * new, case["heads"], case["dim"])).astype(np.float32)
    scale = np.float32(case["dim"] ** -0.5)
    want, tol, sums = c.attend(0, q, float(scale), starts)
    got = attend(gpu, c, 0, q, scale, weights=True, decay=0.5)
    check(got, want, beside(want, tol, c.lens, new, c.v))
    check_weights(c, sums, 0.5)
    dq, out, stream = hip.DeviceBuffer.from_numpy(q), hip.DeviceBuffer(q.nbytes), hip.Stream()
    hip.device_synchronize()
    graph = hip.Graph(stream, lambda s: gpu.attn_device(c.cache, c.seqs, 0, case["heads"], dq.ptr, out.ptr, scale, weights=True, decay=0.0, stream=s.ptr))
    for change in (lens, [min(x, 2 + i % 30) for i, x in enumerate(lens)], [x // 2 for x in lens], lens):
        c.dl.upload(np.array(change, np.uint32))
        hip.device_synchronize()
        eager = attend(gpu, c, 0, q, scale, weights=True, decay=0.0)
        eager_w = c.down()[2]
        out.fill_byte(0)
        hip.device_synchronize()
        graph.launch()
        stream.synchronize()
        assert np.array_equal(out.to_numpy(np.float32).reshape(q.shape), eager) and np.array_equal(c.down()[2], eager_w)
    assert np.array_equal(eager, got)
    graph.destroy()
    stream.destroy()


def chosen(gpu, hip, case, lens, starts):
    kind = KINDS[case["type"]]
    rng = np.random.default_rng(case["dim"] + case["block"])
    c = cache_of(kind, rng, 1, case["heads_kv"], case["dim"], case["block"], lens)
    c.tables[0, 7] = NOWHERE
    c.up(starts, max_new=int(np.diff(starts).max()) if starts else 1)
    q = (rng.normal(0, 1, (starts[-1] if starts else len(lens), case["heads"], case["dim"])) * 1.5).astype(np.float32)
    check_chosen(gpu, hip, c, kind, 0, q, case["select"], 1, 2, starts, bounds_of(c, kind))


@pytest.mark.parametrize("case", LISTS_WHOLE, ids=name_of)
def test_long_lists_of_many_rows(gpu, hip, case):
    """More rows than compute units, each with a list of hundreds of positions of its own."""
    chosen(gpu, hip, case, [case["len"], case["len"] // 2 + 1], [0, case["new"], case["new"] + 1])


@pytest.mark.parametrize("case", LISTS_SHARED + LISTS_MANY, ids=name_of)
def test_lists_of_few_rows(gpu, hip, case):
    """Lists in shares, and lists of a row's many query heads."""
    chosen(gpu, hip, case, [case["len"], case["len"] // 3], None)
