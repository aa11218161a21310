"""Sessions over the paged-cache operators against the llama forward pass in 64 bits and against the sessions beside them: f32 and
f16 caches, windows with first tokens, prompts in chunks, reused prefixes.

Logits of an f32 cache are held to 2e-4 of the largest, the bound of every session against the 64-bit forward pass.  An f16 cache
rounds K and V once (half a step); the forward pass below rounds the same way, and where a value lies so near the middle of two that
f32 and f64 round it apart - one in some hundred, an f32 error being 2^-10 of an f16 step or so - it is one step off: a quarter of what all
the roundings together change, which is added to the bound, is many times what those few change."""
import importlib

import numpy as np
import pytest

import oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def llama(pkg):
    return importlib.import_module("llama-rust_amd.llama")


def forward(llama, path, hp, tokens, window=0, sinks=0, half=False, evict=None, gaps=None):
    """Logits of every position in float64 (langtax/src/decode.rs:2710-3099), a token seeing a window and the first tokens, K and V
    rounded to f16 where they are kept so.  evict (behind, keep, first, recent): after `behind` tokens every layer and K/V head keeps
    those positions; gaps gets how far the lightest weight that stays and the heaviest that goes are apart, relative."""
    blob = np.fromfile(path, dtype=np.uint8)
    by = {t[0]: t for t in llama.gguf_tensors(blob)}

    def mat(name):
        _, ty, (n_cols, n_rows), start, end = by[name]
        return oracle.dequant(ty, n_cols, blob[start:end], n_rows).astype(np.float64)

    def norm(x, name):
        return x / np.sqrt((x ** 2).mean(axis=-1, keepdims=True) + float(hp.rms_eps)) * blob[by[name][3]:by[name][4]].view(np.float32)

    def rotated(v):
        angle = np.arange(len(tokens))[:, None] * float(hp.rope_base) ** (-2.0 * np.arange(hp.n_rot // 2) / hp.n_rot)[None, :]
        z = (v[..., 0:hp.n_rot:2] + 1j * v[..., 1:hp.n_rot:2]) * np.exp(1j * angle)[:, None, :]
        out = v.copy()
        out[..., 0:hp.n_rot:2], out[..., 1:hp.n_rot:2] = z.real, z.imag
        return out

    def kept(v):
        return v.astype(np.float16).astype(np.float64) if half else v

    n, hd, group = len(tokens), hp.head_dim, hp.n_head // hp.n_head_kv
    p, t = np.arange(n)[:, None], np.arange(n)[None, :]
    sees = (t <= p) & ((t > p - window) | (t < sinks) if window else True)
    x = mat("token_embd.weight")[np.asarray(tokens)]
    for li in range(hp.n_layer):
        b = f"blk.{li}."
        h = norm(x, b + "attn_norm.weight")
        q = rotated((h @ mat(b + "attn_q.weight").T).reshape(n, hp.n_head, hd))
        k = kept(rotated((h @ mat(b + "attn_k.weight").T).reshape(n, hp.n_head_kv, hd)))
        v = kept((h @ mat(b + "attn_v.weight").T).reshape(n, hp.n_head_kv, hd))
        att = np.empty((n, hp.n_head, hd))
        for hkv in range(hp.n_head_kv):
            scores = [q[:, head] @ k[:, hkv].T / np.sqrt(hd) for head in range(hkv * group, (hkv + 1) * group)]

            def softmax(s, sees):
                e = np.exp(np.where(sees, s, -np.inf) - np.where(sees, s, -np.inf).max(axis=1, keepdims=True))
                return e / e.sum(axis=1, keepdims=True)
            stays = sees
            if evict is not None and evict[0] > evict[1]:
                behind, keep, first, recent = evict
                weight = sum(softmax(s, sees)[:behind, :behind].sum(axis=0) for s in scores)
                middle = np.arange(first, behind - recent)
                order = middle[np.argsort(-weight[middle], kind="stable")]
                left, gone = order[:keep - first - recent], order[keep - first - recent:]
                if gaps is not None and len(left) and len(gone):
                    gaps.append(weight[left[-1]] / weight[gone[0]] - 1)
                dropped = np.zeros(n, bool)
                dropped[gone] = True
                stays = sees & ~(dropped[None, :] & (p >= behind))
            for i, s in enumerate(scores):
                att[:, hkv * group + i] = softmax(s, stays) @ v[:, hkv]
        x = x + att.reshape(n, -1) @ mat(b + "attn_output.weight").T
        h = norm(x, b + "ffn_norm.weight")
        g = h @ mat(b + "ffn_gate.weight").T
        x = x + (g / (1 + np.exp(-g)) * (h @ mat(b + "ffn_up.weight").T)) @ mat(b + "ffn_down.weight").T
    return norm(x, "output_norm.weight") @ mat("output.weight").T


MODELS = {"groups of four": dict(n_embd=512, n_head=8, n_head_kv=2), "heads of 128": dict(n_embd=512, n_head=4, n_head_kv=4),
          "heads of 256": dict(n_embd=512, n_head=2, n_head_kv=1)}


@pytest.fixture(scope="module", params=list(MODELS))
def model(request, llama, tmp_path_factory):
    path = tmp_path_factory.mktemp("paged") / "small.gguf"
    llama.write_synthetic_llama(path, n_layer=2, n_ff=1024, n_vocab=512, block_type=8, embd_type=8, output_type=8, weight_std=0.06, seed=11, **MODELS[request.param])
    return llama.Llama(path=path), path


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (9, 0), (16, 4), (400, 2)])
def test_steps_and_prompts_against_the_forward_pass(pkg, llama, model, half, window, sinks):
    """Three tokens, then one at a time, then a prompt's remainder, then one at a time again."""
    m, path = model
    tokens = np.random.default_rng(window + half).integers(0, 512, 90).tolist()
    want = forward(llama, path, m.hparams, tokens, window, sinks, half)
    tol = 2e-4 * np.abs(want).max()
    if half:
        tol += np.abs(want - forward(llama, path, m.hparams, tokens, window, sinks)).max() / 4
    s = m.session(kv_block=5, device_positions=90, kv_type=pkg.F16 if half else pkg.F32, window=window, sinks=sinks)
    done = 0
    for upto in [3, 4, 5, 6, 7, 80] + list(range(81, 91)):
        got = s.forward(tokens[done:upto])
        assert np.abs(got - want[upto - 1]).max() <= tol, upto
        done = upto
    with pytest.raises(llama.LlamaError, match="outgrew"):
        s.forward([1])


@pytest.mark.parametrize("half", [False, True])
def test_a_long_prompt_in_chunks(pkg, llama, model, half):
    """1100 tokens are three chunks, each behind the ones before."""
    m, path = model
    tokens = np.random.default_rng(5).integers(0, 512, 1100).tolist()
    kind = pkg.F16 if half else pkg.F32
    for window, sinks in ((0, 0), (200, 4)):
        want = forward(llama, path, m.hparams, tokens, window, sinks, half)[-1]
        tol = 2e-4 * np.abs(want).max()
        if half:
            tol += np.abs(want - forward(llama, path, m.hparams, tokens, window, sinks)[-1]).max() / 4
        assert np.abs(m.session(device_positions=1200, kv_type=kind, window=window, sinks=sinks).forward(tokens) - want).max() <= tol


def test_the_same_tokens_as_the_other_sessions(pkg, llama, model):
    """An f32 cache without a window, blocks in any order: the tokens of the host's session and of the device's own kernels."""
    m, _ = model
    prompt = np.random.default_rng(8).integers(0, 512, 37).tolist()
    host, _, _ = m.session().generate_greedy(prompt, 24)
    beside, _, _ = m.session(device_positions=64).generate_greedy(prompt, 24)
    here, _, _ = m.session(kv_block=4, block_ids=list(range(16))[::-1], device_positions=61, kv_type=pkg.F32).generate_greedy(prompt, 24)
    assert here.tolist() == beside.tolist() == host.tolist()


def test_a_prompt_keeps_its_prefix(pkg, llama, model):
    m, _ = model
    prompt = np.random.default_rng(9).integers(0, 512, 60).tolist()
    s = m.session(device_positions=128, kv_type=pkg.F16, window=16, sinks=4)
    s.prompt(prompt)
    other = prompt[:33] + [7, 8, 9]
    got, hit = s.prompt(other)
    assert hit == 33
    fresh, _ = m.session(device_positions=128, kv_type=pkg.F16, window=16, sinks=4).prompt(other)
    assert np.abs(got - fresh).max() <= 2e-4 * np.abs(fresh).max()


def test_sessions_of_one_model_take_turns(pkg, llama, model):
    """Their graphs share the executor's workspace, which the second, larger session made anew."""
    m, _ = model
    tokens = np.random.default_rng(10).integers(0, 512, 40).tolist()
    a = m.session(device_positions=64, kv_type=pkg.F16)
    b = m.session(device_positions=5000, kv_type=pkg.F32)
    alone = m.session(device_positions=64, kv_type=pkg.F16)
    want = [alone.forward([t]) for t in tokens]
    for t, w in zip(tokens, want):
        got = a.forward([t])
        b.forward([t])
        assert np.array_equal(got, w)


def test_a_table_longer_than_the_other_sessions_take(pkg, llama, model):
    m, _ = model
    tokens = np.random.default_rng(12).integers(0, 512, 50).tolist()
    want = m.session(device_positions=64, kv_type=pkg.F32).forward(tokens)
    got = m.session(kv_block=1, device_positions=1 << 16, kv_type=pkg.F32).forward(tokens)
    assert np.abs(got - want).max() <= 1e-4 * np.abs(want).max()


def test_refusals(pkg, llama, model, tmp_path):
    m, _ = model
    with pytest.raises(llama.LlamaError, match="f32 or f16"):
        m.session(device_positions=16, kv_type=pkg.Q8_0)
    with pytest.raises(llama.LlamaError, match="sinks without one"):
        m.session(device_positions=16, kv_type=pkg.F16, sinks=4)
    with pytest.raises(llama.LlamaError, match="31 bits"):
        m.session(device_positions=16, kv_type=pkg.F16, window=1 << 31)
    with pytest.raises(llama.LlamaError, match="kv_type"):
        m.session(device_positions=16, window=4)
    with pytest.raises(llama.LlamaError, match="device_positions"):
        m.session(kv_type=pkg.F16)
    path = tmp_path / "narrow.gguf"
    llama.write_synthetic_llama(path, n_layer=1, n_embd=768, n_head=64, n_head_kv=64, n_ff=256, n_vocab=256, block_type=8, embd_type=8, output_type=8)
    narrow = llama.Llama(path=path)
    assert len(narrow.session(device_positions=16).forward([1, 2])) == 256
    with pytest.raises(llama.LlamaError, match="multiple of 8"):
        narrow.session(device_positions=16, kv_type=pkg.F32)


LENGTHS = [40, 1, 1, 300, 7, 2, 513, 1, 90, 33]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 3)])
def test_a_batch_equals_its_sequences_alone(pkg, llama, model, half, window, sinks):
    """Prompts of one token to more than a chunk, chunks that end one prompt and begin another: the tokens that the batch picks are those
    whose logits are largest in the forward pass over what it picked before, to the sessions' bound."""
    m, path = model
    rng = np.random.default_rng(14)
    prompts = [rng.integers(0, 512, n).tolist() for n in LENGTHS]
    kind = pkg.F16 if half else pkg.F32
    batch = m.batch_session(len(prompts), 530, kv_block=9, kv_type=kind, window=window, sinks=sinks)
    got, _, _ = batch.generate_greedy(prompts, 12)
    again, _, _ = batch.generate_greedy(prompts[::-1], 12)  # other lengths through the same graph
    for prompt, tokens, other in zip(prompts, got, again[::-1]):
        for picked in (tokens, other):
            whole = prompt + picked.tolist()
            want = forward(llama, path, m.hparams, whole, window, sinks, half)
            tol = 2e-4 * np.abs(want).max()
            if half:
                tol += np.abs(want - forward(llama, path, m.hparams, whole, window, sinks)).max() / 4
            for i, t in enumerate(picked):
                logits = want[len(prompt) - 1 + i]
                assert logits[t] >= logits.max() - 2 * tol, (len(prompt), i)


def test_a_batch_of_the_largest_size(pkg, llama, model):
    m, _ = model
    prompts = [[int(x) for x in np.random.default_rng(i).integers(0, 512, 1 + i % 5)] for i in range(128)]
    beside, _, _ = m.batch_session(128, 64).generate_greedy(prompts, 8)
    here, _, _ = m.batch_session(128, 64, kv_type=pkg.F32).generate_greedy(prompts, 8)
    assert np.array_equal(here, beside)


def test_batch_refusals(pkg, llama, model):
    m, _ = model
    with pytest.raises(llama.LlamaError, match="f32 or f16"):
        m.batch_session(2, 16, kv_type=pkg.Q8_0)
    with pytest.raises(llama.LlamaError, match="sinks without one"):
        m.batch_session(2, 16, kv_type=pkg.F16, sinks=1)
    with pytest.raises(llama.LlamaError, match="kv_type"):
        m.batch_session(2, 16, window=1)
    s = m.batch_session(2, 16, kv_type=pkg.F16)
    with pytest.raises(llama.LlamaError, match="outgrew"):
        s.generate_greedy([[1] * 10, [2]], 8)
    assert s.generate_greedy([[1] * 9, [2]], 8)[0].shape == (2, 8)


def test_an_evicted_cache_goes_on(pkg, llama, model):
    """A prompt, some steps, an eviction, a prompt's remainder and steps again, against the forward pass in which later tokens do not
    see what each layer and head dropped.  What stays is decided by weights that lie apart by far more than their errors (the
    attention's bound, 2^-23 times a few hundred)."""
    m, path = model
    tokens = np.random.default_rng(21).integers(0, 512, 140).tolist()
    behind, keep, first, recent = 90, 60, 4, 20
    gaps = []
    want = forward(llama, path, m.hparams, tokens, evict=(behind, keep, first, recent), gaps=gaps)
    plain = forward(llama, path, m.hparams, tokens)
    assert min(gaps) > 1e-4
    tol = 2e-4 * np.abs(want).max()
    assert np.abs(want - plain)[behind:].max() > 4 * tol  # the eviction shows
    s = m.session(kv_block=7, device_positions=140, kv_type=pkg.F32, cache_positions=110, weights=True)
    assert np.abs(s.forward(tokens[:80]) - want[79]).max() <= tol
    for i in range(80, behind):
        assert np.abs(s.forward([tokens[i]]) - want[i]).max() <= tol
    assert s.evict(200) == behind  # nothing to do
    assert s.evict(keep, first, recent) == keep
    done = behind
    for upto in [91, 92, 120] + list(range(121, 141)):
        got = s.forward(tokens[done:upto])
        assert np.abs(got - want[upto - 1]).max() <= tol, upto
        done = upto
    with pytest.raises(llama.LlamaError, match="outgrew"):
        s.forward([1])


@pytest.mark.parametrize("half", [False, True])
def test_more_tokens_than_the_cache_holds(pkg, llama, model, half):
    """Evictions let a sequence pass the cache's size; a prompt that does not go on where it is starts anew, one that does goes on."""
    m, _ = model
    kind = pkg.F16 if half else pkg.F32
    s = m.session(device_positions=400, kv_type=kind, cache_positions=64, weights=True)
    prompt = np.random.default_rng(22).integers(0, 512, 40).tolist()
    out = []
    s.prompt(prompt)
    last = prompt[-1]
    for _ in range(40):
        tokens, _, _ = s.generate_greedy([last], 9)
        out += tokens.tolist()
        last = out[-1]
        assert s.evict(48, 4, 24) == 48
    assert len(out) == 360 and all(0 <= t < 512 for t in out)
    with pytest.raises(llama.LlamaError, match="positions"):
        s.forward([1])
    fresh, hit = s.prompt(prompt)
    assert hit == 0
    want, _ = m.session(device_positions=400, kv_type=kind, cache_positions=64, weights=True).prompt(prompt)
    assert np.array_equal(fresh, want)
    s.evict(32, 4, 4)
    more, hit = s.prompt(prompt + [5, 6, 7])
    assert hit == 40 and np.all(np.isfinite(more))
    assert s.evict(64) == 35
    with pytest.raises(llama.LlamaError, match="cache"):
        s.forward([1] * 30)
    assert s.evict(0) == 0
    assert np.all(np.isfinite(s.forward([1, 2, 3])))


def test_weights_leave_the_results_as_they_are(pkg, llama, model):
    m, _ = model
    tokens = np.random.default_rng(23).integers(0, 512, 300).tolist()
    for kind in (pkg.F32, pkg.F16):
        a, b = (m.session(device_positions=320, kv_type=kind, weights=w) for w in (False, True))
        assert np.array_equal(a.forward(tokens), b.forward(tokens))
        assert np.array_equal(a.generate_greedy([7], 12)[0], b.generate_greedy([7], 12)[0])


@pytest.mark.parametrize("variable", ["LLAMA_HIP_DECODE_EAGER", "LLAMA_HIP_DECODE_UNFUSED", "LLAMA_HIP_DECODE_STEP_PREFILL"])
def test_the_sessions_other_ways(pkg, llama, model, monkeypatch, variable):
    m, _ = model
    prompt = np.random.default_rng(24).integers(0, 512, 50).tolist()
    want, _, _ = m.session(device_positions=80, kv_type=pkg.F32, window=20, sinks=4).generate_greedy(prompt, 16)
    monkeypatch.setenv(variable, "1")
    got, _, _ = m.session(device_positions=80, kv_type=pkg.F32, window=20, sinks=4).generate_greedy(prompt, 16)
    assert got.tolist() == want.tolist()


def test_eviction_refusals(pkg, llama, model):
    m, _ = model
    for s in (m.session(), m.session(device_positions=16), m.session(device_positions=16, kv_type=pkg.F16)):
        with pytest.raises(llama.LlamaError, match="keeps weights"):
            s.evict(4)
    s = m.session(device_positions=32, kv_type=pkg.F16, weights=True)
    s.forward(list(range(20)))
    with pytest.raises(llama.LlamaError, match="exceed those to keep"):
        s.evict(10, 6, 6)
    assert s.evict(10, 5, 5) == 10


@pytest.mark.parametrize("half", [False, True])
def test_weights_are_those_of_the_tokens_that_are_there(pkg, llama, model, half):
    """A prompt that leaves another one's path, or repeats it, before any eviction: what an eviction then keeps is what it keeps in a session
    that saw the second prompt alone - tokens that are no longer there, or were run again, count nothing."""
    m, _ = model
    kind = pkg.F16 if half else pkg.F32
    first = np.random.default_rng(25).integers(0, 512, 90).tolist()
    tail = np.random.default_rng(26).integers(0, 512, 6).tolist()

    def session():
        return m.session(device_positions=160, kv_type=kind, weights=True)

    for second in (first[:50] + [7, 8, 9, 10], first, first[:70], first[:1]):
        s, alone = session(), session()
        s.prompt(first)
        for t in tail[:3]:
            s.forward([t])
        got, hit = s.prompt(second)
        want, _ = alone.prompt(second)
        assert hit == 0 and np.array_equal(got, want)
        keep = len(second) // 2
        assert s.evict(keep, 0, 1 if keep else 0) == alone.evict(keep, 0, 1 if keep else 0) == keep
        for t in tail:
            assert np.array_equal(s.forward([t]), alone.forward([t]))
    # one that goes on where the cache is keeps it, evicted or not
    s = session()
    s.prompt(first)
    assert s.prompt(first + tail)[1] == len(first)
    s.evict(40, 4, 4)
    assert s.prompt(first + tail + [3])[1] == len(first + tail)
