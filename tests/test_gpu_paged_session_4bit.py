"""Sessions whose cache is held in 4 bits, against the llama forward pass in 64 bits with K and V packed where they are kept: steps, prompts in
chunks, windows, evictions, batches.

Logits are held to 2e-4 of the largest, the bound of every session, and a quarter of what all the packing together changes: where a number
lies so near the middle between two codes that f32 and f64 pack it apart (x / d is known to some 1e-6 of 8, so one in 1e5), one element is a step
off, where packing leaves every element a third of a step off on average, and there are tens of thousands of them."""
import importlib

import numpy as np
import pytest

import oracle
from paged4 import pack, unpack

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def llama(pkg):
    return importlib.import_module("llama-rust_amd.llama")


@pytest.fixture(scope="module", params=[dict(n_embd=512, n_head=8, n_head_kv=2), dict(n_embd=512, n_head=4, n_head_kv=4), dict(n_embd=256, n_head=8, n_head_kv=8)])
def model(request, llama, tmp_path_factory):
    path = tmp_path_factory.mktemp("packed") / "small.gguf"
    llama.write_synthetic_llama(path, n_layer=2, n_ff=1024, n_vocab=512, block_type=8, embd_type=8, output_type=8, weight_std=0.06, seed=11, **request.param)
    return llama.Llama(path=path), path


def packed(v):
    return unpack(*pack(v.astype(np.float32))).astype(np.float64)


def forward(llama, path, hp, tokens, kept=packed, window=0, sinks=0, evict=None, gaps=None):
    """Logits of every position in float64 (langtax/src/decode.rs:2710-3099).  evict (behind, keep, first, recent): after `behind` tokens every layer
    and K/V head keeps those positions; gaps gets how far the lightest weight that stays and the heaviest that goes are apart, relative."""
    blob = np.fromfile(path, dtype=np.uint8)
    by = {t[0]: t for t in llama.gguf_tensors(blob)}

    def mat(name):
        _, ty, (n_cols, n_rows), start, end = by[name]
        return oracle.dequant(ty, n_cols, blob[start:end], n_rows).astype(np.float64)

    def norm(x, name):
        return x / np.sqrt((x ** 2).mean(axis=-1, keepdims=True) + float(hp.rms_eps)) * blob[by[name][3]:by[name][4]].view(np.float32)

    n, hd, group = len(tokens), hp.head_dim, hp.n_head // hp.n_head_kv
    turn = np.exp(1j * np.arange(n)[:, None] * float(hp.rope_base) ** (-2.0 * np.arange(hp.n_rot // 2) / hp.n_rot)[None, :])[:, None, :]

    def rotated(v):
        z = (v[..., 0:hp.n_rot:2] + 1j * v[..., 1:hp.n_rot:2]) * turn
        out = v.copy()
        out[..., 0:hp.n_rot:2], out[..., 1:hp.n_rot:2] = z.real, z.imag
        return out

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
        def softmax(s, sees):
            e = np.exp(np.where(sees, s, -np.inf) - np.where(sees, s, -np.inf).max(axis=1, keepdims=True))
            return e / e.sum(axis=1, keepdims=True)

        for hkv in range(hp.n_head_kv):
            heads, stays = range(hkv * group, (hkv + 1) * group), sees
            scores = [q[:, head] @ k[:, hkv].T / np.sqrt(hd) for head in heads]
            if evict is not None:
                behind, keep, first, recent = evict
                weight = sum(softmax(s, sees)[:behind, :behind].sum(axis=0) for s in scores)
                middle = np.arange(first, behind - recent)
                order = middle[np.argsort(-weight[middle], kind="stable")]
                left, gone = order[:keep - first - recent], order[keep - first - recent:]
                if gaps is not None:
                    gaps.append(weight[left[-1]] / weight[gone[0]] - 1)
                dropped = np.zeros(n, bool)
                dropped[gone] = True
                stays = sees & ~(dropped[None, :] & (p >= behind))
            for head, s in zip(heads, scores):
                att[:, head] = softmax(s, stays) @ v[:, hkv]
        x = x + att.reshape(n, -1) @ mat(b + "attn_output.weight").T
        h = norm(x, b + "ffn_norm.weight")
        g = h @ mat(b + "ffn_gate.weight").T
        x = x + (g / (1 + np.exp(-g)) * (h @ mat(b + "ffn_up.weight").T)) @ mat(b + "ffn_down.weight").T
    return norm(x, "output_norm.weight") @ mat("output.weight").T


def wanted(llama, path, hp, tokens, **kw):
    """Logits and what they may be off by."""
    want, plain = forward(llama, path, hp, tokens, **kw), forward(llama, path, hp, tokens, kept=lambda v: v, **kw)
    assert np.abs(want - plain).max() > 1e-2 * np.abs(want).max()  # the packing shows
    return want, 2e-4 * np.abs(want).max() + np.abs(want - plain).max() / 4


@pytest.mark.parametrize("window,sinks", [(0, 0), (9, 0), (16, 4)])
def test_steps_and_prompts_against_the_forward_pass(pkg, llama, model, window, sinks):
    m, path = model
    tokens = np.random.default_rng(window).integers(0, 512, 90).tolist()
    want, tol = wanted(llama, path, m.hparams, tokens, window=window, sinks=sinks)
    s = m.session(kv_block=5, device_positions=90, kv_type=pkg.Q4_0, window=window, sinks=sinks)
    done = 0
    for upto in [3, 4, 5, 6, 7, 80] + list(range(81, 91)):
        got = s.forward(tokens[done:upto])
        assert np.abs(got - want[upto - 1]).max() <= tol, upto
        done = upto
    with pytest.raises(llama.LlamaError, match="outgrew"):
        s.forward([1])


def test_a_long_prompt_in_chunks(pkg, llama, model):
    m, path = model
    tokens = np.random.default_rng(5).integers(0, 512, 700).tolist()
    for window, sinks in ((0, 0), (200, 4)):
        want, tol = wanted(llama, path, m.hparams, tokens, window=window, sinks=sinks)
        assert np.abs(m.session(device_positions=700, kv_type=pkg.Q4_0, window=window, sinks=sinks).forward(tokens) - want[-1]).max() <= tol


def test_a_prompt_keeps_its_prefix(pkg, llama, model):
    m, path = model
    tokens = np.random.default_rng(6).integers(0, 512, 60).tolist()
    s = m.session(device_positions=64, kv_type=pkg.Q4_0)
    s.prompt(tokens[:40])
    got, hit = s.prompt(tokens[:30] + tokens[45:])
    assert hit == 30
    want, tol = wanted(llama, path, m.hparams, tokens[:30] + tokens[45:])
    assert np.abs(got - want[-1]).max() <= tol


@pytest.mark.parametrize("variable", ["LLAMA_HIP_DECODE_EAGER", "LLAMA_HIP_DECODE_STEP_PREFILL"])
def test_the_sessions_other_ways(pkg, llama, model, monkeypatch, variable):
    """Captured steps are the eager ones; prompts in chunks pack what steps pack, but for what the order of sums moves across a code's border."""
    m, path = model
    prompt = np.random.default_rng(7).integers(0, 512, 40).tolist()
    s = m.session(device_positions=64, kv_type=pkg.Q4_0)
    first = s.forward(prompt)
    then = [s.forward([t]) for t in (3, 4, 5)]
    monkeypatch.setenv(variable, "1")
    o = m.session(device_positions=64, kv_type=pkg.Q4_0)
    same = [o.forward(prompt)] + [o.forward([t]) for t in (3, 4, 5)]
    if variable.endswith("EAGER"):
        assert all(np.array_equal(x, y) for x, y in zip([first] + then, same))
    _, tol = wanted(llama, path, m.hparams, prompt + [3, 4, 5])
    assert all(np.abs(x - y).max() <= tol for x, y in zip([first] + then, same))


@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 2)])
def test_a_batch_equals_its_sequences_alone(pkg, llama, model, window, sinks):
    """Prompts of different lengths, one of a single token, decoded together: the logits behind the chosen tokens lie with those of the forward pass
    over every sequence's own tokens."""
    m, path = model
    rng = np.random.default_rng(9)
    prompts = [rng.integers(0, 512, n).tolist() for n in (1, 17, 300, 5)]
    out, _, _ = m.batch_session(4, 320, kv_block=16, kv_type=pkg.Q4_0, window=window, sinks=sinks).generate_greedy(prompts, 6)
    for b, prompt in enumerate(prompts):
        tokens = prompt + out[b].tolist()
        want, tol = wanted(llama, path, m.hparams, tokens, window=window, sinks=sinks)
        for i, token in enumerate(out[b]):
            logits = want[len(prompt) - 1 + i]
            assert logits[token] >= logits.max() - 2 * tol


def test_an_evicted_cache_goes_on(pkg, llama, model):
    """A prompt, some steps, an eviction, a prompt's remainder and steps again: later tokens are turned by their positions, not by the places they
    take.  What stays is decided by weights that lie apart by far more than their errors."""
    m, path = model
    tokens = np.random.default_rng(23).integers(0, 512, 140).tolist()
    evict = (90, 60, 4, 20)
    gaps = []
    want = forward(llama, path, m.hparams, tokens, evict=evict, gaps=gaps)
    assert min(gaps) > 1e-4
    _, tol = wanted(llama, path, m.hparams, tokens)
    assert np.abs(want - forward(llama, path, m.hparams, tokens))[90:].max() > 2 * tol  # the eviction shows
    s = m.session(kv_block=7, device_positions=140, kv_type=pkg.Q4_0, cache_positions=110, weights=True)
    assert np.abs(s.forward(tokens[:80]) - want[79]).max() <= tol
    for i in range(80, 90):
        assert np.abs(s.forward([tokens[i]]) - want[i]).max() <= tol
    assert s.evict(200) == 90  # nothing to do
    assert s.evict(*evict[1:]) == 60
    done = 90
    for upto in [91, 92, 120] + list(range(121, 141)):
        got = s.forward(tokens[done:upto])
        assert np.abs(got - want[upto - 1]).max() <= tol, upto
        done = upto
    with pytest.raises(llama.LlamaError, match="outgrew"):
        s.forward([1])


def test_refusals(pkg, llama, tmp_path):
    path = tmp_path / "odd.gguf"
    llama.write_synthetic_llama(path, n_layer=1, n_embd=320, n_head=8, n_head_kv=8, n_ff=256, n_vocab=64, block_type=8, embd_type=8, output_type=8)
    m = llama.Llama(path=path)
    for make in (lambda: m.session(device_positions=16, kv_type=pkg.Q4_0), lambda: m.batch_session(2, 16, kv_type=pkg.Q4_0)):
        with pytest.raises(llama.LlamaError, match="multiple of 32"):
            make()
