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


def forward(llama, path, hp, tokens, window=0, sinks=0, half=False):
    """Logits of every position in float64 (langtax/src/decode.rs:2710-3099), a token seeing a window and the first tokens, K and V
    rounded to f16 where they are kept so."""
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
        for head in range(hp.n_head):
            s = np.where(sees, q[:, head] @ k[:, head // group].T / np.sqrt(hd), -np.inf)
            e = np.exp(s - s.max(axis=1, keepdims=True))
            att[:, head] = e / e.sum(axis=1, keepdims=True) @ v[:, head // group]
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
