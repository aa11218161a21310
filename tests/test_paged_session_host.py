"""What a session over the paged-cache operators refuses: before a GPU is asked for anything, so that it is shown without one."""
import importlib

import pytest

HUGE = (1 << 64) - 1


@pytest.fixture(scope="module")
def llama(pkg):
    return importlib.import_module("llama-rust_amd.llama")


@pytest.fixture(scope="module")
def model(llama, tmp_path_factory):
    path = tmp_path_factory.mktemp("paged") / "tiny.gguf"
    llama.write_synthetic_llama(path, n_layer=2, n_embd=256, n_head=4, n_head_kv=2, n_ff=256, n_vocab=96, block_type=8, embd_type=8, output_type=8)
    return llama.Llama(path=path, products=llama.CALLBACK, matmul=lambda *a: None)


def both(m, match, llama, positions=16, kv_block=16, sequences=2, **kw):
    with pytest.raises(llama.LlamaError, match=match):
        m.session(kv_block=kv_block, device_positions=positions, **kw)
    with pytest.raises(llama.LlamaError, match=match):
        m.batch_session(sequences, positions, kv_block=kv_block, **kw)


def test_arguments(pkg, llama, model):
    for kind in (pkg.Q8_0, pkg.Q4_K, 77):
        both(model, "f32 or f16", llama, kv_type=kind)
    both(model, "sinks without one", llama, kv_type=pkg.F16, sinks=4)
    both(model, "kv_type", llama, window=4)
    both(model, "kv_type", llama, sinks=4)
    both(model, "window or sinks exceed", llama, kv_type=pkg.F16, window=1 << 31)
    both(model, "window or sinks exceed", llama, kv_type=pkg.F32, window=8, sinks=HUGE)
    with pytest.raises(llama.LlamaError, match="device_positions"):
        model.session(kv_type=pkg.F16)
    both(model, "zero K/V block", llama, kv_block=0, kv_type=pkg.F16)
    # fine as far as it goes: the model's products are not the GPU's
    both(model, "resident product route", llama, kv_type=pkg.F16, window=8, sinks=4)


@pytest.mark.parametrize("positions,kv_block", [(HUGE, 16), (16, HUGE), (HUGE, HUGE), (1 << 31, 16), (16, 1 << 31), ((1 << 31) - 4096, (1 << 31) - 4097), (1 << 40, 1)])
def test_positions_beyond_31_bits(pkg, llama, model, positions, kv_block):
    both(model, "exceed 31 bits", llama, positions=positions, kv_block=kv_block, kv_type=pkg.F16)


def test_a_cache_of_too_many_rows(pkg, llama, model):
    with pytest.raises(llama.LlamaError, match="2\\^31 rows"):
        model.session(device_positions=(1 << 29) + 16, kv_type=pkg.F16)
    with pytest.raises(llama.LlamaError, match="resident product route"):
        model.session(device_positions=1 << 29, kv_type=pkg.F16)
    with pytest.raises(llama.LlamaError, match="2\\^31 rows"):
        model.batch_session(128, (1 << 22) + 16, kv_type=pkg.F16)
    with pytest.raises(llama.LlamaError, match="2\\^31 rows"):
        model.batch_session(HUGE, 16, kv_type=pkg.F16)


def test_head_sizes(pkg, llama, tmp_path):
    path = tmp_path / "narrow.gguf"
    llama.write_synthetic_llama(path, n_layer=1, n_embd=768, n_head=64, n_head_kv=64, n_ff=256, n_vocab=256, block_type=8, embd_type=8, output_type=8)
    both(llama.Llama(path=path, products=llama.CALLBACK, matmul=lambda *a: None), "multiple of 8", llama, kv_type=pkg.F32)


def test_a_bounded_cache(pkg, llama, model):
    for kw, match in ((dict(window=4, weights=True), "without a window"), (dict(cache_positions=17), "more positions than the session"),
                      (dict(cache_positions=HUGE), "more positions than the session"), (dict(cache_positions=16, weights=True), "resident product route")):
        with pytest.raises(llama.LlamaError, match=match):
            model.session(device_positions=16, kv_type=pkg.F16, **kw)
    for kw in (dict(weights=True), dict(cache_positions=8)):
        with pytest.raises(llama.LlamaError, match="kv_type"):
            model.session(device_positions=16, **kw)
    # positions beyond the cache cost no rows of it
    with pytest.raises(llama.LlamaError, match="resident product route"):
        model.session(device_positions=(1 << 29) + 16, kv_type=pkg.F16, cache_positions=1 << 20)
    with pytest.raises(llama.LlamaError, match="keeps weights"):
        model.session().evict(4)
