"""Contexts with the 8-bit cache on models with 64-wide heads, alone and grouped.  The bound is that of
test_gpu_kv8.py: a stored value is off by at most 2^-4 of itself, half an E4M3 step, and softmax(QK)V averages
independent errors, so logits (mean absolute change over mean absolute value) move by less than that (needs a
B200)."""
import numpy as np
import pytest

from conftest import MINI_DREAM, MINI_LLADA
from test_gpu_kv8 import moved

pytestmark = pytest.mark.gpu

LLADA64 = dict(MINI_LLADA, n_head=16, n_head_kv=16)
DREAM64 = dict(MINI_DREAM, n_head=28, n_head_kv=4)


@pytest.fixture(scope="module")
def models(pkg, model_dir):
    return {"llada": pkg.synth_model(model_dir / "kv8_llada64.gguf", LLADA64, "q4_k_m", seed=41, n_layer=2),
            "dream": pkg.synth_model(model_dir / "kv8_dream64.gguf", DREAM64, "q4_k_m", seed=42, n_layer=2)}


@pytest.mark.parametrize("name,n", [("llada", 1), ("llada", 65), ("llada", 600), ("dream", 64), ("dream", 330)])
def test_forward(pkg, models, name, n):
    model = pkg.Model(models[name])
    f32, kv8 = pkg.Context(model, 0), pkg.Context(model, 16, kv_bits=8)
    toks = np.random.default_rng(n).integers(0, model.hparams.n_vocab - 2, n).astype(np.int32)
    want, got = f32.forward(toks), kv8.forward(toks)
    assert 0 < moved(got, want) < 2.0 ** -4
    assert (kv8.forward(toks) == got).all()
    kv8.close(); f32.close(); model.close()


@pytest.mark.parametrize("name", ["llada", "dream"])
def test_generation_and_cached_step(pkg, models, name):
    model = pkg.Model(models[name])
    p = pkg.SamplerParams(n_steps=6, remasking=0, use_cache=1, seed=1)
    prompt = np.random.default_rng(6).integers(0, model.hparams.n_vocab - 2, 100).astype(np.int32)
    rows = {}
    for bits in (32, 8):
        ctx = pkg.Context(model, 0, kv_bits=bits)
        ctx.gen_begin(prompt, 50, p)
        ctx.gen_step(0, 0, True)
        assert ctx.gen_step(1, 0, False)["used_cache"] == 1
        rows[bits] = ctx.logits_rows(100, 50)
        out = ctx.generate(prompt, 50, p)
        assert ((out >= 0) & (out < model.hparams.n_vocab)).all()
        ctx.close()
    assert 0 < moved(rows[8], rows[32]) < 2.0 ** -4
    model.close()
