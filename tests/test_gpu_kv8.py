"""Contexts with the 8-bit K/V cache against contexts with the f32 one.

What can be said without the model's whole arithmetic: a stored value is off by at most 2^-4 of itself
(half an E4M3 step), errors of different keys and dimensions are independent, and softmax(QK)V averages
them, so logits (mean absolute change over mean absolute value) move by less than 2^-4; a row, head,
page or sequence taken for another one changes them by about their own size."""
import numpy as np
import pytest

from conftest import MINI_DREAM, MINI_LLADA, write_tiny_gguf

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def models(pkg, model_dir):
    return {"llada": pkg.synth_model(model_dir / "kv8_llada.gguf", MINI_LLADA, "q4_k_m", seed=31, n_layer=2),
            "dream": pkg.synth_model(model_dir / "kv8_dream.gguf", MINI_DREAM, "q4_k_m", seed=32, n_layer=2),
            "tiny": write_tiny_gguf(model_dir / "kv8_tiny.gguf")}


def moved(a, b):
    return float(np.abs(a - b).mean() / np.abs(b).mean())


@pytest.mark.parametrize("name,n", [("llada", 1), ("llada", 63), ("llada", 700), ("dream", 65), ("dream", 330)])
def test_forward(pkg, models, name, n):
    model = pkg.Model(models[name])
    f32, kv8 = pkg.Context(model, 0), pkg.Context(model, 16, kv_bits=8)
    toks = np.random.default_rng(n).integers(0, model.hparams.n_vocab - 2, n).astype(np.int32)
    want, got = f32.forward(toks), kv8.forward(toks)
    print(f"{name} {n}: logits move by {moved(got, want):.2e}")
    assert 0 < moved(got, want) < 2.0 ** -4
    assert (kv8.forward(toks[: max(n // 2, 1)]) != 0).any()  # other segments in between
    assert (kv8.forward(toks) == got).all()
    s8 = kv8.score(toks, toks, top_k=1)
    assert np.isfinite(s8["logprob"]).all() and np.isfinite(s8["entropy"]).all()
    kv8.close(); f32.close(); model.close()


@pytest.mark.parametrize("name", ["llada", "dream"])
def test_generation_runs_and_repeats(pkg, models, name):
    model = pkg.Model(models[name])
    p = pkg.SamplerParams(n_steps=8, remasking=0, use_cache=1, seed=1)
    prompt = np.random.default_rng(5).integers(0, model.hparams.n_vocab - 2, 90).astype(np.int32)
    runs = []
    for _ in range(2):
        ctx = pkg.Context(model, 0, kv_bits=8)
        out, tr = ctx.generate(prompt, 60, p, trace=True)
        runs.append((out, ctx.logits_rows(0, 150)))
        assert ((out >= 0) & (out < model.hparams.n_vocab) & (out != model.hparams.mask_token_id)).all()
        assert tr["n_active"][1] < 150  # the cached steps compute the changed and masked positions only
        ctx.close()
    assert (runs[0][0] == runs[1][0]).all() and (runs[0][1] == runs[1][1]).all()
    model.close()


@pytest.mark.parametrize("name", ["llada", "dream"])
def test_cached_step_logits(pkg, models, name):
    """A full step that commits nothing, then a step over the masked positions against the stored rest."""
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
        ctx.close()
    assert 0 < moved(rows[8], rows[32]) < 2.0 ** -4
    model.close()


def test_batch_of_sequences(pkg, models):
    model = pkg.Model(models["dream"])
    ctx, alone = pkg.Context(model, 0, kv_bits=8), pkg.Context(model, 0)
    rng = np.random.default_rng(7)
    prompts = [rng.integers(0, model.hparams.n_vocab - 2, n).astype(np.int32) for n in (3, 130, 64)]
    p = pkg.SamplerParams(n_steps=4, remasking=0, use_cache=1)
    ctx.gen_begin_batch(prompts, 20, p)
    ctx.gen_step_batch(0, [0, 0, 0], True)
    ctx.gen_step_batch(1, [0, 0, 0], False)
    at = 0
    for prompt in prompts:
        alone.gen_begin(prompt, 20, p)
        alone.gen_step(0, 0, True)
        alone.gen_step(1, 0, False)
        n = prompt.size
        assert moved(ctx.logits_rows(at + n, 20), alone.logits_rows(n, 20)) < 2.0 ** -4
        at += n + 20
    outs = ctx.generate_batch(prompts, 20, p)
    assert outs.shape == (3, 20) and ((outs >= 0) & (outs < model.hparams.n_vocab)).all()
    ctx.close(); alone.close(); model.close()


def test_refusals_and_switching_back(pkg, models):
    tiny = pkg.Model(models["tiny"])
    with pytest.raises(pkg.DiffuseError):
        pkg.Context(tiny, 0, kv_bits=8)
    with pytest.raises(ValueError):
        pkg.Context(tiny, 0, kv_bits=16)
    tiny.close()
    model = pkg.Model(models["llada"])
    ctx, f32 = pkg.Context(model, 40, kv_bits=8), pkg.Context(model, 40)
    toks = np.arange(33, dtype=np.int32)
    a = ctx.forward(toks)
    lib = pkg.native()[0]
    assert lib.dfb_ctx_set_kv8(ctx.engine, 0) == 0
    want = f32.forward(toks)
    assert (ctx.forward(toks) == want).all()
    assert lib.dfb_ctx_set_kv8(ctx.engine, 1) == 0
    assert (ctx.forward(toks) == a).all()
    ctx.close(); f32.close(); model.close()
