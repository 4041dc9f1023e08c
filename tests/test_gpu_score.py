"""Context.score: a forward whose logits stay on the GPU, then log probabilities, entropies and
alternatives.  The reference is the softmax in f64 of the logits that Context.forward copies out.

Tolerance.  The kernel holds y = (x - m) log2 e (three roundings of 2^-24 relative, |y| <= 1.45 range),
exponentials of 2 units in the last place, a sum of n positive terms by at most ~n / 256 + 20 steps in a
row, and one logarithm: with range r = max - min of a row and n <= 32768 that is an absolute error below
2^-24 * (4 r + n / 128 + 64 + |log p|) for a log probability; the entropy weighs the same errors by the
probabilities, each term 2^y |y| once more: four times the bound."""
import numpy as np
import pytest

from conftest import MINI_DREAM, MINI_LLADA, write_tiny_gguf

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def models(pkg, model_dir):
    return {"llada": pkg.synth_model(model_dir / "score_llada.gguf", MINI_LLADA, "q4_k_m", seed=21, n_layer=2),
            "dream": pkg.synth_model(model_dir / "score_dream.gguf", MINI_DREAM, "q4_k_m", seed=22, n_layer=2),
            "tiny": write_tiny_gguf(model_dir / "score_tiny.gguf")}


@pytest.mark.parametrize("name,n,top_k", [("llada", 1, 3), ("llada", 97, 5), ("dream", 70, 32), ("dream", 1, 0), ("tiny", 40, 1)])
def test_score_matches_softmax_of_the_logits(pkg, models, name, n, top_k):
    model = pkg.Model(models[name])
    ctx = pkg.Context(model, 0)
    V = model.hparams.n_vocab
    rng = np.random.default_rng(n)
    toks, targets = rng.integers(0, V - 2, n).astype(np.int32), rng.integers(0, V, n).astype(np.int32)
    targets[n // 2] = -1 if n > 1 else targets[n // 2]
    got = ctx.score(toks, targets, top_k=top_k)
    logits = ctx.forward(toks).astype(np.float64)
    if name == "dream":  # position i is predicted by the row before
        logits = logits[np.maximum(np.arange(n) - 1, 0)]
    m = logits.max(-1, keepdims=True)
    logp = (logits - m) - np.log(np.exp(logits - m).sum(-1, keepdims=True))
    want = np.where(targets < 0, 0.0, logp[np.arange(n), np.maximum(targets, 0)])
    spread = (logits.max(-1) - logits.min(-1))
    tol = 2.0 ** -24 * (4 * spread + V / 128 + 64 + np.abs(want))
    assert (np.abs(got["logprob"] - want) <= tol).all()
    assert (np.abs(got["entropy"] + (np.exp(logp) * logp).sum(-1)) <= 4 * tol).all()
    assert got["top_ids"].shape == got["top_logprob"].shape == (n, top_k)
    if top_k:
        order = np.argsort(-logits, axis=-1, kind="stable")[:, :top_k]
        assert (got["top_ids"] == order).all()
        ref = np.take_along_axis(logp, order, -1)
        assert (np.abs(got["top_logprob"] - ref) <= tol[:, None] + 2.0 ** -24 * np.abs(ref)).all()
    only = ctx.score(toks)
    assert only["logprob"] is None and (only["entropy"] == got["entropy"]).all()
    ctx.close(); model.close()


def test_score_then_generate_and_growing_texts(pkg, models):
    model = pkg.Model(models["llada"])
    ctx, other = pkg.Context(model, 0), pkg.Context(model, 0)
    p = pkg.SamplerParams(n_steps=4, remasking=0, use_cache=1)
    prompt = np.arange(1, 17, dtype=np.int32)
    want = other.generate(prompt, 16, p)
    want = want[0] if isinstance(want, tuple) else want
    small = ctx.score(prompt, prompt, top_k=4)
    big = ctx.score(np.resize(prompt, 200), top_k=4)  # the context's buffers grow
    assert big["top_ids"].shape == (200, 4)
    out = ctx.generate(prompt, 16, p)
    out = out[0] if isinstance(out, tuple) else out
    assert (np.asarray(out) == np.asarray(want)).all()
    again = ctx.score(prompt, prompt, top_k=4)
    assert all((small[k] == again[k]).all() for k in small)
    ctx.close(); other.close(); model.close()


def test_score_refusals(pkg, models):
    model = pkg.Model(models["tiny"])
    ctx = pkg.Context(model, 0)
    V = model.hparams.n_vocab
    for bad in (dict(tokens=[]), dict(tokens=[1, 2], targets=[1]), dict(tokens=[1], top_k=33), dict(tokens=[1], top_k=-1)):
        with pytest.raises(ValueError):
            ctx.score(**bad)
    for bad in (dict(tokens=[V]), dict(tokens=[-1]), dict(tokens=[1], targets=[V])):
        with pytest.raises(pkg.DiffuseError):
            ctx.score(**bad)
    assert ctx.score([1], [0])["logprob"].shape == (1,)
    ctx.close(); model.close()
