"""What one call of a context finds wrong is that call's error and not a later one's (needs a B200)."""
import ctypes as C

import gguf
import numpy as np
import pytest

from conftest import MINI_LLADA

pytestmark = pytest.mark.gpu

ERR_TIMEOUT = -5
BAD = MINI_LLADA["mask_token_id"]  # its embedding is infinite: the K, V and logits of masked positions are not numbers
GOOD = np.arange(20, 52, dtype=np.int32)


@pytest.fixture(scope="module")
def model(pkg, model_dir):
    path = pkg.synth_model(model_dir / "errors.gguf", MINI_LLADA, "f16", seed=9, n_layer=2)
    reader = gguf.GGUFReader(path, "r+")
    t = next(t for t in reader.tensors if t.name == "token_embd.weight")
    assert t.tensor_type == gguf.GGMLQuantizationType.F16
    t.data[BAD] = np.inf
    reader.data.flush()
    del reader, t
    model = pkg.Model(path)
    yield model
    model.close()


def failing_step(pkg, ctx):
    ctx.gen_begin(GOOD, 8, pkg.SamplerParams(n_steps=4, remasking=0, use_cache=1))
    with pytest.raises(pkg.DiffuseError):
        ctx.gen_step(0, 2, True)


@pytest.mark.parametrize("bits", [8, 32])
def test_an_error_is_reported_once(pkg, model, bits):
    ctx = pkg.Context(model, 64, kv_bits=bits)
    want = ctx.forward(GOOD)
    for _ in range(2):
        failing_step(pkg, ctx)
        assert (ctx.forward(GOOD) == want).all()  # (this call has nothing wrong)
    ctx.close()


def test_a_time_out_does_not_hide_behind_bad_values(pkg, model):
    ctx = pkg.Context(model, 64, kv_bits=8)
    dfb, _ = pkg.native()
    want = ctx.forward(GOOD)
    failing_step(pkg, ctx)
    with pytest.raises(pkg.DiffuseError):
        ctx.forward(np.full(9, BAD, np.int32))
    x = np.random.default_rng(3).standard_normal((17, MINI_LLADA["n_ff"])).astype(np.float32)
    y = np.zeros((17, MINI_LLADA["n_embd"]), np.float32)
    rc = dfb.dfb_debug_stalled_linear(ctx.engine, pkg.DOWN, 1, x.ctypes.data_as(C.c_void_p), 17, y.ctypes.data_as(C.c_void_p), 20_000_000)
    assert rc == ERR_TIMEOUT, (rc, dfb.dfb_last_error())
    assert (ctx.forward(GOOD) == want).all()
    ctx.close()


def test_a_failed_allocation_is_reported_once(pkg, model):
    ctx = pkg.Context(model, 0)
    want = ctx.forward(GOOD)
    # no GPU holds the activations of so many positions: the first allocation fails
    with pytest.raises(pkg.DiffuseError, match="memory"):
        ctx.score(np.zeros(60_000_000, np.int32))
    assert (ctx.forward(GOOD) == want).all()
    ctx.close()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_generation_ends_when_its_buffers_go(pkg, model, bits):
    """A call that replaces a context's buffers and fails, or drops them, leaves no generation that a step could
    go on with."""
    ctx = pkg.Context(model, 0, kv_bits=bits)
    p = pkg.SamplerParams(n_steps=4, remasking=0, use_cache=1)
    want = ctx.forward(GOOD)

    def refused():
        with pytest.raises(pkg.DiffuseError, match="gen_begin"):
            ctx.gen_step(1, 2, False)

    def begun():
        ctx.gen_begin(np.zeros(0, np.int32), 8, p)

    # no GPU holds the activations of so many positions: the first allocation fails
    many = np.zeros(60_000_000, np.int32)
    begun()
    with pytest.raises(pkg.DiffuseError):
        ctx.gen_begin(many, 8, p)
    refused()
    assert (ctx.forward(GOOD) == want).all()
    begun()
    with pytest.raises(pkg.DiffuseError):
        ctx.score(many)
    refused()
    begun()
    assert pkg.native()[0].dfb_ctx_set_kv8(ctx.engine, int(bits == 8)) == 0
    refused()
    assert (ctx.forward(GOOD) == want).all()
    begun()
    ctx.linear(pkg.WO, 0, np.ones((300, MINI_LLADA["n_embd"]), np.float32))  # more rows than the context had buffers for
    refused()
    assert (ctx.forward(GOOD) == want).all()
    ctx.close()
