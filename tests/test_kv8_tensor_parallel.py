"""The 8-bit cache is refused on a tensor-parallel model: a rank's error would leave the others waiting."""
import multiprocessing as mp
import os
import types

import pytest

from conftest import MINI_LLADA, load_package
from test_gpu_tp import _device_count

ARCH = dict(MINI_LLADA, n_ff=2048)  # (halves are multiples of the K-quants' 256 values)


def test_refused_before_a_context_is_made(pkg):
    model = types.SimpleNamespace(tp_size=2, _h=None)
    with pytest.raises(pkg.DiffuseError, match="tensor-parallel"):
        pkg.Context(model, 0, kv_bits=8)


def _rank(rank, nid, path, q):
    try:
        os.environ["DIFFUSE_DEVICE"] = str(rank)
        pkg = load_package()
        model = pkg.Model(path, tp=(rank, 2, nid))
        ctx = pkg.Context(model, 0)
        q.put((rank, pkg.native()[0].dfb_ctx_set_kv8(ctx.engine, 1), pkg.native()[0].dfb_ctx_set_kv8(ctx.engine, 0)))
        ctx.close()
        model.close()
    except Exception as e:  # reported to the parent
        q.put((rank, "error", repr(e)))


@pytest.mark.gpu
def test_refused_by_the_library(pkg, model_dir):
    if _device_count(pkg) < 2:
        pytest.skip("needs 2 GPUs")
    path = pkg.synth_model(model_dir / "tp_kv8.gguf", ARCH, "q4_k_m", seed=21, n_layer=2)
    ctxm = mp.get_context("spawn")
    nid, q = pkg.tp_unique_id(), ctxm.Queue()
    procs = [ctxm.Process(target=_rank, args=(r, nid, str(path), q)) for r in range(2)]
    for p in procs:
        p.start()
    try:
        got = [q.get(timeout=300) for _ in range(2)]
    finally:
        for p in procs:
            p.join(timeout=60)
            if p.is_alive():
                p.terminate()
    assert sorted(got) == [(0, -6, 0), (1, -6, 0)], got
