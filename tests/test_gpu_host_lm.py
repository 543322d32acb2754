"""The C++ host layers around the MoE layer (omega-ai_amd/host/LmLayers.hpp): a whole training step, the same bits as the Python layers'.
The demo binary is built by __graft_entry__.build()."""
import importlib
import os
import subprocess
import tempfile

import numpy as np
import pytest

from tests.test_gpu_lm_step import D, H, V, Model, batch

pytestmark = pytest.mark.gpu
P = importlib.import_module("omega-ai_amd")

DEMO = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "omega-ai_amd", "host", "lm_host_demo")


def test_a_training_step_gives_the_bits_of_the_python_layers():
    assert os.path.exists(DEMO), "build omega-ai_amd/host/lm_host_demo first (__graft_entry__.build())"
    T, E, K = 200, 4, 2
    ctx = P.Context(0)
    m = Model(ctx, "f32", E=E, K=K)
    assert m.scale == 16.0
    idb, yb, ids, y = batch(ctx, np.random.default_rng(9), T)
    with tempfile.TemporaryDirectory() as td:
        at = lambda name: os.path.join(td, name)
        for name, a, t in (("table", m.table, "<f4"), ("gamma", m.gamma, "<f4"), ("beta", m.beta, "<f4"), ("ids", ids, "<i4"), ("targets", y, "<i4")):
            a.astype(t).tofile(at(name + ".bin"))
        with open(at("block.bin"), "wb") as f:
            m.moe.saveModelBlock(f)
        r = subprocess.run([DEMO, td, str(T), str(V), str(D), str(E), str(K), str(H), "0.25"], capture_output=True, text=True, timeout=100)
        assert r.returncode == 0, r.stderr
        loss = m.forward(idb, yb).to_numpy()
        m.back()
        c = m.clip()
        norm = c.clip(0.25).to_numpy()
        m.moe.updateAdamW(1e-3, 1)
        with open(at("mine.bin"), "wb") as f:
            m.moe.saveModelBlock(f)
        want = dict(loss=loss, mean=m.head.mean.to_numpy(), norm=norm, tied=m.head.diffW.to_numpy(), dgamma=m.ln.diffGamma.to_numpy(),
                    dbeta=m.ln.diffBeta.to_numpy(), block_step=np.fromfile(at("mine.bin"), "<f4"))
        for k, a in want.items():
            assert np.array_equal(np.fromfile(at(k + ".bin"), "<f4"), a.ravel()), k
    assert norm[0] > 0.25 and norm[1] < 1
    c.close()
    m.close()
    ctx.close()
