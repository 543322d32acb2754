"""The C++ host layers around the experts (omega-ai_amd/host/BlockLayers.hpp): a block's step, the same bits as the Python layers'.
The demo binary is built by __graft_entry__.build()."""
import importlib
import os
import subprocess
import tempfile

import numpy as np
import pytest

from tests.test_gpu_block_step import D, E, H, K, Block, inputs

pytestmark = pytest.mark.gpu
P = importlib.import_module("omega-ai_amd")

DEMO = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "omega-ai_amd", "host", "block_host_demo")


def test_a_blocks_step_gives_the_bits_of_the_python_layers():
    assert os.path.exists(DEMO), "build omega-ai_amd/host/block_host_demo first (__graft_entry__.build())"
    T = 77
    ctx = P.Context(0)
    b = Block(ctx, "f32")
    b.moe.set_training(False)
    (x, res, dout), (xb, rb, db) = inputs(ctx, np.random.default_rng(9), T, "f32")
    with tempfile.TemporaryDirectory() as td:
        at = lambda name: os.path.join(td, name)  # noqa: E731
        for name, a in (("x", x), ("res", res), ("dout", dout), ("gamma1", b.gammas[0]), ("gamma2", b.gammas[1])):
            a.astype("<f4").tofile(at(name + ".bin"))
        with open(at("moe.bin"), "wb") as f:
            b.moe.saveModel(f)
        r = subprocess.run([DEMO, td, str(T), str(D), str(E), str(K), str(H)], capture_output=True, text=True, timeout=100)
        assert r.returncode == 0, r.stderr
        h = b.norm1.forward(xb, rb)
        m = b.moe.forward(h)
        y = b.norm2.forward(m, b.norm1.sum).to_numpy()
        d2 = b.norm2.back(db)
        dx = b.norm1.back(b.moe.back(d2), d2).to_numpy()
        b.moe.balance(0.01)
        with open(at("mine.bin"), "wb") as f:
            b.moe.saveModel(f)
        bias = P.DeviceBuffer.from_numpy(ctx, np.zeros(E, np.float32), "f32")
        route = P.RoutingLayer(E, K, score="sigmoid", scale=2.5, nGroups=4, topGroups=2, ctx=ctx, bias=bias)
        logits = P.DeviceBuffer.from_numpy(ctx, np.ascontiguousarray(x[:, :E]), "f32")
        w = route.forward(logits)
        want = dict(y=y, dx=dx, dgamma1=b.norm1.diffGamma.to_numpy(), dgamma2=b.norm2.diffGamma.to_numpy(), moe_out=np.fromfile(at("mine.bin"), "<f4"), w=w.to_numpy(),
                    dlogits=route.back(w).to_numpy())
        route.balance(0.5)
        keep = P.Keep8Layer(D, form="mx", ctx=ctx)
        keep.save(xb)
        want.update(bias=bias.to_numpy(), x8=keep.load().to_numpy())
        for k, a in want.items():
            assert np.array_equal(np.fromfile(at(k + ".bin"), "<f4"), a.ravel()), k
        for k, a in (("ids", route.ids), ("counts", route.counts)):
            assert np.array_equal(np.fromfile(at(k + ".bin"), "<i4"), a.to_numpy().ravel()), k
    for o in (b, route, keep):
        o.close()
    ctx.close()
