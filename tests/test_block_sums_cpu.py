"""A norm that keeps its input in 8 bits holds neither x nor the sum, without a GPU: the C ABI compiled for the host against stand-ins."""
import gc
import os
import subprocess
import weakref

import pytest

from tests.conftest import ROOT
from tests.test_block_host_logic import lib  # noqa: F401  (the host's build of the C ABI)
from tests.test_block_layers_cpu import D, P, T, buf, ctx, free, launched, refused  # noqa: F401


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_nothing_of_the_input_is_held(ctx, dtype):  # noqa: F811
    g, dy = buf(ctx, D), buf(ctx, T, D, dtype=dtype)
    layer = P.RMSLayer(D, ctx=ctx, dtype=dtype, gamma=g, keep8=True)
    for residual, own in ((False, False), (True, False), (True, True)):
        x, r = buf(ctx, T, D, dtype=dtype), buf(ctx, T, D, dtype=dtype) if residual else None
        before = ctx.lib.host_live_bytes()
        launched(ctx, lambda: layer.forward(x, r, None if own or r is None else r), b"rms\n")
        size = T * D * (2 if dtype == "bf16" else 4)
        if not residual:          # out, rstd, codes, scales
            assert ctx.lib.host_live_bytes() - before <= size + T * 4 + T * D + T * 2 * 4
        else:                     # nothing more but the sum, where no buffer was given for it
            assert ctx.lib.host_live_bytes() - before == (size if own else 0) and layer.sum.shape == (T, D) and (layer.sum is r) != own
        assert layer.input is None
        free(x, *([r] if r else []))
        gone = weakref.ref(x)
        del x, r
        gc.collect()
        assert gone() is None
        launched(ctx, lambda: layer.back(dy, dy), b"rms_back ws\n")
    layer.close()
    refused(ctx, lambda: layer.back(dy), "without a forward")
    free(g, dy)


@pytest.mark.parametrize("keep8", [False, True])
def test_a_buffer_for_the_sum(ctx, keep8):  # noqa: F811
    g, dy, x, r, s = buf(ctx, D), buf(ctx, T, D), buf(ctx, T, D), buf(ctx, T, D), buf(ctx, T, D)
    wrong = [buf(ctx, T, D, dtype="bf16"), buf(ctx, T, D - 1), buf(ctx, T + 1, D), buf(ctx, D)]
    layer = P.RMSLayer(D, ctx=ctx, gamma=g, keep8=keep8)
    refused(ctx, lambda: layer.forward(x, sum=s), "without a residual")
    for bad in wrong:
        refused(ctx, lambda: layer.forward(x, r, bad), "sum shape")
    for into in (s, x, r):
        launched(ctx, lambda: layer.forward(x, r, sum=into), b"rms\n")
        assert layer.sum is into and layer.input is (None if keep8 else into)
        launched(ctx, lambda: layer.back(dy), b"rms_back ws\n")
    refused(ctx, lambda: layer.forward(x, r, sum=g), "sum shape")
    launched(ctx, lambda: layer.forward(x, r), b"rms\n")                 # its own again
    mine = layer.sum
    assert mine not in (s, x, r)
    launched(ctx, lambda: layer.forward(mine, r, sum=mine), b"rms\n")
    out = layer.forward(x, r, sum=s)
    refused(ctx, lambda: layer.forward(x, r, sum=out), "overlap")
    refused(ctx, lambda: layer.back(dy), "without a forward")            # a refused forward leaves none behind
    free(s)
    refused(ctx, lambda: layer.forward(x, r, sum=s), "sum has been freed")
    layer.close()
    free(g, dy, x, r, *wrong)


def test_the_cpp_layer(tmp_path):
    csrc, exe = os.path.join(ROOT, "omega-ai_amd", "csrc"), str(tmp_path / "sums")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-g", "-w", "-D__HIP_PLATFORM_AMD__", "-D__align__(n)=__attribute__((aligned(n)))", "-DHIP_SYMBOL(x)=((const void *)(x))",
                           "-I/opt/rocm/include", "-I" + os.path.join(ROOT, "include"), "-I" + csrc,
                           "-I" + os.path.join(ROOT, "omega-ai_amd", "host"), "-o", exe, "-x", "c++"]
                          + [os.path.join(csrc, f) for f in ("api.hip", "ops_api.hip", "block_api.hip")]
                          + [os.path.join(ROOT, "tests", f) for f in ("host_runtime.cpp", "host_ops.cpp", "host_block.cpp", "host_block_sums.cpp")])
    got = subprocess.run([exe], capture_output=True, text=True)
    assert got.returncode == 0 and got.stdout.endswith("0 failed\n"), got.stdout + got.stderr
