"""Argument checks and the shared workspace of the operators around the layer, without a GPU: ops_api.hip and api.hip compiled for
the host against stand-ins (host_runtime.cpp, host_ops.cpp).  A refused call launches nothing and says why."""
import ctypes as C
import os
import subprocess

import pytest

from tests.conftest import ROOT, load_pkg

L = load_pkg("_lib")
F32, BF16 = L.DTYPE_F32, L.DTYPE_BF16
BAD, OOM = L.ERR_INVALID_ARG, L.ERR_OOM
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("host") / "ops_logic.so")
    csrc = os.path.join(ROOT, "omega-ai_amd", "csrc")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-g", "-w", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__",
                           "-D__align__(n)=__attribute__((aligned(n)))", "-DHIP_SYMBOL(x)=((const void *)(x))",
                           "-I/opt/rocm/include", "-I" + os.path.join(ROOT, "include"), "-I" + csrc, "-o", so, "-x", "c++",
                           os.path.join(csrc, "api.hip"), os.path.join(csrc, "ops_api.hip"), os.path.join(ROOT, "tests", "host_runtime.cpp"),
                           os.path.join(ROOT, "tests", "host_ops.cpp")])
    lib = C.CDLL(so)
    for name, (res, args) in L.SIGNATURES.items():
        if hasattr(lib, name):
            getattr(lib, name).restype, getattr(lib, name).argtypes = res, args
    lib.host_live_bytes.restype = C.c_size_t
    lib.host_take_ops.restype = C.c_char_p
    return lib


@pytest.fixture
def ctx(lib):
    h = C.c_void_p()
    assert lib.omega_hip_ctx_create(0, C.byref(h)) == 0
    lib.host_take_ops()
    yield h
    assert lib.omega_hip_ctx_destroy(h) == 0 and lib.host_live_bytes() == 0     # the workspace goes with the context


A, B, D, E, F, G, H = (0x10000000 * k for k in range(1, 8))      # addresses that nothing follows


def embedding(lib, ctx, **kw):
    a = dict(table=A, dtype=BF16, V=100, d=8, ids=B, T=5, scale=1.0, out=D)
    a.update(kw)
    return lib.omega_hip_embedding_forward(ctx, a["table"], a["dtype"], a["V"], a["d"], a["ids"], a["T"], a["scale"], a["out"])


def embedding_back(lib, ctx, **kw):
    a = dict(ids=B, T=5, dout=A, dtype=BF16, V=100, d=8, scale=1.0, add=0, dtable=D, grad=F32)
    a.update(kw)
    return lib.omega_hip_embedding_backward(ctx, a["ids"], a["T"], a["dout"], a["dtype"], a["V"], a["d"], a["scale"], a["add"], a["dtable"], a["grad"])


def norm(lib, ctx, **kw):
    a = dict(x=A, dtype=BF16, T=5, d=8, gamma=B, beta=D, eps=1e-5, out=E, mean=F, rstd=G)
    a.update(kw)
    return lib.omega_hip_layernorm_forward(ctx, a["x"], a["dtype"], a["T"], a["d"], a["gamma"], a["beta"], a["eps"], a["out"], a["mean"], a["rstd"])


def norm_back(lib, ctx, **kw):
    a = dict(x=A, dout=B, dtype=BF16, T=5, d=8, gamma=D, mean=E, rstd=F, dx=G, dgamma=H, dbeta=H + 4096)
    a.update(kw)
    return lib.omega_hip_layernorm_backward(ctx, a["x"], a["dout"], a["dtype"], a["T"], a["d"], a["gamma"], a["mean"], a["rstd"], a["dx"], a["dgamma"], a["dbeta"])


def head(lib, ctx, **kw):
    a = dict(x=A, w=B, dtype=BF16, T=5, V=100, d=8, targets=D, loss=E, stats=F, mean=G)
    a.update(kw)
    return lib.omega_hip_head_loss_forward(ctx, a["x"], a["w"], a["dtype"], a["T"], a["V"], a["d"], a["targets"], a["loss"], a["stats"], a["mean"])


def head_back(lib, ctx, **kw):
    a = dict(x=A, w=B, dtype=BF16, T=5, V=100, d=8, targets=D, stats=E, mean=F, dloss=None, dx=G, dw=H)
    a.update(kw)
    return lib.omega_hip_head_loss_backward(ctx, a["x"], a["w"], a["dtype"], a["T"], a["V"], a["d"], a["targets"], a["stats"], a["mean"], a["dloss"], a["dx"], a["dw"])


REFUSED = [
    (embedding, [dict(table=None), dict(ids=None), dict(out=None), dict(dtype=2), dict(V=0), dict(d=0), dict(T=-1), dict(V=-5), dict(d=(1 << 20) + 1),
                 dict(table=A + 1), dict(out=D + 1), dict(ids=B + 2), dict(dtype=F32, table=A + 2), dict(out=A), dict(out=A + 100 * 16 - 2), dict(out=B),
                 dict(table=D + 16)]),
    (embedding_back, [dict(ids=None), dict(dout=None), dict(dtable=None), dict(dtype=-1), dict(grad=3), dict(V=0), dict(T=-1), dict(dtable=D + 2),
                      dict(dtable=A), dict(dtable=B), dict(dout=A + 1), dict(dout=D + 64)]),
    (norm, [dict(x=None), dict(gamma=None), dict(beta=None), dict(out=None), dict(eps=-1.0), dict(eps=NAN), dict(eps=INF), dict(dtype=9), dict(d=0), dict(T=-1),
            dict(out=A), dict(out=A + 2), dict(mean=G), dict(rstd=E), dict(mean=B), dict(gamma=B + 2), dict(mean=F + 1), dict(x=A + 1)]),
    (norm_back, [dict(x=None), dict(dout=None), dict(gamma=None), dict(mean=None), dict(rstd=None), dict(dx=None), dict(dgamma=None), dict(dbeta=None), dict(d=-1),
                 dict(dx=A), dict(dx=B), dict(dgamma=D), dict(dbeta=H), dict(dbeta=H + 28), dict(dgamma=H + 1)]),
    (head, [dict(x=None), dict(w=None), dict(targets=None), dict(loss=None), dict(mean=None), dict(V=0), dict(T=-1), dict(d=0), dict(dtype=5), dict(loss=D),
            dict(stats=E + 4), dict(mean=F + 36), dict(w=B + 1), dict(targets=D + 1), dict(loss=B + 8)]),
    (head_back, [dict(x=None), dict(w=None), dict(targets=None), dict(stats=None), dict(mean=None), dict(V=0), dict(T=-1), dict(dx=A), dict(dw=B), dict(dx=H),
                 dict(dw=A + 16), dict(dloss=G), dict(dloss=A + 1), dict(dx=G + 1), dict(dw=E)]),
]


@pytest.mark.parametrize("call,cases", REFUSED, ids=[c.__name__ for c, _ in REFUSED])
def test_refusals(lib, ctx, call, cases):
    assert call(lib, ctx) == 0 and len(lib.host_take_ops().splitlines()) == 1
    for kw in cases:
        assert call(lib, ctx, **kw) == BAD, kw
        assert lib.omega_hip_last_error(ctx).startswith(b"Error code 1:") and lib.host_take_ops() == b"", kw
    assert call(lib, None) == BAD
    assert call(lib, ctx) == 0                                          # a refusal leaves the context as it was


def test_optional_buffers_and_empty_calls(lib, ctx):
    assert norm(lib, ctx, mean=None, rstd=None) == 0 and head(lib, ctx, stats=None) == 0
    assert head_back(lib, ctx, dx=None) == 0 and head_back(lib, ctx, dw=None) == 0 and head_back(lib, ctx, dloss=0x70000000 + 0x8000) == 0
    lib.host_take_ops()
    assert head_back(lib, ctx, dx=None, dw=None) == 0 and lib.host_take_ops() == b""
    # no rows: only what is written all the same is asked for
    assert embedding(lib, ctx, T=0, ids=None, out=None) == 0 and embedding_back(lib, ctx, T=0, ids=None, dout=None, add=1) == 0
    assert norm(lib, ctx, T=0, x=None, out=None) == 0 and lib.host_take_ops() == b""
    assert embedding_back(lib, ctx, T=0, ids=None, dout=None) == 0 and b"gradient" in lib.host_take_ops()       # a gradient of zeros
    assert norm_back(lib, ctx, T=0, x=None, dout=None, gamma=None, mean=None, rstd=None, dx=None) == 0 and b"norm_back" in lib.host_take_ops()
    assert head(lib, ctx, T=0, x=None, targets=None, loss=None, stats=None) == 0 and b"head" in lib.host_take_ops()


def test_one_workspace_grows_and_is_shared(lib, ctx):
    assert norm_back(lib, ctx) == 0
    small = lib.host_live_bytes()
    assert norm_back(lib, ctx) == 0 and lib.host_live_bytes() == small
    assert head_back(lib, ctx, T=64) == 0
    large = lib.host_live_bytes()
    assert large >= 64 * 4096
    assert embedding_back(lib, ctx) == 0 and head(lib, ctx) == 0 and lib.host_live_bytes() == large
    lib.host_take_ops()
    # no room: nothing is launched, nothing half there, and the next call that fits runs
    lib.host_fail_allocation(1)
    assert head_back(lib, ctx, T=1000) == OOM and lib.host_take_ops() == b"" and lib.host_live_bytes() < large
    assert norm_back(lib, ctx) == 0 and head_back(lib, ctx, T=1000) == 0
    assert all(b"ws=1" in s for s in lib.host_take_ops().splitlines())


def test_a_context_of_its_own_has_a_workspace_of_its_own(lib, ctx):
    other = C.c_void_p()
    assert lib.omega_hip_ctx_create(0, C.byref(other)) == 0
    assert head_back(lib, ctx) == 0
    one = lib.host_live_bytes()
    assert head_back(lib, other) == 0 and lib.host_live_bytes() == 2 * one
    assert lib.omega_hip_ctx_destroy(other) == 0 and lib.host_live_bytes() == one


def clip(lib, ctx, tensors, limit=1.0, norm_out=None, layers=None):
    T = L.GradTensorStruct
    ls = (C.c_void_p * max(len(layers or []), 1))(*(layers or []))
    return lib.omega_hip_clip_grad_norm(ctx, (T * max(len(tensors), 1))(*[T(*t) for t in tensors]), len(tensors), ls, len(layers or []), limit, norm_out)


def test_clip_refusals(lib, ctx):
    ok = [(A, A, 100, F32, 0), (B, D, 10, BF16, 0), (None, None, 0, F32, 0), (A + 400, A + 400, 7, F32, 0)]
    assert clip(lib, ctx, ok, norm_out=E) == 0 and clip(lib, ctx, []) == 0 and clip(lib, ctx, ok, limit=INF) == 0 and clip(lib, ctx, ok, limit=0.0) == 0
    lib.host_take_ops()
    bad = [[(A, A, 10, F32, 0), (A, A, 10, F32, 0)],           # a tensor twice
           [(A, A, 10, F32, 0), (A + 36, A + 36, 4, F32, 0)],  # tensors that overlap
           [(A, D, 10, F32, 0), (B, D, 10, F32, 0)],           # one destination for two
           [(A, B, 10, F32, 0), (B, B, 10, F32, 0)],           # a destination that another reads
           [(A, A + 4, 10, F32, 0)],                           # ... or itself, shifted
           [(A, A, 10, 2, 0)], [(A, A, 10, F32, 1)], [(None, A, 10, F32, 0)], [(A, None, 10, F32, 0)],
           [(A + 2, A + 2, 10, F32, 0)], [(A + 1, A + 1, 10, BF16, 0)], [(A, A, 1 << 60, F32, 0)]]
    for tensors in bad:
        assert clip(lib, ctx, tensors) == BAD and lib.host_take_ops() == b"", tensors
    assert clip(lib, ctx, ok, limit=-1.0) == BAD and clip(lib, ctx, ok, limit=NAN) == BAD
    assert clip(lib, ctx, ok, norm_out=A + 8) == BAD and clip(lib, ctx, ok, norm_out=E + 2) == BAD
    assert lib.omega_hip_clip_grad_norm(ctx, None, 1, None, 0, 1.0, None) == BAD and lib.omega_hip_clip_grad_norm(ctx, None, 0, None, 1, 1.0, None) == BAD
    assert lib.omega_hip_clip_grad_norm(ctx, None, -1, None, 0, 1.0, None) == BAD and clip(lib, None, ok) == BAD
    # two tensors may share a source that nobody writes
    assert clip(lib, ctx, [(A, B, 10, F32, 0), (A, D, 10, F32, 0)]) == 0


def test_clip_takes_the_gradients_of_layers(lib, ctx):
    cfg = L.MoEConfigStruct(0, 256, 4, 2, 256, 1, 1, 1, F32, L.ROUTER_EXACT)
    layer, other, foreign = C.c_void_p(), C.c_void_p(), C.c_void_p()
    assert lib.omega_moe_create(ctx, C.byref(cfg), C.byref(layer)) == 0
    assert lib.omega_hip_ctx_create(0, C.byref(other)) == 0 and lib.omega_moe_create(other, C.byref(cfg), C.byref(foreign)) == 0
    assert clip(lib, ctx, [], layers=[layer]) == BAD                       # no backward has run
    assert lib.omega_moe_forward(layer, A, 8, B) == 0 and lib.omega_moe_backward(layer, A, D, 8, E) == 0
    lib.host_take_ops()
    assert clip(lib, ctx, [(F, F, 10, F32, 0)], layers=[layer]) == 0
    n = 3 * 5 * 256 * 256 + 4 * 256 + 4 + 256                              # the layer's gradient block
    assert lib.host_take_ops() == b"clip ws=1 bytes=%d\n" % (256 + 10 + n)
    assert clip(lib, ctx, [], layers=[layer, layer]) == BAD and clip(lib, ctx, [], layers=[None]) == BAD
    assert lib.omega_moe_forward(foreign, A, 8, B) == 0 and lib.omega_moe_backward(foreign, A, D, 8, E) == 0
    assert clip(lib, ctx, [], layers=[foreign]) == BAD                     # a layer of another context
    assert lib.omega_moe_destroy(foreign) == 0 and lib.omega_hip_ctx_destroy(other) == 0 and lib.omega_moe_destroy(layer) == 0
