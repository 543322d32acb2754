"""Argument checks of the operators around the experts, and the routing that a MoE layer holds, without a GPU: block_api.hip beside api.hip and
ops_api.hip compiled for the host against stand-ins (host_runtime.cpp, host_ops.cpp, host_block.cpp).  A refused call launches nothing and says why."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from tests.conftest import ROOT, load_pkg

P, L = load_pkg(), load_pkg("_lib")
F32, BF16 = L.DTYPE_F32, L.DTYPE_BF16
BAD, OOM = L.ERR_INVALID_ARG, L.ERR_OOM
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("host") / "block_logic.so")
    csrc = os.path.join(ROOT, "omega-ai_amd", "csrc")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-g", "-w", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__",
                           "-D__align__(n)=__attribute__((aligned(n)))", "-DHIP_SYMBOL(x)=((const void *)(x))",
                           "-I/opt/rocm/include", "-I" + os.path.join(ROOT, "include"), "-I" + csrc, "-o", so, "-x", "c++"]
                          + [os.path.join(csrc, f) for f in ("api.hip", "ops_api.hip", "block_api.hip")]
                          + [os.path.join(ROOT, "tests", f) for f in ("host_runtime.cpp", "host_ops.cpp", "host_block.cpp")])
    lib = C.CDLL(so)
    for name, (res, args) in L.SIGNATURES.items():
        if hasattr(lib, name):
            getattr(lib, name).restype, getattr(lib, name).argtypes = res, args
    lib.host_live_bytes.restype = C.c_size_t
    lib.host_take_block.restype = lib.host_take_log.restype = C.c_char_p
    return lib


@pytest.fixture
def ctx(lib):
    h = C.c_void_p()
    assert lib.omega_hip_ctx_create(0, C.byref(h)) == 0
    lib.host_take_block()
    yield h
    assert lib.omega_hip_ctx_destroy(h) == 0 and lib.host_live_bytes() == 0     # the workspace goes with the context


A, B, D, E, F, G, H = (0x10000000 * k for k in range(1, 8))      # addresses that nothing follows
I, J = 0x80000000, 0x90000000


def rms(lib, ctx, **kw):
    a = dict(x=A, res=B, dtype=BF16, T=5, d=200, gamma=D, eps=1e-6, sum=E, out=F, o8=G, o8s=H, k8=I, k8s=J, rstd=J + 4096)
    a.update(kw)
    return lib.omega_hip_rmsnorm_forward(ctx, a["x"], a["res"], a["dtype"], a["T"], a["d"], a["gamma"], a["eps"], a["sum"], a["out"], a["o8"], a["o8s"], a["k8"], a["k8s"],
                                         a["rstd"])


def rms_back(lib, ctx, **kw):
    a = dict(h=A, k8=None, k8s=None, dout=B, dsum=D, dtype=BF16, T=5, d=200, gamma=E, rstd=F, dx=G, dgamma=H)
    a.update(kw)
    return lib.omega_hip_rmsnorm_backward(ctx, a["h"], a["k8"], a["k8s"], a["dout"], a["dsum"], a["dtype"], a["T"], a["d"], a["gamma"], a["rstd"], a["dx"], a["dgamma"])


def save(lib, ctx, **kw):
    a = dict(x=A, dtype=BF16, T=5, d=200, form=L.KEEP8_INT8, codes=B, scales=D)
    a.update(kw)
    return lib.omega_hip_keep8_save(ctx, a["x"], a["dtype"], a["T"], a["d"], a["form"], a["codes"], a["scales"])


def load(lib, ctx, **kw):
    a = dict(codes=A, scales=B, form=L.KEEP8_INT8, T=5, d=200, out=D, dtype=BF16)
    a.update(kw)
    return lib.omega_hip_keep8_load(ctx, a["codes"], a["scales"], a["form"], a["T"], a["d"], a["out"], a["dtype"])


CONFIG = dict(E=16, K=4, score=0, renorm=1, groups=4, top_groups=2, group_best=2, scale=1.0)
WRONG = [dict(E=0), dict(E=513, groups=1, top_groups=1), dict(E=-1), dict(K=0), dict(K=65), dict(K=9), dict(score=2), dict(score=-1), dict(renorm=2), dict(groups=0),
         dict(groups=3), dict(groups=65, E=65, top_groups=65), dict(top_groups=0), dict(top_groups=5), dict(group_best=0), dict(group_best=3), dict(scale=0.0), dict(scale=-1.0),
         dict(scale=NAN), dict(scale=INF)]


def config(**kw):
    c = dict(CONFIG)
    c.update(kw)
    return L.RouteConfigStruct(*[c[n] for n, _ in L.RouteConfigStruct._fields_])


def route(lib, ctx, cfg=None, **kw):
    a = dict(z=A, T=5, bias=B, ids=D, w=E, counts=F)
    a.update(kw)
    return lib.omega_hip_route_forward(ctx, C.byref(cfg or config()), a["z"], a["T"], a["bias"], a["ids"], a["w"], a["counts"])


def route_back(lib, ctx, cfg=None, **kw):
    a = dict(z=A, T=5, ids=B, w=D, dw=E, dz=F)
    a.update(kw)
    return lib.omega_hip_route_backward(ctx, C.byref(cfg or config(score=1)), a["z"], a["T"], a["ids"], a["w"], a["dw"], a["dz"])


def balance(lib, ctx, **kw):
    a = dict(counts=A, E=16, rate=0.1, bias=B)
    a.update(kw)
    return lib.omega_hip_route_balance(ctx, a["counts"], a["E"], a["rate"], a["bias"])


REFUSED = [
    (rms, [dict(x=None), dict(gamma=None), dict(out=None, o8=None, o8s=None), dict(o8=None), dict(o8s=None), dict(k8=None), dict(k8s=None), dict(res=None), dict(dtype=2),
           dict(T=-1), dict(d=0), dict(d=(1 << 20) + 1), dict(eps=-1.0), dict(eps=NAN), dict(eps=INF), dict(x=A + 1), dict(res=B + 1), dict(sum=E + 1), dict(out=F + 1),
           dict(gamma=D + 2), dict(k8s=J + 2), dict(rstd=J + 4097), dict(out=A), dict(out=B), dict(sum=A + 2), dict(sum=B - 2), dict(out=E), dict(o8=F + 1999), dict(o8s=G + 999),
           dict(k8=G), dict(k8s=D + 796), dict(rstd=J + 36), dict(x=B, sum=B)]),
    (rms_back, [dict(h=None), dict(k8=I, k8s=J), dict(h=None, k8=I), dict(h=None, k8s=J), dict(dout=None), dict(gamma=None), dict(rstd=None), dict(dx=None), dict(dgamma=None),
                dict(dtype=7), dict(d=0), dict(T=-1), dict(dx=A), dict(dx=B), dict(dx=D + 2), dict(dgamma=E), dict(dgamma=G + 1996), dict(h=A + 1), dict(dsum=D + 1), dict(dx=G + 1),
                dict(dgamma=H + 2), dict(h=None, k8=I, k8s=J + 2)]),
    (save, [dict(x=None), dict(codes=None), dict(scales=None), dict(dtype=2), dict(form=2), dict(form=-1), dict(T=-1), dict(d=0), dict(x=A + 1), dict(scales=D + 2), dict(codes=A),
            dict(scales=B + 999), dict(scales=A + 1996)]),
    (load, [dict(codes=None), dict(scales=None), dict(out=None), dict(dtype=2), dict(form=2), dict(T=-1), dict(d=0), dict(out=D + 1), dict(scales=B + 1), dict(out=A), dict(out=B)]),
    (route, [dict(z=None), dict(ids=None), dict(w=None), dict(T=-1), dict(z=A + 2), dict(bias=B + 1), dict(ids=D + 2), dict(w=E + 1), dict(counts=F + 2), dict(ids=A), dict(w=D + 76),
             dict(counts=B), dict(counts=E)] + [dict(cfg=config(**kw)) for kw in WRONG]),
    (route_back, [dict(z=None), dict(ids=None), dict(w=None), dict(dw=None), dict(dz=None), dict(T=-1), dict(z=A + 2), dict(dz=F + 1), dict(dz=A), dict(dz=B), dict(dz=E + 76),
                  dict(z=None, cfg=config(renorm=0))] + [dict(cfg=config(**kw)) for kw in WRONG]),
    (balance, [dict(counts=None), dict(bias=None), dict(E=0), dict(rate=-0.1), dict(rate=NAN), dict(rate=INF), dict(counts=A + 2), dict(bias=B + 2), dict(bias=A + 60)]),
]


@pytest.mark.parametrize("call,cases", REFUSED, ids=[c.__name__ for c, _ in REFUSED])
def test_refusals(lib, ctx, call, cases):
    assert call(lib, ctx) == 0 and len(lib.host_take_block().splitlines()) == 1
    for kw in cases:
        assert call(lib, ctx, **kw) == BAD, kw
        assert lib.omega_hip_last_error(ctx).startswith(b"Error code 1:") and lib.host_take_block() == b"", kw
    assert call(lib, None) == BAD
    assert call(lib, ctx) == 0                                          # a refusal leaves the context as it was


def test_what_may_be_left_out_or_lie_in_place(lib, ctx):
    none = dict(o8=None, o8s=None, k8=None, k8s=None)
    for kw in (none, dict(none, res=None, sum=None), dict(none, sum=None, rstd=None), dict(out=None), dict(sum=A), dict(sum=B), dict(x=B), dict(k8=None, k8s=None, o8=G + 1, o8s=H + 3)):
        assert rms(lib, ctx, **kw) == 0, kw
    for kw in (dict(dsum=None), dict(dx=D), dict(h=None, k8=I, k8s=J), dict(h=None, k8=I + 1, k8s=J, dsum=None)):
        assert rms_back(lib, ctx, **kw) == 0, kw
    assert save(lib, ctx, form=L.KEEP8_MX, codes=B + 1, scales=D + 3) == 0 and load(lib, ctx, form=L.KEEP8_MX, codes=A + 1, scales=B + 1) == 0
    assert route(lib, ctx, bias=None) == 0 and route(lib, ctx, counts=None) == 0
    assert route_back(lib, ctx, z=None, cfg=config()) == 0              # softmax with renorm needs no logits
    lib.host_take_block()
    # no rows: only what is written all the same is asked for
    assert rms(lib, ctx, T=0, x=None, out=None) == 0 and save(lib, ctx, T=0, x=None) == 0 and load(lib, ctx, T=0, out=None) == 0
    assert route(lib, ctx, T=0, z=None, ids=None, w=None, counts=None) == 0 and route_back(lib, ctx, T=0, z=None, ids=None, w=None, dw=None, dz=None) == 0
    assert lib.host_take_block() == b""
    assert rms_back(lib, ctx, T=0, h=None, dout=None, gamma=None, rstd=None, dx=None, dsum=None) == 0 and lib.host_take_block() == b"rms_back ws\n"
    assert route(lib, ctx, T=0, z=None, ids=None, w=None) == 0 and lib.host_take_block() == b"route ws\n"


def test_no_room_for_the_workspace(lib, ctx):
    lib.host_fail_allocation(1)
    assert rms_back(lib, ctx) == OOM and lib.host_take_block() == b""
    assert rms_back(lib, ctx) == 0
    lib.host_fail_allocation(1)
    assert route(lib, ctx, T=1000) == OOM and lib.host_take_block() == b"rms_back ws\n"
    assert route(lib, ctx, T=1000) == 0


def layer_of(lib, ctx, dtype=F32, E=16, K=4, T_max=0):
    cfg = L.MoEConfigStruct(T_max, 256, E, K, 256, 0, 1, 1, dtype, L.ROUTER_EXACT)
    m = C.c_void_p()
    assert lib.omega_moe_create(ctx, C.byref(cfg), C.byref(m)) == 0
    return m


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_layers_routing(lib, ctx, dtype):
    m = layer_of(lib, ctx, dtype)
    host = np.zeros(16, np.float32)
    kept = lambda call, *a: call(m, *a)  # noqa: E731
    weights = lambda f: kept(f, L.W_BALANCE, 0, host.ctypes.data, 0)  # noqa: E731
    assert weights(lib.omega_moe_get_weights) == BAD and weights(lib.omega_moe_set_weights) == BAD and kept(lib.omega_moe_balance, 0.1) == BAD
    for cfg in [config(**kw) for kw in WRONG] + [config(E=32), config(K=3)]:
        assert kept(lib.omega_moe_set_routing, C.byref(cfg), 1) == BAD
    assert weights(lib.omega_moe_get_weights) == BAD                    # a refused routing leaves nothing
    before = lib.host_live_bytes()
    assert lib.omega_moe_forward(m, A, 40, B) == 0
    workspace = lib.host_live_bytes()
    # bias and logits come with the routing, and go with it
    lib.host_fail_allocation(2)
    assert kept(lib.omega_moe_set_routing, C.byref(config()), 1) == OOM and lib.host_live_bytes() == workspace
    assert lib.omega_moe_backward(m, A, D, 40, E) == 0                  # the old routing's batch is still there
    workspace = lib.host_live_bytes()
    assert kept(lib.omega_moe_set_routing, C.byref(config()), 1) == 0 and lib.host_live_bytes() == workspace + 64 + 40 * 64
    assert weights(lib.omega_moe_set_weights) == 0 and weights(lib.omega_moe_get_weights) == 0
    for call in (lambda: lib.omega_moe_backward(m, A, D, 40, E), lambda: lib.omega_moe_dispatch(m, A, 40), lambda: lib.omega_moe_combine(m, 40, B), lambda: kept(lib.omega_moe_balance, 0.1)):
        assert call() == BAD                                            # ... of another routing
    assert lib.omega_moe_forward(m, A, 40, B) == 0 and kept(lib.omega_moe_balance, -0.1) == BAD and kept(lib.omega_moe_balance, NAN) == BAD
    lib.host_take_block()
    assert kept(lib.omega_moe_balance, 0.1) == 0 and lib.host_take_block() == b"balance\n"
    assert lib.omega_moe_backward(m, A, D, 40, E) == 0                  # a step of the bias leaves the batch as it is
    assert lib.omega_moe_get_grad(m, L.W_BALANCE, 0, host.ctypes.data, 0) == BAD    # it has no gradient
    assert lib.omega_moe_forward(m, A, 100, B) == 0                     # a larger batch: the logits grow with the workspace
    assert kept(lib.omega_moe_set_routing, C.byref(config(groups=1, top_groups=1)), 0) == 0
    assert weights(lib.omega_moe_get_weights) == BAD and lib.omega_moe_forward(m, A, 100, B) == 0 and kept(lib.omega_moe_balance, 0.1) == BAD
    assert kept(lib.omega_moe_set_routing, None, 1) == 0 and weights(lib.omega_moe_get_weights) == BAD
    assert lib.omega_moe_forward(m, A, 100, B) == 0 and lib.omega_moe_backward(m, A, D, 100, E) == 0
    assert lib.omega_moe_set_routing(None, C.byref(config()), 0) == BAD and lib.omega_moe_balance(None, 0.1) == BAD
    assert lib.omega_moe_destroy(m) == 0
    assert before > 0


def test_a_layers_masters_outlive_its_bias(lib, ctx):
    """The bias for balance has no master copy: setting it does not make a bf16 layer forget the masters of its weights."""
    m = layer_of(lib, ctx, BF16)
    assert lib.omega_moe_set_routing(m, C.byref(config()), 1) == 0
    assert lib.omega_moe_forward(m, A, 70, B) == 0 and lib.omega_moe_backward(m, A, D, 70, E) == 0 and lib.omega_moe_update(m, 0.1) == 0
    lib.host_take_log()

    def second_update():
        assert lib.omega_moe_forward(m, A, 70, B) == 0 and lib.omega_moe_backward(m, A, D, 70, E) == 0
        lib.host_take_log()
        assert lib.omega_moe_update(m, 0.1) == 0
        return lib.host_take_log()

    kept = second_update()
    host = np.zeros(16, np.float32)
    assert lib.omega_moe_set_weights(m, L.W_BALANCE, 0, host.ctypes.data, 0) == 0 and second_update() == kept
    assert lib.omega_moe_destroy(m) == 0
