"""The operators around the experts of a transformer block, as cases that can be measured: routing to experts, RMS norm with the
residual's addition, and activations kept in 8 bits and used in the backward pass.

`run` computes them in elementary torch operations, or, where `own` is true, with this repository's kernels.
"""
import importlib
import math

import torch

own = False

EPS = 1e-6          # RMS norm
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
INT8_GROUP, MX_GROUP = 128, 32   # elements of a row that share a scale
E4M3_MAX = 448.0


def listed():
    return [
        # a decode step's tokens, one for each of 64 sequences: latency
        dict(name="route_decode", op="route", do="forward", T=64, E=128, K=8, score="softmax", bias=False, groups=1, top_groups=1, best=1, renorm=True,
             scale=1.0, closed=0.0, pad=0.0),
        # the prompt tokens of a batch, experts in groups, balanced by a bias
        dict(name="route_prefill", op="route", do="forward", T=16384, E=256, K=8, score="sigmoid", bias=True, groups=8, top_groups=4, best=2, renorm=True,
             scale=2.5, closed=0.0, pad=0.0),
        # weights and gradient of a training batch
        dict(name="route_train", op="route", do="train", T=16384, E=128, K=8, score="softmax", bias=False, groups=1, top_groups=1, best=1, renorm=True,
             scale=1.0, closed=0.0, pad=0.0),
        # the same at odd sizes, weights as they are, experts that are not offered to a token, a padded batch
        dict(name="route_train_odd", op="route", do="train", T=8191, E=60, K=6, score="softmax", bias=True, groups=5, top_groups=3, best=1, renorm=False,
             scale=1.0, closed=0.05, pad=0.1),
        # norm in front of the experts in a decode step
        dict(name="norm_decode", op="norm", do="forward", T=64, d=4096, dtype="bf16", residual=True),
        # forward and backward of a training batch
        dict(name="norm_train", op="norm", do="train", T=16384, d=2048, dtype="bf16", residual=True),
        # the same in fp32 at odd sizes, a network's last norm (nothing added)
        dict(name="norm_train_odd_f32", op="norm", do="train", T=4001, d=1023, dtype="f32", residual=False),
        # rows for products in 8 bits, and what those products then read
        dict(name="norm_out8", op="norm", do="out8", T=16384, d=4096, dtype="bf16", residual=True),
        # a block's input kept for the backward pass, and brought back
        dict(name="keep_int8", op="keep", do="hold", T=16384, d=4096, dtype="bf16", form="int8"),
        # the same of fp32 rows at odd sizes, in the 8-bit floating form
        dict(name="keep_mx_odd_f32", op="keep", do="hold", T=2999, d=1333, dtype="f32", form="mx"),
        # norm of a training batch that keeps its input in 8 bits and goes back from them
        dict(name="keep_train", op="keep", do="train", T=16384, d=2048, dtype="bf16", residual=True),
        # the same of a small batch, fp32 rows of odd width
        dict(name="keep_train_odd_f32", op="keep", do="train", T=513, d=1411, dtype="f32", residual=False),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = max(work(c)["bytes"] for c in listed())
    while True:
        op = rng.choice(["route", "route", "norm", "norm", "keep"])
        if op == "route":
            groups = rng.choice([1, 1, 2, 4, 5, 8, 16])
            E = groups * _spread(rng, 4 if groups > 1 else 2, 512 // groups)
            top = rng.randint(1, groups)
            K = _spread(rng, 1, min(16, top * (E // groups)))
            c = dict(op=op, do=rng.choice(["forward", "train"]), T=_spread(rng, 1, 65536), E=E, K=K, score=rng.choice(["softmax", "sigmoid"]),
                     bias=rng.random() < 0.5, groups=groups, top_groups=top, best=rng.choice([1, 2]), renorm=rng.random() < 0.6, scale=rng.choice([1.0, 2.5]),
                     closed=rng.choice([0.0, 0.0, 0.05]), pad=rng.choice([0.0, 0.0, 0.1]))
        else:
            dtype = rng.choice(["bf16", "bf16", "f32"])
            d = _spread(rng, 64, 8192) if rng.random() < 0.3 else 8 * _spread(rng, 8, 1024)
            do = rng.choice(["forward", "train", "out8"] if op == "norm" else ["hold", "train"])
            c = dict(op=op, do=do, T=_spread(rng, 1, 16384), d=d, dtype=dtype)
            if do == "hold":
                c["form"] = rng.choice(["int8", "mx"])
            else:
                c["residual"] = rng.random() < 0.5
        if work(c)["bytes"] <= most:
            return c


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(std)

    def share(p, *shape):
        return torch.rand(*shape, generator=gen, device="cuda") < p

    s = {"case": case}
    T = case["T"]
    if case["op"] == "route":
        E = case["E"]
        # experts that are liked more or less by every token, and each token's own view
        s["logits"] = normal(T, E, std=1.2) + normal(E, std=0.6)
        if case["closed"]:
            s["logits"].masked_fill_(share(case["closed"], T, E), -math.inf)   # experts that a token is not offered
        if case["pad"]:
            s["logits"].masked_fill_(share(case["pad"], T, 1), -math.inf)      # padding of the batch
        s["bias"] = normal(E, std=0.1 if case["score"] == "sigmoid" else 0.5 / E) if case["bias"] else None
        if case["do"] == "train":
            s["dw"] = normal(T, case["K"], std=1e-3)
    else:
        d, dt = case["d"], TYPES[case["dtype"]]
        # rows of different sizes and a few columns that stand out, as in a deep network's residual stream
        x = normal(T, d) * torch.exp(normal(T, 1, std=0.5))
        x[:, share(0.005, d)] *= 20.0
        s["x"] = x.to(dt)
        s["residual"] = (normal(T, d) * torch.exp(normal(T, 1, std=0.5))).to(dt) if case.get("residual") else None
        if case["do"] != "hold":
            s["gamma"] = normal(d, std=0.1) + 1.0
        if case["do"] == "train":
            s["dout"] = normal(T, d, std=1e-3).to(dt)
            s["dsum"] = normal(T, d, std=1e-3).to(dt) if case["residual"] else None
    if own:
        s["own"] = _Own(case, s)
    torch.cuda.synchronize()
    return s


# ---- plain forms

def _route(case, s):
    T, E, K, groups = case["T"], case["E"], case["K"], case["groups"]
    # (in 64 bits: which of two nearly equal experts is the larger one decides what a token gets)
    z = s["logits"].double()
    open_ = z > -math.inf
    top = z.max(1, keepdim=True).values.clamp(min=-1e30)
    if case["score"] == "softmax":
        score = torch.exp(z - top)
        score = score / score.sum(1, keepdim=True).clamp(min=1e-30)
    else:
        score = 1.0 / (1.0 + torch.exp(-z))
    worth = torch.where(open_, score if s["bias"] is None else score + s["bias"].double(), -math.inf)
    key = z if s["bias"] is None else worth
    if groups > 1:
        best = worth.view(T, groups, E // groups).sort(dim=2, descending=True).values[:, :, :case["best"]]
        of_group = torch.where(best[:, :, 0] > -math.inf, torch.where(best > -math.inf, best, 0.0).sum(2), -math.inf)
        order = of_group.sort(dim=1, descending=True, stable=True).indices
        stays = torch.zeros(T, groups, dtype=torch.bool, device="cuda").scatter_(1, order[:, :case["top_groups"]], True)
        key = torch.where(stays.repeat_interleave(E // groups, 1), key, -math.inf)
    key, ids = key.sort(dim=1, descending=True, stable=True)
    held, ids = key[:, :K] > -math.inf, ids[:, :K]
    chosen = torch.where(held, score.gather(1, ids), 0.0)
    total = chosen.sum(1, keepdim=True)
    w = torch.where(held, chosen / total, 0.0) if case["renorm"] else chosen
    counts = torch.zeros(E, dtype=torch.int64, device="cuda").index_add_(0, ids.reshape(-1), held.reshape(-1).long())
    got = {"ids": torch.where(held, ids, -1).int(), "w": (w * case["scale"]).float(), "counts": counts.int()}
    if case["do"] == "train":
        dw = torch.where(held, s["dw"].double(), 0.0) * case["scale"]
        if case["renorm"]:
            g = w * (dw - (dw * w).sum(1, keepdim=True))
        else:
            g = dw * w
        dz = torch.zeros_like(z).scatter_add_(1, ids, g)
        if case["score"] == "sigmoid":
            dz = dz * (1.0 - score)
        elif not case["renorm"]:
            dz = dz - score * g.sum(1, keepdim=True)
        got["dlogits"] = dz.float()
    return got


def _in_groups(x, n):
    """x [T,d] as [T, groups of n elements, n], filled up with zeros."""
    return torch.nn.functional.pad(x, (0, -x.shape[1] % n)).view(x.shape[0], -1, n)


def _through_int8(x):
    """The values that an 8-bit whole number and a scale hold of x."""
    g = _in_groups(x.float(), INT8_GROUP)
    scale = (g.abs().amax(2, keepdim=True) / 127.0).clamp(min=2.0 ** -126)
    code = torch.round(g.double() / scale.double()).float()   # (64 bits: quotients next to a half)
    return (code * scale).view(x.shape[0], -1)[:, :x.shape[1]]


def _through_mx(x):
    """The values that an 8-bit floating number and a power of two hold of x (in 32 bits or 64)."""
    g = _in_groups(x, MX_GROUP)
    most = g.abs().amax(2, keepdim=True)
    mantissa, exponent = torch.frexp(most)                    # most = mantissa * 2^exponent, mantissa in [0.5, 1)
    k = torch.where(most > 0, exponent - 9 + (mantissa > E4M3_MAX / 512.0).int(), -127).clamp(min=-127)
    g = torch.ldexp(g, -k)
    # four significant bits, multiples of 2^-9 below 2^-6
    step = torch.frexp(g.abs().clamp(min=2.0 ** -6)).exponent - 4
    code = torch.ldexp(torch.round(torch.ldexp(g, -step)), step)
    return torch.ldexp(code, k).view(x.shape[0], -1)[:, :x.shape[1]]


def _norm_forward(s, of=torch.float32):
    """What is normed, 1 / root mean square, and the normed rows."""
    h = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    v = h.to(of)
    r = torch.rsqrt((v * v).mean(1, keepdim=True) + EPS)
    return h, r, v * r * s["gamma"]


def _norm_backward(s, v, r):
    dy = s["dout"].float()
    xh = v * r
    g = dy * s["gamma"]
    dx = r * (g - xh * (g * xh).mean(1, keepdim=True))
    if s["dsum"] is not None:
        dx = dx + s["dsum"].float()
    return {"dx": dx.to(s["x"].dtype), "dgamma": (dy * xh).sum(0)}


def _norm(case, s):
    eight = case["do"] == "out8"
    h, r, y = _norm_forward(s, torch.float64 if eight else torch.float32)   # (64 bits: values next to a border of the 8)
    # (four significant bits and a power of two: bf16 holds them)
    got = {"out": _through_mx(y).to(torch.bfloat16) if eight else y.to(h.dtype)}
    if case["residual"]:
        got["sum"] = h
    if case["do"] == "train":
        got.update(_norm_backward(s, h.float(), r))
    return got


def _keep(case, s):
    if case["do"] == "hold":
        return {"x": (_through_int8 if case["form"] == "int8" else _through_mx)(s["x"].float()).to(s["x"].dtype)}
    h, r, y = _norm_forward(s)
    got = {"out": y.to(h.dtype), **_norm_backward(s, _through_int8(h), r)}
    if case["residual"]:
        got["sum"] = h
    return got


# ---- this repository's operators

_ctx = None


class _Held:
    """A layer, given back with the last tensor that looks at its buffers."""

    def __init__(self, layer):
        self.layer = layer

    def __del__(self):
        self.layer.close()


class _Memory:
    """Device memory of a library buffer, for torch.as_tensor (no copy)."""

    def __init__(self, held, buf):
        self.held = held
        self.__cuda_array_interface__ = {"version": 2, "shape": tuple(buf.shape), "data": (buf.ptr.value, False),
                                         "typestr": {"bf16": "<i2", "i32": "<i4", "f32": "<f4"}[buf.dtype], "strides": None}


class _Own:
    """The layer of a case and its buffers, as a program keeps them."""

    def __init__(self, case, s):
        global _ctx
        self.P = P = importlib.import_module("omega-ai_amd")
        if _ctx is None:
            _ctx = P.Context(0)
        self.seen = {}
        if case["op"] == "route":
            self.layer = P.RoutingLayer(case["E"], case["K"], score=case["score"], renorm=case["renorm"], scale=case["scale"], nGroups=case["groups"],
                                        topGroups=case["top_groups"], groupBest=case["best"], ctx=_ctx,
                                        bias=self.buffer(s["bias"]))
            self.logits, self.dw = self.buffer(s["logits"]), self.buffer(s.get("dw"))
        else:
            if case["do"] == "hold":
                self.layer = P.Keep8Layer(case["d"], form=case["form"], ctx=_ctx, dtype=case["dtype"])
            else:
                self.layer = P.RMSLayer(case["d"], eps=EPS, ctx=_ctx, dtype=case["dtype"], gamma=self.buffer(s["gamma"]), out8=case["do"] == "out8",
                                        keep8=case["op"] == "keep")
            self.x, self.residual = self.buffer(s["x"]), self.buffer(s["residual"])
            self.dout, self.dsum = self.buffer(s.get("dout")), self.buffer(s.get("dsum"))
        self.held = _Held(self.layer)

    def buffer(self, t):
        if t is None:
            return None
        return self.P.DeviceBuffer.wrap(_ctx, t.data_ptr(), tuple(t.shape), {torch.bfloat16: "bf16", torch.float32: "f32"}[t.dtype])

    def tensor(self, buf):
        t = self.seen.get(buf.ptr.value)
        if t is None:
            t = torch.as_tensor(_Memory(self.held, buf), device="cuda")
            t = self.seen[buf.ptr.value] = t.view(torch.bfloat16) if buf.dtype == "bf16" else t
        return t

    def run(self, case):
        layer, tensor = self.layer, self.tensor
        if case["op"] == "route":
            got = {"w": tensor(layer.forward(self.logits)), "ids": tensor(layer.ids), "counts": tensor(layer.counts)}
            if case["do"] == "train":
                got["dlogits"] = tensor(layer.back(self.dw))
            return got
        if case["do"] == "hold":
            layer.save(self.x)
            return {"x": tensor(layer.load())}
        out = layer.forward(self.x, self.residual)
        got = {"out": tensor(layer.read8(out) if case["do"] == "out8" else out)}
        if case["residual"]:
            got["sum"] = tensor(layer.sum)
        if case["do"] == "train":
            got["dx"], got["dgamma"] = tensor(layer.back(self.dout, self.dsum)), tensor(layer.diffGamma)
        return got


_PLAIN = {"route": _route, "norm": _norm, "keep": _keep}


def run(state):
    case = state["case"]
    return state["own"].run(case) if own else _PLAIN[case["op"]](case, state)


def work(case):
    T = case["T"]
    if case["op"] == "route":
        E, K = case["E"], case["K"]
        rows, picks = 4 * T * E, 4 * T * K
        n = {"bytes": rows + 2 * picks + 8 * E, "flops": T * E * 12}
        if case["do"] == "train":   # (the logits again where every score has a part in the gradient)
            n["bytes"] += 3 * picks + rows + (rows if case["score"] == "softmax" and not case["renorm"] else 0)
            n["flops"] += T * E * 4
        return n
    d, b = case["d"], 2 if case["dtype"] == "bf16" else 4
    whole, eight = T * d * b, T * d + (T * -(-d // INT8_GROUP) * 4 if case.get("form") != "mx" else T * -(-d // MX_GROUP))
    if case["do"] == "hold":
        return {"bytes": 2 * whole + 2 * eight, "flops": 8 * T * d}
    added = 2 if case["residual"] else 0   # the residual in, the sum out
    n = {"bytes": (1 + added) * whole + 4 * d, "flops": 8 * T * d}
    if case["do"] == "out8":
        n["bytes"] += 2 * T * d + 2 * (T * d + T * -(-d // MX_GROUP))
        return n
    n["bytes"] += whole
    if case["do"] == "train":   # rows, the output's and the sum's gradient in, the input's out
        n["bytes"] += (2 + added // 2) * whole + (2 * eight if case["op"] == "keep" else whole) + 8 * T + 4 * d
        n["flops"] += 12 * T * d
    return n


def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64
    if case["op"] == "route":
        T, E, K, G = case["T"], case["E"], case["K"], case["groups"]
        z = s["logits"].to(f)
        live = torch.isfinite(z)
        if case["score"] == "softmax":
            p = torch.where(live, z - torch.logsumexp(z, 1, keepdim=True), -math.inf).exp()
        else:
            p = torch.sigmoid(z)
        merit = torch.where(live, p + (0.0 if s["bias"] is None else s["bias"].to(f)), -math.inf)
        rank_by = merit if s["bias"] is not None else z.clone()
        if G > 1:
            m = merit.view(T, G, -1)
            first, at = m.max(2)
            if case["best"] == 2:
                second = m.scatter(2, at[:, :, None], -math.inf).amax(2)
                first = first + torch.where(torch.isfinite(second), second, torch.zeros_like(second))
            # a group stays if fewer than top_groups are better, or as good and in front of it
            a, b = first[:, :, None], first[:, None, :]
            i = torch.arange(G, device="cuda")
            better = (b > a) | ((b == a) & (i[None, :] < i[:, None]))
            rank_by.view(T, G, -1)[better.sum(2) >= case["top_groups"]] = -math.inf
        picks = []
        for _ in range(K):
            v = rank_by.amax(1, keepdim=True)
            e = (rank_by == v).int().argmax(1, keepdim=True)
            picks.append(torch.where(torch.isfinite(v), e, -1))
            rank_by.scatter_(1, e, -math.inf)
        ids = torch.cat(picks, 1)
        mine = torch.zeros(T, E, dtype=torch.bool, device="cuda")
        for k in range(K):
            mine |= torch.arange(E, device="cuda")[None] == ids[:, k:k + 1]
        share = torch.where(mine, p, torch.zeros_like(p))
        total = share.sum(1, keepdim=True)
        dense = torch.where(total > 0, share / total, torch.zeros_like(share)) if case["renorm"] else share
        at, none = ids.clamp(min=0), ids < 0
        got = {"ids": None, "w": (dense.gather(1, at) * case["scale"]).masked_fill(none, 0.0), "counts": None}
        if case["do"] == "train":
            # gradient of the dense weights, then by the rules of quotient, softmax and sigmoid
            dd = torch.zeros(T, E, dtype=f, device="cuda").scatter_add_(1, at, (s["dw"].to(f) * case["scale"]).masked_fill(none, 0.0))
            if case["renorm"]:
                dp = torch.where(mine, (dd - (dd * dense).sum(1, keepdim=True)) / torch.where(total > 0, total, torch.ones_like(total)), torch.zeros_like(dd))
            else:
                dp = torch.where(mine, dd, torch.zeros_like(dd))
            got["dlogits"] = p * (dp - (p * dp).sum(1, keepdim=True)) if case["score"] == "softmax" else dp * p * (1.0 - p)
        return got

    def int8(x):
        T, d = x.shape
        v = torch.zeros(T, -(-d // INT8_GROUP) * INT8_GROUP, dtype=f, device="cuda")
        v[:, :d] = x.to(f)
        v = v.view(T, -1, INT8_GROUP)
        # (the scale is a number of 32 bits)
        step = torch.clamp((v.abs().amax(2, keepdim=True).float() / 127.0), min=2.0 ** -126).to(f)
        n = torch.floor(v / step + 0.5)
        n = n - ((v / step + 0.5 == n) & (n.remainder(2) == 1)).to(f)
        return (n * step).reshape(T, -1)[:, :d]

    def mx(x):
        T, d = x.shape
        v = torch.zeros(T, -(-d // MX_GROUP) * MX_GROUP, dtype=f, device="cuda")
        v[:, :d] = x.to(f)
        v = v.view(T, -1, MX_GROUP)
        most = v.abs().amax(2, keepdim=True)
        k = torch.ceil(torch.log2(torch.clamp(most, min=2.0 ** -140) / E4M3_MAX)).clamp(min=-127)
        k = torch.where(E4M3_MAX * torch.exp2(k - 1) >= most, k - 1, k)   # (a logarithm next to a whole number)
        k = torch.where(E4M3_MAX * torch.exp2(k) < most, k + 1, k).clamp(min=-127)
        u = v / torch.exp2(k)
        # the nearest of what the format holds: 8 fractions of each power of two from 2^-6 on, multiples of 2^-9 below
        held = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8)][:-1]
        held = torch.tensor(held, dtype=f, device="cuda")
        up = torch.searchsorted(held, u.abs().contiguous()).clamp(max=len(held) - 1)
        low = (up - 1).clamp(min=0)
        a, b = u.abs() - held[low], held[up] - u.abs()
        at = torch.where((a < b) | ((a == b) & (low % 2 == 0)), low, up)
        return (torch.sign(v) * held[at] * torch.exp2(k)).reshape(T, -1)[:, :d]

    if case["do"] == "hold":
        return {"x": (int8 if case["form"] == "int8" else mx)(s["x"])}
    h = s["x"] if s["residual"] is None else (s["x"].to(f) + s["residual"].to(f)).to(s["x"].dtype)
    v, gamma = h.to(f), s["gamma"].to(f)
    rms = torch.sqrt(v.square().mean(1, keepdim=True) + EPS)
    y = v / rms * gamma
    got = {"out": mx(y) if case["do"] == "out8" else y}
    if case["residual"]:
        got["sum"] = s["x"].to(f) + s["residual"].to(f)
    if case["do"] == "train":
        u = int8(h) if case["op"] == "keep" else v
        dn = s["dout"].to(f) * gamma
        # gradient of u / rms, by way of the root mean square
        drms = -(dn * u).sum(1, keepdim=True) / rms ** 2
        dx = dn / rms + drms * u / (case["d"] * rms)
        got["dx"] = dx if s["dsum"] is None else dx + s["dsum"].to(f)
        got["dgamma"] = (s["dout"].to(f) * u / rms).sum(0)
    return got
