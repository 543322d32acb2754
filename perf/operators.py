"""The operators of a language model around its layers, as cases that can be measured: token embedding and its gradient,
layer norm, the head with its softmax cross entropy, and the clipping of all gradients by their global norm.

`run` computes them in elementary torch operations, or, where `own` is true, with this repository's kernels.
"""
import importlib
import math
import random

import torch

own = False

EPS = 1e-5          # layer norm
CLIP_EPS = 1e-6     # clipping: max_norm / (norm + CLIP_EPS)
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # a decode step's tokens, one for each of 64 sequences: latency
        dict(name="embed_decode", op="embedding", do="lookup", T=64, V=32000, d=4096, dtype="bf16", scale=1.0, pad=0.0),
        # the prompt tokens of a batch, scaled rows
        dict(name="embed_prefill", op="embedding", do="lookup", T=16384, V=128000, d=2048, dtype="bf16", scale=45.25, pad=0.0),
        # gradient of a training batch with hot tokens, fp32 parameter gradients
        dict(name="embed_grad", op="embedding", do="grad", T=16384, V=128000, d=2048, dtype="bf16", scale=45.25, pad=0.05),
        # the same in fp32 at odd sizes, a padded batch
        dict(name="embed_grad_odd_f32", op="embedding", do="grad", T=2999, V=50021, d=333, dtype="f32", scale=1.0, pad=0.3),
        # norm in front of the head in a decode step
        dict(name="norm_decode", op="layer_norm", do="forward", T=64, d=4096, dtype="bf16"),
        # forward and backward of a training batch
        dict(name="norm_train", op="layer_norm", do="train", T=16384, d=2048, dtype="bf16"),
        # the same in fp32 at odd sizes
        dict(name="norm_train_odd_f32", op="layer_norm", do="train", T=4001, d=1023, dtype="f32"),
        # log probability of one token: the head's weights are read once
        dict(name="head_score_one", op="head_loss", do="score", T=1, V=128000, d=4096, dtype="bf16", pad=0.0),
        # a text scored by its tokens' losses (perplexity), odd sizes
        dict(name="head_score", op="head_loss", do="score", T=777, V=50021, d=2048, dtype="bf16", pad=0.1),
        # loss and gradients of a training batch
        dict(name="head_train", op="head_loss", do="train", T=4096, V=128000, d=4096, dtype="bf16", pad=0.05),
        # the same in fp32, the reference's type
        dict(name="head_train_f32", op="head_loss", do="train", T=1500, V=32000, d=1024, dtype="f32", pad=0.05),
        # every gradient of a network of 24 blocks
        dict(name="clip_network", op="clip", tensors=219, values=400_000_003, dtype="f32", limit=1.0),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(case):
    """Rough seconds of a pass."""
    w = work(case)
    return w["flops"] / (8e13 if case["dtype"] == "f32" else 8e14) + w["bytes"] / 3e12


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["embedding", "layer_norm", "head_loss", "head_loss", "clip"])
        dtype = rng.choice(["bf16", "bf16", "f32"])
        width = lambda hi: _spread(rng, 64, hi) if rng.random() < 0.3 else 8 * _spread(rng, 8, hi // 8)  # noqa: E731
        if op == "embedding":
            do = rng.choice(["lookup", "grad"])
            c = dict(op=op, do=do, T=_spread(rng, 1, 32768), V=_spread(rng, 1000, 128000), d=width(4096), dtype=dtype,
                     scale=rng.choice([1.0, 45.25]), pad=rng.choice([0.0, 0.0, 0.2]))
        elif op == "layer_norm":
            c = dict(op=op, do=rng.choice(["forward", "train"]), T=_spread(rng, 1, 16384), d=width(8192), dtype=dtype)
        elif op == "head_loss":
            do = rng.choice(["score", "train"])
            c = dict(op=op, do=do, T=_spread(rng, 1 if do == "score" else 64, 4096), V=_spread(rng, 1000, 128000), d=width(4096),
                     dtype=dtype, pad=rng.choice([0.0, 0.1, 0.5]))
        else:
            c = dict(op=op, tensors=_spread(rng, 1, 400), values=_spread(rng, 20_000, 400_000_000), dtype=dtype,
                     limit=rng.choice([1.0, 0.5]))
        if _cost(c) <= most:
            return c


def _sizes(case):
    """Lengths of the gradient tensors: matrices of a model beside its vectors, over four decades."""
    n, total = case["tensors"], case["values"]
    r = random.Random(n)
    w = [math.exp(r.uniform(0.0, math.log(1e4))) for _ in range(n)]
    s = [max(1, int(total * x / sum(w))) for x in w]
    s[s.index(max(s))] += total - sum(s)
    return s


def _tokens(case, gen):
    """Token numbers with the frequencies of text (the most frequent one several times in a hundred), -1 where a batch is padded."""
    T, V = case["T"], case["V"]
    u = torch.rand(T, generator=gen, device="cuda", dtype=torch.float64)
    rank = torch.exp(u * math.log(V + 1.0)).long().clamp(1, V) - 1
    ids = torch.randperm(V, generator=gen, device="cuda")[rank]
    if case["pad"]:
        ids = torch.where(torch.rand(T, generator=gen, device="cuda") < case["pad"], torch.full_like(ids, -1), ids)
    return ids.to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(std)

    s = {"case": case}
    if case["op"] == "embedding":
        T, V, d = case["T"], case["V"], case["d"]
        s["ids"] = _tokens(case, gen)
        if case["do"] == "lookup":
            s["table"] = normal(V, d, std=0.02).to(dt)
        else:
            s["dout"] = normal(T, d, std=1e-3).to(dt)
    elif case["op"] == "layer_norm":
        T, d = case["T"], case["d"]
        # rows of different sizes and a few columns that stand out, as in a deep network's residual stream
        x = normal(T, d) * torch.exp(normal(T, 1, std=0.5)) + 0.2
        x[:, torch.rand(d, generator=gen, device="cuda") < 0.005] *= 20.0
        s["x"] = x.to(dt)
        s["gamma"], s["beta"] = normal(d, std=0.1) + 1.0, normal(d, std=0.1)
        if case["do"] == "train":
            s["dout"] = normal(T, d, std=1e-3).to(dt)
    elif case["op"] == "head_loss":
        T, V, d = case["T"], case["V"], case["d"]
        s["w"] = normal(V, d, std=d ** -0.5).to(dt)
        s["targets"] = _tokens(case, gen)
        # rows that know their target more or less: its logit stands 0 to 12 over the others
        sure = torch.rand(T, 1, generator=gen, device="cuda") * 12.0
        s["x"] = (normal(T, d) + sure * s["w"][s["targets"].long().clamp(min=0)].float()).to(dt)
    else:
        s["grads"] = normal(case["values"], std=1e-3).to(dt)
    if own:
        s["own"] = _Own(case, s)
    torch.cuda.synchronize()
    return s


# ---- plain forms

def _embedding(case, s):
    ids = s["ids"].long()
    held = (ids >= 0) & (ids < case["V"])
    if case["do"] == "lookup":
        rows = s["table"][torch.where(held, ids, torch.zeros_like(ids))].float() * case["scale"]
        return {"out": torch.where(held[:, None], rows, torch.zeros_like(rows)).to(s["table"].dtype)}
    grad = torch.zeros(case["V"] + 1, case["d"], device="cuda")
    grad.index_add_(0, torch.where(held, ids, torch.full_like(ids, case["V"])), s["dout"].float())
    return {"dtable": grad[:-1].mul_(case["scale"])}


def _layer_norm(case, s):
    x = s["x"].float()
    xc = x - x.mean(1, keepdim=True)
    r = torch.rsqrt((xc * xc).mean(1, keepdim=True) + EPS)
    xh = xc * r
    got = {"out": (xh * s["gamma"] + s["beta"]).to(s["x"].dtype)}
    if case["do"] == "train":
        dy = s["dout"].float()
        g = dy * s["gamma"]
        dx = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
        got.update(dx=dx.to(s["x"].dtype), dgamma=(dy * xh).sum(0), dbeta=dy.sum(0))
    return got


def _head_loss(case, s):
    x, w, y = s["x"].float(), s["w"].float(), s["targets"].long()
    held = (y >= 0) & (y < case["V"])
    at = torch.where(held, y, torch.zeros_like(y))[:, None]
    logits = x @ w.t()
    top = logits.max(1, keepdim=True).values
    e = torch.exp(logits - top)
    total = e.sum(1, keepdim=True)
    loss = torch.where(held, (top + torch.log(total) - logits.gather(1, at))[:, 0], torch.zeros_like(total[:, 0]))
    n = held.sum().clamp(min=1)
    got = {"loss": loss, "mean": loss.sum() / n}
    if case["do"] == "train":
        p = e / total
        p.scatter_add_(1, at, -torch.ones_like(total))
        p *= (held / n).to(p.dtype)[:, None]
        got.update(dx=(p @ w).to(s["x"].dtype), dw=(p.t() @ x).to(s["w"].dtype))
    return got


def _clip(case, s):
    g = s["grads"].float()
    norm = torch.sqrt(g.square().sum(dtype=torch.float64))
    coef = torch.clamp(case["limit"] / (norm + CLIP_EPS), max=1.0).float()
    return {"norm": norm.float(), "clipped": (g * coef).to(s["grads"].dtype)}


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
                                         "typestr": "<i2" if buf.dtype == "bf16" else "<f4", "strides": None}


class _Own:
    """The layer of a case and its buffers, as a program keeps them."""

    def __init__(self, case, s):
        global _ctx
        self.P = P = importlib.import_module("omega-ai_amd")
        if _ctx is None:
            _ctx = P.Context(0)
        self.seen = {}
        if case["op"] == "embedding":
            self.layer = P.EmbeddingLayer(case["V"], case["d"], scale=case["scale"], ctx=_ctx, dtype=case["dtype"],
                                          weight=self.buffer(s["table"]) if "table" in s else None)
            self.ids = self.buffer(s["ids"])
        elif case["op"] == "layer_norm":
            self.layer = P.LNLayer(case["d"], eps=EPS, ctx=_ctx, dtype=case["dtype"], gamma=self.buffer(s["gamma"]),
                                   beta=self.buffer(s["beta"]))
            self.x = self.buffer(s["x"])
        elif case["op"] == "head_loss":
            self.layer = P.HeadLossLayer(case["V"], case["d"], ctx=_ctx, dtype=case["dtype"], weight=self.buffer(s["w"]))
            self.x, self.targets = self.buffer(s["x"]), self.buffer(s["targets"])
        else:
            self.out = torch.empty_like(s["grads"])
            sizes = _sizes(case)
            self.layer = P.GradClip(_ctx, [self.buffer(t) for t in s["grads"].split(sizes)],
                                    out=[self.buffer(t) for t in self.out.split(sizes)])
        self.held = _Held(self.layer)
        if "dout" in s:
            self.dout = self.buffer(s["dout"])

    def buffer(self, t):
        dtype = {torch.bfloat16: "bf16", torch.float32: "f32", torch.int32: "i32"}[t.dtype]
        return self.P.DeviceBuffer.wrap(_ctx, t.data_ptr(), tuple(t.shape), dtype)

    def tensor(self, buf):
        t = self.seen.get(buf.ptr.value)
        if t is None:
            t = torch.as_tensor(_Memory(self.held, buf), device="cuda")
            t = self.seen[buf.ptr.value] = t.view(torch.bfloat16) if buf.dtype == "bf16" else t
        return t

    def run(self, case):
        if case["op"] == "embedding":
            if case["do"] == "lookup":
                return {"out": self.tensor(self.layer.forward(self.ids))}
            return {"dtable": self.tensor(self.layer.back(self.dout, self.ids))}
        if case["op"] == "layer_norm":
            got = {"out": self.tensor(self.layer.forward(self.x))}
            if case["do"] == "train":
                got["dx"] = self.tensor(self.layer.back(self.dout))
                got["dgamma"], got["dbeta"] = self.tensor(self.layer.diffGamma), self.tensor(self.layer.diffBeta)
            return got
        if case["op"] == "head_loss":
            got = {"loss": self.tensor(self.layer.forward(self.x, self.targets)), "mean": self.tensor(self.layer.mean)[0]}
            if case["do"] == "train":
                got["dx"] = self.tensor(self.layer.back())
                got["dw"] = self.tensor(self.layer.diffW)
            return got
        return {"norm": self.tensor(self.layer.clip(case["limit"]))[0], "clipped": self.out}


_PLAIN = {"embedding": _embedding, "layer_norm": _layer_norm, "head_loss": _head_loss, "clip": _clip}


def run(state):
    case = state["case"]
    return state["own"].run(case) if own else _PLAIN[case["op"]](case, state)


def work(case):
    b = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "clip":
        return {"bytes": 2 * case["values"] * b, "flops": 3 * case["values"]}
    T, d = case["T"], case["d"]
    if case["op"] == "layer_norm":
        # x in, y out; training: the output's gradient in, the input's and the parameters' out
        return {"bytes": (4 if case["do"] == "train" else 2) * T * d * b + (16 if case["do"] == "train" else 8) * d,
                "flops": (20 if case["do"] == "train" else 8) * T * d}
    V = case["V"]
    if case["op"] == "embedding":
        if case["do"] == "lookup":
            return {"bytes": 2 * T * d * b + 4 * T, "flops": T * d}
        return {"bytes": T * d * b + 4 * T + 4 * V * d, "flops": 2 * T * d}
    if case["do"] == "score":
        return {"bytes": (T + V) * d * b + 8 * T, "flops": 2 * T * V * d}
    return {"bytes": 2 * (T + V) * d * b + 8 * T, "flops": 6 * T * V * d}


def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64
    if case["op"] == "embedding":
        ids, V = s["ids"].long(), case["V"]
        keep = torch.nonzero((ids >= 0) & (ids < V))[:, 0]
        src = (s["table"] if case["do"] == "lookup" else s["dout"]).to(f)
        if case["do"] == "lookup":
            out = torch.zeros(case["T"], case["d"], device="cuda", dtype=f)
            out[keep] = src[ids[keep]] * case["scale"]
            return {"out": out}
        out = torch.zeros(V, case["d"], device="cuda", dtype=f)
        return {"dtable": out.index_add_(0, ids[keep], src[keep] * case["scale"])}
    if case["op"] == "layer_norm":
        x, gamma = s["x"].to(f), s["gamma"].to(f)
        var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
        std = torch.sqrt(var + EPS)
        n = (x - mean) / std
        got = {"out": n * gamma + s["beta"].to(f)}
        if case["do"] == "train":
            dy = s["dout"].to(f)
            dn = dy * gamma
            # gradient of (x - mean) / std, by way of the two moments
            dvar = -0.5 * (dn * (x - mean)).sum(1, keepdim=True) / std ** 3
            dmean = -dn.sum(1, keepdim=True) / std
            got.update(dx=dn / std + (2.0 * dvar * (x - mean) + dmean) / case["d"], dgamma=(dy * n).sum(0), dbeta=dy.sum(0))
        return got
    if case["op"] == "head_loss":
        x, w, y = s["x"].to(f), s["w"].to(f), s["targets"].long()
        keep = torch.nonzero((y >= 0) & (y < case["V"]))[:, 0]
        n = max(1, keep.numel())
        logp = torch.log_softmax(x[keep] @ w.t(), 1)
        rows = torch.arange(keep.numel(), device="cuda")
        loss = torch.zeros(case["T"], device="cuda", dtype=f)
        loss[keep] = -logp[rows, y[keep]]
        got = {"loss": loss, "mean": loss.sum() / n}
        if case["do"] == "train":
            p = logp.exp_()
            p[rows, y[keep]] -= 1.0
            dx = torch.zeros(case["T"], case["d"], device="cuda", dtype=f)
            dx[keep] = p @ w / n
            got.update(dx=dx, dw=p.t() @ x[keep] / n)
        return got
    g = s["grads"].to(f)
    norm = torch.linalg.vector_norm(g)
    return {"norm": norm, "clipped": g * torch.clamp(case["limit"] / (norm + CLIP_EPS), max=1.0)}
