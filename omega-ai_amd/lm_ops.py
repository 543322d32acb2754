"""The parts of a language model around its MoE layers, over the C ABI: token embedding, layer norm, the head with its softmax
cross entropy, and the clipping of all gradients of a network by their global norm.

Classes keep the house style of the layers (moe_layer.py): forward(input) returns the layer's own output buffer, back(delta) the
input gradient, parameter gradients lie beside the parameters (diffW, diffGamma, ...); a parameter may be a buffer of the caller
(weight=..., gamma=...), so that a table can be tied to the head.  A non-zero status raises RuntimeError("Error code N:msg").
"""
import ctypes as C

from . import _lib as L
from .moe_layer import Context, DeviceBuffer

_DT = {"f32": L.DTYPE_F32, "bf16": L.DTYPE_BF16}


def _want(cond, what):
    if not cond:
        raise RuntimeError("Error code 1:" + what)


class _Param:
    """A parameter of a layer, a buffer of the caller: looked at whenever it is set, since the kernels read it with the layer's sizes.  (One
    that is freed later has no address, which the calls refuse.  Reading it is an ordinary look into the layer: this class has no __get__,
    which would cost a decode step's lookup 0.25 of 4 us.)"""

    def __init__(self, shape, dtype):
        self.shape, self.dtype = shape, dtype   # functions of the layer

    def __set_name__(self, owner, name):
        self.name = name

    def __set__(self, layer, buf):
        if buf is not None:
            _want(buf.shape == self.shape(layer) and buf.dtype == self.dtype(layer), self.name + " shape or dtype")
            _want(buf.ptr, self.name + " has been freed")
        layer.__dict__[self.name] = buf


class _Layer:
    """Buffers of a layer: made when a batch of another size comes (Layer.init), given back by close()."""

    def __init__(self, ctx, dtype):
        _want(dtype in _DT, "dtype is f32 or bf16")
        self.ctx = ctx or Context(0)
        self.lib, self.dtype, self._owned = self.ctx.lib, dtype, {}

    def _buffer(self, name, shape, dtype):
        buf = self._owned.get(name)
        if buf is None or buf.shape != shape or buf.dtype != dtype:
            if buf is not None:
                buf.free()
            self._owned[name] = None
            buf = self._owned[name] = DeviceBuffer(self.ctx, shape, dtype)
        return buf

    def close(self):
        for buf in self._owned.values():
            if buf is not None:
                buf.free()
        self._owned = {}
        for view in (getattr(self, "diffGamma", None), getattr(self, "diffBeta", None)):
            if view is not None:
                view.free()   # (into a buffer that has gone)
        self.input = self.diffW = self.diffGamma = self.diffBeta = None


class EmbeddingLayer(_Layer):
    """out[t] = scale * weight[ids[t]] (an id outside 0..nVocab-1: zeros) and its gradient by sorted tokens
    (EmbeddingFW / EmbeddingGrad, J/engine/nn/layer/gpu/EmbeddingKernel.cu:13-56)."""

    weight = _Param(lambda layer: (layer.nVocab, layer.embedDim), lambda layer: layer.dtype)

    def __init__(self, nVocab, embedDim, scale=1.0, ctx=None, dtype="f32", weight=None, gradDtype="f32"):
        super().__init__(ctx, dtype)
        _want(gradDtype in _DT, "gradDtype is f32 or bf16")
        self.nVocab, self.embedDim, self.scale, self.gradDtype = nVocab, embedDim, float(scale), gradDtype
        self.weight = weight
        self.input = self.diffW = None

    def forward(self, ids):
        _want(ids.dtype == "i32" and len(ids.shape) == 1, "ids are a vector of i32")
        _want(self.weight is not None, "the layer has no weight")
        self.input, T = None, ids.shape[0]   # (until the call has succeeded)
        out = self._buffer("out", (T, self.embedDim), self.dtype)
        self.ctx.check(self.lib.omega_hip_embedding_forward(self.ctx.handle, self.weight.ptr, _DT[self.dtype], self.nVocab, self.embedDim, ids.ptr, T,
                                                            self.scale, out.ptr))
        self.input = ids
        return out

    def back(self, delta, ids=None, diffW=None):
        """Gradient of the weight from the output's gradient `delta`, for the ids of the last forward() or for `ids`: into the layer's
        own diffW (gradDtype, overwritten), or added to the buffer `diffW` of the caller (a tied head's gradient)."""
        ids = self.input if ids is None else ids
        _want(ids is not None, "back without a forward")
        _want(ids.dtype == "i32" and len(ids.shape) == 1, "ids are a vector of i32")
        _want(delta.shape == (ids.shape[0], self.embedDim) and delta.dtype == self.dtype, "delta shape or dtype does not match the output")
        add = diffW is not None
        if add:
            _want(diffW.shape == (self.nVocab, self.embedDim) and diffW.dtype in _DT, "diffW shape or dtype")
        else:
            diffW = self._buffer("diffW", (self.nVocab, self.embedDim), self.gradDtype)
        self.diffW = diffW
        self.ctx.check(self.lib.omega_hip_embedding_backward(self.ctx.handle, ids.ptr, ids.shape[0], delta.ptr, _DT[self.dtype], self.nVocab, self.embedDim,
                                                             self.scale, int(add), diffW.ptr, _DT[diffW.dtype]))
        return diffW


class LNLayer(_Layer):
    """Layer norm over the last dimension (J/engine/nn/layer/normalization): gamma and beta fp32, as the RMSNorm's gamma of the MoE layer."""

    gamma = _Param(lambda layer: (layer.embedDim,), lambda layer: "f32")
    beta = _Param(lambda layer: (layer.embedDim,), lambda layer: "f32")

    def __init__(self, embedDim, eps=1e-5, ctx=None, dtype="f32", gamma=None, beta=None):
        super().__init__(ctx, dtype)
        self.embedDim, self.eps = embedDim, float(eps)
        self.gamma, self.beta = gamma, beta
        self.input = self.diffGamma = self.diffBeta = None

    def forward(self, x):
        _want(len(x.shape) == 2 and x.shape[1] == self.embedDim and x.dtype == self.dtype, "input shape or dtype")
        _want(self.gamma is not None and self.beta is not None, "the layer has no gamma or beta")
        self.input, T = None, x.shape[0]
        out = self._buffer("out", x.shape, self.dtype)
        stats = self._buffer("stats", (2, T), "f32")   # mean, then rstd
        self.ctx.check(self.lib.omega_hip_layernorm_forward(self.ctx.handle, x.ptr, _DT[self.dtype], T, self.embedDim, self.gamma.ptr, self.beta.ptr, self.eps,
                                                            out.ptr, stats.ptr, stats.ptr.value + 4 * T))
        self.input = x
        return out

    def back(self, delta):
        """Input gradient for the input of the last forward(); the parameters' gradients are diffGamma and diffBeta."""
        x = self.input
        _want(x is not None, "back without a forward")
        _want(delta.shape == x.shape and delta.dtype == self.dtype, "delta shape or dtype does not match the output")
        dx = self._buffer("diff", x.shape, self.dtype)
        if self.diffGamma is None:
            both = self._buffer("diffParams", (2, self.embedDim), "f32")
            self.diffGamma, self.diffBeta = (DeviceBuffer.wrap(self.ctx, both.ptr.value + 4 * k * self.embedDim, (self.embedDim,), "f32") for k in (0, 1))
        stats, T = self._owned["stats"], x.shape[0]
        self.ctx.check(self.lib.omega_hip_layernorm_backward(self.ctx.handle, x.ptr, delta.ptr, _DT[self.dtype], x.shape[0], self.embedDim, self.gamma.ptr,
                                                             stats.ptr, stats.ptr.value + 4 * T, dx.ptr, self.diffGamma.ptr, self.diffBeta.ptr))
        return dx


class HeadLossLayer(_Layer):
    """logits = x weight^T, softmax cross entropy against targets and its gradients, in pieces of the vocabulary: no logits are kept
    (FullyLayer.output and the softmax of J/engine/gpu/SoftmaxKernel.cu:4-24 in one)."""

    weight = _Param(lambda layer: (layer.nVocab, layer.embedDim), lambda layer: layer.dtype)

    def __init__(self, nVocab, embedDim, ctx=None, dtype="f32", weight=None):
        super().__init__(ctx, dtype)
        self.nVocab, self.embedDim = nVocab, embedDim
        self.weight = weight
        self.input = self.targets = self.mean = self.diffW = None

    def forward(self, x, targets):
        """loss [T] (0 where the target is outside 0..nVocab-1); mean [2] = mean loss over the tokens with a target, their number."""
        _want(len(x.shape) == 2 and x.shape[1] == self.embedDim and x.dtype == self.dtype, "input shape or dtype")
        _want(targets.shape == (x.shape[0],) and targets.dtype == "i32", "targets are one i32 a row")
        _want(self.weight is not None, "the layer has no weight")
        self.input, self.targets, T = None, targets, x.shape[0]
        loss, stats = self._buffer("loss", (T,), "f32"), self._buffer("stats", (2, T), "f32")
        self.mean = self._buffer("mean", (2,), "f32")
        self.ctx.check(self.lib.omega_hip_head_loss_forward(self.ctx.handle, x.ptr, self.weight.ptr, _DT[self.dtype], T, self.nVocab, self.embedDim, targets.ptr,
                                                            loss.ptr, stats.ptr, self.mean.ptr))
        self.input = x
        return loss

    def back(self, dloss=None, input_gradient=True, weight_gradient=True):
        """Gradients of dloss * mean loss (dloss: a buffer of one f32, None = 1) of the last forward(): returns the input's, diffW is the
        weight's (both of the layer's dtype)."""
        x = self.input
        _want(x is not None, "back without a forward")
        _want(dloss is None or (dloss.shape == (1,) and dloss.dtype == "f32" and dloss.ptr), "dloss is one f32")   # (no address would mean 1)
        dx = self._buffer("diff", x.shape, self.dtype) if input_gradient else None
        self.diffW = self._buffer("diffW", (self.nVocab, self.embedDim), self.dtype) if weight_gradient else None
        self.ctx.check(self.lib.omega_hip_head_loss_backward(self.ctx.handle, x.ptr, self.weight.ptr, _DT[self.dtype], x.shape[0], self.nVocab, self.embedDim,
                                                             self.targets.ptr, self._owned["stats"].ptr, self.mean.ptr, dloss.ptr if dloss else None,
                                                             dx.ptr if dx else None, self.diffW.ptr if self.diffW else None))
        return dx


class GradClip:
    """Network.clipGradNorm (J/engine/nn/network/Network.java:379-432) over the gradient buffers of a network and its MoE layers, without
    a copy to the host: tensors are scaled in place, or into `out`; the layers' gradients in place."""

    def __init__(self, ctx, tensors, layers=(), out=None):
        self.ctx, self.lib = ctx, ctx.lib
        out = tensors if out is None else out
        _want(len(out) == len(tensors), "as many outputs as tensors")
        self._kept = (list(tensors), list(out), list(layers))   # (their memory stays while the list does)
        self._list = (L.GradTensorStruct * max(len(tensors), 1))()
        for e, src, dst in zip(self._list, tensors, out):
            _want(src.dtype in _DT and dst.dtype == src.dtype and dst.shape == src.shape, "gradient shape or dtype")
            e.src, e.dst, e.n, e.dtype, e.reserved = src.ptr.value, dst.ptr.value, src.size, _DT[src.dtype], 0
        self._layers = (C.c_void_p * max(len(layers), 1))()
        self.norm = DeviceBuffer(ctx, (2,), "f32")

    def clip(self, maxNorm):
        """Scales by min(1, maxNorm / (norm + 1e-6)); returns the buffer of norm and coefficient."""
        tensors, out, layers = self._kept
        _want(self.norm.ptr, "the clip has been closed")
        _want(all(b.ptr for b in tensors) and all(b.ptr for b in out), "a gradient buffer has been freed")
        for i, layer in enumerate(layers):
            self._layers[i] = layer.handle   # (None once it is closed: refused)
        self.ctx.check(self.lib.omega_hip_clip_grad_norm(self.ctx.handle, self._list, len(tensors), self._layers, len(layers), float(maxNorm), self.norm.ptr))
        return self.norm

    def close(self):
        self.norm.free()
