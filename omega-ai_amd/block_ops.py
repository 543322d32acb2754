"""What stands around the experts of a transformer block, over the C ABI: routing to experts, RMS norm with the residual's addition, rows
kept in 8 bits.

Classes in the manner of lm_ops.py: forward(input) returns the layer's own output buffer, back(delta) the input gradient, parameter
gradients lie beside the parameters.
"""
import ctypes as C

from . import _lib as L
from .lm_ops import _DT, _Layer, _Param, _want

_SCORES = {"softmax": L.ROUTE_SOFTMAX, "sigmoid": L.ROUTE_SIGMOID}


def route_config(nExperts, topK, score="softmax", renorm=True, scale=1.0, nGroups=1, topGroups=None, groupBest=2):
    """omega_route_config: scores (softmax or sigmoid) of nExperts in nGroups groups, of which the topGroups (None: all) with the best sum of their
    groupBest best stay; topK chosen, their weights times scale, divided by their sum with renorm."""
    _want(score in _SCORES, "score is softmax or sigmoid")
    return L.RouteConfigStruct(nExperts, topK, _SCORES[score], int(bool(renorm)), nGroups, nGroups if topGroups is None else topGroups, groupBest, float(scale))


class RoutingLayer(_Layer):
    """Routing of tokens to experts from the logits of a gate (fp32; the reference has no router): forward(logits) returns the weights of the chosen
    experts [T,topK], ids [T,topK] are their numbers (-1 where none was open) and counts [nExperts] the tokens of each.

    bias: the caller's buffer for balance; it takes part in the choice only, and balance(rate) moves it by the last counts."""

    bias = _Param(lambda layer: (layer.nExperts,), lambda layer: "f32")

    def __init__(self, nExperts, topK, score="softmax", renorm=True, scale=1.0, nGroups=1, topGroups=None, groupBest=2, ctx=None, bias=None):
        super().__init__(ctx, "f32")
        self.nExperts, self.topK = nExperts, topK
        self._config = route_config(nExperts, topK, score, renorm, scale, nGroups, topGroups, groupBest)
        self._by = C.byref(self._config)
        self.bias = bias
        self.input = self.w = self.ids = self.counts = None

    def forward(self, logits):
        shape = logits.shape
        _want(len(shape) == 2 and shape[1] == self.nExperts and logits.dtype == "f32", "logits shape or dtype")
        bias = self.bias
        _want(bias is None or bias.ptr, "bias has been freed")   # (no address would mean none)
        self.input, T = None, shape[0]   # (until the call has succeeded)
        w, ids = self._buffer("w", (T, self.topK), "f32"), self._buffer("ids", (T, self.topK), "i32")
        counts = self._buffer("counts", (self.nExperts,), "i32")
        self.ctx.check(self.lib.omega_hip_route_forward(self.ctx.handle, self._by, logits.ptr, T, bias.ptr if bias else None, ids.ptr, w.ptr, counts.ptr))
        self.input, self.w, self.ids, self.counts = logits, w, ids, counts
        return w

    def back(self, delta):
        """Gradient of the logits of the last forward() from that of its weights."""
        x = self.input
        _want(x is not None, "back without a forward")
        _want(delta.shape == self.w.shape and delta.dtype == "f32", "delta shape or dtype does not match the weights")
        dx = self._buffer("diff", x.shape, "f32")
        self.ctx.check(self.lib.omega_hip_route_backward(self.ctx.handle, self._by, x.ptr, x.shape[0], self.ids.ptr, self.w.ptr, delta.ptr, dx.ptr))
        return dx

    def balance(self, rate):
        """bias -+= rate for the experts that the last forward() gave more or fewer tokens than the mean."""
        _want(self.bias is not None and self.counts is not None, "balance without a bias or a forward")
        self.ctx.check(self.lib.omega_hip_route_balance(self.ctx.handle, self.counts.ptr, self.nExperts, float(rate), self.bias.ptr))

    def close(self):
        super().close()
        self.w = self.ids = self.counts = None


_FORMS = {"int8": L.KEEP8_INT8, "mx": L.KEEP8_MX}
_GROUP = {"int8": 128, "mx": 32}


class Rows8:
    """Rows held in 8 bits: codes [T,d] and a scale for every group of a row (form "int8": of 128 elements, fp32; "mx": of 32, a byte)."""

    def __init__(self, form, shape, codes, scales):
        _want(form in _FORMS, "form is int8 or mx")
        _want(len(shape) == 2 and codes.shape == tuple(shape) and codes.dtype == "u8", "codes shape or dtype")
        _want((scales.shape, scales.dtype) == _scales(form, shape), "scales shape or dtype")
        self.form, self.shape, self.codes, self.scales = form, codes.shape, codes, scales


def _scales(form, shape):
    """Shape and dtype of the scales of rows of `shape`."""
    return (shape[0], -(-shape[1] // _GROUP[form])), "f32" if form == "int8" else "u8"


def _rows8(layer, name, form, shape):
    """The layer's own buffers of that name for rows of `shape`."""
    rows = layer.__dict__.get(name)
    if rows is None or rows.shape != shape or not rows.codes.ptr:
        layer.__dict__[name] = None
        codes = layer._buffer(name, shape, "u8")
        rows = layer.__dict__[name] = Rows8(form, shape, codes, layer._buffer(name + "_scales", *_scales(form, shape)))
    return rows


def _load8(layer, name, rows, dtype):
    """`rows` as elements of dtype, in the layer's own buffer of that name."""
    out = layer._buffer(name, rows.shape, dtype)
    layer.ctx.check(layer.lib.omega_hip_keep8_load(layer.ctx.handle, rows.codes.ptr, rows.scales.ptr, _FORMS[rows.form], rows.shape[0], rows.shape[1], out.ptr,
                                                   _DT[dtype]))
    return out


class RMSLayer(_Layer):
    """RMS norm over the last dimension (RMSLayer, J/engine/nn/layer/normalization/RMSLayer.java), with the addition in front of it
    (LlamaTransformerBlock.output, J/engine/nn/layer/llama/LlamaTransformerBlock.java:129-136): sum = x + residual, out = norm(sum).

    out8: the output is Rows8 of the form "mx" (read8 brings them back); keep8: the forward pass keeps what was normed in 8 bits and the
    backward pass reads those.  Then the layer holds neither x nor the sum after forward(); the sum takes no memory of its own where forward() is given a
    buffer for it, which may be the residual."""

    gamma = _Param(lambda layer: (layer.embedDim,), lambda layer: "f32")

    def __init__(self, embedDim, eps=1e-6, ctx=None, dtype="f32", gamma=None, out8=False, keep8=False):
        super().__init__(ctx, dtype)
        self.embedDim, self.eps, self.out8, self.keep8 = embedDim, float(eps), bool(out8), bool(keep8)
        self.gamma = gamma
        self.input = self.sum = self.kept = self.diffGamma = self._for = self._rows = None

    def _ready(self, x, summed):
        """What a batch like x is written to: sum (the layer's own), rstd, out, out8, kept.  (Made, and x looked at, when another batch comes: both again for every call would cost a
        decode step's 1.5 of 5 us.)"""
        shape = x.shape
        _want(len(shape) == 2 and shape[1] == self.embedDim and x.dtype == self.dtype, "input shape or dtype")
        self.input = self._rows = self._for = None
        self._held = (self._buffer("sum", shape, self.dtype) if summed else None, self._buffer("rstd", (shape[0],), "f32"),
                      None if self.out8 else self._buffer("out", shape, self.dtype), _rows8(self, "rows8_out", "mx", shape) if self.out8 else None,
                      _rows8(self, "rows8_kept", "int8", shape) if self.keep8 else None)

    def forward(self, x, residual=None, sum=None):
        """norm(x + residual); the sum is self.sum (None without a residual), written to the buffer `sum` of the caller (x or residual themselves, say) or
        to the layer's own."""
        shape, gamma, ctx = x.shape, self.gamma, self.ctx
        _want(gamma is not None, "the layer has no gamma")
        if residual is not None:
            _want(residual.shape == shape and residual.dtype == x.dtype and residual.ptr, "residual shape or dtype")   # (no address would mean none)
        if sum is not None:
            _want(residual is not None, "a sum without a residual")
            _want(sum.shape == shape and sum.dtype == x.dtype, "sum shape or dtype")
        batch = (shape, x.dtype, residual is None or sum is not None, self.out8, self.keep8)
        if batch != self._for:
            self._ready(x, not batch[2])
            self._for = batch
        h, rstd, out, o8, kept = self._held
        if sum is not None:
            h = sum
        self.input, self._rows, self.sum = None, None, h   # (no rows until the call has succeeded)
        if h is not None:
            _want(h.ptr, "sum has been freed")
        st = self.lib.omega_hip_rmsnorm_forward(
            ctx.handle, x.ptr, residual.ptr if h else None, _DT[x.dtype], shape[0], shape[1], gamma.ptr, self.eps, h.ptr if h else None,
            out.ptr if out else None, o8.codes.ptr if o8 else None, o8.scales.ptr if o8 else None, kept.codes.ptr if kept else None,
            kept.scales.ptr if kept else None, rstd.ptr)
        if st:
            ctx.check(st)
        self._rows, self.kept = shape, kept
        if kept is None:
            self.input = x if h is None else h
        return out or o8

    def read8(self, rows, dtype="bf16"):
        """Rows8 as elements of dtype (bf16 holds every value of the form "mx")."""
        _want(dtype in _DT, "dtype is f32 or bf16")
        return _load8(self, "read8", rows, dtype)

    def back(self, delta, dsum=None):
        """Gradient of x and of the residual alike, for the last forward(); dsum: the gradient that reaches the sum past the norm.  gamma's is diffGamma."""
        h, rows, kept = self.input, self._rows, self.kept
        _want(rows is not None, "back without a forward")
        _want(delta.shape == rows and delta.dtype == self.dtype, "delta shape or dtype does not match the output")
        _want(dsum is None or (dsum.shape == rows and dsum.dtype == self.dtype and dsum.ptr), "dsum shape or dtype does not match the sum")
        _want(self.gamma is not None, "the layer has no gamma")
        dx = self._buffer("diff", rows, self.dtype)
        self.diffGamma = dg = self._buffer("diffGamma", (self.embedDim,), "f32")
        self.ctx.check(self.lib.omega_hip_rmsnorm_backward(
            self.ctx.handle, None if kept else h.ptr, kept.codes.ptr if kept else None, kept.scales.ptr if kept else None, delta.ptr,
            dsum.ptr if dsum else None, _DT[self.dtype], rows[0], self.embedDim, self.gamma.ptr, self._owned["rstd"].ptr, dx.ptr, dg.ptr))
        return dx

    def close(self):
        super().close()
        self.sum = self.kept = self._for = self._held = self._rows = None


class Keep8Layer(_Layer):
    """Rows kept in 8 bits between a forward pass and its backward pass: save(x) keeps them, load() brings them back (the reference keeps
    activations whole)."""

    def __init__(self, embedDim, form="int8", ctx=None, dtype="f32"):
        super().__init__(ctx, dtype)
        _want(form in _FORMS, "form is int8 or mx")
        self.embedDim, self.form, self.kept = embedDim, form, None

    def save(self, x):
        _want(len(x.shape) == 2 and x.shape[1] == self.embedDim and x.dtype == self.dtype, "input shape or dtype")
        self.kept = None
        rows = _rows8(self, "rows8", self.form, x.shape)
        self.ctx.check(self.lib.omega_hip_keep8_save(self.ctx.handle, x.ptr, _DT[self.dtype], x.shape[0], x.shape[1], _FORMS[self.form], rows.codes.ptr,
                                                     rows.scales.ptr))
        self.kept = rows
        return rows

    def load(self):
        """The rows of the last save()."""
        _want(self.kept is not None, "load without a save")
        return _load8(self, "out", self.kept, self.dtype)

    def close(self):
        super().close()
        self.kept = None
