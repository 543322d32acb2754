// C++ host side of the parts of a language model around its MoE layers, over the C ABI of libomega_hip.so, in the manner of MoELayer.hpp
// (fp32 tensors as the reference's; bf16 buffers go through the C ABI itself):
//
//   omega::EmbeddingLayer  out[t] = scale * weight[ids[t]] and the weight's gradient (EmbeddingFW / EmbeddingGrad,
//                          J/engine/nn/layer/gpu/EmbeddingKernel.cu:13-56; whole ids instead of float-coded ones)
//   omega::LNLayer         layer norm over the width (J/engine/nn/layer/normalization)
//   omega::HeadLossLayer   logits = x weight^T with softmax cross entropy, no logits kept (FullyLayer.output and
//                          J/engine/gpu/SoftmaxKernel.cu:4-24 in one)
//   omega::clipGradNorm    Network.clipGradNorm over tensors and MoE layers (J/engine/nn/network/Network.java:379-432)
//
// Parameters are tensors of the caller (a table can be tied to the head); gradients lie in the layers.
#pragma once
#include "MoELayer.hpp"

namespace omega {

// whole numbers on the device (token ids, targets)
class Ids {
public:
    Ids(const std::vector<int32_t> &v, Context *cx) : n((int)v.size()), ctx(cx)
    {
        check(ctx->get(), omega_hip_malloc(ctx->get(), v.empty() ? 4 : v.size() * 4, &ptr_));
        if (n) check(ctx->get(), omega_hip_memcpy_h2d(ctx->get(), ptr_, v.data(), v.size() * 4));
    }
    ~Ids() { omega_hip_free(ctx->get(), ptr_); }
    Ids(const Ids &) = delete;
    Ids &operator=(const Ids &) = delete;
    const int32_t *gpuData() const { return (const int32_t *)ptr_; }
    const int n;
    Context *const ctx;

private:
    void *ptr_ = nullptr;
};

namespace detail {
inline void want(bool cond, const char *what)
{
    if (!cond) throw std::runtime_error(std::string("Error code 1:") + what);
}
// a layer's own tensor, made when a batch of another size comes (Layer.init)
inline Tensor &sized(std::unique_ptr<Tensor> &t, int number, int width, Context *ctx)
{
    if (!t || t->number != number || t->width != width) t.reset(new Tensor(number, 1, 1, width, ctx, true));
    return *t;
}
inline void rows_of(const Tensor &t, int width, const char *what) { want(t.width == width && t.channel * t.height == 1 && t.isHasGPU(), what); }
}  // namespace detail

class EmbeddingLayer {
public:
    EmbeddingLayer(int nVocab, int embedDim, Tensor &weight, float scale = 1.0f) : V_(nVocab), d_(embedDim), scale_(scale), w_(weight)
    {
        detail::rows_of(weight, embedDim, "weight shape");
        detail::want(weight.number == nVocab, "weight shape");
    }
    Tensor &forward(const Ids &ids)
    {
        ids_ = nullptr;  // (until the call has succeeded)
        Tensor &out = detail::sized(out_, ids.n, d_, w_.ctx);
        check(w_.ctx->get(), omega_hip_embedding_forward(w_.ctx->get(), w_.gpuData, OMEGA_DTYPE_F32, V_, d_, ids.gpuData(), ids.n, scale_, out.gpuData));
        ids_ = &ids;
        return out;
    }
    // gradient of the weight for the ids of the last forward: into the layer's own tensor, or added to `tied` (a head's gradient)
    Tensor &back(Tensor &delta, Tensor *tied = nullptr)
    {
        detail::want(ids_, "back without a forward");
        detail::rows_of(delta, d_, "delta shape does not match the output");
        detail::want(delta.number == ids_->n, "delta shape does not match the output");
        if (tied) {
            detail::rows_of(*tied, d_, "gradient shape");
            detail::want(tied->number == V_, "gradient shape");
        }
        Tensor &g = tied ? *tied : detail::sized(diffW_, V_, d_, w_.ctx);
        check(w_.ctx->get(), omega_hip_embedding_backward(w_.ctx->get(), ids_->gpuData(), ids_->n, delta.gpuData, OMEGA_DTYPE_F32, V_, d_, scale_, tied != nullptr,
                                                          g.gpuData, OMEGA_DTYPE_F32));
        return g;
    }

private:
    int V_, d_;
    float scale_;
    Tensor &w_;
    const Ids *ids_ = nullptr;
    std::unique_ptr<Tensor> out_, diffW_;
};

class LNLayer {
public:
    LNLayer(int embedDim, Tensor &gamma, Tensor &beta, float eps = 1e-5f) : d_(embedDim), eps_(eps), gamma_(gamma), beta_(beta)
    {
        for (Tensor *p : {&gamma, &beta}) {
            detail::rows_of(*p, embedDim, "gamma or beta shape");
            detail::want(p->number == 1, "gamma or beta shape");
        }
    }
    Tensor &forward(Tensor &x)
    {
        detail::rows_of(x, d_, "input shape");
        x_ = nullptr;
        Tensor &out = detail::sized(out_, x.number, d_, gamma_.ctx), &st = detail::sized(stats_, 2, x.number, gamma_.ctx);  // mean, rstd
        check(gamma_.ctx->get(), omega_hip_layernorm_forward(gamma_.ctx->get(), x.gpuData, OMEGA_DTYPE_F32, x.number, d_, (const float *)gamma_.gpuData,
                                                             (const float *)beta_.gpuData, eps_, out.gpuData, (float *)st.gpuData, (float *)st.gpuData + x.number));
        x_ = &x;
        return out;
    }
    Tensor &back(Tensor &delta)
    {
        detail::want(x_, "back without a forward");
        detail::rows_of(delta, d_, "delta shape does not match the output");
        detail::want(delta.number == x_->number, "delta shape does not match the output");
        Tensor &dx = detail::sized(diff_, x_->number, d_, gamma_.ctx), &dg = detail::sized(diffGamma_, 1, d_, gamma_.ctx), &db = detail::sized(diffBeta_, 1, d_, gamma_.ctx);
        const float *st = (const float *)stats_->gpuData;
        check(gamma_.ctx->get(), omega_hip_layernorm_backward(gamma_.ctx->get(), x_->gpuData, delta.gpuData, OMEGA_DTYPE_F32, x_->number, d_, (const float *)gamma_.gpuData,
                                                              st, st + x_->number, dx.gpuData, (float *)dg.gpuData, (float *)db.gpuData));
        return dx;
    }
    Tensor *getDiffGamma() { return diffGamma_.get(); }
    Tensor *getDiffBeta() { return diffBeta_.get(); }

private:
    int d_;
    float eps_;
    Tensor &gamma_, &beta_;
    Tensor *x_ = nullptr;
    std::unique_ptr<Tensor> out_, stats_, diff_, diffGamma_, diffBeta_;
};

class HeadLossLayer {
public:
    HeadLossLayer(int nVocab, int embedDim, Tensor &weight) : V_(nVocab), d_(embedDim), w_(weight)
    {
        detail::rows_of(weight, embedDim, "weight shape");
        detail::want(weight.number == nVocab, "weight shape");
    }
    // loss of every token (0 without a target); getMean() = mean loss over the tokens with a target, their number
    Tensor &forward(Tensor &x, const Ids &targets)
    {
        detail::rows_of(x, d_, "input shape");
        detail::want(targets.n == x.number, "targets are one a row");
        x_ = nullptr;
        Tensor &loss = detail::sized(loss_, 1, x.number, w_.ctx), &st = detail::sized(stats_, 2, x.number, w_.ctx), &mean = detail::sized(mean_, 1, 2, w_.ctx);
        check(w_.ctx->get(), omega_hip_head_loss_forward(w_.ctx->get(), x.gpuData, w_.gpuData, OMEGA_DTYPE_F32, x.number, V_, d_, targets.gpuData(), (float *)loss.gpuData,
                                                         (float *)st.gpuData, (float *)mean.gpuData));
        x_ = &x;
        y_ = &targets;
        return loss;
    }
    // gradients of the mean loss: the input's is returned, getDiffW() the weight's
    Tensor &back()
    {
        detail::want(x_, "back without a forward");
        Tensor &dx = detail::sized(diff_, x_->number, d_, w_.ctx), &dw = detail::sized(diffW_, V_, d_, w_.ctx);
        check(w_.ctx->get(), omega_hip_head_loss_backward(w_.ctx->get(), x_->gpuData, w_.gpuData, OMEGA_DTYPE_F32, x_->number, V_, d_, y_->gpuData(),
                                                          (const float *)stats_->gpuData, (const float *)mean_->gpuData, nullptr, dx.gpuData, dw.gpuData));
        return dx;
    }
    Tensor *getMean() { return mean_.get(); }
    Tensor *getDiffW() { return diffW_.get(); }

private:
    int V_, d_;
    Tensor &w_;
    Tensor *x_ = nullptr;
    const Ids *y_ = nullptr;
    std::unique_ptr<Tensor> loss_, stats_, mean_, diff_, diffW_;
};

// every tensor and the gradients of every layer times min(1, maxNorm / (norm + 1e-6)), in place; norm: two floats, the norm and the factor
inline void clipGradNorm(Context &ctx, const std::vector<Tensor *> &tensors, const std::vector<MoELayer *> &layers, float maxNorm, Tensor *norm = nullptr)
{
    std::vector<omega_grad_tensor> t;
    for (Tensor *p : tensors) t.push_back({p->gpuData, p->gpuData, p->dataLength(), OMEGA_DTYPE_F32, 0});
    std::vector<omega_moe *> l;
    for (MoELayer *m : layers) l.push_back(m->handle());
    detail::want(!norm || norm->dataLength() == 2, "norm is two floats");
    check(ctx.get(), omega_hip_clip_grad_norm(ctx.get(), t.data(), (int)t.size(), l.data(), (int)l.size(), maxNorm, norm ? (float *)norm->gpuData : nullptr));
}

}  // namespace omega
