// C++ host side of what stands around the experts of a transformer block, over the C ABI of libomega_hip.so, in the manner of LmLayers.hpp
// (fp32 tensors as the reference's; bf16 buffers go through the C ABI itself):
//
//   omega::RMSLayer      RMS norm with the addition in front of it: sum = x + residual, out = norm(sum) (RMSLayer,
//                        J/engine/nn/layer/normalization/RMSLayer.java; the additions of LlamaTransformerBlock.java:129-136); may keep
//                        what it normed in 8 bits and go back from those, and then holds neither x nor the sum
//   omega::Keep8Layer    rows kept in 8 bits and brought back
//   omega::RoutingLayer  routing to experts from a gate's logits (the reference has no router)
#pragma once
#include "LmLayers.hpp"

namespace omega {

namespace detail {
// device memory of a layer's own, made when more is asked for
class Memory {
public:
    explicit Memory(Context *ctx) : ctx_(ctx) {}
    ~Memory() { omega_hip_free(ctx_->get(), ptr_); }
    Memory(const Memory &) = delete;
    Memory &operator=(const Memory &) = delete;
    void *of(size_t bytes)
    {
        if (bytes > bytes_) {
            check(ctx_->get(), omega_hip_free(ctx_->get(), ptr_));
            ptr_ = nullptr;
            bytes_ = 0;
            check(ctx_->get(), omega_hip_malloc(ctx_->get(), bytes, &ptr_));
            bytes_ = bytes;
        }
        return ptr_;
    }
    void *get() const { return ptr_; }

private:
    Context *ctx_;
    void *ptr_ = nullptr;
    size_t bytes_ = 0;
};
}  // namespace detail

class RMSLayer {
public:
    RMSLayer(int embedDim, Tensor &gamma, float eps = 1e-6f, bool keep8 = false)
        : d_(embedDim), eps_(eps), keep_(keep8), gamma_(gamma), codes_(gamma.ctx), scales_(gamma.ctx)
    {
        detail::rows_of(gamma, embedDim, "gamma shape");
        detail::want(gamma.number == 1, "gamma shape");
    }
    // sum: where x + residual goes (x or residual themselves, say); nullptr: the layer's own tensor
    Tensor &forward(Tensor &x, Tensor *residual = nullptr, Tensor *sum = nullptr)
    {
        detail::rows_of(x, d_, "input shape");
        if (residual) {
            detail::rows_of(*residual, d_, "residual shape");
            detail::want(residual->number == x.number, "residual shape");
        }
        if (sum) {
            detail::want(residual, "a sum without a residual");
            detail::rows_of(*sum, d_, "sum shape");
            detail::want(sum->number == x.number, "sum shape");
        }
        h_ = summed_ = nullptr;
        ran_ = false;  // (until the call has succeeded)
        Tensor &out = detail::sized(out_, x.number, d_, gamma_.ctx), &st = detail::sized(rstd_, 1, x.number, gamma_.ctx);
        Tensor *h = sum ? sum : residual ? &detail::sized(sum_, x.number, d_, gamma_.ctx) : nullptr;  // (an older sum stays: x may be it)
        summed_ = h;
        uint8_t *codes = keep_ ? (uint8_t *)codes_.of((size_t)x.number * d_) : nullptr;
        float *scales = keep_ ? (float *)scales_.of((size_t)x.number * ((d_ + 127) / 128) * 4) : nullptr;
        check(gamma_.ctx->get(), omega_hip_rmsnorm_forward(gamma_.ctx->get(), x.gpuData, residual ? residual->gpuData : nullptr, OMEGA_DTYPE_F32, x.number, d_,
                                                           (const float *)gamma_.gpuData, eps_, h ? h->gpuData : nullptr, out.gpuData, nullptr, nullptr,
                                                           codes, scales, (float *)st.gpuData));
        if (!keep_) h_ = h ? h : &x;
        rows_ = x.number;
        ran_ = true;
        return out;
    }
    // gradient of the input and of the residual alike; dsum: the gradient that reaches the sum past the norm
    Tensor &back(Tensor &delta, Tensor *dsum = nullptr)
    {
        detail::want(ran_, "back without a forward");
        detail::rows_of(delta, d_, "delta shape does not match the output");
        detail::want(delta.number == rows_, "delta shape does not match the output");
        if (!keep_) {
            detail::rows_of(*h_, d_, "the input has another shape than in the forward pass");
            detail::want(h_->number == rows_, "the input has another shape than in the forward pass");
        }
        if (dsum) {
            detail::rows_of(*dsum, d_, "dsum shape does not match the sum");
            detail::want(dsum->number == rows_, "dsum shape does not match the sum");
        }
        Tensor &dx = detail::sized(diff_, rows_, d_, gamma_.ctx), &dg = detail::sized(diffGamma_, 1, d_, gamma_.ctx);
        check(gamma_.ctx->get(), omega_hip_rmsnorm_backward(gamma_.ctx->get(), keep_ ? nullptr : h_->gpuData, keep_ ? (const uint8_t *)codes_.get() : nullptr,
                                                            keep_ ? (const float *)scales_.get() : nullptr, delta.gpuData, dsum ? dsum->gpuData : nullptr,
                                                            OMEGA_DTYPE_F32, rows_, d_, (const float *)gamma_.gpuData, (const float *)rstd_->gpuData, dx.gpuData,
                                                            (float *)dg.gpuData));
        return dx;
    }
    Tensor *getSum() { return summed_; }
    Tensor *getDiffGamma() { return diffGamma_.get(); }

private:
    int d_, rows_ = 0;
    float eps_;
    bool keep_, ran_ = false;
    Tensor &gamma_, *h_ = nullptr, *summed_ = nullptr;  // what back() reads, where that is not the kept rows; the last sum
    detail::Memory codes_, scales_;
    std::unique_ptr<Tensor> out_, sum_, rstd_, diff_, diffGamma_;
};

class Keep8Layer {
public:
    // form: OMEGA_KEEP8_INT8 or OMEGA_KEEP8_MX
    Keep8Layer(int embedDim, Context &ctx, int form = OMEGA_KEEP8_INT8) : d_(embedDim), form_(form), ctx_(ctx), codes_(&ctx), scales_(&ctx) {}
    void save(Tensor &x)
    {
        detail::rows_of(x, d_, "input shape");
        rows_ = -1;
        const size_t groups = form_ == OMEGA_KEEP8_MX ? (size_t)((d_ + 31) / 32) : (size_t)((d_ + 127) / 128) * 4;
        check(ctx_.get(), omega_hip_keep8_save(ctx_.get(), x.gpuData, OMEGA_DTYPE_F32, x.number, d_, form_, (uint8_t *)codes_.of((size_t)x.number * d_),
                                               scales_.of((size_t)x.number * groups)));
        rows_ = x.number;
    }
    Tensor &load()
    {
        detail::want(rows_ >= 0, "load without a save");
        Tensor &out = detail::sized(out_, rows_, d_, &ctx_);
        check(ctx_.get(), omega_hip_keep8_load(ctx_.get(), (const uint8_t *)codes_.get(), scales_.get(), form_, rows_, d_, out.gpuData, OMEGA_DTYPE_F32));
        return out;
    }

private:
    int d_, form_, rows_ = -1;
    Context &ctx_;
    detail::Memory codes_, scales_;
    std::unique_ptr<Tensor> out_;
};

class RoutingLayer {
public:
    // bias [1,E]: the caller's, for balance; nullptr: none
    RoutingLayer(const omega_route_config &config, Context &ctx, Tensor *bias = nullptr) : c_(config), ctx_(ctx), bias_(bias), ids_(&ctx), counts_(&ctx)
    {
        if (bias) {
            detail::rows_of(*bias, c_.E, "bias shape");
            detail::want(bias->number == 1, "bias shape");
        }
    }
    // weights [T,K] of the chosen experts
    Tensor &forward(Tensor &logits)
    {
        detail::rows_of(logits, c_.E, "logits shape");
        x_ = nullptr;  // (until the call has succeeded)
        Tensor &w = detail::sized(w_, logits.number, c_.K, &ctx_);
        check(ctx_.get(), omega_hip_route_forward(ctx_.get(), &c_, (const float *)logits.gpuData, logits.number, bias_ ? (const float *)bias_->gpuData : nullptr,
                                                  (int32_t *)ids_.of((size_t)logits.number * c_.K * 4), (float *)w.gpuData, (int32_t *)counts_.of((size_t)c_.E * 4)));
        x_ = &logits;
        rows_ = logits.number;
        return w;
    }
    Tensor &back(Tensor &delta)
    {
        detail::want(x_, "back without a forward");
        detail::rows_of(delta, c_.K, "delta shape does not match the weights");
        detail::want(delta.number == rows_, "delta shape does not match the weights");
        detail::rows_of(*x_, c_.E, "the logits have another shape than in the forward pass");
        detail::want(x_->number == rows_, "the logits have another shape than in the forward pass");
        Tensor &dx = detail::sized(diff_, rows_, c_.E, &ctx_);
        check(ctx_.get(), omega_hip_route_backward(ctx_.get(), &c_, (const float *)x_->gpuData, rows_, (const int32_t *)ids_.get(), (const float *)w_->gpuData,
                                                   (const float *)delta.gpuData, (float *)dx.gpuData));
        return dx;
    }
    void balance(float rate)
    {
        detail::want(x_ && bias_, "balance without a bias or a forward");
        check(ctx_.get(), omega_hip_route_balance(ctx_.get(), (const int32_t *)counts_.get(), c_.E, rate, (float *)bias_->gpuData));
    }
    std::vector<int32_t> getIds() const { return host(ids_, (size_t)(x_ ? rows_ : 0) * c_.K); }
    std::vector<int32_t> getCounts() const { return host(counts_, x_ ? (size_t)c_.E : 0); }

private:
    std::vector<int32_t> host(const detail::Memory &m, size_t n) const
    {
        std::vector<int32_t> v(n);
        if (n) check(ctx_.get(), omega_hip_memcpy_d2h(ctx_.get(), v.data(), m.get(), n * 4));
        return v;
    }
    omega_route_config c_;
    Context &ctx_;
    Tensor *bias_, *x_ = nullptr;
    int rows_ = 0;
    detail::Memory ids_, counts_;
    std::unique_ptr<Tensor> w_, diff_;
};

}  // namespace omega
