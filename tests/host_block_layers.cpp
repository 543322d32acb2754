// The C++ layers around the experts against the stand-ins of the C ABI's launchers: inputs that are a layer's own buffers, and refusals.
#include <cstdio>

#include "BlockLayers.hpp"

static int g_failed = 0;
#define EXPECT(c)                                                                   \
    do {                                                                            \
        if (!(c)) { printf("line %d: %s\n", __LINE__, #c); ++g_failed; }            \
    } while (0)
template <class F> static bool refuses(F f, const char *what)
{
    try {
        f();
    } catch (const std::runtime_error &e) {
        return std::string(e.what()).find(what) != std::string::npos;
    }
    return false;
}

int main()
{
    omega::Context ctx(0);
    auto rows = [&](int n, int d) { return std::unique_ptr<omega::Tensor>(new omega::Tensor(n, 1, 1, d, &ctx, true)); };
    auto x = rows(6, 40), r = rows(6, 40), more = rows(7, 40), wide = rows(6, 41), gamma = rows(1, 40);
    {
        omega::RMSLayer norm(40, *gamma);
        EXPECT(refuses([&] { norm.back(*x); }, "without a forward"));
        EXPECT(refuses([&] { norm.forward(*wide); }, "input shape"));
        EXPECT(refuses([&] { norm.forward(*x, more.get()); }, "residual shape"));
        norm.forward(*x, r.get());
        omega::Tensor *sum = norm.getSum();
        EXPECT(sum && sum->number == 6);
        EXPECT(&norm.back(*x, r.get()) != nullptr && norm.getDiffGamma());
        norm.forward(*sum);             // the sum as the next input, with nothing added
        EXPECT(norm.getSum() == nullptr && sum->number == 6 && sum->gpuData);
        norm.back(*x);
        norm.forward(*sum, r.get());    // in place
        EXPECT(norm.getSum() == sum);
        EXPECT(refuses([&] { norm.back(*more); }, "delta shape"));
        EXPECT(refuses([&] { norm.back(*x, more.get()); }, "dsum shape"));
        norm.forward(*x);
        x->number = 5;
        EXPECT(refuses([&] { norm.back(*r); }, "another shape"));
        x->number = 6;
        omega::RMSLayer kept(40, *gamma, 1e-6f, true);
        auto gone = rows(6, 40);
        kept.forward(*gone);
        gone.reset();
        kept.back(*x);                  // the kept rows are enough
    }
    {
        omega::Keep8Layer keep(40, ctx, OMEGA_KEEP8_MX);
        EXPECT(refuses([&] { keep.load(); }, "without a save"));
        keep.save(*x);
        EXPECT(keep.load().number == 6);
        EXPECT(refuses([&] { keep.save(*wide); }, "input shape"));
        EXPECT(keep.load().number == 6);
    }
    {
        auto z = rows(6, 16), dw = rows(6, 4), bias = rows(1, 16);
        omega_route_config c = {16, 4, OMEGA_ROUTE_SOFTMAX, 1, 4, 2, 2, 1.0f};
        EXPECT(refuses([&] { omega::RoutingLayer bad(c, ctx, x.get()); }, "bias shape"));
        omega::RoutingLayer route(c, ctx, bias.get()), plain(c, ctx);
        EXPECT(refuses([&] { route.back(*dw); }, "without a forward") && refuses([&] { route.balance(0.1f); }, "without a bias or a forward"));
        EXPECT(route.getIds().empty() && route.getCounts().empty());
        route.forward(*z);
        plain.forward(*z);
        EXPECT(route.getIds().size() == 24 && route.getCounts().size() == 16);
        route.back(*dw);
        route.balance(0.1f);
        EXPECT(refuses([&] { plain.balance(0.1f); }, "without a bias"));
        EXPECT(refuses([&] { route.back(*z); }, "delta shape"));
        z->number = 5;
        EXPECT(refuses([&] { route.back(*dw); }, "another shape"));
        z->number = 6;
        c.K = 9;                        // (the layer's own copy stays)
        route.forward(*z);
        omega::RoutingLayer bad(c, ctx);
        EXPECT(refuses([&] { bad.forward(*z); }, "K exceeds"));
        EXPECT(refuses([&] { bad.back(*dw); }, "without a forward"));
    }
    printf("%d failed\n", g_failed);
    return g_failed != 0;
}
