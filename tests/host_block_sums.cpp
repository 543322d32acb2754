// The C++ norm with a tensor of the caller for the sum, against the stand-ins of the C ABI's launchers: with its input kept in 8 bits nothing of x or the
// sum is held.
#include <cstdio>

#include "BlockLayers.hpp"

extern "C" size_t host_live_bytes(void);
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
    auto dy = rows(6, 40), more = rows(7, 40), wide = rows(6, 41), gamma = rows(1, 40);
    for (bool keep : {false, true}) {
        omega::RMSLayer norm(40, *gamma, 1e-6f, keep);
        auto x = rows(6, 40), r = rows(6, 40), s = rows(6, 40);
        EXPECT(refuses([&] { norm.forward(*x, nullptr, s.get()); }, "without a residual"));
        EXPECT(refuses([&] { norm.forward(*x, r.get(), more.get()); }, "sum shape"));
        EXPECT(refuses([&] { norm.forward(*x, r.get(), wide.get()); }, "sum shape"));
        EXPECT(refuses([&] { norm.back(*dy); }, "without a forward") && norm.getSum() == nullptr);
        norm.forward(*x);
        const size_t live = host_live_bytes();
        for (omega::Tensor *into : {s.get(), x.get(), r.get()}) {
            norm.forward(*x, r.get(), into);
            EXPECT(norm.getSum() == into && host_live_bytes() == live);
        }
        norm.forward(*x, r.get());
        EXPECT(norm.getSum() && norm.getSum() != s.get() && host_live_bytes() == live + 6 * 40 * 4);
        norm.forward(*x, r.get(), r.get());
        if (keep) {
            x.reset();
            r.reset();
            s.reset();
        }
        norm.back(*dy, dy.get());
        EXPECT(refuses([&] { norm.back(*more); }, "delta shape"));
        EXPECT(refuses([&] { norm.forward(*wide); }, "input shape"));
        norm.back(*dy);  // (refused before anything was given up)
    }
    printf("%d failed\n", g_failed);
    return g_failed != 0;
}
