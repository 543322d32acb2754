// A block's training step through the C++ layers: norm with the residual's addition that keeps its sum in 8 bits, experts with a routing of
// their own, the next norm, all the way back, the step of the bias for balance; used by tests/test_gpu_host_block.py, which compares against
// the same step in Python.
//   block_host_demo <dir> T d E K H
#include <cstdlib>

#include "BlockLayers.hpp"

static std::vector<float> read_all(const std::string &path, size_t n)
{
    std::vector<float> v(n);
    FILE *f = fopen(path.c_str(), "rb");
    if (!f || fread(v.data(), 4, n, f) != n) throw std::runtime_error("cannot read " + path);
    fclose(f);
    return v;
}
template <class T> static void write_all(const std::string &path, const std::vector<T> &v)
{
    FILE *f = fopen(path.c_str(), "wb");
    if (!f || fwrite(v.data(), sizeof(T), v.size(), f) != v.size()) throw std::runtime_error("cannot write " + path);
    fclose(f);
}
static void write_all(const std::string &path, omega::Tensor &t)
{
    t.syncHost();
    write_all(path, t.data);
}

int main(int argc, char **argv)
{
    if (argc != 7) { fprintf(stderr, "usage: %s dir T d E K H\n", argv[0]); return 2; }
    try {
        const std::string dir = std::string(argv[1]) + "/";
        const int T = atoi(argv[2]), d = atoi(argv[3]), E = atoi(argv[4]), K = atoi(argv[5]), H = atoi(argv[6]);
        omega::Context ctx(0);
        auto tensor = [&](const char *name, int number, int width) {
            std::unique_ptr<omega::Tensor> t(new omega::Tensor(number, 1, 1, width, &ctx, true));
            t->data = read_all(dir + name, t->data.size());
            t->hostToDevice();
            return t;
        };
        auto x = tensor("x.bin", T, d), res = tensor("res.bin", T, d), dout = tensor("dout.bin", T, d), gamma1 = tensor("gamma1.bin", 1, d), gamma2 = tensor("gamma2.bin", 1, d);
        omega::MoELayer moe(d, H, E, K, true, 0, false, ctx);
        const omega_route_config route = {E, K, OMEGA_ROUTE_SIGMOID, 1, 4, 2, 2, 2.5f};
        moe.setRouting(&route, true);
        FILE *f = fopen((dir + "moe.bin").c_str(), "rb");
        if (!f) throw std::runtime_error("cannot open moe.bin");
        moe.loadModel(f);
        fclose(f);
        omega::RMSLayer norm1(d, *gamma1, 1e-6f, true), norm2(d, *gamma2);
        omega::Tensor &h = norm1.forward(*x, res.get());
        static_cast<omega::Layer &>(moe).forward(h);
        write_all(dir + "y.bin", norm2.forward(*moe.getOutput(), norm1.getSum()));
        omega::Tensor &d2 = norm2.back(*dout);
        static_cast<omega::Layer &>(moe).back(d2);
        write_all(dir + "dx.bin", norm1.back(*moe.getDiff(), &d2));
        write_all(dir + "dgamma1.bin", *norm1.getDiffGamma());
        write_all(dir + "dgamma2.bin", *norm2.getDiffGamma());
        moe.balance(0.01f);
        f = fopen((dir + "moe_out.bin").c_str(), "wb");
        moe.saveModel(f);
        fclose(f);
        // the operator on its own, on the first E columns of rows that are at hand, and rows through 8 bits
        omega::Tensor logits(T, 1, 1, E, &ctx, true), bias(1, 1, 1, E, &ctx, true);
        for (int t = 0; t < T; ++t)
            for (int e = 0; e < E; ++e) logits.data[(size_t)t * E + e] = x->data[(size_t)t * d + e];
        logits.hostToDevice();
        bias.hostToDevice();
        omega::RoutingLayer router(route, ctx, &bias);
        omega::Tensor &w = router.forward(logits);
        write_all(dir + "w.bin", w);
        write_all(dir + "ids.bin", router.getIds());
        write_all(dir + "counts.bin", router.getCounts());
        write_all(dir + "dlogits.bin", router.back(w));
        router.balance(0.5f);
        write_all(dir + "bias.bin", bias);
        omega::Keep8Layer mx(d, ctx, OMEGA_KEEP8_MX);
        mx.save(*x);
        write_all(dir + "x8.bin", mx.load());

        // refusals are exceptions
        omega::Tensor bad(T, 1, 1, d + 1, &ctx, true);
        omega_route_config odd = route;
        odd.groups = 3;
        int raised = 0;
        try { norm1.forward(bad); } catch (const std::runtime_error &) { ++raised; }
        try { norm2.back(*dout, &bad); } catch (const std::runtime_error &) { ++raised; }
        try { omega::RMSLayer(d, *x); } catch (const std::runtime_error &) { ++raised; }
        try { router.forward(*x); } catch (const std::runtime_error &) { ++raised; }
        try { omega::RoutingLayer(odd, ctx).forward(logits); } catch (const std::runtime_error &) { ++raised; }
        try { moe.setRouting(&odd); } catch (const std::runtime_error &) { ++raised; }
        try { omega::Keep8Layer(d, ctx).load(); } catch (const std::runtime_error &) { ++raised; }
        try { mx.save(bad); } catch (const std::runtime_error &) { ++raised; }
        if (raised != 8) throw std::runtime_error("a call that does not fit was accepted");
        printf("ok T=%d\n", T);
        return 0;
    } catch (const std::exception &e) {
        fprintf(stderr, "block_host_demo: %s\n", e.what());
        return 1;
    }
}
