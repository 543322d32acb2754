// One training step of a small language model through the C++ layers: embedding -> MoE block -> layer norm -> tied head with its loss, all
// the way back, the clip and the MoE layer's update; used by tests/test_gpu_host_lm.py, which compares against the same step in Python.
//   lm_host_demo <dir> T V d E K H maxNorm
#include <cstdlib>

#include "LmLayers.hpp"

template <class T> static std::vector<T> read_all(const std::string &path, size_t n)
{
    std::vector<T> v(n);
    FILE *f = fopen(path.c_str(), "rb");
    if (!f || fread(v.data(), sizeof(T), n, f) != n) throw std::runtime_error("cannot read " + path);
    fclose(f);
    return v;
}
static void write_all(const std::string &path, omega::Tensor &t)
{
    t.syncHost();
    FILE *f = fopen(path.c_str(), "wb");
    if (!f || fwrite(t.data.data(), 4, t.data.size(), f) != t.data.size()) throw std::runtime_error("cannot write " + path);
    fclose(f);
}

int main(int argc, char **argv)
{
    if (argc != 9) { fprintf(stderr, "usage: %s dir T V d E K H maxNorm\n", argv[0]); return 2; }
    try {
        const std::string dir = std::string(argv[1]) + "/";
        const int T = atoi(argv[2]), V = atoi(argv[3]), d = atoi(argv[4]), E = atoi(argv[5]), K = atoi(argv[6]), H = atoi(argv[7]);
        omega::Context ctx(0);
        auto param = [&](const char *name, int number, int width) {
            std::unique_ptr<omega::Tensor> t(new omega::Tensor(number, 1, 1, width, &ctx, true));
            t->data = read_all<float>(dir + name, t->data.size());
            t->hostToDevice();
            return t;
        };
        auto table = param("table.bin", V, d), gamma = param("gamma.bin", 1, d), beta = param("beta.bin", 1, d);
        omega::Ids ids(read_all<int32_t>(dir + "ids.bin", T), &ctx), targets(read_all<int32_t>(dir + "targets.bin", T), &ctx);
        omega::MoELayer moe(d, H, E, K, true, 0, false, ctx);
        FILE *f = fopen((dir + "block.bin").c_str(), "rb");
        if (!f) throw std::runtime_error("cannot open block.bin");
        moe.loadModelBlock(f);
        fclose(f);
        omega::EmbeddingLayer emb(V, d, *table, 16.0f);
        omega::LNLayer ln(d, *gamma, *beta);
        omega::HeadLossLayer head(V, d, *table);

        omega::Tensor &e = emb.forward(ids);
        moe.forwardBlock(e);
        omega::Tensor &n = ln.forward(*moe.getOutput());
        write_all(dir + "loss.bin", head.forward(n, targets));
        write_all(dir + "mean.bin", *head.getMean());
        moe.backBlock(ln.back(head.back()));
        omega::Tensor &tied = emb.back(*moe.getDiff(), head.getDiffW());
        omega::Tensor norm(1, 1, 1, 2, &ctx, true);
        omega::clipGradNorm(ctx, {&tied, ln.getDiffGamma(), ln.getDiffBeta()}, {&moe}, (float)atof(argv[8]), &norm);
        write_all(dir + "norm.bin", norm);
        write_all(dir + "tied.bin", tied);
        write_all(dir + "dgamma.bin", *ln.getDiffGamma());
        write_all(dir + "dbeta.bin", *ln.getDiffBeta());
        moe.updateAdamW(1e-3f, 1);
        f = fopen((dir + "block_step.bin").c_str(), "wb");
        moe.saveModelBlock(f);
        fclose(f);

        // refusals are exceptions
        omega::Tensor bad(T, 1, 1, d + 1, &ctx, true);
        int raised = 0;
        try { ln.forward(bad); } catch (const std::runtime_error &) { ++raised; }
        try { head.forward(bad, targets); } catch (const std::runtime_error &) { ++raised; }
        try { emb.back(bad); } catch (const std::runtime_error &) { ++raised; }
        try { omega::HeadLossLayer(V + 1, d, *table); } catch (const std::runtime_error &) { ++raised; }
        try { omega::clipGradNorm(ctx, {&tied, &tied}, {}, 1.0f); } catch (const std::runtime_error &) { ++raised; }
        if (raised != 5) throw std::runtime_error("a call that does not fit was accepted");
        printf("ok T=%d\n", T);
        return 0;
    } catch (const std::exception &e) {
        fprintf(stderr, "lm_host_demo: %s\n", e.what());
        return 1;
    }
}
