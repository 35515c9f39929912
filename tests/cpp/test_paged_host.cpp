// test_paged_host.cpp -- GPU tests of the C++ host mirror's paged caches
// (HipPool, HipSequence over it) against contiguous caches of the same model.
//
// Run by tests/test_gpu_host_paged.py on a machine with a GPU; built by
// tests/cpp/Makefile (called from the package build).
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <stdexcept>
#include <vector>

#include "../../oracle/ftx_oracle.h"
#include "../../xwfes_amd/host/hip_backend.hpp"

using namespace ftx_host;

static int g_checks = 0;
#define CHECK(cond, msg)                                                   \
    do {                                                                   \
        ++g_checks;                                                        \
        if (!(cond)) {                                                     \
            std::fprintf(stderr, "CHECK failed: %s (%s:%d)\n", msg, __FILE__, \
                         __LINE__);                                        \
            std::exit(1);                                                  \
        }                                                                  \
    } while (0)

static std::mt19937_64 rng_gen(777);
static float rnd() { return std::normal_distribution<float>(0.f, 1.f)(rng_gen); }

struct Model {
    ModelConfig c;
    ModelWeights w;
    std::vector<std::vector<uint8_t>> keep;

    HostTensor add(DType dt, int64_t rows, int64_t cols, float scale, float mean = 0.f) {
        const int64_t rb = orc_row_bytes((int)dt, cols);
        keep.emplace_back((size_t)(rb * rows));
        std::vector<float> row((size_t)cols);
        for (int64_t r = 0; r < rows; ++r) {
            for (auto& v : row) v = mean + rnd() * scale;
            CHECK(orc_quantize_row(keep.back().data() + r * rb, row.data(), (int)dt, cols) == 0, "quantise");
        }
        HostTensor t;
        t.ne[0] = cols;
        t.ne[1] = rows;
        t.n_dims = 2;
        t.dtype = dt;
        t.data = keep.back().data();
        t.nbytes = keep.back().size();
        return t;
    }
    Model() {
        c.n_layer = 2;
        c.n_embd = 256;
        c.n_head = 4;
        c.n_head_kv = 2;
        c.head_dim = 64;
        c.n_ff = 512;
        c.vocab = 256;
        c.rope_theta = 10000.0;
        w.tok_embd = add(DType::F32, c.vocab, c.n_embd, 1.f);
        w.out_norm = add(DType::F32, 1, c.n_embd, 0.3f, 1.f);
        w.output = add(DType::Q8_0, c.vocab, c.n_embd, 0.05f);
        const int64_t kdim = c.n_head_kv * c.head_dim, qdim = c.n_head * c.head_dim;
        for (int64_t l = 0; l < c.n_layer; ++l)
            w.layers.push_back({add(DType::F32, 1, c.n_embd, 0.3f, 1.f), add(DType::Q8_0, qdim, c.n_embd, 0.05f),
                                add(DType::Q8_0, kdim, c.n_embd, 0.05f), add(DType::Q8_0, kdim, c.n_embd, 0.05f),
                                add(DType::Q8_0, c.n_embd, qdim, 0.05f), add(DType::F32, 1, c.n_embd, 0.3f, 1.f),
                                add(DType::Q8_0, c.n_ff, c.n_embd, 0.05f), add(DType::Q8_0, c.n_ff, c.n_embd, 0.05f),
                                add(DType::Q8_0, c.n_ff, c.n_embd, 0.05f)});
    }
};

// the same step over both caches: the largest difference of a row's logits
// relative to its largest
static double step_diff(HipBackend& be, HipVerifier& ver, HipSequence& a, HipSequence& b,
                        const std::vector<int32_t>& props, const std::vector<int32_t>& parents, bool advance) {
    const size_t V = (size_t)ver.config().vocab, n = props.size() * V;
    std::vector<float> out[2];
    HipSequence* seqs[2] = {&a, &b};
    for (int s = 0; s < 2; ++s) {
        float* d = (float*)be.alloc_staging(n * sizeof(float));
        HipVerifier::BatchItem it;
        it.seq = seqs[s];
        it.props = props;
        it.parents = parents;
        it.logits = d;
        it.advance = advance;
        ver.verify_batch({it});
        out[s].resize(n);
        be.stage(out[s].data(), d, n * sizeof(float));
        be.free_staging(d);
    }
    double worst = 0;
    for (size_t m = 0; m < props.size(); ++m) {
        double num = 0, den = 1e-30;
        for (size_t v = 0; v < V; ++v) {
            num = std::max(num, (double)std::fabs(out[0][m * V + v] - out[1][m * V + v]));
            den = std::max(den, (double)std::fabs(out[0][m * V + v]));
        }
        worst = std::max(worst, num / den);
    }
    return worst;
}

static void test_paged_equals_contiguous(HipBackend& be, HipVerifier& ver) {
    const int64_t cap = 200;
    HipPool pool(ver, 6);
    CHECK(pool.available() == 6, "a new pool is free");
    {
        HipSequence paged(ver, pool, cap), plain(ver, cap);
        std::vector<int32_t> chain(61);
        for (size_t i = 0; i < chain.size(); ++i) chain[i] = (int32_t)((i * 37) % 256);
        CHECK(step_diff(be, ver, plain, paged, chain, {}, true) < 1e-3, "a prompt");
        CHECK(pool.available() == 5 && paged.npast() == 61, "its page");
        CHECK(step_diff(be, ver, plain, paged, {7}, {}, true) < 1e-3, "one token");
        const std::vector<int32_t> tree = {3, 9, 27, 81, 200, 11}, par = {-1, 0, 0, 1, 1, 2};
        CHECK(step_diff(be, ver, plain, paged, tree, par, false) < 1e-3, "a tree over a page's end");
        CHECK(pool.available() == 4, "the second page");
        plain.commit({0, 1, 4});
        paged.commit({0, 1, 4});
        CHECK(paged.npast() == 65, "the committed path");
        CHECK(step_diff(be, ver, plain, paged, {42, 43}, {}, true) < 1e-3, "after the commit");
        plain.truncate_to(20);
        paged.truncate_to(20);
        CHECK(pool.available() == 5, "a page given back");
        CHECK(step_diff(be, ver, plain, paged, {42, 43, 44}, {}, true) < 1e-3, "after the truncation");
    }
    CHECK(pool.available() == 6, "every page came back");
}

static void test_pool_runs_out(HipBackend& be, HipVerifier& ver) {
    HipPool pool(ver, 1, true);
    HipSequence a(ver, pool, 200, 16, 4);
    std::vector<int32_t> chain(64, 5);
    HipVerifier::BatchItem it;
    it.seq = &a;
    it.props = chain;
    it.advance = true;
    ver.verify_batch({it});
    it.props = {1};
    bool threw = false;
    try {
        ver.verify_batch({it});
    } catch (const std::runtime_error&) {
        threw = true;
    }
    CHECK(threw && a.npast() == 64, "no page for the next token");
    a.truncate_to(63);
    ver.verify_batch({it});
    be.sync();
    CHECK(a.npast() == 64, "room in the page");
}

int main() {
    HipBackend be(0);
    Model m;
    HipVerifier ver(be, m.c, m.w, 200, 64);
    test_paged_equals_contiguous(be, ver);
    test_pool_runs_out(be, ver);
    std::printf("all %d checks passed\n", g_checks);
    return 0;
}
