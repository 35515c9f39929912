// test_paged_rows.cpp -- GPU tests of the C++ host mirror's paged caches whose rows
// are held in 4 bits (HipPool of KvRows::Bits4).
//
// Run by tests/test_gpu_host_paged_rows.py on a machine with a GPU; built by
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

// rows that a cache in 4 bits shows are off by half a step of their block, at most
// 1/14 of its largest value (and the step's cover: one in 255 of the row's largest need)
static void test_rows_come_back(HipBackend& be, HipVerifier& ver) {
    const ModelConfig& c = ver.config();
    const int64_t cap = 130, w = c.n_head_kv * c.head_dim, n = c.n_layer * cap * w;
    HipPool pool(ver, 3, KvRows::Bits4);
    HipSequence seq(ver, pool, cap);
    std::vector<float> k((size_t)n), v((size_t)n), k2((size_t)n), v2((size_t)n);
    for (auto* x : {&k, &v})
        for (auto& y : *x) y = rnd();
    seq.write_kv(k.data(), v.data());
    CHECK(pool.available() == 0, "pages for all of the cache");
    seq.truncate_to(cap);
    seq.read_kv(k2.data(), v2.data());
    be.sync();
    bool near = true;
    double off = 0, size = 0;
    for (int64_t r = 0; r < n / c.head_dim; ++r)
        for (auto* p : {&k, &v}) {
            const float* x = p->data() + r * c.head_dim;
            const float* y = (p == &k ? k2 : v2).data() + r * c.head_dim;
            float row = 0;
            for (int64_t d = 0; d < c.head_dim; ++d) row = std::fmax(row, std::fabs(x[d]));
            for (int64_t d = 0; d < c.head_dim; ++d) {
                float blk = 0;
                for (int64_t e = d / 32 * 32; e < d / 32 * 32 + 32; ++e) blk = std::fmax(blk, std::fabs(x[e]));
                near = near && std::fabs(x[d] - y[d]) <= 0.501f * (blk / 7 + row / 7 / 255);
                off += (x[d] - y[d]) * (x[d] - y[d]);
                size += x[d] * x[d];
            }
        }
    CHECK(near, "every value within half a step");
    CHECK(off > 0 && std::sqrt(off / size) < 0.12, "steps of a quarter of a block's spread, evenly rounded");
}

// a prompt, steps, a tree's commit and a truncation: pages come and go, and a step
// over the same rows gives the same logits
static void test_steps(HipBackend& be, HipVerifier& ver) {
    const size_t V = (size_t)ver.config().vocab;
    HipPool pool(ver, 6, KvRows::Bits4);
    HipSequence a(ver, pool, 200), b(ver, pool, 200);
    float* d = (float*)be.alloc_staging(2 * V * sizeof(float));
    std::vector<int32_t> chain(61);
    for (size_t i = 0; i < chain.size(); ++i) chain[i] = (int32_t)((i * 37) % 256);
    for (auto* s : {&a, &b}) {
        HipVerifier::BatchItem it;
        it.seq = s;
        it.props = chain;
        it.advance = true;
        ver.verify_batch({it});
        it.props = {3, 9, 27, 81, 200, 11};
        it.parents = {-1, 0, 0, 1, 1, 2};
        it.advance = false;
        ver.verify_batch({it});
        s->commit({0, 1, 4});
    }
    CHECK(a.npast() == 64 && pool.available() == 2, "a path up to its page's end, the tree's second page kept");
    std::vector<HipVerifier::BatchItem> both(2);
    for (int s = 0; s < 2; ++s) {
        both[s].seq = s ? &b : &a;
        both[s].props = {42};
        both[s].advance = true;
        both[s].logits = d + s * V;
    }
    ver.verify_batch(both);
    CHECK(pool.available() == 2 && a.npast() == 65 && b.npast() == 65, "the next token in the second page");
    std::vector<float> out(2 * V);
    be.stage(out.data(), d, 2 * V * sizeof(float));
    bool same = true, finite = true;
    for (size_t i = 0; i < V; ++i) {
        same = same && out[i] == out[V + i];
        finite = finite && std::isfinite(out[i]);
    }
    CHECK(same && finite, "the same rows, the same logits");
    a.truncate_to(20);
    CHECK(pool.available() == 3, "a page given back");
    be.free_staging(d);
}

int main() {
    HipBackend be(0);
    Model m;
    HipVerifier ver(be, m.c, m.w, 200, 64);
    test_rows_come_back(be, ver);
    test_steps(be, ver);
    std::printf("all %d checks passed\n", g_checks);
    return 0;
}
