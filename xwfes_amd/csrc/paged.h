// paged.h -- paged KV caches: the host side of a plan (checks of a step's
// sequences and the division of the attention's work, no device calls) and
// what the kernels of k_paged.hip take.
#pragma once

#include <string>
#include <vector>

#include "ftx_internal.h"

// ---------------------------------------------------------------- page layout
// One block per (layer, page, kv head): K values, V values, FTX_PAGE K scales,
// FTX_PAGE V scales (fp32), all in the order the attention's MFMA operands are
// loaded, so that every wave load of 16 bytes per lane is one contiguous KB.
// Slot of a page: slot = 16 st + m (K: row m of score tile st);
// slot = 16 st + 4 kq + r (V: the slots whose scores lane (q row, kq) holds).
//   halves: K unit (dc 4 + st) 64 + 16 kq + m: slot 16 st + m, dims 32 dc + 8 kq ..+7
//           V unit (2 dt + sp) 64 + 16 kq + dl: dim 16 dt + dl, slots 16 (2 sp + i / 4) + 4 kq + i % 4
//   8 bit:  K unit (4 j + st) 64 + 16 kq + m: slot 16 st + m, dims 64 j + 16 kq ..+15
//           V unit 64 dt + 16 kq + dl: dim 16 dt + dl, byte 4 st + r: slot 16 st + 4 kq + r
__host__ __device__ inline int64_t paged_values_bytes(int hd, int q8) {
    return (int64_t)FTX_PAGE * hd * (q8 ? 1 : 2);
}
__host__ __device__ inline int64_t paged_block_bytes(int hd, int q8) {
    return 2 * paged_values_bytes(hd, q8) + 2 * FTX_PAGE * 4;
}
// byte offsets of element (slot, d) in the K and in the V values of a block
__host__ __device__ inline int paged_k_at(int slot, int d, int q8) {
    const int st = slot >> 4, m = slot & 15;
    return q8 ? (((d >> 6) * 4 + st) * 64 + ((d >> 4) & 3) * 16 + m) * 16 + (d & 15)
              : ((((d >> 5) * 4 + st) * 64 + ((d >> 3) & 3) * 16 + m) * 8 + (d & 7)) * 2;
}
__host__ __device__ inline int paged_v_at(int slot, int d, int q8) {
    const int st = slot >> 4, kq = (slot >> 2) & 3, r = slot & 3;
    const int lane = kq * 16 + (d & 15);
    return q8 ? ((d >> 4) * 64 + lane) * 16 + 4 * st + r
              : ((((d >> 4) * 2 + (st >> 1)) * 64 + lane) * 8 + 4 * (st & 1) + r) * 2;
}

// ---------------------------------------------------------------- a plan's tables
struct PagedSeq {
    int32_t npast, M;
    int32_t tok0;        // its first row in the packed new rows
    int32_t tab0, ntab;  // its pages in the table array
    int32_t dep0;        // its node depths in the depth array, -1: a chain
    int32_t anc0, aw;    // its mask words in the mask array, words a node
    int64_t all0;        // its first row when contexts are read back
};
// A row tile (query rows of a kv head: row r = token r / gqa, head r % gqa;
// PAGED_TR, PAGED_TR_MANY or twice that many of them) over entries i0 .. i1 - 1 of its page
// list: pages 0 .. s - 1 (the first tokens'), then pages a, a + 1, ..  q: its
// sequence, held here so that a workgroup's first page is two loads away and
// not three
struct PagedItem {
    int32_t seq, row0, i0, i1, s, a;
    int32_t part;  // its partials' place (in blocks of PAGED_TR rows), or -1: the whole list, results go to out
    int32_t nt;    // 0: PAGED_TR rows; 1: PAGED_TR_MANY; 2: twice that
    PagedSeq q;
    int32_t fill[6];  // to 96 bytes
};
// the partials part0, part0 + step, .. (n of them) of PAGED_TR rows; tok0, M:
// its sequence's
struct PagedComb {
    int32_t seq, row0, part0, n, step, tok0, M, pad;
};
constexpr int PAGED_TR = 16, PAGED_TR_MANY = 128;

struct PagedGeom {
    int64_t n_kv = 0, hd = 0, n_pages = 0;
    const uint8_t* taken = nullptr;
    int cu = 0;
};
struct PagedTables {
    int64_t n_head = 0, window = 0, sinks = 0;
    int64_t tokens = 0, rows = 0;  // new tokens, positions of all contexts
    int64_t longest = 0;            // new tokens of one sequence
    int64_t max_new_pages = 0, max_pages = 0;  // of one sequence
    int64_t parts = 0;   // in blocks of PAGED_TR rows
    int64_t comb_max = 0;  // most partials of a row
    int64_t few = 0;     // items of PAGED_TR rows, before the others
    bool wide = false;   // by workgroups of eight waves
    bool absent = false;  // a page below npast + M is absent
    double seen = 0, pages_read = 0;  // visible (row, slot) pairs bound, pages of all items
    std::vector<PagedSeq> seqs;
    std::vector<int32_t> table, depth;
    std::vector<uint32_t> anc;
    std::vector<PagedItem> items;
    std::vector<PagedComb> combs;
};
// The tables of a step, or an FTX_E_* code and its message.  `mark`: scratch
// of the caller, kept from call to call with `epoch`.
int paged_tables(const PagedGeom& g, const ftx_plan_args& a, std::vector<uint32_t>& mark,
                 uint32_t& epoch, PagedTables& out, std::string& err);

// The same with plain arrays, no context and no device: up to max_out row-tile
// items (PagedItem) and joins (PagedComb) of a pool of `n_pages` pages
extern "C" int paged_probe(const ftx_plan_args* a, int64_t n_kv, int64_t hd, int64_t n_pages, const uint8_t* taken,
                           int cu, PagedItem* items, int64_t* n_items, PagedComb* combs, int64_t* n_combs,
                           int64_t max_out, char* msg, int64_t msg_bytes);

// For tests: the row tiles of sequences of many rows in the calling thread's plans
// from now on, 16, 128 or 256 (heads of 256 dims: 128), 0: by the estimate
extern "C" void paged_force_rows(int rows);

// ---------------------------------------------------------------- launches
// a launch has fewer than 2^32 threads along its x
inline bool paged_grid_fits(int64_t workgroups, int64_t threads) { return workgroups * threads < (int64_t)1 << 32; }

struct PagedView {
    uint8_t* data;  // the layer's first block
    int64_t block;  // bytes of a block
    int n_kv, hd, q8;
    const PagedSeq* seqs;
    const int32_t* table;
    int nseq;
};
hipError_t launch_paged_write(hipStream_t st, const PagedView& p, int64_t max_new_pages,
                              const float* k, int64_t ldk, const float* v, int64_t ldv);
hipError_t launch_paged_read(hipStream_t st, const PagedView& p, int64_t max_pages, int context,
                             float* k, int64_t ldk, float* v, int64_t ldv);
struct PagedAttn {
    PagedView p;
    const int32_t* depth;
    const uint32_t* anc;
    const PagedItem* items;
    const PagedComb* combs;
    int n_few, n_many, n_combs;
    bool wide;  // few: eight waves a workgroup
    int rows_max, comb_max;  // query rows of the longest sequence, most partials of a row
    int gqa;
    int window, sinks;
    const float* q;
    float* out;
    int64_t ldq, ldo;
    float* part;  // [parts][n_kv][PAGED_TR][hd] normalised outputs
    float* pml;   // [parts][n_kv][PAGED_TR][2]: maximum (base 2), sum
};
hipError_t launch_paged_attention(hipStream_t st, const PagedAttn& a);

// rows of a committed path: slots src[i] move to dst[i] (page * FTX_PAGE +
// slot), in order, every layer and kv head
struct PagedMove {
    uint8_t* data;
    int64_t block, n_pages;
    int n_kv, hd, q8, n_layer, n;
    int32_t src[256], dst[256];
};
hipError_t launch_paged_move(hipStream_t st, const PagedMove& m);

// ---------------------------------------------------------------- the verify step's use
// The plan of the pool's running step (one a pool, its calls in stream order)
int paged_step_plan(ftx_ctx* ctx, ftx_pool* p, const ftx_plan_args& a, ftx_plan** out);
// the layer as the plan's kernels see it, for steps whose RoPE stores the rows
// (up to PAGED_ROWS_FEW new tokens a sequence, where rows are stored one by one)
constexpr int PAGED_ROWS_FEW = 15;
PagedView paged_view(const ftx_plan* pl, int64_t layer);
int paged_write_rows(ftx_plan* pl, int64_t layer, const float* k, int64_t ldk, const float* v, int64_t ldv);
int paged_read_rows(ftx_plan* pl, int64_t layer, int context, float* k, int64_t ldk, float* v, int64_t ldv);
int paged_attend_rows(ftx_plan* pl, int64_t layer, const float* q, int64_t ldq, float* out, int64_t ldo);
