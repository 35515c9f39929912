// paged.h -- paged KV caches: the host side of a plan (checks of a step's
// sequences and the division of the attention's work, no device calls) and
// what the kernels of k_paged.hip take.
#pragma once

#include <string>
#include <vector>

#include "ftx_internal.h"

// ---------------------------------------------------------------- page layout
// One block per (layer, page, kv head): K values, V values, FTX_PAGE K scales,
// FTX_PAGE V scales (fp32), and for 4-bit rows K's and V's multipliers (a byte
// for each 32 dims of a slot), all in the order the attention's MFMA operands
// are loaded, so that every wave load of 16 bytes per lane is one contiguous KB.
// Slot of a page: slot = 16 st + m (K: row m of score tile st);
// slot = 16 st + 4 kq + r (V: the slots whose scores lane (q row, kq) holds).
//   halves: K unit (dc 4 + st) 64 + 16 kq + m: slot 16 st + m, dims 32 dc + 8 kq ..+7
//           V unit (2 dt + sp) 64 + 16 kq + dl: dim 16 dt + dl, slots 16 (2 sp + i / 4) + 4 kq + i % 4
//   8 bit:  K unit (4 j + st) 64 + 16 kq + m: slot 16 st + m, dims 64 j + 16 kq ..+15
//           V unit 64 dt + 16 kq + dl: dim 16 dt + dl, byte 4 st + r: slot 16 st + 4 kq + r
//   4 bit:  K unit (2 (dc / 2) + st / 2) 64 + 16 kq + m, word 2 (st % 2) + dc % 2: slot 16 st + m,
//             dims 32 dc + 8 kq ..+7 as nibbles 0 4 1 5 2 6 3 7 (nibble n + 4 in the high half)
//           V unit 64 g + 16 kq + dl, word st, bytes of slots 16 st + 4 kq + 0 2 1 3:
//             dim 32 g + dl in the low nibble, 32 g + 16 + dl in the high one
//           (so that a row's bytes are its own, and a nibble of both halves of a word is two
//           neighbours of an operand)
//           multiplier of slot 16 st + 4 kq + r, dims 32 g ..+31: byte 64 g + 16 kq + 4 st + r
enum { PT_F16 = 0, PT_Q8 = 1, PT_Q4 = 2 };
__host__ __device__ constexpr int64_t paged_values_bytes(int hd, int kt) {
    return (int64_t)FTX_PAGE * hd * (kt == PT_F16 ? 4 : kt == PT_Q8 ? 2 : 1) / 2;
}
__host__ __device__ constexpr int64_t paged_mult_bytes(int hd, int kt) {
    return kt == PT_Q4 ? (int64_t)FTX_PAGE * hd / 32 : 0;
}
__host__ __device__ constexpr int64_t paged_block_bytes(int hd, int kt) {
    return 2 * paged_values_bytes(hd, kt) + 2 * FTX_PAGE * 4 + 2 * paged_mult_bytes(hd, kt);
}
// byte offsets of element (slot, d) in the K and in the V values of a block
__host__ __device__ inline int paged_k_at(int slot, int d, int kt) {
    const int st = slot >> 4, m = slot & 15;
    if (kt == PT_Q4)
        return (((d >> 6) * 2 + (st >> 1)) * 64 + ((d >> 3) & 3) * 16 + m) * 16 + (st & 1) * 8 + ((d >> 5) & 1) * 4 +
               (d & 1) * 2 + ((d >> 2) & 1);
    return kt == PT_Q8 ? (((d >> 6) * 4 + st) * 64 + ((d >> 4) & 3) * 16 + m) * 16 + (d & 15)
                       : ((((d >> 5) * 4 + st) * 64 + ((d >> 3) & 3) * 16 + m) * 8 + (d & 7)) * 2;
}
__host__ __device__ inline int paged_v_at(int slot, int d, int kt) {
    const int st = slot >> 4, kq = (slot >> 2) & 3, r = slot & 3;
    const int lane = kq * 16 + (d & 15);
    if (kt == PT_Q4) return ((d >> 5) * 64 + lane) * 16 + 4 * st + (r & 1) * 2 + (r >> 1);
    return kt == PT_Q8 ? ((d >> 4) * 64 + lane) * 16 + 4 * st + r
                       : ((((d >> 4) * 2 + (st >> 1)) * 64 + lane) * 8 + 4 * (st & 1) + r) * 2;
}
// of 4-bit rows: the byte of slot `slot`'s multiplier for dims 32 g ..+31, and the
// dim in the low nibble of byte t of a row (the other is d + 2 in K, d + 16 in V)
__host__ __device__ inline int paged_c_at(int slot, int g) {
    return 64 * g + ((slot >> 2) & 3) * 16 + (slot >> 4) * 4 + (slot & 3);
}
__host__ __device__ inline int paged_k_dim(int t) { return (t >> 2) * 8 + ((t >> 1) & 1) + (t & 1) * 4; }
__host__ __device__ inline int paged_v_dim(int t) { return (t >> 4) * 32 + (t & 15); }

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
// A page that new tokens go to, in tables built on the GPU: its id (-1: none), their
// slots s0 .. s1 - 1 and the row that slot 0 would be in the packed new rows
struct PagedTouch {
    int32_t page, s0, s1, pad;
    int64_t row, pad2;
};
constexpr int PAGED_TR = 16, PAGED_TR_MANY = 128;
// Sequences of at least this many query rows a kv head may go to the kernel
// that shares each page among 128 or 256 rows
constexpr int PAGED_MANY = 65;

struct PagedGeom {
    int64_t n_kv = 0, hd = 0, n_pages = 0;
    const uint8_t* taken = nullptr;
    int cu = 0;
    int kt = PT_F16;
};
struct PagedTables {
    int64_t n_head = 0, window = 0, sinks = 0;
    int64_t tokens = 0, rows = 0;  // new tokens, positions of all contexts
    int64_t longest = 0;            // new tokens of one sequence
    int64_t max_new_pages = 0, max_pages = 0;  // of one sequence
    int64_t parts = 0;   // in blocks of PAGED_TR rows
    int64_t comb_max = 0;  // most partials of a row
    int64_t few = 0;     // items of PAGED_TR rows, before the others
    int64_t few_rows = 0;  // most query rows (a kv head) of a sequence that has such an item
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

// ---------------------------------------------------------------- tables built on the GPU
constexpr int PAGED_ROOM_SEQS = 4096;
// What a plan of lengths that the GPU holds has room for
struct PagedRoom {
    int32_t nseq, tokens, most, n_pages;  // sequences, new tokens of all, of one; pages of one
    int32_t pool_pages, n_kv, gqa;        // gqa = 0: no attention
    int32_t window, sinks;
    // parts that lists of many rows are cut into beyond one each (seq_per); of few
    // rows: workgroups a kv head that fill the chip, and the most such parts
    int32_t cut_many, slots, cut_few;
    int32_t wide;               // lists of few rows stay whole, for workgroups of eight waves
    int32_t few, many, combs, parts, touch;  // entries
};
// from ftx_plan_room, or an FTX_E_* code and its message
int paged_room(const PagedGeom& g, const ftx_plan_room& a, PagedRoom& r, std::string& err);

struct PagedBuild {
    PagedRoom r;
    int nseq;
    // the caller's
    const int32_t *npast, *M, *free_pages, *used;
    int32_t *tables, *used_after, *starts, *slots, *positions, *status;
    int64_t ldt, n_free;
    // the plan's
    PagedSeq* seqs;
    int32_t* table;  // [r.nseq][r.n_pages]
    PagedTouch* touch;
    PagedItem* items;  // r.few, then r.many; seq = -1: none (seq_none)
    PagedComb* combs;  // M = 0: none
    int32_t* codes;    // [r.nseq]: what the first kernel says of each sequence, then the pages used before
};
hipError_t launch_paged_build(hipStream_t st, const PagedBuild& b);
// its kernel's LDS on the current device, before the first
hipError_t paged_build_limits();

// The same lists for plain arrays, no context and no device: items (r.few + r.many
// of them) and joins (r.combs) of sequences whose lengths fit the room
extern "C" int paged_build_probe(const ftx_plan_room* a, int64_t n_kv, int64_t hd, int64_t pool_pages, int cu,
                                 const int32_t* npast, const int32_t* M, int64_t nseq, PagedRoom* room, PagedItem* items,
                                 PagedComb* combs, int64_t max_out, char* msg, int64_t msg_bytes);

// ---------------------------------------------------------------- launches
// a launch has fewer than 2^32 threads along its x
inline bool paged_grid_fits(int64_t workgroups, int64_t threads) { return workgroups * threads < (int64_t)1 << 32; }

struct PagedView {
    uint8_t* data;  // the layer's first block
    int64_t block;  // bytes of a block
    int n_kv, hd, kt;
    const PagedSeq* seqs;
    const int32_t* table;
    int nseq;
    // of tables built on the GPU: the pages that new tokens go to, one after the
    // other (else a launch covers every sequence's most such pages)
    const PagedTouch* touch;
    int n_touch;
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
    int few_rows;            // query rows of the longest sequence of the n_few items
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
    int n_kv, hd, kt, n_layer, n;
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
