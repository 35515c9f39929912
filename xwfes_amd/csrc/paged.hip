// paged.hip -- paged KV caches: the page pool, a step's plan and the C ABI's
// calls over them (include/ftx.h).  The kernels are in k_paged.hip.
#include "paged.h"

#include <algorithm>
#include <chrono>
#include <cstdio>
#include <cstring>
#include <new>
#include <thread>

#include "paged_pool.h"

// ---------------------------------------------------------------- plan tables

// Sequences of at least this many query rows a kv head may go to the kernel
// that shares each page among 128 or 256 rows
constexpr int64_t PAGED_MANY = 65;
// Row tiles beyond which such sequences do so without a look at tiles of 16
constexpr int64_t FEW_MOST = 4096;
// Pages of a list beyond which few rows are not given to eight waves unsplit
constexpr int64_t WIDE_MOST = 48;

namespace {

thread_local int forced_rows = 0;  // (paged_force_rows)

struct Tile {
    int32_t seq, row0, rows, s, a, n;  // n pages: 0 .. s - 1, then a, a + 1, ..
    int tiles() const { return rows > PAGED_TR_MANY ? 2 : 1; }  // of many rows: a wave's
};

// us that a launch takes whose lists are split into parts of up to `per` pages,
// `slots` workgroups at a time, each `fix` and `page` for a page (1.74 times
// that for two row tiles a wave); a join's launch, its partials written and read
// at 6 TB/s, what passes 128 MB slower.  Lists of one length go round by round,
// others fill the gaps of each other.
struct LaunchCost {
    int64_t n_kv, hd, slots;
    double fix, page;
    double operator()(const std::vector<Tile>& tiles, int64_t per) const {
        double total = 0, longest = 0;
        int64_t n = 0, rows = 0;
        for (const Tile& t : tiles) {
            const int64_t np = (t.n + per - 1) / per;
            const bool two = t.tiles() == 2;
            const double c = fix + (two ? 3 : 0) + (double)((t.n + np - 1) / np) * page * (two ? 1.74 : 1);
            total += (double)np * c;
            longest = std::max(longest, c);
            n += np;
            if (np > 1) rows += np * t.rows;
        }
        if (n == 0) return 0;  // (no launch)
        const double mean = total / (double)n, whole = total * (double)n_kv / (double)slots;
        double e = longest;
        if (n * n_kv > slots) {
            const double rounds = (double)((n * n_kv + slots - 1) / slots) * mean;
            e = std::max(e, whole + (rounds - whole) * std::max(0., 1 - 4 * (1 - mean / longest)));
        }
        if (rows == 0) return e;
        const double b = (double)(rows * n_kv * hd) * 8;
        return e + 4 + b / 6e6 + std::max(0., b - 128e6) / 4e6;
    }
};

}  // namespace

int paged_tables(const PagedGeom& g, const ftx_plan_args& a, std::vector<uint32_t>& mark,
                 uint32_t& epoch, PagedTables& o, std::string& err) {
    auto fail = [&](int code, const char* what) {
        err = std::string("plan: ") + what;
        return code;
    };
    o = PagedTables{};
    if (!a.seqs) return fail(FTX_E_INVALID, "null argument");
    if (a.nseq < 1 || a.nseq > 65535) return fail(FTX_E_INVALID, "nseq out of range (1 .. 65535)");
    if (a.n_head < 0 || a.n_head % g.n_kv || a.n_head > 65535)
        return fail(FTX_E_INVALID, "n_head must be a multiple of the pool's kv heads");
    if (a.window < 0 || a.sinks < 0) return fail(FTX_E_INVALID, "negative window or sinks");
    // (positions stay below 2^30)
    constexpr int64_t FAR = (int64_t)1 << 30;
    const int64_t W = std::min(a.window, FAR), sinks = W ? std::min(a.sinks, FAR) : 0;
    o.n_head = a.n_head;
    o.window = W;
    o.sinks = sinks;
    if ((int64_t)mark.size() != g.n_pages) mark.assign((size_t)g.n_pages, 0u);
    if (epoch >= 0xFFFFFFF0u) {
        std::fill(mark.begin(), mark.end(), 0u);
        epoch = 0;
    }
    // marks of this call: named once / written / written and named
    const uint32_t named = epoch + 1, written = epoch + 2;
    epoch += 2;
    const int64_t gqa = a.n_head / g.n_kv;
    for (int64_t s = 0; s < a.nseq; ++s) {
        const ftx_paged_seq& q = a.seqs[s];
        if (q.npast < 0 || q.M < 0 || q.npast > FAR || q.M > FAR || q.npast + q.M > FAR)
            return fail(FTX_E_RANGE, "npast and M must be >= 0, npast + M <= 2^30");
        if (q.parents && q.M > 256) return fail(FTX_E_INVALID, "a draft tree has at most 256 nodes");
        const int64_t ntab = (q.npast + q.M + FTX_PAGE - 1) / FTX_PAGE;
        if (q.n_pages < ntab || (ntab && !q.pages))
            return fail(FTX_E_INVALID, "too few pages for npast + M");
        PagedSeq d{};
        d.npast = (int32_t)q.npast;
        d.M = (int32_t)q.M;
        d.tok0 = (int32_t)o.tokens;
        d.tab0 = (int32_t)o.table.size();
        d.ntab = (int32_t)ntab;
        d.dep0 = -1;
        d.all0 = o.rows;
        o.tokens += q.M;
        o.longest = std::max(o.longest, q.M);
        o.rows += q.npast + q.M;
        if (o.tokens * std::max<int64_t>(a.n_head, 1) >= (int64_t)1 << 31 ||
            (int64_t)o.table.size() + ntab >= (int64_t)1 << 31 || ntab * 2 * g.n_kv >= (int64_t)1 << 31)
            return fail(FTX_E_RANGE, "too many tokens or pages in one plan");
        const int64_t first_new = q.M ? q.npast / FTX_PAGE : ntab;
        for (int64_t i = 0; i < ntab; ++i) {
            const int32_t pg = q.pages[i];
            o.table.push_back(pg);
            if (pg == -1) {
                if (i >= first_new) return fail(FTX_E_INVALID, "a page of new tokens is absent");
                o.absent = true;
                continue;
            }
            if (pg < 0 || pg >= g.n_pages) return fail(FTX_E_RANGE, "page id out of range");
            if (!g.taken[pg]) return fail(FTX_E_INVALID, "a page is not taken from the pool");
            uint32_t& mk = mark[(size_t)pg];
            if (mk == written || (mk == named && i >= first_new))
                return fail(FTX_E_INVALID, "a page that new tokens go to occurs twice");
            mk = i >= first_new ? written : named;
        }
        if (q.M) o.max_new_pages = std::max(o.max_new_pages, ntab - first_new);
        o.max_pages = std::max(o.max_pages, ntab);
        if (q.parents) {
            d.dep0 = (int32_t)o.depth.size();
            d.aw = (int32_t)((q.M + 31) / 32);
            d.anc0 = (int32_t)o.anc.size();
            o.anc.resize(o.anc.size() + (size_t)(q.M * d.aw), 0u);
            uint32_t* anc = o.anc.data() + d.anc0;
            for (int64_t i = 0; i < q.M; ++i) {
                const int32_t p = q.parents[i];
                if (p < -1 || p >= i) return fail(FTX_E_INVALID, "parents[i] must be in [-1, i)");
                o.depth.push_back(p < 0 ? 0 : o.depth[(size_t)(d.dep0 + p)] + 1);
                if (p >= 0) std::copy(anc + p * d.aw, anc + (p + 1) * d.aw, anc + i * d.aw);
                anc[i * d.aw + i / 32] |= 1u << (i % 32);
            }
            // (the ancestors are complete: what the window hides goes last)
            const int32_t* dep = o.depth.data() + d.dep0;
            for (int64_t i = 0; W && i < q.M; ++i)
                for (int64_t j = 0; j < i; ++j)
                    if (dep[i] - dep[j] >= W && q.npast + dep[j] >= sinks)
                        anc[i * d.aw + j / 32] &= ~(1u << (j % 32));
        }
        o.seqs.push_back(d);
    }
    if (!paged_grid_fits(o.max_new_pages * 2 * g.n_kv, 256))
        return fail(FTX_E_RANGE, "too many new tokens of one sequence in one plan");
    if (a.n_head == 0) return FTX_OK;
    // The row tiles and the pages each sees: of TR rows for the sequences of
    // PAGED_MANY rows and more (big) or the others.  false: a page is absent.
    auto tile_all = [&](std::vector<Tile>& tiles, bool big, int64_t TR) -> bool {
        for (int64_t s = 0; s < a.nseq; ++s) {
            const PagedSeq& d = o.seqs[(size_t)s];
            const int64_t R = d.M * gqa;
            if ((R >= PAGED_MANY) != big) continue;
            int64_t checked_s = 0, checked_a = d.ntab;  // pages seen so far: [0, checked_s), [checked_a, ..)
            for (int64_t row0 = 0; row0 < R; row0 += TR) {
                const int64_t t0 = row0 / gqa, t1 = (std::min(R, row0 + TR) - 1) / gqa;
                // (a tree's nodes are all looked at: a node's position is below its slot)
                int64_t lo = 0;
                if (W) lo = std::max<int64_t>(0, d.npast + (d.dep0 >= 0 ? 0 : t0) - W + 1);
                const int64_t pa = lo / FTX_PAGE, pe = (d.npast + t1) / FTX_PAGE + 1;
                const int64_t ps = std::min((sinks + FTX_PAGE - 1) / FTX_PAGE, pa);
                tiles.push_back(Tile{(int32_t)s, (int32_t)row0, (int32_t)std::min(R - row0, TR), (int32_t)ps,
                                     (int32_t)pa, (int32_t)(ps + pe - pa)});
                for (; checked_s < ps; ++checked_s)
                    if (o.table[(size_t)(d.tab0 + checked_s)] < 0) return false;
                for (; checked_a > pa; --checked_a)
                    if (o.table[(size_t)(d.tab0 + checked_a - 1)] < 0) return false;
            }
        }
        return true;
    };
    const int64_t cu = std::max(g.cu, 1);
    // Few rows: lists are split so that a launch has some four workgroups a CU (1
    // to 4 are within 5%, 8 are 8% slower for one token over 131072), no finer
    // than four pages, one a wave; or, where the launch has at most a workgroup a
    // CU, stay whole for workgroups of eight waves and need no join.  Whole / split,
    // us, for sequences x pages (one token, 8-bit 128 dims, 8 kv heads): 1 x 7 8.8 /
    // 9.9, 1 x 17 11.6 / 10.0, 8 x 12 10.1 / 10.5, 8 x 22 14.7 / 12.4, 16 x 46
    // 23.8 / 27.5, 32 x 17 16.7 / 22.7; 64 dims: 1 x 12 7.2 / 8.8, 8 x 17 8.9 /
    // 8.8, 16 x 46 17.2 / 17.9.  Halves, of twice the bytes a page, go by the same rule.
    struct Few {
        bool wide;
        int64_t per;
        double us;
    };
    auto few_plan = [&](const std::vector<Tile>& tiles) {
        int64_t total = 0, longest = 0;
        for (const Tile& t : tiles) {
            total += t.n;
            longest = std::max<int64_t>(longest, t.n);
        }
        const double load = (double)(total * g.n_kv) / (double)cu;  // pages a CU
        if (g.hd <= 128 && longest > 4 && longest <= WIDE_MOST && (int64_t)tiles.size() * g.n_kv <= cu &&
            (double)longest <= (g.hd == 64 ? 15 : 10) + 1.6 * load)
            return Few{true, INT32_MAX, 6 + std::max((0.17 + 0.17 * (double)g.hd / 128) * (double)longest, 0.6 * load)};
        const int64_t per = std::max<int64_t>(4, (total * g.n_kv + 4 * cu - 1) / (4 * cu));
        return Few{false, per, LaunchCost{g.n_kv, g.hd, 2 * cu, 8, 0.8 * (double)g.hd / 128}(tiles, per)};
    };
    std::vector<Tile> tiles[2], big;  // of PAGED_TR rows, of many
    int64_t per[2] = {INT32_MAX, INT32_MAX}, big_rows = 0;
    bool present = tile_all(tiles[0], false, PAGED_TR);
    for (const PagedSeq& d : o.seqs)
        if (d.M * gqa >= PAGED_MANY) big_rows += d.M * gqa;
    if (present && big_rows) {
        // Sequences of many rows: tiles of 256, 128 or 16 rows (the kernel of
        // few), their lists split as it is estimated fastest.  Measured, us, for
        // rows x context (8-bit, 128 dims, 8 kv heads), by 256 / 128 / 16 rows:
        // 16 x 1024 over 4000: 508 / 581 / 753; 16 x 768 over 4000 (256 rows
        // leave a third of the second round empty): 545 / 480 / -; 4 x 68 over
        // 4000: - / 29 / 34; 256 over 300: 22 / 15 / 11.
        const double page = 0.75 + 1.5 * (double)g.hd / 128;
        double best = 1e300;
        int64_t bestp = 0, chosen = 0;
        const int force = forced_rows;
        const int64_t most = g.hd <= 128 && (force == 0 || force > PAGED_TR_MANY) ? 2 * PAGED_TR_MANY : PAGED_TR_MANY;
        for (int64_t TR = most; present && TR >= PAGED_TR_MANY; TR /= 2) {
            if (force && TR < most) break;
            big.clear();
            present = tile_all(big, true, TR);
            const LaunchCost cost{g.n_kv, g.hd, cu, 8, page};
            int64_t longest = 0;
            for (const Tile& t : big) longest = std::max<int64_t>(longest, t.n);
            const bool full = (int64_t)big.size() * g.n_kv >= 4 * cu;
            for (int64_t k = 1; k <= 64; k += 1 + k / 6) {
                const int64_t p = (longest + k - 1) / k;
                if (k > 1 && (full || p < 2)) break;
                const double us = cost(big, p);
                if (us >= best) continue;
                best = us;
                bestp = p;
                chosen = TR;
            }
            if (chosen == TR) {
                tiles[1] = big;
                per[1] = bestp;
            }
        }
        if (present && (force ? force == PAGED_TR : big_rows / PAGED_TR <= FEW_MOST)) {
            big = tiles[0];
            present = tile_all(big, true, PAGED_TR);
            if (present && (force || few_plan(big).us - few_plan(tiles[0]).us < best)) {
                tiles[0] = big;
                tiles[1].clear();
            }
        }
    }
    if (!present) return fail(FTX_E_INVALID, "a page that a new token sees is absent");
    const Few few = few_plan(tiles[0]);
    per[0] = few.per;
    o.wide = few.wide;
    o.pages_read = 0;
    for (int many = 0; many < 2; ++many) {
        for (const Tile& t : tiles[many]) {
            o.pages_read += t.n;
            const int nt = many ? t.tiles() : 0;
            const int64_t np = (t.n + per[many] - 1) / per[many], blocks = many ? nt * PAGED_TR_MANY / PAGED_TR : 1;
            for (int64_t k = 0; k < np; ++k)
                o.items.push_back(PagedItem{t.seq, t.row0, (int32_t)(t.n * k / np), (int32_t)(t.n * (k + 1) / np), t.s,
                                            t.a, np > 1 ? (int32_t)(o.parts + k * blocks) : -1, nt,
                                            o.seqs[(size_t)t.seq], {}});
            if (np == 1) continue;
            o.comb_max = std::max(o.comb_max, np);
            for (int64_t r = 0; r < t.rows; r += PAGED_TR)
                o.combs.push_back(PagedComb{t.seq, (int32_t)(t.row0 + r), (int32_t)(o.parts + r / PAGED_TR), (int32_t)np,
                                            (int32_t)blocks, o.seqs[(size_t)t.seq].tok0, o.seqs[(size_t)t.seq].M, 0});
            o.parts += np * blocks;
        }
        // the longest first (two row tiles a wave: 7 for 4)
        auto work = [](const PagedItem& x) { return (x.i1 - x.i0) * (int64_t)(x.nt == 2 ? 7 : 4); };
        std::stable_sort(o.items.begin() + o.few, o.items.end(),
                         [&](const PagedItem& x, const PagedItem& y) { return work(x) > work(y); });
        if (!many) o.few = (int64_t)o.items.size();
    }
    if (!paged_grid_fits(o.few * g.n_kv, o.wide ? 512 : 256) ||
        !paged_grid_fits(((int64_t)o.items.size() - o.few) * g.n_kv, 512) ||
        !paged_grid_fits((int64_t)o.combs.size() * g.n_kv, 256) || o.parts >= (int64_t)1 << 31)
        return fail(FTX_E_RANGE, "too many tokens or pages in one plan");
    return FTX_OK;
}

extern "C" void paged_force_rows(int rows) { forced_rows = rows; }

extern "C" int paged_probe(const ftx_plan_args* a, int64_t n_kv, int64_t hd, int64_t n_pages, const uint8_t* taken,
                           int cu, PagedItem* items, int64_t* n_items, PagedComb* combs, int64_t* n_combs,
                           int64_t max_out, char* msg, int64_t msg_bytes) {
    try {
        PagedGeom g;
        g.n_kv = n_kv;
        g.hd = hd;
        g.n_pages = n_pages;
        g.taken = taken;
        g.cu = cu;
        std::vector<uint32_t> mark;
        uint32_t epoch = 0;
        PagedTables t;
        std::string err;
        const int rc = paged_tables(g, *a, mark, epoch, t, err);
        snprintf(msg, (size_t)msg_bytes, "%s", err.c_str());
        if (rc) return rc;
        *n_items = (int64_t)t.items.size();
        *n_combs = (int64_t)t.combs.size();
        if (*n_items > max_out || *n_combs > max_out) return FTX_E_RANGE;
        std::copy(t.items.begin(), t.items.end(), items);
        std::copy(t.combs.begin(), t.combs.end(), combs);
        return FTX_OK;
    } catch (...) {
        return FTX_E_NOMEM;
    }
}

// ---------------------------------------------------------------- pool and plan

namespace {

// the context's device made current for a scope
struct OnDevice {
    int prev = -1;
    bool ok = true;
    explicit OnDevice(int dev) {
        if (hipGetDevice(&prev) != hipSuccess) prev = -1;
        if (prev == dev) {
            prev = -1;
            return;
        }
        ok = hipSetDevice(dev) == hipSuccess;
        if (!ok) (void)hipGetLastError();
    }
    ~OnDevice() {
        if (prev >= 0) (void)hipSetDevice(prev);
    }
};

bool capturing(hipStream_t st) {
    hipStreamCaptureStatus s = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(st, &s) != hipSuccess) {
        (void)hipGetLastError();
        return false;
    }
    return s != hipStreamCaptureStatusNone;
}

// device memory of the context's own device
bool on_device(const ftx_ctx* ctx, const void* p) {
    hipPointerAttribute_t at;
    if (hipPointerGetAttributes(&at, p) != hipSuccess) {
        (void)hipGetLastError();
        return false;
    }
    return (at.type == hipMemoryTypeDevice && at.device == ctx->device) || at.type == hipMemoryTypeManaged;
}

// No events of the trace go into a captured graph
struct NoTrace {
    ftx_ctx* ctx;
    bool was;
    NoTrace(ftx_ctx* c, bool off) : ctx(c), was(c->trace) { c->trace = was && !off; }
    ~NoTrace() { ctx->trace = was; }
};

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace

struct ftx_plan {
    ftx_ctx* ctx = nullptr;
    ftx_pool* pool = nullptr;
    PagedTables t;
    bool ready = false;     // the device block holds t
    bool captured = false;  // a graph holds calls of this plan
    std::vector<uint32_t> mark;
    uint32_t epoch = 0;
    uint8_t* dev = nullptr;
    size_t dev_bytes = 0;
    float* part = nullptr;
    size_t part_floats = 0;
    // the tables' host copies, in turn; an event after each copy guards its reuse
    static constexpr int RING = 2;
    uint8_t* pin[RING] = {};
    size_t pin_bytes[RING] = {};
    hipEvent_t ev[RING] = {};
    int next = 0;
    hipEvent_t up = nullptr;  // the last copy's
    bool landed = false;      // the host has waited for it
    // of the last set or call outside of captures: another stream waits for the
    // copy, a set on another for everything
    hipStream_t stream = nullptr;
    // the parts of the device block
    size_t o_seq = 0, o_tab = 0, o_dep = 0, o_anc = 0, o_item = 0, o_comb = 0, o_serial = 0;
    size_t bytes = 0;     // of the last set's tables
    uint64_t serial = 0;  // its number
};

static void plan_release(ftx_plan* pl) {
    if (pl->dev) (void)hipFree(pl->dev);
    if (pl->part) (void)hipFree(pl->part);
    for (int i = 0; i < ftx_plan::RING; ++i) {
        if (pl->pin[i]) (void)hipHostFree(pl->pin[i]);
        if (pl->ev[i]) (void)hipEventDestroy(pl->ev[i]);
    }
    if (pl->pool) --pl->pool->users;
    delete pl;
}

// pl->t to the device
static int plan_upload(ftx_plan* pl) {
    ftx_ctx* ctx = pl->ctx;
    const PagedTables& t = pl->t;
    pl->ready = false;
    size_t at = 0;
    auto place = [&](size_t& off, size_t bytes) {
        off = at;
        at += up256(bytes);
    };
    place(pl->o_seq, t.seqs.size() * sizeof(PagedSeq));
    place(pl->o_tab, t.table.size() * 4);
    place(pl->o_dep, t.depth.size() * 4);
    place(pl->o_anc, t.anc.size() * 4);
    place(pl->o_item, t.items.size() * sizeof(PagedItem));
    place(pl->o_comb, t.combs.size() * sizeof(PagedComb));
    place(pl->o_serial, sizeof pl->serial);
    const size_t bytes = pl->bytes = at;
    ++pl->serial;
    const size_t pf = (size_t)t.parts * pl->pool->n_kv * PAGED_TR * (pl->pool->hd + 2);
    hipStream_t st = ctx->stream;
    auto grow = [&](void** p, size_t& have, size_t need, size_t unit) -> int {
        if (need <= have) return FTX_OK;
        if (*p) {
            // calls on this block may still run
            FTX_HIP(ctx, hipDeviceSynchronize());
            FTX_HIP(ctx, hipFree(*p));
            *p = nullptr;
            have = 0;
        }
        need += need / 4;
        if (hipMalloc(p, need * unit + 256) != hipSuccess) {
            (void)hipGetLastError();
            *p = nullptr;
            return ftx_fail(ctx, FTX_E_NOMEM, "plan: device allocation failed");
        }
        have = need;
        return FTX_OK;
    };
    int rc = grow((void**)&pl->dev, pl->dev_bytes, bytes, 1);
    if (!rc) rc = grow((void**)&pl->part, pl->part_floats, pf, sizeof(float));
    if (rc) return rc;
    if (pl->up && pl->stream != st) FTX_HIP(ctx, hipDeviceSynchronize());
    const int k = pl->next;
    if (pl->ev[k]) FTX_HIP(ctx, hipEventSynchronize(pl->ev[k]));
    if (!pl->ev[k]) FTX_HIP(ctx, hipEventCreateWithFlags(&pl->ev[k], hipEventDisableTiming));
    if (bytes > pl->pin_bytes[k]) {
        if (pl->pin[k]) FTX_HIP(ctx, hipHostFree(pl->pin[k]));
        pl->pin[k] = nullptr;
        pl->pin_bytes[k] = 0;
        if (hipHostMalloc((void**)&pl->pin[k], bytes + bytes / 4, hipHostMallocDefault) != hipSuccess) {
            (void)hipGetLastError();
            pl->pin[k] = nullptr;
            return ftx_fail(ctx, FTX_E_NOMEM, "plan: host allocation failed");
        }
        pl->pin_bytes[k] = bytes + bytes / 4;
    }
    uint8_t* h = pl->pin[k];
    auto put = [&](size_t off, const void* src, size_t n) {
        if (n) memcpy(h + off, src, n);
    };
    put(pl->o_seq, t.seqs.data(), t.seqs.size() * sizeof(PagedSeq));
    put(pl->o_tab, t.table.data(), t.table.size() * 4);
    put(pl->o_dep, t.depth.data(), t.depth.size() * 4);
    put(pl->o_anc, t.anc.data(), t.anc.size() * 4);
    put(pl->o_item, t.items.data(), t.items.size() * sizeof(PagedItem));
    put(pl->o_comb, t.combs.data(), t.combs.size() * sizeof(PagedComb));
    put(pl->o_serial, &pl->serial, sizeof pl->serial);
    FTX_HIP(ctx, hipMemcpyAsync(pl->dev, h, bytes, hipMemcpyHostToDevice, st));
    FTX_HIP(ctx, hipEventRecord(pl->ev[k], st));
    pl->up = pl->ev[k];
    pl->landed = false;
    pl->stream = st;
    pl->next = (k + 1) % ftx_plan::RING;
    pl->ready = true;
    return FTX_OK;
}

PagedView paged_view(const ftx_plan* pl, int64_t layer) {
    const ftx_pool* p = pl->pool;
    PagedView v{};
    v.block = p->block;
    v.data = p->data + layer * p->n_pages * p->n_kv * p->block;
    v.n_kv = (int)p->n_kv;
    v.hd = (int)p->hd;
    v.q8 = p->q8;
    v.seqs = (const PagedSeq*)(pl->dev + pl->o_seq);
    v.table = (const int32_t*)(pl->dev + pl->o_tab);
    v.nseq = (int)pl->t.seqs.size();
    return v;
}

// The last set's tables in device memory, seen from the host: read back on a
// stream of its own and compared (their event is no help, HIP refuses one whose
// stream is being captured).  The serial number tells them from an older set's.
static hipError_t tables_landed(const ftx_plan* pl) {
    std::vector<uint8_t> got(pl->bytes);
    const uint8_t* want = pl->pin[(pl->next + ftx_plan::RING - 1) % ftx_plan::RING];
    hipStream_t st;
    hipError_t e = hipStreamCreateWithFlags(&st, hipStreamNonBlocking);
    if (e != hipSuccess) return e;
    for (;;) {
        e = hipMemcpyAsync(got.data(), pl->dev, pl->bytes, hipMemcpyDeviceToHost, st);
        if (e == hipSuccess) e = hipStreamSynchronize(st);
        if (e != hipSuccess || memcmp(got.data(), want, pl->bytes) == 0) break;
        std::this_thread::sleep_for(std::chrono::microseconds(50));
    }
    (void)hipStreamDestroy(st);
    return e;
}

// the tables' copy ahead of a call on another stream than its own, and of a
// captured one on any: the copy is not in the graph, which may be launched on
// another stream than the captured one, so the host waits
static int plan_order(ftx_plan* pl) {
    ftx_ctx* ctx = pl->ctx;
    if (!capturing(ctx->stream)) {
        if (ctx->stream == pl->stream) return FTX_OK;
        FTX_HIP(ctx, hipStreamWaitEvent(ctx->stream, pl->up, 0));
        pl->stream = ctx->stream;
        return FTX_OK;
    }
    pl->captured = true;
    if (pl->landed) return FTX_OK;
    OnDevice od(ctx->device);
    hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
    FTX_HIP(ctx, hipThreadExchangeStreamCaptureMode(&mode));
    hipError_t e;
    try {
        e = tables_landed(pl);
    } catch (...) {
        e = hipErrorOutOfMemory;
    }
    FTX_HIP(ctx, hipThreadExchangeStreamCaptureMode(&mode));
    FTX_HIP(ctx, e);
    pl->landed = true;
    return FTX_OK;
}

// what every call of a plan checks, before plan_order; *ld: 0 becomes `width`
static int plan_call(ftx_plan* pl, int64_t layer, const void* x, int64_t* ldx, int64_t xw, const void* y,
                     int64_t* ldy, int64_t yw) {
    ftx_ctx* ctx = pl->ctx;
    if (!pl->ready) return ftx_fail(ctx, FTX_E_INVALID, "the plan has no sequences");
    if (layer < 0 || layer >= pl->pool->n_layer) return ftx_fail(ctx, FTX_E_RANGE, "layer out of range");
    if (!x || !y) return ftx_fail(ctx, FTX_E_INVALID, "null argument");
    if (*ldx == 0) *ldx = xw;
    if (*ldy == 0) *ldy = yw;
    if (*ldx < xw || *ldy < yw) return ftx_fail(ctx, FTX_E_INVALID, "row stride shorter than a row");
    if (((uintptr_t)x | (uintptr_t)y) & 3) return ftx_fail(ctx, FTX_E_INVALID, "rows must be 4-byte aligned");
    if (!on_device(ctx, x) || !on_device(ctx, y))
        return ftx_fail(ctx, FTX_E_INVALID, "rows must be memory of the context's device");
    return FTX_OK;
}

// whether n rows of w floats, ldx and ldy apart, at x and y share a float
static bool rows_overlap(const float* x, int64_t ldx, const float* y, int64_t ldy, int64_t w, int64_t n) {
    const intptr_t x0 = (intptr_t)x / 4, y0 = (intptr_t)y / 4;
    if (n <= 0 || x0 + (n - 1) * ldx + w <= y0 || y0 + (n - 1) * ldy + w <= x0) return false;
    if (ldx != ldy) return true;
    // two column ranges of one matrix
    const intptr_t r = ((y0 - x0) % ldx + ldx) % ldx;
    return r < w || r > ldx - w;
}

extern "C" {

int ftx_pool_create(ftx_ctx* ctx, int64_t n_layer, int64_t n_head_kv, int64_t head_dim, int64_t n_pages,
                    int kv_dtype, ftx_pool** out) {
    if (!ctx || !out) return ftx_fail(ctx, FTX_E_INVALID, "null argument");
    *out = nullptr;
    if (n_layer < 1 || n_layer > 65535 || n_head_kv < 1 || n_head_kv > 1024 || n_pages < 1 ||
        n_pages > (int64_t)1 << 24)
        return ftx_fail(ctx, FTX_E_INVALID, "pool: layers, kv heads or pages out of range");
    if (head_dim != 64 && head_dim != 128 && head_dim != 256)
        return ftx_fail(ctx, FTX_E_UNSUPPORTED, "pool: head_dim must be 64, 128 or 256");
    if (kv_dtype != FTX_KV_F16 && kv_dtype != FTX_KV_Q8)
        return ftx_fail(ctx, FTX_E_UNSUPPORTED, "pool: kv dtype must be F16 or Q8");
    OnDevice od(ctx->device);
    if (!od.ok) return ftx_fail(ctx, FTX_E_DEVICE, "the context's device could not be made current");
    ftx_pool* p = new (std::nothrow) ftx_pool;
    if (!p) return ftx_fail(ctx, FTX_E_NOMEM, "host allocation failed");
    p->ctx = ctx;
    p->n_layer = n_layer;
    p->n_kv = n_head_kv;
    p->hd = head_dim;
    p->n_pages = n_pages;
    p->q8 = kv_dtype == FTX_KV_Q8;
    p->block = paged_block_bytes((int)head_dim, p->q8);
    p->free_pages = n_pages;
    try {
        p->taken.assign((size_t)n_pages, 0);
    } catch (...) {
        delete p;
        return ftx_fail(ctx, FTX_E_NOMEM, "host allocation failed");
    }
    // (up to 2^66: past 64 bits the product would come round to a small size)
    const int64_t blocks = n_layer * n_pages * n_head_kv;
    const size_t bytes = blocks <= ((int64_t)1 << 62) / p->block ? (size_t)(blocks * p->block) : 0;
    if (bytes == 0 || hipMalloc((void**)&p->data, bytes) != hipSuccess) {
        (void)hipGetLastError();
        delete p;
        return ftx_fail(ctx, FTX_E_NOMEM, "pool allocation failed");
    }
    // finite values everywhere: slots that a row does not see still meet its P.V product
    if (hipMemset(p->data, 0, bytes) != hipSuccess || hipDeviceSynchronize() != hipSuccess) {
        (void)hipGetLastError();
        (void)hipFree(p->data);
        delete p;
        return ftx_fail(ctx, FTX_E_DEVICE, "pool: clearing failed");
    }
    *out = p;
    return FTX_OK;
}

int ftx_pool_free(ftx_pool* p) {
    if (!p) return FTX_OK;
    if (p->users) return ftx_fail(p->ctx, FTX_E_INVALID, "pool: a plan or cache of it lives");
    OnDevice od(p->ctx->device);
    (void)hipStreamSynchronize(p->ctx->stream);
    if (p->step) {
        ++p->users;
        plan_release(p->step);
    }
    if (p->data) (void)hipFree(p->data);
    delete p;
    return FTX_OK;
}

int64_t ftx_pool_available(const ftx_pool* p) { return p ? p->free_pages : 0; }

int ftx_pool_take(ftx_pool* p, int64_t n, int32_t* pages) {
    if (!p) return FTX_E_INVALID;
    if (n < 0 || (n && !pages)) return ftx_fail(p->ctx, FTX_E_INVALID, "pool_take: bad argument");
    if (n > p->free_pages) return ftx_fail(p->ctx, FTX_E_NOMEM, "pool_take: not enough free pages");
    p->take(n, pages);
    return FTX_OK;
}

int ftx_pool_give(ftx_pool* p, const int32_t* pages, int64_t n) {
    if (!p) return FTX_E_INVALID;
    if (n < 0 || (n && !pages)) return ftx_fail(p->ctx, FTX_E_INVALID, "pool_give: bad argument");
    return p->give(pages, n) ? FTX_OK
                             : ftx_fail(p->ctx, FTX_E_INVALID, "pool_give: a page is not taken or named twice");
}

int ftx_plan_set(ftx_plan* pl, const ftx_plan_args* a) {
    if (!pl) return FTX_E_INVALID;
    ftx_ctx* ctx = pl->ctx;
    if (!a) return ftx_fail(ctx, FTX_E_INVALID, "null argument");
    if (pl->captured) return ftx_fail(ctx, FTX_E_INVALID, "plan: a graph holds calls of this plan");
    if (capturing(ctx->stream)) return ftx_fail(ctx, FTX_E_INVALID, "plan: set while the stream is captured");
    OnDevice od(ctx->device);
    if (!od.ok) return ftx_fail(ctx, FTX_E_DEVICE, "the context's device could not be made current");
    try {
        PagedGeom g;
        g.n_kv = pl->pool->n_kv;
        g.hd = pl->pool->hd;
        g.n_pages = pl->pool->n_pages;
        g.taken = pl->pool->taken.data();
        g.cu = ctx->cu_count;
        PagedTables t;
        std::string err;
        const int rc = paged_tables(g, *a, pl->mark, pl->epoch, t, err);
        if (rc) return ftx_fail(ctx, rc, err);
        std::swap(pl->t, t);
        return plan_upload(pl);
    } catch (...) {
        pl->ready = false;
        return ftx_fail(ctx, FTX_E_NOMEM, "host allocation failed");
    }
}

int ftx_plan_create(ftx_ctx* ctx, ftx_pool* p, const ftx_plan_args* a, ftx_plan** out) {
    if (!ctx || !p || !a || !out) return ftx_fail(ctx, FTX_E_INVALID, "null argument");
    *out = nullptr;
    if (p->ctx != ctx) return ftx_fail(ctx, FTX_E_INVALID, "plan: the pool is another context's");
    ftx_plan* pl = new (std::nothrow) ftx_plan;
    if (!pl) return ftx_fail(ctx, FTX_E_NOMEM, "host allocation failed");
    pl->ctx = ctx;
    pl->pool = p;
    ++p->users;
    const int rc = ftx_plan_set(pl, a);
    if (rc) {
        plan_release(pl);
        return rc;
    }
    *out = pl;
    return FTX_OK;
}

int ftx_plan_free(ftx_plan* pl) {
    if (!pl) return FTX_OK;
    OnDevice od(pl->ctx->device);
    (void)hipStreamSynchronize(pl->ctx->stream);
    plan_release(pl);
    return FTX_OK;
}

int ftx_paged_write(ftx_plan* pl, int64_t layer, const float* k, int64_t ldk, const float* v, int64_t ldv) {
    if (!pl) return FTX_E_INVALID;
    const int64_t w = pl->pool->n_kv * pl->pool->hd;
    if (pl->ready && pl->t.tokens == 0) return FTX_OK;
    int rc = plan_call(pl, layer, k, &ldk, w, v, &ldv, w);
    if (!rc) rc = plan_order(pl);
    return rc ? rc : paged_write_rows(pl, layer, k, ldk, v, ldv);
}

int ftx_paged_read(ftx_plan* pl, int64_t layer, int context, float* k, int64_t ldk, float* v, int64_t ldv) {
    if (!pl) return FTX_E_INVALID;
    const int64_t w = pl->pool->n_kv * pl->pool->hd;
    const int64_t n = context ? pl->t.rows : pl->t.tokens;
    if (pl->ready && n == 0) return FTX_OK;
    int rc = plan_call(pl, layer, k, &ldk, w, v, &ldv, w);
    if (rc) return rc;
    if (context && !paged_grid_fits(pl->t.max_pages * 2 * pl->pool->n_kv, 256))
        return ftx_fail(pl->ctx, FTX_E_RANGE, "paged_read: too many positions of one sequence");
    if (context && pl->t.absent) return ftx_fail(pl->ctx, FTX_E_RANGE, "paged_read: a page is absent");
    if (rows_overlap(k, ldk, v, ldv, w, n)) return ftx_fail(pl->ctx, FTX_E_INVALID, "paged_read: k and v overlap");
    rc = plan_order(pl);
    return rc ? rc : paged_read_rows(pl, layer, context, k, ldk, v, ldv);
}

int ftx_paged_attention(ftx_plan* pl, int64_t layer, const float* q, int64_t ldq, float* out, int64_t ldo) {
    if (!pl) return FTX_E_INVALID;
    if (pl->ready && pl->t.n_head == 0) return ftx_fail(pl->ctx, FTX_E_INVALID, "the plan has no query heads");
    if (pl->ready && pl->t.tokens == 0) return FTX_OK;
    const int64_t w = pl->t.n_head * pl->pool->hd;
    int rc = plan_call(pl, layer, q, &ldq, w, out, &ldo, w);
    if (rc) return rc;
    if (rows_overlap(q, ldq, out, ldo, w, pl->t.tokens))
        return ftx_fail(pl->ctx, FTX_E_INVALID, "paged_attention: q and out overlap");
    rc = plan_order(pl);
    return rc ? rc : paged_attend_rows(pl, layer, q, ldq, out, ldo);
}

}  // extern "C"

// ---------------------------------------------------------------- launches of a plan

// bytes that n rows of K and V move
static double rows_bytes(const ftx_pool* p, double n) {
    return n * p->n_kv * (8.0 * p->hd + (double)p->block / FTX_PAGE);
}

int paged_write_rows(ftx_plan* pl, int64_t layer, const float* k, int64_t ldk, const float* v, int64_t ldv) {
    ftx_ctx* ctx = pl->ctx;
    OnDevice od(ctx->device);
    NoTrace nt(ctx, ctx->trace && capturing(ctx->stream));
    TraceScope ts(ctx);
    FTX_HIP(ctx, launch_paged_write(ctx->stream, paged_view(pl, layer), pl->t.max_new_pages, k, ldk, v, ldv));
    ts.end(TK_PAGED_KV, rows_bytes(pl->pool, (double)pl->t.tokens));
    return FTX_OK;
}

int paged_read_rows(ftx_plan* pl, int64_t layer, int context, float* k, int64_t ldk, float* v, int64_t ldv) {
    ftx_ctx* ctx = pl->ctx;
    OnDevice od(ctx->device);
    NoTrace nt(ctx, ctx->trace && capturing(ctx->stream));
    TraceScope ts(ctx);
    FTX_HIP(ctx, launch_paged_read(ctx->stream, paged_view(pl, layer),
                                   context ? pl->t.max_pages : pl->t.max_new_pages, context, k, ldk, v, ldv));
    ts.end(TK_PAGED_KV, rows_bytes(pl->pool, (double)(context ? pl->t.rows : pl->t.tokens)));
    return FTX_OK;
}

int paged_attend_rows(ftx_plan* pl, int64_t layer, const float* q, int64_t ldq, float* out, int64_t ldo) {
    ftx_ctx* ctx = pl->ctx;
    const PagedTables& t = pl->t;
    const ftx_pool* p = pl->pool;
    OnDevice od(ctx->device);
    PagedAttn a{};
    a.p = paged_view(pl, layer);
    a.depth = (const int32_t*)(pl->dev + pl->o_dep);
    a.anc = (const uint32_t*)(pl->dev + pl->o_anc);
    a.items = (const PagedItem*)(pl->dev + pl->o_item);
    a.combs = (const PagedComb*)(pl->dev + pl->o_comb);
    a.n_few = (int)t.few;
    a.n_many = (int)((int64_t)t.items.size() - t.few);
    a.n_combs = (int)t.combs.size();
    a.wide = t.wide;
    a.gqa = (int)(t.n_head / p->n_kv);
    a.rows_max = (int)(t.longest * a.gqa);
    a.comb_max = (int)std::min<int64_t>(t.comb_max, INT32_MAX);
    a.window = (int)t.window;
    a.sinks = (int)t.sinks;
    a.q = q;
    a.out = out;
    a.ldq = ldq;
    a.ldo = ldo;
    a.part = pl->part;
    a.pml = pl->part + (size_t)t.parts * p->n_kv * PAGED_TR * p->hd;
    NoTrace nt(ctx, ctx->trace && capturing(ctx->stream));
    TraceScope ts(ctx);
    FTX_HIP(ctx, launch_paged_attention(ctx->stream, a));
    ts.end(TK_ATTENTION, t.pages_read * p->n_kv * (double)p->block + 8.0 * t.tokens * t.n_head * p->hd);
    return FTX_OK;
}

int paged_step_plan(ftx_ctx* ctx, ftx_pool* p, const ftx_plan_args& a, ftx_plan** out) {
    if (!p->step) {
        const int rc = ftx_plan_create(ctx, p, &a, &p->step);
        if (rc) return rc;
        --p->users;  // the pool's own
        *out = p->step;
        return FTX_OK;
    }
    *out = p->step;
    return ftx_plan_set(p->step, &a);
}
