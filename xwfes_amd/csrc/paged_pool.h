// paged_pool.h -- the page pool's host side: which pages are taken.
#pragma once

#include <cstdint>
#include <vector>

struct ftx_ctx;
struct ftx_plan;

struct ftx_pool {
    ftx_ctx* ctx = nullptr;
    int64_t n_layer = 0, n_kv = 0, hd = 0, n_pages = 0;
    int kt = 0;  // how rows are stored (PT_F16, ..)
    int64_t block = 0;  // bytes of one (layer, page, kv head)
    uint8_t* data = nullptr;  // [n_layer][n_pages][n_kv] blocks
    std::vector<uint8_t> taken;
    int64_t free_pages = 0, low = 0;  // no free page below `low`
    int users = 0;  // plans and caches
    ftx_plan* step = nullptr;  // of the verify steps over the pool

    // n <= free_pages of them, the lowest ids
    void take(int64_t n, int32_t* pages) {
        int64_t i = low;
        for (int64_t k = 0; k < n; ++i)
            if (!taken[(size_t)i]) {
                taken[(size_t)i] = 1;
                pages[k++] = (int32_t)i;
            }
        low = i;
        free_pages -= n;
    }
    // all of them, or none and false
    bool give(const int32_t* pages, int64_t n) {
        for (int64_t k = 0; k < n; ++k) {
            const int32_t pg = pages[k];
            if (pg < 0 || pg >= n_pages || !taken[(size_t)pg]) {
                for (int64_t j = 0; j < k; ++j) taken[(size_t)pages[j]] = 1;
                return false;
            }
            taken[(size_t)pg] = 0;  // (a page named twice is free the second time)
        }
        for (int64_t k = 0; k < n; ++k)
            if (pages[k] < low) low = pages[k];
        free_pages += n;
        return true;
    }
};
