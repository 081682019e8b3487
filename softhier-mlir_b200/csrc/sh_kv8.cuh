// What the entry points of the paged 8-bit K / V cache (sh_cuda_kv8_t) share: the checks of its descriptor.
#pragma once

#include "sh_internal.cuh"

namespace sh {

inline bool kv8_page_ok(uint32_t page) { return page == 16 || page == 32 || page == 64 || page == 128; }
inline uint32_t kv8_shift(uint32_t page) { return page == 16 ? 4u : page == 32 ? 5u : page == 64 ? 6u : 7u; }

// arrays of 32-bit words lie on whole words
inline bool words_ok(uint64_t a, uint64_t b = 0, uint64_t c = 0, uint64_t d = 0) { return ((a | b | c | d) & 3) == 0; }

// 0, or -1 / -3 with the reason recorded
inline int kv8_check(const sh_cuda_kv8_t *c, const char *who) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || !aligned16(c->k) || !aligned16(c->v) ||
        (c->k_scale & 3) || (c->v_scale & 3)) {
        set_error(-1, "[%s] null cache or arrays, or codes not 16-byte aligned", who);
        return -1;
    }
    if (c->fmt != SH_INT8 && c->fmt != SH_FP8) {
        set_error(-3, "[%s] fmt %u is neither SH_INT8 nor SH_FP8", who, c->fmt);
        return -3;
    }
    if (!kv8_page_ok(c->page) || (c->dh != 64 && c->dh != 128) || c->heads == 0 || c->pages == 0 ||
        (uint64_t)c->pages * c->page >= (1ull << 31)) {
        set_error(-1, "[%s] need page 16, 32, 64 or 128, dh 64 or 128, heads > 0, 0 < pages * page < 2^31 (page=%u dh=%u "
                  "heads=%u pages=%u)", who, c->page, c->dh, c->heads, c->pages);
        return -1;
    }
    if (c->page_stride % 16 || c->page_stride < (uint64_t)c->heads * c->page * c->dh) {
        set_error(-1, "[%s] page_stride %llu is not a multiple of 16 or less than heads * page * dh", who,
                  (unsigned long long)c->page_stride);
        return -1;
    }
    return 0;
}

}  // namespace sh
