// The paged 8-bit K / V cache of a decode step: block tables and slot maps from request lengths (sh_cuda_kv_tables) and
// the quantising append (sh_cuda_kv8_append). The attention that reads the cache is in sh_attention_kv8.cu.
#include "sh_kv8.cuh"

namespace {

// ================================================================================================================
// Tables. Every CTA scans all R requests (three running sums: new tokens, new pages, pages given back) into shared
// memory, so a token's request is a binary search there and no CTA waits for another; CTA c then fills its share of the
// slot map. The pages a call takes come from the ring's head and those it gets back go to its tail, so no entry
// that one CTA reads is written by another. lens / pool may be updated in place: each CTA draws a ticket once it has
// read them, and the CTA with the last one writes the new state.
// Bound by latency: one round trip for the lengths, one for the table. A second launch for the slot map would cost as much
// again.
// ================================================================================================================
constexpr uint32_t kTabThreads = 512, kTabMaxR = 8192;

struct TablesArgs {
    const int *lens, *add;
    int *table, *ring;
    const uint32_t *pool;
    uint32_t *pool_out;
    int *lens_out, *q_start, *slots, *pos;
    uint32_t R, page_shift, ld_table, pages, t_cap;
    uint32_t vec;   // slots / pos take 16-byte stores
};

// inclusive sums over the block of three values per thread
__device__ __forceinline__ void block_scan3(uint32_t &a, uint32_t &b, uint32_t &c, uint32_t (*part)[3]) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o),
                       z = __shfl_up_sync(0xffffffffu, c, o);
        if (lane >= (uint32_t)o) a += x, b += y, c += z;
    }
    if (lane == 31) part[warp][0] = a, part[warp][1] = b, part[warp][2] = c;
    __syncthreads();
    uint32_t x = 0, y = 0, z = 0;
    if (lane < kTabThreads / 32 && lane < warp) x = part[lane][0], y = part[lane][1], z = part[lane][2];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        x += __shfl_xor_sync(0xffffffffu, x, o);
        y += __shfl_xor_sync(0xffffffffu, y, o);
        z += __shfl_xor_sync(0xffffffffu, z, o);
    }
    a += x, b += y, c += z;
}

// first index with v[index] > i (v rises), or n
__device__ __forceinline__ uint32_t upper_bound(const uint32_t *v, uint32_t n, uint32_t i) {
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) >> 1;
        if (v[mid] > i) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

struct Req {   // what a request's length and new tokens make of it, before the ring is looked at
    uint32_t len, n, have, need, back;
    bool ended, too_long;
};
__device__ __forceinline__ Req request(int len, int add, uint32_t shift, uint32_t ld) {
    Req q;
    q.len = (uint32_t)max(len, 0);
    q.ended = add < 0;
    q.n = (uint32_t)max(add, 0);
    const uint32_t page1 = (1u << shift) - 1;
    q.have = (q.len + page1) >> shift;                 // < 2^31 + 128: no wrap
    const uint32_t total = (uint32_t)(((uint64_t)q.len + q.n + page1) >> shift);
    q.too_long = total > ld;
    q.need = q.ended || q.too_long ? 0u : total - q.have;
    q.back = q.ended ? min(q.have, ld) : 0u;
    return q;
}

template <uint32_t PER>
__global__ void __launch_bounds__(kTabThreads) k_kv_tables(TablesArgs a) {
    extern __shared__ uint32_t sm[];
    __shared__ uint32_t part[kTabThreads / 32][3];
    __shared__ uint32_t s_taken, s_off, s_last;
    uint32_t *s_len = sm, *s_tok = sm + a.R, *s_need = s_tok + a.R, *s_back = s_need + a.R;   // sums are inclusive
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t t = threadIdx.x, R = a.R;
    const uint32_t head = a.pool[0] % a.pages, count = min(a.pool[1], a.pages);
    if (t == 0) s_taken = 0, s_off = 0, s_last = 0;
    const uint32_t per = (R + kTabThreads - 1) / kTabThreads, r0 = min(t * per, R), r1 = min(r0 + per, R);
    uint32_t tok = 0, need = 0, back = 0;
    for (uint32_t r = r0; r < r1; ++r) {
        const Req q = request(a.lens[r], a.add[r], a.page_shift, a.ld_table);
        s_len[r] = q.len;
        s_tok[r] = tok += q.n;
        s_need[r] = need += q.need;
        s_back[r] = back += q.back;
    }
    const uint32_t tok1 = tok, need1 = need, back1 = back;
    block_scan3(tok, need, back, part);
    uint32_t taken = 0;
    // the thread's own sums become the block's: add what the threads before it had
    const uint32_t tok0 = tok - tok1, need0 = need - need1, back0 = back - back1;
    for (uint32_t r = r0; r < r1; ++r) {
        s_tok[r] += tok0;
        s_need[r] += need0;
        s_back[r] += back0;
        if (s_need[r] <= count) taken = s_need[r];     // rises with r: the pages that the ring can give
    }
    if (taken) atomicMax(&s_taken, taken);
    __syncthreads();
    if (t == 0 && gridDim.x > 1) s_last = atom_add_acq_rel_gpu(a.pool_out + 7, 1u) == gridDim.x - 1;

    // ---- the slot map: PER neighbouring tokens per thread, their look-ups in flight together (new table entries also of
    // tokens past t_cap) ------------------------------------------------------------------------------------------------
    const uint32_t page1 = (1u << a.page_shift) - 1, total = s_tok[R - 1], stop = max(total, a.t_cap);
    auto wrap = [&](uint32_t i) { return i < a.pages ? i : i - a.pages; };      // i < 2 pages
    for (uint64_t i0 = (uint64_t)PER * ((uint64_t)blockIdx.x * kTabThreads + t); i0 < stop;
         i0 += (uint64_t)PER * gridDim.x * kTabThreads) {
        int slot[PER], pos[PER];
        int *entry[PER];            // the token's table entry, to be written when its page is new and the token is its first
        const int *from[PER];       // where the page's id is
        bool fresh[PER];
        uint32_t r = upper_bound(s_tok, R, (uint32_t)i0);
#pragma unroll
        for (uint32_t j = 0; j < PER; ++j) {
            const uint32_t i = (uint32_t)i0 + j;
            slot[j] = -1, pos[j] = 0, from[j] = nullptr, entry[j] = nullptr, fresh[j] = false;
            if (i >= total) continue;
            while (r < R - 1 && s_tok[r] <= i) ++r;
            const uint32_t before = r ? s_tok[r - 1] : 0u, nb = r ? s_need[r - 1] : 0u, len = s_len[r];
            const uint32_t have = (len + page1) >> a.page_shift, need_r = s_need[r] - nb, n = s_tok[r] - before;
            const uint32_t p = len + (i - before), b = p >> a.page_shift;
            pos[j] = (int)p;
            const bool fits = (((uint64_t)len + n + page1) >> a.page_shift) <= a.ld_table;
            if (!fits || b >= a.ld_table || (need_r && s_need[r] > count)) continue;   // put off
            entry[j] = a.table + (size_t)r * a.ld_table + b;
            fresh[j] = b >= have;
            from[j] = fresh[j] ? a.ring + wrap(head + min(nb + (b - have), a.pages - 1)) : entry[j];
        }
        int pid[PER];
#pragma unroll
        for (uint32_t j = 0; j < PER; ++j) pid[j] = from[j] ? *from[j] : 0;
#pragma unroll
        for (uint32_t j = 0; j < PER; ++j) {
            const uint32_t in = (uint32_t)pos[j] & page1;
            if (from[j]) slot[j] = (int)(((uint32_t)pid[j] << a.page_shift) + in);
            if (fresh[j] && in == 0) *entry[j] = pid[j];
        }
        if (PER == 4 && a.vec && i0 + PER <= a.t_cap) {
            constexpr uint32_t j1 = PER > 1 ? 1 : 0, j2 = PER > 2 ? 2 : 0;
            *reinterpret_cast<int4 *>(a.slots + i0) = make_int4(slot[0], slot[j1], slot[j2], slot[PER - 1]);
            *reinterpret_cast<int4 *>(a.pos + i0) = make_int4(pos[0], pos[j1], pos[j2], pos[PER - 1]);
        } else {
#pragma unroll
            for (uint32_t j = 0; j < PER; ++j)
                if (i0 + j < a.t_cap) a.slots[i0 + j] = slot[j], a.pos[i0 + j] = pos[j];
        }
    }
    // ---- pages given back, four look-ups of a thread in flight --------------------------------------------------------
    const uint32_t gone = s_back[R - 1], step = gridDim.x * kTabThreads;
    for (uint64_t i0 = (uint64_t)blockIdx.x * kTabThreads + t; i0 < gone; i0 += 4ull * step) {
        int id[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const uint64_t i = i0 + (uint64_t)j * step;
            if (i >= gone) continue;
            const uint32_t r = upper_bound(s_back, R, (uint32_t)i), before = r ? s_back[r - 1] : 0u;
            id[j] = a.table[(size_t)r * a.ld_table + ((uint32_t)i - before)];
        }
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const uint64_t i = i0 + (uint64_t)j * step;
            if (i < gone) a.ring[((uint64_t)head + count + i) % a.pages] = id[j];
        }
    }
    // ---- the new state: by the CTA that was the last to read the old one ---------------------------------------------
    __syncthreads();
    if (blockIdx.x == 0)
        for (uint32_t r = t; r < R; r += kTabThreads) {
            if (r == 0) a.q_start[0] = 0;
            a.q_start[r + 1] = (int)s_tok[r];
        }
    if (gridDim.x > 1 && !s_last) return;
    uint32_t put_off = 0;
    for (uint32_t r = t; r < R; r += kTabThreads) {
        const uint32_t n = s_tok[r] - (r ? s_tok[r - 1] : 0u), nb = r ? s_need[r - 1] : 0u;
        const bool ended = a.add[r] < 0;
        const bool fits = (((uint64_t)s_len[r] + n + page1) >> a.page_shift) <= a.ld_table;
        const bool served = fits && !(s_need[r] > nb && s_need[r] > count);
        a.lens_out[r] = ended ? 0 : (int)(served ? s_len[r] + n : s_len[r]);
        put_off += !ended && !served && n;
    }
    if (put_off) atomicAdd(&s_off, put_off);
    __syncthreads();
    if (t == 0) {
        a.pool_out[0] = (head + s_taken) % a.pages;
        a.pool_out[1] = count - s_taken + gone;
        a.pool_out[2] = s_off;
        if (gridDim.x > 1) a.pool_out[7] = 0;
    }
}

// ================================================================================================================
// Append. The scale of a page and head covers all of its tokens, so the new tokens of a page are handled by one
// CTA per head and per K / V: the CTA of the page's first new token (its "leader"). A CTA owns `chunk` rows of the slot
// map and takes the pages whose leader is among them, reading on past its rows to the end of the last such page. Phases:
// runs of one page from the slots, max |x| per run (rows read once from HBM), the new scale, codes (rows still in
// registers, or again from L2 when there are more than a batch), older codes of pages whose scale grew. DH / 8 lanes hold a
// row, 16 bytes each.
// Bound by latency for single tokens. Prompts (6 bytes per element; 4 x 2048 tokens of 8 heads of 128, e4m3, 12.4 us where the
// bytes take 4.2) issue 57 % of the time: each of the 2 heads CTAs of a chunk finds its window, runs and minima anew, behind six
// barriers.
// ================================================================================================================
constexpr uint32_t kAppThreads = 256, kAppWin = 256 + 1;

struct AppendArgs {
    uint8_t *codes[2];
    float *scale[2];
    const __half *x[2];
    uint32_t ld[2];
    const int *slots;
    uint64_t page_stride;
    uint32_t T, pages, page_shift, heads, chunk;
    int *err;
};

// the next fp32 value with 8 significant bits, for x >= 0
__device__ __forceinline__ float up8(float x) { return __uint_as_float((__float_as_uint(x) + 0xFFFFu) & ~0xFFFFu); }

// x / s from r = 1 / s (correctly rounded) and one correction by the exact remainder, Markstein's method: a quotient that is
// representable (a border between two codes, which has at most 9 bits) comes out as it is, and the scale's 8 bits keep all others
// further from a border than this is off. No operand here is near over- or underflow.
__device__ __forceinline__ float divide(float x, float s, float r) {
    const float q = x * r;
    return fmaf(fmaf(-q, s, x), r, q);
}
// the codes of four quotients, |y| <= qmax
template <bool FP8>
__device__ __forceinline__ uint32_t encode4(float y0, float y1, float y2, float y3) {
    if (FP8) {
        uint16_t lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(y1), "f"(y0));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(y3), "f"(y2));
        return (uint32_t)lo | (uint32_t)hi << 16;
    }
    // adding 1.5 2^23 rounds to a whole number, to nearest even, and leaves its two's complement in the low byte
    const uint32_t a = __float_as_uint(y0 + 12582912.f), b = __float_as_uint(y1 + 12582912.f);
    const uint32_t c = __float_as_uint(y2 + 12582912.f), d = __float_as_uint(y3 + 12582912.f);
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
template <bool FP8>
__device__ __forceinline__ float decode(uint32_t c) {
    if (FP8) {
        uint32_t h2;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)c));
        return __half2float(__ushort_as_half((uint16_t)h2));
    }
    return (float)(int8_t)c;
}

// 8 fp16 values of a row
template <bool VEC>
__device__ __forceinline__ void raw8(uint32_t (&w)[4], const __half *p) {
    if (VEC) {
        const uint4 v = __ldcg(reinterpret_cast<const uint4 *>(p));
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            w[j] = (uint32_t)__half_as_ushort(p[2 * j]) | (uint32_t)__half_as_ushort(p[2 * j + 1]) << 16;
    }
}
// NaN becomes 0 and infinities the largest fp16; returns the largest magnitude
__device__ __forceinline__ float clean8(uint32_t (&w)[4]) {
    auto largest = [&]() {
        __half2 m = __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t abs2 = w[j] & 0x7FFF7FFFu;
            m = __hmax2_nan(m, *reinterpret_cast<const __half2 *>(&abs2));
        }
        return __half2float(__hmax_nan(__low2half(m), __high2half(m)));
    };
    float m = largest();
    if (!(m <= 65504.f)) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t h = w[j] >> (16 * e) & 0xFFFFu;
                if ((h & 0x7C00u) != 0x7C00u) continue;
                const uint32_t to = h & 0x3FFu ? 0u : (h & 0x8000u) | 0x7BFFu;
                w[j] = (w[j] & ~(0xFFFFu << (16 * e))) | to << (16 * e);
            }
        m = largest();
    }
    return m;
}

template <int DH, bool FP8, bool VEC>
__global__ void __launch_bounds__(kAppThreads) k_kv8_append(AppendArgs a) {
    constexpr uint32_t LPR = DH / 8, kRows = kAppThreads / LPR;   // lanes per row, rows per pass
    constexpr float kQmax = FP8 ? 448.f : 127.f;
    __shared__ int s_slot[kAppWin];
    __shared__ int s_run[kAppWin];             // window index of the row's leader, -1: no row of this CTA
    __shared__ uint32_t s_amax[kAppWin], s_min[kAppWin];
    __shared__ float s_old[kAppWin], s_new[kAppWin];
    __shared__ int s_lead[kAppThreads / 32];
    __shared__ uint32_t s_end, s_grown_n;
    __shared__ uint8_t s_grown[kAppThreads];       // leaders whose page's scale grew over older rows, as window index - 1
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const uint32_t h = blockIdx.y >> 1, kv = blockIdx.y & 1, first = blockIdx.x * a.chunk;
    const uint32_t page = 1u << a.page_shift, win = min(a.chunk + page, a.T - first);   // <= 256
    const int last_slot = (int)(a.pages << a.page_shift);
    // window index 0 is the row before the chunk
    for (uint32_t j = t; j <= win; j += kAppThreads) s_slot[j] = first + j == 0 ? -1 : a.slots[first + j - 1];
    if (t == 0) s_end = 0, s_grown_n = 0;
    __syncthreads();

    // a leader is a valid row whose predecessor is not of the same page
    const uint32_t j = t + 1;
    bool good = false, goes_on = false;
    int slot = -1;
    if (j <= win) {
        slot = s_slot[j];
        const int prev = s_slot[j - 1];
        const bool in = slot >= 0 && slot < last_slot;
        const bool same = in && prev >= 0 && prev < last_slot && (prev >> a.page_shift) == (slot >> a.page_shift);
        good = in && !(same && slot <= prev);
        // bad slots are reported by the CTA that owns the row
        if (slot >= 0 && !good && t < a.chunk && blockIdx.y == 0) atomicCAS(a.err, 0, (int)sh::kErrBadArgs);
        goes_on = same;
        s_amax[j] = 0;
        s_min[j] = 0xFFFFFFFFu;
    }
    const uint32_t b1 = __ballot_sync(0xffffffffu, !goes_on);   // rows that begin a page, and rows of none
    if (lane == 31) s_lead[warp] = b1 ? (int)(warp * 32 + 32 - __clz(b1)) : 0;   // window index, 0: none in this warp
    __syncthreads();
    int lead = 0;
    {
        const uint32_t upto = b1 & (0xffffffffu >> (31 - lane));
        if (upto) lead = (int)(warp * 32 + 32 - __clz(upto));
        for (int w = (int)warp - 1; lead == 0 && w >= 0; --w) lead = s_lead[w];
    }
    // lead: where the row's page began in this window (0: before it). Ours if that is a leader among the chunk's rows.
    bool ours = j <= win && good && lead >= 1 && lead <= (int)a.chunk && (uint32_t)(j - lead) < page;
    if (ours) {
        const int s = s_slot[lead];
        ours = s >= 0 && s < last_slot;
    }
    __syncthreads();
    if (j <= win) s_run[j] = ours ? lead : -1;
    if (ours) {
        atomicMin(&s_min[lead], (uint32_t)slot & (page - 1));
        atomicMax(&s_end, j + 1);
    }
    __syncthreads();
    const uint32_t end = s_end;
    if (end == 0) return;

    const __half *x = (kv ? a.x[1] : a.x[0]) + (size_t)h * DH;
    const uint32_t ld = kv ? a.ld[1] : a.ld[0], l = t % LPR, rw = t / LPR;
    // rows of this thread, kBatch at a time so that their loads are in flight together; one batch is held in registers
    constexpr uint32_t kBatch = 8;
    uint32_t w[kBatch][4];
    auto load_batch = [&](uint32_t r0, float (&m)[kBatch]) {
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b) {
            const uint32_t i = r0 + b * kRows + rw;
            m[b] = 0.f;
            if (i < end && s_run[i] >= 0) raw8<VEC>(w[b], x + (size_t)(first + i - 1) * ld + l * 8);
        }
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b) {
            const uint32_t i = r0 + b * kRows + rw;
            if (i < end && s_run[i] >= 0) m[b] = clean8(w[b]);
        }
    };
    float m[kBatch];
    for (uint32_t r0 = 1; r0 < end; r0 += kBatch * kRows) {    // every lane walks the loop: the reductions are warp-wide
        load_batch(r0, m);
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b) {
            if (r0 + b * kRows >= end) break;
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) m[b] = fmaxf(m[b], __shfl_xor_sync(0xffffffffu, m[b], o));
            const uint32_t i = r0 + b * kRows + rw;
            if (l == 0 && i < end && s_run[i] >= 0) atomicMax(&s_amax[s_run[i]], __float_as_uint(m[b]));
        }
    }
    __syncthreads();
    float *scale = kv ? a.scale[1] : a.scale[0];
    if (j <= win && ours && lead == (int)j) {
        float *sp = scale + (size_t)(slot >> a.page_shift) * a.heads + h;
        const float old = s_min[j] ? *sp : 0.f;
        const float now = fmaxf(old, up8(__fdiv_rn(__uint_as_float(s_amax[j]), kQmax)));
        s_old[j] = old;
        s_new[j] = now;
        *sp = now;
        if (s_min[j] && now > old) s_grown[atomicAdd(&s_grown_n, 1u)] = (uint8_t)t;
    }
    __syncthreads();
    uint8_t *codes = kv ? a.codes[1] : a.codes[0];
    const size_t head_off = (size_t)h << a.page_shift;
    for (uint32_t r0 = 1; r0 < end; r0 += kBatch * kRows) {
        if (end > 1 + kBatch * kRows) load_batch(r0, m);
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b) {
            const uint32_t i = r0 + b * kRows + rw;
            const int run = i < end ? s_run[i] : -1;
            if (run < 0) continue;
            const float s = s_new[run], r1 = s > 0.f ? __frcp_rn(s) : 0.f;      // scale 0: all values are
            uint32_t c[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float2 a0 = __half22float2(*reinterpret_cast<const __half2 *>(&w[b][2 * e]));
                const float2 a1 = __half22float2(*reinterpret_cast<const __half2 *>(&w[b][2 * e + 1]));
                c[e] = encode4<FP8>(divide(a0.x, s, r1), divide(a0.y, s, r1), divide(a1.x, s, r1), divide(a1.y, s, r1));
            }
            const uint32_t sl = (uint32_t)s_slot[i];
            uint8_t *dst = codes + (size_t)(sl >> a.page_shift) * a.page_stride + (head_off + (sl & (page - 1))) * DH + l * 8;
            *reinterpret_cast<uint2 *>(dst) = make_uint2(c[0], c[1]);
        }
    }
    // older rows of pages whose scale grew: code s / s', rounded once more
    for (uint32_t k = 0; k < s_grown_n; ++k) {
        const uint32_t q = s_grown[k] + 1u;
        const float so = s_old[q], sn = s_new[q], r1 = __frcp_rn(sn);
        uint8_t *base = codes + (size_t)((uint32_t)s_slot[q] >> a.page_shift) * a.page_stride + head_off * DH;
        for (uint32_t row = rw; row < s_min[q]; row += kRows) {
            uint2 *p = reinterpret_cast<uint2 *>(base + (size_t)row * DH + l * 8);
            const uint2 c = *p;
            const uint32_t cw[2] = {c.x, c.y};
            uint32_t w[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float y[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = divide(decode<FP8>(cw[e] >> (8 * j) & 0xFFu) * so, sn, r1);
                w[e] = encode4<FP8>(y[0], y[1], y[2], y[3]);
            }
            *p = make_uint2(w[0], w[1]);
        }
    }
}

template <int DH, bool FP8>
cudaError_t append_launch(const AppendArgs &a, bool vec, dim3 grid, cudaStream_t st) {
    return sh::launch_pdl(vec ? k_kv8_append<DH, FP8, true> : k_kv8_append<DH, FP8, false>, grid, dim3(kAppThreads), 0, st, a);
}

}  // namespace

extern "C" {

int sh_cuda_kv_tables(uint64_t lens, uint64_t add, uint32_t R, uint32_t page, uint64_t table, uint32_t ld_table,
                      uint64_t ring, uint32_t pages, uint64_t pool, uint64_t pool_out, uint64_t lens_out,
                      uint64_t q_start, uint64_t slots, uint64_t pos, uint32_t t_cap) {
    if (!sh::kv8_page_ok(page) || pages == 0 || (uint64_t)pages * page >= (1ull << 31) || R > kTabMaxR) {
        sh::set_error(-1, "[sh_cuda_kv_tables] need page 16, 32, 64 or 128, 0 < pages * page < 2^31, R <= %u (page=%u "
                      "pages=%u R=%u)", kTabMaxR, page, pages, R);
        return -1;
    }
    if (R && (!lens || !add || !table || !ring || !pool || !pool_out || !lens_out || !q_start || ld_table == 0 ||
              ld_table >= (1u << 31) / page || (t_cap && (!slots || !pos)) || t_cap >= (1u << 31) ||
              !sh::words_ok(lens, add, table, ring) || !sh::words_ok(pool, pool_out, lens_out, q_start) ||
              !sh::words_ok(slots, pos))) {
        sh::set_error(-1, "[sh_cuda_kv_tables] a null or misaligned array, or ld_table * page or t_cap past 2^31 (ld_table=%u "
                      "t_cap=%u)", ld_table, t_cap);
        return -1;
    }
    if (R == 0) return 0;
    const sh::DeviceState &s = sh::state();
    TablesArgs a = {(const int *)lens, (const int *)add, (int *)table, (int *)ring, (const uint32_t *)pool,
                    (uint32_t *)pool_out, (int *)lens_out, (int *)q_start, (int *)slots, (int *)pos, R,
                    sh::kv8_shift(page), ld_table, pages, t_cap, sh::aligned16(slots) && sh::aligned16(pos)};
    // one token per thread while that fills no GPU, four (16-byte stores) beyond
    const uint32_t cap = s.num_sms > 0 ? s.num_sms : 1, per = t_cap > cap * kTabThreads ? 4 : 1;
    const uint64_t want = ((uint64_t)t_cap + per * kTabThreads - 1) / (per * kTabThreads);
    const uint32_t grid = want < 1 ? 1 : want < cap ? (uint32_t)want : cap;
    const size_t smem = (size_t)R * 16;
    auto kernel = per == 4 ? k_kv_tables<4> : k_kv_tables<1>;
    if (!sh::cuda_ok(per == 4 ? sh::allow_smem<k_kv_tables<4>>(kTabMaxR * 16) : sh::allow_smem<k_kv_tables<1>>(kTabMaxR * 16),
                     "sh_cuda_kv_tables"))
        return -1;
    return sh::cuda_ok(sh::launch_pdl(kernel, dim3(grid), dim3(kTabThreads), smem, s.stream, a), "sh_cuda_kv_tables") ? 0 : -1;
}

int sh_cuda_kv8_append(const sh_cuda_kv8_t *c, uint64_t k, uint64_t v, uint32_t T, uint32_t ldk, uint32_t ldv,
                       uint64_t slots) {
    const int bad = sh::kv8_check(c, "sh_cuda_kv8_append");
    if (bad) return bad;
    const uint64_t w = (uint64_t)c->heads * c->dh;
    if (T && (!k || !v || !slots || ((k | v) & 1) || !sh::words_ok(slots) || ldk < w || ldv < w || T >= (1u << 31))) {
        sh::set_error(-1, "[sh_cuda_kv8_append] null or odd k / v, null or misaligned slots, or ldk, ldv < heads * dh (ldk=%u "
                      "ldv=%u)", ldk, ldv);
        return -1;
    }
    if (T == 0) return 0;
    sh::DeviceState &s = sh::state();
    AppendArgs a = {{(uint8_t *)c->k, (uint8_t *)c->v}, {(float *)c->k_scale, (float *)c->v_scale},
                    {(const __half *)k, (const __half *)v}, {ldk, ldv}, (const int *)slots, c->page_stride, T, c->pages,
                    sh::kv8_shift(c->page), c->heads, 0, s.dev_err};
    // A prompt's pages hold up to `page` new rows each: 64 rows per CTA and at least a page (4096 tokens, 8 heads of 64,
    // pages of 16: 9 us, 21 us with 16 rows). Few rows are mostly one per page: eight rows per CTA spread them over the GPU, 16 in
    // between (1024 rows 4.9 us, 6.2 us with eight).
    const uint32_t many = c->page > 64 ? c->page : 64;
    const uint64_t ctas = (uint64_t)((T + many - 1) / many) * c->heads * 2;
    a.chunk = ctas >= 2ull * s.num_sms ? many : ctas * 4 >= 2ull * s.num_sms ? 16u : 8u;
    const uint32_t gx = (T + a.chunk - 1) / a.chunk;
    if (c->heads * 2ull > 65535) {
        sh::set_error(-1, "[sh_cuda_kv8_append] heads %u > 32767", c->heads);
        return -1;
    }
    const bool vec = sh::aligned16(k) && sh::aligned16(v) && ldk % 8 == 0 && ldv % 8 == 0;
    const dim3 grid(gx, c->heads * 2);
    const bool fp8 = c->fmt == SH_FP8;
    auto launch = c->dh == 64 ? (fp8 ? append_launch<64, true> : append_launch<64, false>)
                              : (fp8 ? append_launch<128, true> : append_launch<128, false>);
    return sh::cuda_ok(launch(a, vec, grid, s.stream), "sh_cuda_kv8_append") ? 0 : -1;
}

}  // extern "C"
