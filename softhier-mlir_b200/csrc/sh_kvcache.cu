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

    // ---- the slot map: four neighbouring tokens per thread (new table entries also of tokens past t_cap) ---------------
    const uint32_t page1 = (1u << a.page_shift) - 1, total = s_tok[R - 1], stop = max(total, a.t_cap);
    for (uint64_t i0 = 4ull * ((uint64_t)blockIdx.x * kTabThreads + t); i0 < stop; i0 += 4ull * gridDim.x * kTabThreads) {
        int slot[4], pos[4];
        uint32_t r = upper_bound(s_tok, R, (uint32_t)i0);
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const uint32_t i = (uint32_t)i0 + j;
            slot[j] = -1, pos[j] = 0;
            if (i >= total) continue;
            while (r < R - 1 && s_tok[r] <= i) ++r;
            const uint32_t before = r ? s_tok[r - 1] : 0u, nb = r ? s_need[r - 1] : 0u, len = s_len[r];
            const uint32_t have = (len + page1) >> a.page_shift, need_r = s_need[r] - nb, n = s_tok[r] - before;
            const uint32_t p = len + (i - before), b = p >> a.page_shift;
            pos[j] = (int)p;
            const bool fits = (((uint64_t)len + n + page1) >> a.page_shift) <= a.ld_table;
            if (!fits || b >= a.ld_table || (need_r && s_need[r] > count)) continue;   // put off
            uint32_t pid;
            if (b < have)
                pid = (uint32_t)a.table[(size_t)r * a.ld_table + b];
            else {
                pid = (uint32_t)a.ring[(head + nb + (b - have)) % a.pages];
                if ((p & page1) == 0) a.table[(size_t)r * a.ld_table + b] = (int)pid;
            }
            slot[j] = (int)((pid << a.page_shift) + (p & page1));
        }
        if (a.vec && i0 + 4 <= a.t_cap) {
            *reinterpret_cast<int4 *>(a.slots + i0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
            *reinterpret_cast<int4 *>(a.pos + i0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
        } else {
            for (uint32_t j = 0; j < 4 && i0 + j < a.t_cap; ++j) a.slots[i0 + j] = slot[j], a.pos[i0 + j] = pos[j];
        }
    }
    // ---- pages given back ------------------------------------------------------------------------------------------
    const uint32_t gone = s_back[R - 1];
    for (uint64_t i = (uint64_t)blockIdx.x * kTabThreads + t; i < gone; i += (uint64_t)gridDim.x * kTabThreads) {
        const uint32_t r = upper_bound(s_back, R, (uint32_t)i), before = r ? s_back[r - 1] : 0u;
        a.ring[((uint64_t)head + count + i) % a.pages] = a.table[(size_t)r * a.ld_table + ((uint32_t)i - before)];
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
// runs of one page from the slots, max |x| per run (rows read once from HBM), the new scale, codes (rows read again from
// L1 / L2), older codes of pages whose scale grew. DH / 8 lanes hold a row, 16 bytes each.
// Bound by HBM for prompts (6 bytes per element) and by latency for single tokens.
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

__device__ __forceinline__ float clean(__half h) {   // NaN -> 0, infinities -> the largest fp16
    const float x = __half2float(h);
    return isnan(x) ? 0.f : fminf(fmaxf(x, -65504.f), 65504.f);
}
// the next fp32 value with 8 significant bits, for x >= 0
__device__ __forceinline__ float up8(float x) { return __uint_as_float((__float_as_uint(x) + 0xFFFFu) & ~0xFFFFu); }

template <bool FP8>
__device__ __forceinline__ uint32_t encode(float y) {   // |y| <= qmax up to rounding
    if (FP8) {
        uint16_t r;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(y));
        return r & 0xFFu;
    }
    return (uint32_t)min(max(__float2int_rn(y), -127), 127) & 0xFFu;
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

template <int DH, bool VEC>
__device__ __forceinline__ void load_row8(float (&f)[8], const __half *row, uint32_t l) {
    __half h[8];
    if (VEC) {
        *reinterpret_cast<uint4 *>(h) = *reinterpret_cast<const uint4 *>(row + l * 8);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = row[l * 8 + j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = clean(h[j]);
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
    __shared__ uint32_t s_end;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const uint32_t h = blockIdx.y >> 1, kv = blockIdx.y & 1, first = blockIdx.x * a.chunk;
    const uint32_t page = 1u << a.page_shift, win = min(a.chunk + page, a.T - first);   // <= 256
    const int last_slot = (int)(a.pages << a.page_shift);
    // window index 0 is the row before the chunk
    for (uint32_t j = t; j <= win; j += kAppThreads) s_slot[j] = first + j == 0 ? -1 : a.slots[first + j - 1];
    if (t == 0) s_end = 0;
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
    for (uint32_t r = 1; r < end; r += kRows) {    // every lane walks the loop: the reductions are warp-wide
        const uint32_t i = r + rw;
        const int run = i < end ? s_run[i] : -1;
        float m = 0.f;
        if (run >= 0) {
            float f[8];
            load_row8<DH, VEC>(f, x + (size_t)(first + i - 1) * ld, l);
#pragma unroll
            for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(f[e]));
        }
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (run >= 0 && l == 0) atomicMax(&s_amax[run], __float_as_uint(m));
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
    }
    __syncthreads();
    uint8_t *codes = kv ? a.codes[1] : a.codes[0];
    const size_t head_off = (size_t)h << a.page_shift;
    for (uint32_t r = 1; r < end; r += kRows) {
        const uint32_t i = r + rw;
        const int run = i < end ? s_run[i] : -1;
        if (run < 0) continue;
        const float s = s_new[run];
        float f[8];
        load_row8<DH, VEC>(f, x + (size_t)(first + i - 1) * ld, l);
        uint32_t w[2] = {0, 0};
        if (s > 0.f) {
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e >> 2] |= encode<FP8>(__fdiv_rn(f[e], s)) << (8 * (e & 3));
        }
        const uint32_t sl = (uint32_t)s_slot[i];
        uint8_t *dst = codes + (size_t)(sl >> a.page_shift) * a.page_stride + (head_off + (sl & (page - 1))) * DH + l * 8;
        *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
    }
    // older rows of pages whose scale grew: code s / s', rounded once more
    for (uint32_t q = 1; q <= min(win, a.chunk); ++q) {
        if (s_run[q] != (int)q || !(s_new[q] > s_old[q])) continue;
        const float so = s_old[q], sn = s_new[q];
        uint8_t *base = codes + (size_t)((uint32_t)s_slot[q] >> a.page_shift) * a.page_stride + head_off * DH;
        for (uint32_t row = rw; row < s_min[q]; row += kRows) {
            uint2 *p = reinterpret_cast<uint2 *>(base + (size_t)row * DH + l * 8);
            const uint2 c = *p;
            const uint32_t cw[2] = {c.x, c.y};
            uint32_t w[2] = {0, 0};
#pragma unroll
            for (int e = 0; e < 8; ++e)
                w[e >> 2] |= encode<FP8>(__fdiv_rn(decode<FP8>((cw[e >> 2] >> (8 * (e & 3))) & 0xFFu) * so, sn))
                             << (8 * (e & 3));
            *p = make_uint2(w[0], w[1]);
        }
    }
}

template <int DH, bool FP8>
void append_launch(const AppendArgs &a, bool vec, dim3 grid, cudaStream_t st) {
    if (vec) sh::launch_pdl(k_kv8_append<DH, FP8, true>, grid, dim3(kAppThreads), 0, st, a);
    else sh::launch_pdl(k_kv8_append<DH, FP8, false>, grid, dim3(kAppThreads), 0, st, a);
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
              ld_table >= (1u << 31) / page || (t_cap && (!slots || !pos)) || t_cap >= (1u << 31))) {
        sh::set_error(-1, "[sh_cuda_kv_tables] a null array, or ld_table * page or t_cap past 2^31 (ld_table=%u t_cap=%u)",
                      ld_table, t_cap);
        return -1;
    }
    if (R == 0) return 0;
    const sh::DeviceState &s = sh::state();
    TablesArgs a = {(const int *)lens, (const int *)add, (int *)table, (int *)ring, (const uint32_t *)pool,
                    (uint32_t *)pool_out, (int *)lens_out, (int *)q_start, (int *)slots, (int *)pos, R,
                    sh::kv8_shift(page), ld_table, pages, t_cap, sh::aligned16(slots) && sh::aligned16(pos)};
    const uint32_t want = (t_cap + 4 * kTabThreads - 1) / (4 * kTabThreads), cap = s.num_sms > 0 ? s.num_sms : 1;
    const uint32_t grid = want < 1 ? 1 : want < cap ? want : cap;
    const size_t smem = (size_t)R * 16;
    if (smem > 48 * 1024 &&
        !sh::cuda_ok(cudaFuncSetAttribute(k_kv_tables, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kTabMaxR * 16)),
                     "sh_cuda_kv_tables"))
        return -1;
    return sh::cuda_ok(sh::launch_pdl(k_kv_tables, dim3(grid), dim3(kTabThreads), smem, s.stream, a),
                       "sh_cuda_kv_tables") ? 0 : -1;
}

int sh_cuda_kv8_append(const sh_cuda_kv8_t *c, uint64_t k, uint64_t v, uint32_t T, uint32_t ldk, uint32_t ldv,
                       uint64_t slots) {
    const int bad = sh::kv8_check(c, "sh_cuda_kv8_append");
    if (bad) return bad;
    const uint64_t w = (uint64_t)c->heads * c->dh;
    if (T && (!k || !v || !slots || (k & 1) || (v & 1) || ldk < w || ldv < w || T >= (1u << 31))) {
        sh::set_error(-1, "[sh_cuda_kv8_append] null or odd k / v, null slots, or ldk, ldv < heads * dh (ldk=%u ldv=%u)",
                      ldk, ldv);
        return -1;
    }
    if (T == 0) return 0;
    sh::DeviceState &s = sh::state();
    AppendArgs a = {{(uint8_t *)c->k, (uint8_t *)c->v}, {(float *)c->k_scale, (float *)c->v_scale},
                    {(const __half *)k, (const __half *)v}, {ldk, ldv}, (const int *)slots, c->page_stride, T, c->pages,
                    sh::kv8_shift(c->page), c->heads, 0, s.dev_err};
    // A prompt's pages hold up to `page` new rows each: one page per CTA. Few rows are mostly one per page: eight rows
    // per CTA spread them over the GPU.
    const uint64_t ctas = (uint64_t)((T + c->page - 1) / c->page) * c->heads * 2;
    a.chunk = ctas >= 2ull * s.num_sms ? c->page : 8u;
    const uint32_t gx = (T + a.chunk - 1) / a.chunk;
    if (c->heads * 2ull > 65535) {
        sh::set_error(-1, "[sh_cuda_kv8_append] heads %u > 32767", c->heads);
        return -1;
    }
    const bool vec = sh::aligned16(k) && sh::aligned16(v) && ldk % 8 == 0 && ldv % 8 == 0;
    const dim3 grid(gx, c->heads * 2);
    const bool fp8 = c->fmt == SH_FP8;
    if (c->dh == 64) fp8 ? append_launch<64, true>(a, vec, grid, s.stream) : append_launch<64, false>(a, vec, grid, s.stream);
    else fp8 ? append_launch<128, true>(a, vec, grid, s.stream) : append_launch<128, false>(a, vec, grid, s.stream);
    return sh::cuda_ok(cudaGetLastError(), "sh_cuda_kv8_append") ? 0 : -1;
}

}  // extern "C"
