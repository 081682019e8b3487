// Attention over the paged 8-bit K / V cache (sh_cuda_attention_kv8): new rows of a batch of requests against all of
// their cached tokens, grouped-query heads, causal among the new rows.
//
// With x_j = scale log2(e) ks_j (q . kcode_j) and w_j = 2^(x_j + log2 vs_j - m), m the running maximum of the exponent,
//     o = (sum_j w_j vcode_j) / (sum_j w_j / vs_j)
// so the value scales ride in the exponent: w_j stays in fp16's range whatever the scales are, and the codes themselves
// (int8 and e4m3 are exact in fp16) are the operands of the second product. The first product is exact up to its
// fp32 sums. The sum of the weights is taken in fp32; for the second product they are fp16 operands, in the kernel for few
// rows with the rest of that rounding as a second operand (the outputs' own rounding is then all there is; it costs 5 of the
// 115 us of a large batch), in the one for many rows without it: each weight is off by up to 2^-11 of itself, as the output is by
// its own rounding. Error against 64 bits 2.9e-4, 2.1e-4 with the rests, which there cost half as many products again (4 x 512 rows
// over up to 8192 tokens 218 us, 182 without). A caller who wants the rests passes a max_q of 1.
#include <math.h>

#include "sh_kv8.cuh"

namespace {

struct KvArgs {
    const __half *q;
    __half *o;
    const uint8_t *k, *v;
    const float *ks, *vs;
    const int *table, *lens, *q_start;
    uint64_t page_stride;
    uint32_t ld_table, R, T, G, heads, pages, page_shift, ldq, ldo;
    float sl2;            // scale * log2(e)
    uint32_t vec;         // q rows take 16-byte loads, o rows 4-byte stores
    uint32_t vec_o;       // o rows take 16-byte stores
    uint32_t box_step, k_at, v_at;      // few rows: bytes from 16 tokens to the next in a stage, K's and V's place there
    uint32_t boxes, box_bytes;          // few rows: copies per step, and their bytes
    uint32_t apart;       // few rows: V comes by a copy of its own, to this place behind K's (0: with K's)
    uint32_t flip;        // sign bits to turn in q: the scale is negative (sl2 is its magnitude then; tiles only)
    uint32_t *counters;   // arrivals per CTA whose last item goes on in others, zero between calls
    float *part;
    int *err;
};

// A request as the kernels see it: lengths that no index leaves the arrays with, whatever the device arrays hold.
struct ReqView {
    uint32_t qs, nq, ctx;
    int base;             // tokens before its first new row (< 0: the first rows have none), at most ctx
};
__device__ __forceinline__ ReqView req_view(const KvArgs &a, uint32_t r) {
    ReqView v;
    const int s = a.q_start[r], e = a.q_start[r + 1], len = max(a.lens[r], 0);
    const int s0 = min(max(s, 0), (int)a.T), e0 = min(max(e, s0), (int)a.T);
    v.qs = (uint32_t)s0;
    v.nq = (uint32_t)(e0 - s0);
    v.ctx = min((uint32_t)len, a.ld_table << a.page_shift);
    // of the length as it is: a row's limit counts tokens past the table, which are then left out. Below -nq and above ctx
    // nothing changes.
    const long long base = (long long)len - max((long long)e - s, 0ll) + (s0 - (long long)s);
    v.base = (int)min(max(base, -(long long)v.nq), (long long)v.ctx);
    return v;
}

// The sum of weights of a row, from token `first` on, that came out as 0: 0 when the row has no keys there (none at all gives
// zeros). Scores that are all -infinity, from an infinity in Q beside keys of one sign, give NaN as beside keys of both signs;
// they are rare, so that Q is looked at here only.
__device__ __forceinline__ float no_weight(const KvArgs &a, const ReqView &v, uint32_t kvh, uint32_t row, uint32_t dh,
                                           uint32_t first) {
    const uint32_t qi = row / a.G, gi = row - qi * a.G;
    if (min(v.base + (int)qi + 1, (int)v.ctx) <= (int)first) return 0.f;
    const __half *q = a.q + (size_t)(v.qs + qi) * a.ldq + ((size_t)kvh * a.G + gi) * dh;
#pragma unroll 1
    for (uint32_t d = 0; d < dh; ++d)
        if ((__half_as_ushort(q[d]) & 0x7FFFu) == 0x7C00u) return NAN;
    return 0.f;
}

__device__ __forceinline__ uint4 lds16(uint32_t at) {
    uint4 r;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at) : "memory");
    return r;
}
__device__ __forceinline__ uint2 lds8(uint32_t at) {
    uint2 r;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(at) : "memory");
    return r;
}
// 4 bytes to shared memory, counted on `bar` with this thread's other copies by cp_async_arrive
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// a box of a K and V map (below)
__device__ __forceinline__ void tma_load_pair(void *dst, const CUtensorMap *map, uint64_t *bar, int row, int page) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %3}], [%2];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(0), "r"(row), "r"(page)
                 : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint64_t *bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// D (16 x 8, fp32) += A (16 x 16, fp16) B (16 x 8, fp16), one warp
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8 x 8 fp16 transpose across the warp (lane 4 r + c holds row r, columns 2 c, 2 c + 1)
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t e4m3x2_to_h2(uint32_t two) {   // low 16 bits: two codes
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
    return r;
}
// (a & b) ^ c in one instruction (written in C, the two constants make it two)
__device__ __forceinline__ uint32_t and_xor(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
// int8: code + 128 in the low byte of the fp16 pattern 0x6400 is 1152 + code, exactly; 1152 comes off again
constexpr uint32_t kMagic = 0x64806480u, kMagicVal = 0x64806480u;   // fp16 1152 = 0x6480 as well

// the four codes of a word as two fp16 pairs: int8 (0, 2), (1, 3); e4m3 (0, 1), (2, 3)
template <bool FP8>
__device__ __forceinline__ void word_to_h2(uint32_t w, uint32_t &p, uint32_t &q) {
    if (FP8) {
        p = e4m3x2_to_h2(w & 0xFFFFu);
        q = e4m3x2_to_h2(w >> 16);
    } else {
        p = hsub2(and_xor(w, 0x00FF00FFu, kMagic), kMagicVal);
        q = hsub2(and_xor(w >> 8, 0x00FF00FFu, kMagic), kMagicVal);
    }
}
// byte B of two words as an fp16 pair (lo from a, hi from b)
template <bool FP8, int B>
__device__ __forceinline__ uint32_t byte_pair(uint32_t a, uint32_t b) {
    if (FP8) return e4m3x2_to_h2(__byte_perm(a, b, B | (4 + B) << 4));
    return hsub2(and_xor(__byte_perm(a, b, B | B << 4 | (4 + B) << 8 | (4 + B) << 12), 0x00FF00FFu, kMagic), kMagicVal);
}

// ================================================================================================================
// Few rows per request (single tokens, drafts). The K / V bytes bound it, so each is read once per tile of up to
// 8 NT (query row, query head) pairs of one kv head. Both products keep the 8-bit side as the 16-row operand of the
// matrix instruction and the rows as its 8 columns:
//     S^T (16 tokens x 8 rows) = K (16 x dh) Q^T,     O^T (16 dims x 8 rows) += V^T (16 x 16 tokens) W^T
// so a group of up to 8 query heads fills the instruction. Its index along the contracted side may be permuted freely when
// both operands agree: a lane takes 16 neighbouring columns of its K rows, and 4 tokens of V with dh / 8 neighbouring
// columns. W^T comes from S^T by an 8 x 8 transpose in registers.
//
// A warp takes 16 tokens of a unit at dh = 128, 32 at dh = 64 (as many bytes); its K and V boxes, both with one instruction
// (swizzled so that neither operand's reads meet in a bank more than two at a time), come by TMA into a ring of its own,
// kStages ahead and across items, so a warp waits for nobody but its own copies until an item ends. The scales come in
// registers as far ahead. What bounds it beside the bytes is the integer pipe: turning int8 codes into fp16 operands takes 112
// of its instructions per 16 tokens and warp at dh = 128, 56 of the 157 cycles that their bytes take, and the rest of a step
// as much again. 64 requests of up to 8192 tokens (32 heads over 8 of 128, int8) take 115 us, the copies alone (no products) 98;
// with heads of 64 (15 over 5) 53 and 39. More warps per SM (20 at dh = 64) are slower. Drafts add what an item's end
// costs: up to 16 rows of partial sums per warp and CTA. Their dh = 128 form has 8 warps per SM with all of their registers
// (32 requests of 4 drafts 70 us; with 12 warps, which spill, 75).
//
// Work is split evenly whatever the lengths are: the units (request, kv head, row tile, block of tokens), in this order,
// are dealt to the CTAs in equal contiguous runs, which every CTA works out from the lengths by itself. An item (request,
// head, tile) that spans CTAs leaves partial sums in the workspace, at most two per CTA; the CTA that arrives last joins
// them in the order of the CTAs, so results do not depend on timing.
// ================================================================================================================
constexpr int kStages = 2;

// A unit in the run of a CTA: where it is, and its item's limits. Every thread of a CTA steps the same cursor.
struct Cursor {
    uint32_t r, kvh, tile, tiles, b, blocks;
    ReqView v;
    int lim_hi;      // keys of the tile's last row
};
template <uint32_t RT, uint32_t KEYS>
__device__ __forceinline__ void cursor_item(Cursor &k, const KvArgs &a) {      // after tile changed
    const uint32_t row0 = k.tile * RT, nrows = min(RT, k.v.nq * a.G - row0);
    k.lim_hi = min(max(k.v.base + (int)((row0 + nrows - 1) / a.G) + 1, 0), (int)k.v.ctx);
}
template <uint32_t RT, uint32_t KEYS>
__device__ __forceinline__ void cursor_sizes(Cursor &k, const KvArgs &a) {     // after the request changed
    k.tiles = (k.v.nq * a.G + RT - 1) / RT, k.blocks = max(1u, (k.v.ctx + KEYS - 1) / KEYS);
}
template <uint32_t RT, uint32_t KEYS>
__device__ __forceinline__ void cursor_next(Cursor &k, const KvArgs &a) {
    if (++k.b < k.blocks) return;
    k.b = 0;
    if (++k.tile == k.tiles) {
        k.tile = 0;
        if (++k.kvh == a.heads) {
            k.kvh = 0;
            do {
                if (++k.r >= a.R) return;
                k.v = req_view(a, k.r);
                cursor_sizes<RT, KEYS>(k, a);
            } while (k.tiles == 0);
        }
    }
    cursor_item<RT, KEYS>(k, a);
}

template <int DH, int NT, int NW>
struct RowsSmem {
    static constexpr uint32_t kTokens = 2048 / DH;                    // of a step: 16 or 32
    static constexpr uint32_t kTile = kTokens * DH;                   // K or V of a step
    static constexpr uint32_t kRing = 0, kO = NW * kStages * 2 * kTile, kM = kO + NW * 8 * NT * (DH + 4) * 4;
    static constexpr uint32_t kL = kM + NW * 8 * NT * 4, kBars = kL + NW * 8 * NT * 4, kPart = kBars + NW * kStages * 8;
    static constexpr uint32_t kMisc = kPart + NW * 8, kBytes = kMisc + 64 + 1024;
};

template <int DH, int NT, int NW, bool FP8>
__global__ void __launch_bounds__(NW * 32, (NT == 1 ? 16 : DH == 64 ? 12 : 8) / NW)
    k_attn_kv8_rows(const __grid_constant__ CUtensorMap mkv, const __grid_constant__ CUtensorMap mv, KvArgs a) {
    using SM = RowsSmem<DH, NT, NW>;
    constexpr uint32_t RT = 8 * NT, kThreads = NW * 32;                     // rows of a tile
    constexpr uint32_t kStep = SM::kTokens, kKeys = kStep * NW;             // keys of a warp's step, of a unit
    constexpr int KC = DH / 64;                     // 16-byte pieces of a K row per lane
    constexpr int VB = DH / 8;                      // V columns per lane
    constexpr int VW = VB / 4;                      // as words
    constexpr uint32_t HF = kStep / 16;             // groups of 16 tokens of a step, each in one page
    extern __shared__ uint8_t smem_raw[];
    uint8_t *sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    // [NW][RT] rows of DH / 2 column pairs: pair i of lane row g (columns VB g + 2 i) at i * 8 + g, so that neither the writes
    // nor the reads of a warp meet in a bank
    float2 *s_o = reinterpret_cast<float2 *>(sm + SM::kO);
    constexpr uint32_t kPitch = DH / 2 + 2;
    float *s_m = reinterpret_cast<float *>(sm + SM::kM), *s_l = reinterpret_cast<float *>(sm + SM::kL);   // [NW][RT]
    typedef unsigned long long u64;
    u64 *s_part = reinterpret_cast<u64 *>(sm + SM::kPart);
    struct Start {       // where this CTA's run begins
        u64 off;
        ReqView v;
        uint32_t r;
    };
    Start &s_start = *reinterpret_cast<Start *>(sm + SM::kMisc);
    uint32_t &s_flag = *reinterpret_cast<uint32_t *>(sm + SM::kMisc + 40);
    volatile int *abort = reinterpret_cast<volatile int *>(sm + SM::kMisc + 44);
    const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5, g = lane >> 2, c = lane & 3;
    const uint32_t page1 = (1u << a.page_shift) - 1;
    uint64_t *full = reinterpret_cast<uint64_t *>(sm + SM::kBars) + warp * kStages;
    if (lane == 0)
        for (int i = 0; i < kStages; ++i) mbar_init(full + i, 1);
    if (t == 0) *abort = 0, prefetch_tmap(&mkv);
    fence_mbar_init();
    fence_proxy_async_smem();
    pdl_launch_dependents();
    pdl_wait();

    // ---- this CTA's run of units ------------------------------------------------------------------------------------
    const uint32_t per_t = (a.R + kThreads - 1) / kThreads, r0 = min(t * per_t, a.R), r1 = min(r0 + per_t, a.R);
    u64 sum = 0;
    for (uint32_t r = r0; r < r1; ++r) {
        const ReqView v = req_view(a, r);
        const uint32_t tiles = (v.nq * a.G + RT - 1) / RT, blocks = max(1u, (v.ctx + kKeys - 1) / kKeys);
        sum += (u64)a.heads * tiles * blocks;
        if (blockIdx.x == 0 && a.lens[r] > (int)(a.ld_table << a.page_shift)) atomicCAS(a.err, 0, (int)sh::kErrBadArgs);
    }
    u64 incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= (uint32_t)o) incl += x;
    }
    if (lane == 31) s_part[warp] = incl;
    __syncthreads();
    u64 total = 0;
#pragma unroll
    for (uint32_t w = 0; w < NW; ++w) {
        if (w < warp) incl += s_part[w];
        total += s_part[w];
    }
    const u64 per = (total + gridDim.x - 1) / gridDim.x;
    const u64 begin = per * blockIdx.x, end = min(total, begin + per);
    if (begin >= end) return;
    if (begin >= incl - sum && begin < incl) {
        u64 off = begin - (incl - sum);
        for (uint32_t r = r0; r < r1; ++r) {
            const ReqView v = req_view(a, r);
            const uint32_t tiles = (v.nq * a.G + RT - 1) / RT, blocks = max(1u, (v.ctx + kKeys - 1) / kKeys);
            const u64 n = (u64)a.heads * tiles * blocks;
            if (off < n) {
                s_start = {off, v, r};
                break;
            }
            off -= n;
        }
    }
    __syncthreads();

    // ---- the copies run ahead of the sums: cursor `p`. Lane i holds the page of the unit that is i units further in p's item
    // than `p_base`; the table is read again, a step before it is needed, when the item or the 32 units end. -----------
    const uint32_t ring = smem_u32(sm) + SM::kRing + warp * (kStages * 2 * SM::kTile);
    Cursor k;
    k.r = s_start.r, k.v = s_start.v;
    cursor_sizes<RT, kKeys>(k, a);
    {
        const uint32_t item = (uint32_t)(s_start.off / k.blocks);
        k.b = (uint32_t)(s_start.off - (u64)item * k.blocks), k.kvh = item / k.tiles, k.tile = item - k.kvh * k.tiles;
    }
    cursor_item<RT, kKeys>(k, a);
    Cursor p = k;
    u64 p_left = end - begin;
    // the warp's tokens of the cursor's unit hold keys
    auto in_use = [&](const Cursor &x) { return (int)(x.b * kKeys + warp * kStep) < x.lim_hi; };
    uint32_t p_base = k.b;
    int p_ids[HF];
    auto lookup = [&]() {
        p_base = p.b;
#pragma unroll
        for (uint32_t f = 0; f < HF; ++f) {
            const uint32_t tok = (p.b + lane) * kKeys + warp * kStep + f * 16;
            p_ids[f] = p_left && (int)tok < p.lim_hi ? a.table[(size_t)p.r * a.ld_table + (tok >> a.page_shift)] : -1;
        }
    };
    lookup();
    auto advance = [&]() {
        cursor_next<RT, kKeys>(p, a);
        --p_left;
        if (p.b == 0 || p.b - p_base == 32) lookup();
    };
    uint32_t p_slot = 0;
    float2 scales[2][HF];      // of the two units on their way, the nearer first; {.., -1}: left out
#pragma unroll
    for (uint32_t f = 0; f < HF; ++f) scales[0][f] = scales[1][f] = make_float2(0.f, -1.f);
    auto issue = [&]() {      // the next unit in which this warp has keys
        while (p_left && !in_use(p)) advance();
        if (p_left == 0) {
#pragma unroll
            for (uint32_t f = 0; f < HF; ++f) scales[0][f] = scales[1][f];
            return;
        }
        int id[HF];
#pragma unroll
        for (uint32_t f = 0; f < HF; ++f) id[f] = __shfl_sync(0xffffffffu, p_ids[f], p.b - p_base);
        const uint32_t tok = p.b * kKeys + warp * kStep;
#pragma unroll
        for (uint32_t f = 0; f < HF; ++f) {
            scales[0][f] = scales[1][f];
            scales[1][f] = make_float2(0.f, -1.f);
            if ((uint32_t)id[f] < a.pages) {
                const size_t at = (size_t)id[f] * a.heads + p.kvh;
                scales[1][f] = make_float2(a.ks[at], a.vs[at]);
            } else if ((int)(tok + f * 16) < p.lim_hi && lane == 0) {
                atomicCAS(a.err, 0, (int)sh::kErrBadArgs);
            }
        }
        if (lane == 0) {
            uint64_t *bar = full + p_slot;
            uint32_t n = 0;
#pragma unroll
            for (uint32_t i = 0; i < HF; ++i) n += i < a.boxes && (uint32_t)id[i] < a.pages;
            mbar_arrive_expect_tx(bar, n * a.box_bytes);
#pragma unroll
            for (uint32_t i = 0; i < HF; ++i)
                if (i < a.boxes && (uint32_t)id[i] < a.pages) {
                    uint8_t *dst = sm + SM::kRing + (warp * kStages + p_slot) * (2 * SM::kTile) + i * SM::kTile;
                    const int row = (int)((p.kvh << a.page_shift) + ((tok + i * 16) & page1));
                    tma_load_pair(dst, &mkv, bar, row, id[i]);
                    if (a.apart) tma_load_pair(dst + a.apart, &mv, bar, row, id[i]);
                }
        }
        p_slot = p_slot + 1 == kStages ? 0 : p_slot + 1;
        advance();
    };
    for (int i = 0; i < kStages; ++i) issue();
    __syncwarp();
    uint32_t slot = 0, phase = 0;

    for (u64 u = begin; u < end;) {
        const ReqView v = k.v;
        const uint32_t kvh = k.kvh, b0 = k.b, blocks = k.blocks, b1 = (uint32_t)min((u64)blocks, (u64)b0 + (end - u));
        const uint32_t row0 = k.tile * RT, nrows = min(RT, v.nq * a.G - row0);
        // keys of the tile's first and last row
        const int ctx = (int)v.ctx, lim_hi = k.lim_hi;
        const int lim_lo = min(max(v.base + (int)(row0 / a.G) + 1, 0), ctx);

        // ---- Q as the column operand: lane (g, c) holds columns 16 c .. of row 8 nt + g ------------------------------
        uint32_t qf[NT][KC * 4][2];
        int lim[NT][2];
        {
            uint32_t w[NT][KC][8];      // all loads before the first use
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const uint32_t n = nt * 8 + g, rr = row0 + n, qi = rr / a.G, gi = rr - qi * a.G;
                const __half *qp = a.q + (size_t)(v.qs + qi) * a.ldq + ((size_t)kvh * a.G + gi) * DH + c * 16;
#pragma unroll
                for (int j = 0; j < KC; ++j) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[nt][j][e] = 0;
                    if (n >= nrows) continue;
                    if (a.vec) {
                        const uint4 x = *reinterpret_cast<const uint4 *>(qp + j * 64);
                        const uint4 y = *reinterpret_cast<const uint4 *>(qp + j * 64 + 8);
                        w[nt][j][0] = x.x, w[nt][j][1] = x.y, w[nt][j][2] = x.z, w[nt][j][3] = x.w;
                        w[nt][j][4] = y.x, w[nt][j][5] = y.y, w[nt][j][6] = y.z, w[nt][j][7] = y.w;
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            w[nt][j][e] = (uint32_t)__half_as_ushort(qp[j * 64 + 2 * e]) |
                                          (uint32_t)__half_as_ushort(qp[j * 64 + 2 * e + 1]) << 16;
                    }
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < KC; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        // columns 4 i .. 4 i + 3 in the order word_to_h2 gives K's
                        const uint32_t x = w[nt][j][2 * i], y = w[nt][j][2 * i + 1];
                        qf[nt][j * 4 + i][0] = FP8 ? x : __byte_perm(x, y, 0x5410);
                        qf[nt][j * 4 + i][1] = FP8 ? y : __byte_perm(x, y, 0x7632);
                    }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t m = nt * 8 + 2 * c + e;
                lim[nt][e] = m < nrows ? min(max(v.base + (int)((row0 + m) / a.G) + 1, 0), ctx) : lim_hi;
            }

        float o[DH / 16][NT][4];
        float m[NT][2], top[NT][2], l[NT][2];      // the maximum (0 before there is one), the maximum + 8, the sum
#pragma unroll
        for (int i = 0; i < DH / 16; ++i)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][nt][e] = 0.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) m[nt][0] = m[nt][1] = l[nt][0] = l[nt][1] = 0.f, top[nt][0] = top[nt][1] = -INFINITY;

        for (uint32_t b = b0; b < b1; ++b) {
            if ((int)(b * kKeys + warp * kStep) >= lim_hi) break;
            if (!mbar_try_wait(full + slot, phase)) mbar_wait(full + slot, phase, abort, a.err);
            const uint32_t ring_at = ring + slot * (2 * SM::kTile);
            slot = slot + 1 == kStages ? 0 : slot + 1;
            phase ^= slot == 0;
#pragma unroll
            for (uint32_t f = 0; f < HF; ++f) {
                const int tok0 = (int)(b * kKeys + warp * kStep + f * 16);
                const float ks = scales[0][f].x, vs = scales[0][f].y;
                if (vs < 0.f) continue;      // no keys of this tile, or no such page: left out
                const uint32_t kt = ring_at + f * a.box_step + a.k_at, vt = ring_at + f * a.box_step + a.v_at;
                float s[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
                for (int j = 0; j < KC; ++j) {
                    // rows g and g + 8, columns 64 j + 16 c ..: 128-byte rows have piece x at x ^ (row % 8), 64-byte rows at
                    // x ^ (row / 2 % 4)
                    const uint32_t at = kt + g * DH + (DH == 128 ? ((j * 4 + c) ^ g) * 16 : (c ^ (g >> 1)) * 16);
                    const uint4 ka4 = lds16(at), kb4 = lds16(at + 8 * DH);
                    const uint32_t ka[4] = {ka4.x, ka4.y, ka4.z, ka4.w}, kb[4] = {kb4.x, kb4.y, kb4.z, kb4.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t a0, a1, a2, a3;
                        word_to_h2<FP8>(ka[i], a0, a2);
                        word_to_h2<FP8>(kb[i], a1, a3);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            mma16816(s[nt], a0, a1, a2, a3, qf[nt][j * 4 + i][0], qf[nt][j * 4 + i][1]);
                    }
                }
                const float ksl = ks * a.sl2, vcl = fmaxf(vs, 0x1p-80f);
                {
                    const float lvs = __log2f(vcl), rvs = __frcp_rn(vcl);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[nt][e] = fmaf(s[nt][e], ksl, lvs);
                    if (tok0 + 16 > lim_lo) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (tok0 + (int)g + 8 * (e >> 1) >= lim[nt][e & 1]) s[nt][e] = -INFINITY;
                    }
                    bool raise = false;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) raise |= fmaxf(s[nt][e], s[nt][e + 2]) > top[nt][e];
                    // the maximum only moves when a weight would pass 2^8 (exact room in fp16), which is rare after the start
                    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                float x = fmaxf(s[nt][e], s[nt][e + 2]);
#pragma unroll
                                for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                                const float was = top[nt][e] - 8.f, now = fmaxf(was, x);
                                const float f = now == -INFINITY ? 1.f : fast_exp2(was - now);
                                top[nt][e] = now + 8.f;
                                m[nt][e] = now == -INFINITY ? 0.f : now;
                                l[nt][e] *= f;
#pragma unroll
                                for (int i = 0; i < DH / 16; ++i) o[i][nt][e] *= f, o[i][nt][e + 2] *= f;
                            }
                    }
                    uint32_t w0[NT], w1[NT], d0[NT], d1[NT];      // weights in fp16, and what that rounding left
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            w[e] = fast_exp2(s[nt][e] - m[nt][e & 1]);
                            l[nt][e & 1] = fmaf(w[e], rvs, l[nt][e & 1]);
                        }
                        const __half2 h0 = __floats2half2_rn(w[0], w[1]), h1 = __floats2half2_rn(w[2], w[3]);
                        const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
                        w0[nt] = movmatrix(*reinterpret_cast<const uint32_t *>(&h0));
                        w1[nt] = movmatrix(*reinterpret_cast<const uint32_t *>(&h1));
                        d0[nt] = movmatrix(pack_h2(w[0] - f0.x, w[1] - f0.y));
                        d1[nt] = movmatrix(pack_h2(w[2] - f1.x, w[3] - f1.y));
                    }
                    uint32_t vr[4][VW];      // tokens 2 c, 2 c + 1, 2 c + 8, 2 c + 9, columns VB g ..
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t tok = 2 * c + (e & 1) + 8 * (e >> 1);
                        if (VW == 4) {
                            const uint4 x = lds16(vt + tok * DH + (g ^ (tok & 7)) * 16);
                            vr[e][0] = x.x, vr[e][1] = x.y, vr[e][VW - 2] = x.z, vr[e][VW - 1] = x.w;
                        } else {
                            const uint2 x = lds8(vt + tok * DH + ((g >> 1) ^ (tok >> 1 & 3)) * 16 + (g & 1) * 8);
                            vr[e][0] = x.x, vr[e][1] = x.y;
                        }
                    }
                    if (tok0 + 16 > lim_hi) {      // rows that are no keys can hold anything
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (tok0 + (int)(2 * c + (e & 1) + 8 * (e >> 1)) >= lim_hi)
#pragma unroll
                                for (int i = 0; i < VW; ++i) vr[e][i] = 0;
                    }
#pragma unroll
                    for (int i = 0; i < VW; ++i) {
                        const uint32_t a00 = byte_pair<FP8, 0>(vr[0][i], vr[1][i]), a02 = byte_pair<FP8, 0>(vr[2][i], vr[3][i]);
                        const uint32_t a01 = byte_pair<FP8, 1>(vr[0][i], vr[1][i]), a03 = byte_pair<FP8, 1>(vr[2][i], vr[3][i]);
                        const uint32_t a10 = byte_pair<FP8, 2>(vr[0][i], vr[1][i]), a12 = byte_pair<FP8, 2>(vr[2][i], vr[3][i]);
                        const uint32_t a11 = byte_pair<FP8, 3>(vr[0][i], vr[1][i]), a13 = byte_pair<FP8, 3>(vr[2][i], vr[3][i]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma16816(o[2 * i][nt], a00, a01, a02, a03, w0[nt], w1[nt]);
                            mma16816(o[2 * i + 1][nt], a10, a11, a12, a13, w0[nt], w1[nt]);
                            mma16816(o[2 * i][nt], a00, a01, a02, a03, d0[nt], d1[nt]);
                            mma16816(o[2 * i + 1][nt], a10, a11, a12, a13, d0[nt], d1[nt]);
                        }
                    }
                }
            }
            __syncwarp();
            issue();      // into the stage just read
        }

        // ---- join the warps --------------------------------------------------------------------------------------------
        __syncthreads();      // s_* of the item before are no longer read
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x = l[nt][e];
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
                const uint32_t n = nt * 8 + 2 * c + e;
                if (g == 0) s_m[warp * RT + n] = top[nt][e] - 8.f, s_l[warp * RT + n] = x;
#pragma unroll
                for (int i = 0; i < DH / 16; ++i)
                    s_o[(warp * RT + n) * kPitch + i * 8 + g] = make_float2(o[i][nt][e], o[i][nt][e + 2]);
            }
        __syncthreads();
        if (NT > 1) {      // many rows: each one's factors of the warps in place of their maxima, and its sum, once
            if (t < RT) {
                float mx = -INFINITY, ll = 0.f;
#pragma unroll
                for (uint32_t w = 0; w < NW; ++w) mx = fmaxf(mx, s_m[w * RT + t]);
#pragma unroll
                for (uint32_t w = 0; w < NW; ++w) {
                    const float mw = s_m[w * RT + t], f = mw == -INFINITY ? 0.f : fast_exp2(mw - mx);
                    ll = fmaf(s_l[w * RT + t], f, ll);
                    s_m[w * RT + t] = f;
                }
                if (ll == 0.f && t < nrows) ll = no_weight(a, v, kvh, row0 + t, DH, b0 * kKeys);
                s_l[t] = ll, s_l[RT + t] = mx;
            }
            __syncthreads();
        }
        auto write_out = [&](uint32_t n, uint32_t d, float x, float y, float ll) {
            const float inv = ll == 0.f ? 0.f : 1.f / ll;
            const uint32_t rr = row0 + n, qi = rr / a.G, gi = rr - qi * a.G;
            __half *op = a.o + (size_t)(v.qs + qi) * a.ldo + ((size_t)kvh * a.G + gi) * DH + d;
            if (a.vec) *reinterpret_cast<__half2 *>(op) = __floats2half2_rn(x * inv, y * inv);
            else op[0] = __float2half_rn(x * inv), op[1] = __float2half_rn(y * inv);
        };
        const bool whole = b0 == 0 && b1 == blocks;
        const uint32_t slot = 2 * blockIdx.x + (b0 == 0 ? 1 : 0);
        float *po = a.part + (size_t)slot * RT * (DH + 2), *pm = po + RT * DH, *pl = pm + RT;
        constexpr uint32_t kRowsPer = kThreads / (DH / 2);      // a thread has one column pair of every kRowsPer-th row
        const uint32_t j = t % (DH / 2), d = (j & 7) * VB + (j >> 3) * 2;
#pragma unroll(NT > 1 ? 4 : 1)
        for (uint32_t n = t / (DH / 2); n < nrows; n += kRowsPer) {
            float mx = NT > 1 ? s_l[RT + n] : -INFINITY, ll = NT > 1 ? s_l[n] : 0.f, x = 0.f, y = 0.f;
            if (NT == 1)
#pragma unroll
                for (uint32_t w = 0; w < NW; ++w) mx = fmaxf(mx, s_m[w * RT + n]);
#pragma unroll
            for (uint32_t w = 0; w < NW; ++w) {
                float f = s_m[w * RT + n];
                if (NT == 1) {
                    f = f == -INFINITY ? 0.f : fast_exp2(f - mx);
                    ll = fmaf(s_l[w * RT + n], f, ll);
                }
                const float2 p = s_o[(w * RT + n) * kPitch + j];
                x = fmaf(p.x, f, x);
                y = fmaf(p.y, f, y);
            }
            if (NT == 1 && ll == 0.f) ll = no_weight(a, v, kvh, row0 + n, DH, b0 * kKeys);
            if (whole) {
                write_out(n, d, x, y, ll);
            } else {
                *reinterpret_cast<float2 *>(po + n * DH + 2 * j) = make_float2(x, y);
                if (j == 0) pm[n] = mx, pl[n] = ll;
            }
        }
        if (!whole) {
            // the item's CTAs: c0 holds its first unit and counts the arrivals
            const u64 u0 = u - b0;
            const uint32_t c0 = (uint32_t)(u0 / per), c1 = (uint32_t)((u0 + blocks - 1) / per);
            __syncthreads();      // the release of thread 0's arrival covers what the CTA has written before this
            if (t == 0) {
                const uint32_t before = atom_add_acq_rel_gpu(a.counters + c0, 1u);
                s_flag = before == c1 - c0;
                if (s_flag) a.counters[c0] = 0;      // for the next call
            }
            __syncthreads();
            if (s_flag) {
                const uint32_t parts = c1 - c0 + 1;
                auto part = [&](uint32_t i) { return a.part + (size_t)(2 * (c0 + i) + (i == 0)) * RT * (DH + 2); };
                // eight loads in flight: a single row's parts, or two of four rows
                constexpr uint32_t kAhead = 8, kR = NT > 1 ? 4 : 1, kP = kAhead / kR;
                // each row's maximum and sum, by eight lanes
                for (uint32_t n = t >> 3; n < (nrows + 3) / 4 * 4; n += kThreads / 8) {      // whole warps: shuffles
                    float mx = -INFINITY, ll = 0.f;
                    for (uint32_t i0 = t & 7; i0 < parts; i0 += 8 * kAhead) {
                        float mi[kAhead], li[kAhead], mb = mx;
#pragma unroll
                        for (uint32_t q = 0; q < kAhead; ++q) {
                            const bool in = n < nrows && i0 + 8 * q < parts;
                            mi[q] = in ? __ldcg(part(i0 + 8 * q) + RT * DH + n) : -INFINITY;
                            li[q] = in ? __ldcg(part(i0 + 8 * q) + RT * DH + RT + n) : 0.f;
                        }
#pragma unroll
                        for (uint32_t q = 0; q < kAhead; ++q) mb = fmaxf(mb, mi[q]);
                        ll *= mx == -INFINITY ? 1.f : fast_exp2(mx - mb);
                        mx = mb;
#pragma unroll
                        for (uint32_t q = 0; q < kAhead; ++q)
                            ll = fmaf(li[q], mi[q] == -INFINITY ? 0.f : fast_exp2(mi[q] - mx), ll);
                    }
                    __syncwarp();
                    float mt = mx;
#pragma unroll
                    for (int d = 4; d > 0; d >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, d));
                    ll *= mx == -INFINITY ? 1.f : fast_exp2(mx - mt);
#pragma unroll
                    for (int d = 4; d > 0; d >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, d);
                    if ((t & 7) == 0 && n < nrows) s_m[n] = mt, s_l[n] = ll;
                }
                __syncthreads();
                for (uint32_t n0 = t / (DH / 2); n0 < nrows; n0 += kR * kRowsPer) {
                    float x[kR], y[kR];
#pragma unroll
                    for (uint32_t r = 0; r < kR; ++r) x[r] = y[r] = 0.f;
                    for (uint32_t i0 = 0; i0 < parts; i0 += kP) {
                        float f[kR][kP];
                        float2 z[kR][kP];
#pragma unroll
                        for (uint32_t r = 0; r < kR; ++r)
#pragma unroll
                            for (uint32_t q = 0; q < kP; ++q) {
                                const uint32_t n = n0 + r * kRowsPer;
                                const float *pi = part(i0 + q);
                                const bool in = n < nrows && i0 + q < parts;
                                f[r][q] = in ? __ldcg(pi + RT * DH + n) : -INFINITY;
                                z[r][q] = in ? __ldcg(reinterpret_cast<const float2 *>(pi + n * DH + 2 * j)) : make_float2(0.f, 0.f);
                            }
#pragma unroll
                        for (uint32_t r = 0; r < kR; ++r)
#pragma unroll
                            for (uint32_t q = 0; q < kP; ++q) {
                                const float mx = s_m[min(n0 + r * kRowsPer, nrows - 1)];
                                const float g = f[r][q] == -INFINITY ? 0.f : fast_exp2(f[r][q] - mx);
                                x[r] = fmaf(z[r][q].x, g, x[r]), y[r] = fmaf(z[r][q].y, g, y[r]);
                            }
                    }
#pragma unroll
                    for (uint32_t r = 0; r < kR; ++r) {
                        const uint32_t n = n0 + r * kRowsPer;
                        if (n < nrows) write_out(n, d, x[r], y[r], s_l[n]);
                    }
                }
            }
        }
        u += b1 - b0;
        k.b = b1 - 1;
        if (u < end) cursor_next<RT, kKeys>(k, a);
    }
    if (*abort)      // a copy did not arrive in time: give those in flight as long again
        for (int i = 0; i < kStages; ++i) drain_wait(full + i, phase ^ (i < (int)slot));
}

// ================================================================================================================
// Many rows per request (prompt chunks): tcgen05. A CTA per SM walks its run of units (request, kv head, 256 rows, block of
// 128 tokens; the blocks behind a tile's last row are left out). 768 threads:
//   warp 0        copies: the pages' K and V boxes (8 bits) and scales into a ring of two blocks, as above
//   warp 1        tcgen05.mma: per block and 128-row tile t  S_t = Q_t K^T (N = 128 tokens), then, when the softmax has
//                 written P_t over S_t, O_t += P_t V with P_t read from tensor memory. The order P V of the block before, S of
//                 this one, for one tile after the other keeps one tile's matrix products under the other's softmax.
//   warps 4..7    turn a block's codes into fp16 operands in the swizzled layout of the matrix unit, once for both tiles
//                 (one key row per lane: neither the reads nor the writes of a quarter-warp meet in a bank); K a block ahead
//   warps 8..23   softmax: eight warps per tile, two threads per row, each with 64 of its scores in registers. A tile's
//                 products wait for its weights and its scores for its products, so the softmax's latency counts: with one
//                 thread per row a block took 5000 cycles.
// The scales of 16 tokens are one multiply-add per 16 scores for the maximum, one per score (x = ks s + log2 vs) and one per
// 16 weights. A block is 2048 cycles of tensor work at its peak rate and as many of the special-function unit's (32768
// exponentials). It takes about 4800: 32 matrix instructions of about 100 cycles each, where the peak rate is 64, and what of the
// softmax they do not cover, as a tile has one buffer for its scores. 4 x 512 rows over up to 8192 tokens: 182 us. The compiler
// reports about 530 bytes of spilled registers at the 80 that all warps start with.
// ================================================================================================================
constexpr uint32_t kTlRows = 128, kTlKeys = 128, kTlItem = 256, kTlThreads = 768, kTlStages = 2;
constexpr uint32_t kTlRegs = 96, kTlRegsOther = 48;      // 512 x 96 + 256 x 48 = 768 x 80, what the block starts with

template <int DH>
struct TilesSmem {
    static constexpr uint32_t kChunk = 128 * 128;                      // 128 rows x 64 fp16 columns
    static constexpr uint32_t kTile = DH / 64 * kChunk, kBox = 16 * DH, kCodes = kTlKeys * DH;
    static constexpr uint32_t kQ = 0, kK = kQ + 2 * kTile, kV = kK + 2 * kTile, kRing = kV + kTile;   // K twice
    static constexpr uint32_t kInfo = kRing + kTlStages * 2 * kCodes;  // [stages][8] {ks, vs, usable}
    static constexpr uint32_t kGroup = kInfo + kTlStages * 128;        // [4][8] {ks scale log2 e, log2 vs, 1 / vs}
    static constexpr uint32_t kRowMax = kGroup + 512;                  // [2 tiles][2][128]
    static constexpr uint32_t kBars = kRowMax + 2048, kMisc = kBars + 20 * 8, kBytes = kMisc + 64;
    static_assert(kBytes <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// A tile of a request in the run of a CTA
struct TileCursor {
    uint32_t r, kvh, tile, tiles, b, blocks;
    ReqView v;
    uint32_t row0, nrows;
    int lim_hi;
};
__device__ __forceinline__ void tile_sizes(TileCursor &k, const KvArgs &a) {      // after tile or request changed
    k.row0 = k.tile * kTlItem, k.nrows = min(kTlItem, k.v.nq * a.G - k.row0);
    k.lim_hi = min(max(k.v.base + (int)((k.row0 + k.nrows - 1) / a.G) + 1, 0), (int)k.v.ctx);
    k.blocks = max(1u, (uint32_t)(k.lim_hi + (int)kTlKeys - 1) / kTlKeys);
}
__device__ __forceinline__ void tile_request(TileCursor &k, const KvArgs &a) {
    k.v = req_view(a, k.r);
    k.tiles = (k.v.nq * a.G + kTlItem - 1) / kTlItem;
}
__device__ __forceinline__ void tile_next(TileCursor &k, const KvArgs &a) {       // the next tile's first block
    k.b = 0;
    if (++k.tile == k.tiles) {
        k.tile = 0;
        if (++k.kvh == a.heads) {
            k.kvh = 0;
            do {
                if (++k.r >= a.R) return;
                tile_request(k, a);
            } while (k.tiles == 0);
        }
    }
    tile_sizes(k, a);
}

template <int DH, bool FP8>
__global__ void __launch_bounds__(kTlThreads, 1)
    k_attn_kv8_tiles(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, KvArgs a) {
    using SM = TilesSmem<DH>;
    typedef unsigned long long u64;
    constexpr uint32_t kTmS = 0, kTmO = 2 * kTlKeys;                   // tensor memory: S_t / P_t, O_t
    extern __shared__ __align__(1024) uint8_t tiles_smem[];      // swizzled tiles from its start: no room to align by hand
    uint8_t *sm = tiles_smem;
    if (smem_u32(sm) & 1023u) {
        if (threadIdx.x == 0) atomicCAS(a.err, 0, (int)sh::kErrBadArgs);
        return;
    }
    uint64_t *bars = reinterpret_cast<uint64_t *>(sm + SM::kBars);
    uint64_t *c_full = bars, *c_empty = bars + 2;                      // ring of codes
    uint64_t *k_full = bars + 4, *k_empty = bars + 18, *v_full = bars + 6, *v_empty = bars + 7;   // K: two each
    uint64_t *q_full = bars + 8, *s_full = bars + 10, *p_full = bars + 12, *o_full = bars + 14, *mdone = bars + 16;
    struct Misc {
        TileCursor first;
        uint32_t flag, tmem;
        int abort;
    };
    static_assert(sizeof(Misc) <= SM::kBytes - SM::kMisc, "shared memory");
    Misc &mi = *reinterpret_cast<Misc *>(sm + SM::kMisc);
    u64 *warp_units = reinterpret_cast<u64 *>(sm + SM::kRowMax);      // read before the first maximum is written
    volatile int *abort = &mi.abort;
    const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const uint32_t page1 = (1u << a.page_shift) - 1;
    if (t == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(c_full + i, 1 + 8), mbar_init(c_empty + i, 4);
            mbar_init(k_full + i, 4), mbar_init(k_empty + i, 1);
            mbar_init(q_full + i, 8), mbar_init(s_full + i, 1), mbar_init(p_full + i, 8), mbar_init(o_full + i, 1);
        }
        mbar_init(v_full, 4), mbar_init(v_empty, 1), mbar_init(mdone, 1);
        mi.abort = 0;
        prefetch_tmap(&mk), prefetch_tmap(&mv);
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(&mi.tmem, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = mi.tmem;
    pdl_launch_dependents();
    pdl_wait();

    // ---- this CTA's run of units ------------------------------------------------------------------------------------
    auto head_units = [&](TileCursor &k) {      // units of one head of a request
        u64 n = 0;
        for (k.tile = 0; k.tile < k.tiles; ++k.tile) {
            tile_sizes(k, a);
            n += k.blocks;
        }
        return n;
    };
    const uint32_t per_t = (a.R + kTlThreads - 1) / kTlThreads, r0 = min(t * per_t, a.R), r1 = min(r0 + per_t, a.R);
    TileCursor k0 = {};
    u64 sum = 0, one = 0;
    for (uint32_t r = r0; r < r1; ++r) {
        k0.r = r;
        tile_request(k0, a);
        one = head_units(k0);
        sum += a.heads * one;
        if (blockIdx.x == 0 && a.lens[r] > (int)(a.ld_table << a.page_shift)) atomicCAS(a.err, 0, (int)sh::kErrBadArgs);
    }
    u64 incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= (uint32_t)o) incl += x;
    }
    if (lane == 31) warp_units[warp] = incl;
    __syncthreads();
    u64 total = 0;
    for (uint32_t w = 0; w < kTlThreads / 32; ++w) {
        if (w < warp) incl += warp_units[w];
        total += warp_units[w];
    }
    const u64 per = (total + gridDim.x - 1) / gridDim.x, begin = per * blockIdx.x, end = min(total, begin + per);
    if (begin < end && begin >= incl - sum && begin < incl) {
        u64 off = begin - (incl - sum);
        for (uint32_t r = r0; r < r1; ++r) {
            if (r1 - r0 > 1) {
                k0.r = r;
                tile_request(k0, a);
                one = head_units(k0);
            }
            if (off < a.heads * one) break;
            off -= a.heads * one;
        }
        k0.kvh = (uint32_t)(off / one);
        off -= k0.kvh * one;
        for (k0.tile = 0; tile_sizes(k0, a), off >= k0.blocks; ++k0.tile) off -= k0.blocks;
        k0.b = (uint32_t)off;
        mi.first = k0;
    }
    __syncthreads();
    k0 = mi.first;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTlRegsOther));
        if (warp == 0) {
            // ---------------- copies: lane i has tokens 16 i .. of a block ----------------
            TileCursor k = k0;
            uint32_t st = 0, ph = 0, n = 0;
            auto lookup = [&]() {
                const uint32_t tok = k.b * kTlKeys + lane * 16;
                return lane < 8 && (int)tok < k.lim_hi ? a.table[(size_t)k.r * a.ld_table + (tok >> a.page_shift)] : -1;
            };
            int id = begin < end ? lookup() : -1;
            for (u64 u = begin; u < end; ++u, ++n) {
                const uint32_t tok = k.b * kTlKeys + lane * 16;
                const bool used = lane < 8 && (int)tok < k.lim_hi, ok = used && (uint32_t)id < a.pages;
                const int row = (int)((k.kvh << a.page_shift) + (tok & page1)), page = id;
                const size_t at = (size_t)(uint32_t)id * a.heads + k.kvh;
                if (u + 1 < end) {
                    if (++k.b == k.blocks) tile_next(k, a);
                    id = lookup();
                }
                if (n >= kTlStages) mbar_wait(c_empty + st, ph ^ 1u, abort, a.err);
                uint64_t *bar = c_full + st;
                const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, ok));
                float *info = reinterpret_cast<float *>(sm + SM::kInfo + (st * 8 + lane) * 16);
                // the lanes' own stores come before lane 0's arrival, which releases them (theirs below only count copies)
                if (lane < 8) info[2] = ok;
                __syncwarp();
                if (lane == 0) mbar_arrive_expect_tx(bar, boxes * 2 * SM::kBox);
                __syncwarp();
                if (lane < 8) {
                    if (ok) {
                        uint8_t *dst = sm + SM::kRing + st * 2 * SM::kCodes + lane * SM::kBox;
                        tma_load_3d(dst, &mk, bar, 0, row, page);
                        tma_load_3d(dst + SM::kCodes, &mv, bar, 0, row, page);
                        cp_async4(smem_u32(info), a.ks + at);
                        cp_async4(smem_u32(info) + 4, a.vs + at);
                    } else if (used) {
                        atomicCAS(a.err, 0, (int)sh::kErrBadArgs);
                    }
                    cp_async_arrive(bar);
                }
                if (++st == kTlStages) st = 0, ph ^= 1u;
            }
            // every copy has landed before the CTA may exit
            for (uint32_t i = 0; i < min(n, kTlStages); ++i) {
                const uint32_t last = n - 1 - i;
                if (lane == 0) drain_wait(c_full + last % kTlStages, last / kTlStages & 1);
            }
        } else if (warp == 1) {
            // ---------------- MMA issue: the whole warp walks the loop, lane 0 issues ----------------
            const uint32_t is0 = lane == 0 ? 1u : 0u;
            constexpr uint32_t idesc_s = umma_idesc_f16(kTlRows, kTlKeys, 0, 0), idesc_o = umma_idesc_f16(kTlRows, DH, 0, 1);
            const uint64_t qd = sw128_desc(smem_u32(sm + SM::kQ), 16, 1024), kd = sw128_desc(smem_u32(sm + SM::kK), 16, 1024);
            const uint64_t vd = sw128_desc(smem_u32(sm + SM::kV), SM::kChunk, 1024);
            uint32_t kn = 0, vn = 0, pn[2] = {0, 0}, qn[2] = {0, 0};      // phases seen of each barrier
            TileCursor k = k0;
            for (u64 u = begin; u < end;) {
                const uint32_t nb = (uint32_t)min((u64)(k.blocks - k.b), end - u), nt = k.nrows > kTlRows ? 2u : 1u;
                // step j: P V of block j - 1, S of block j
                for (uint32_t j = 0; j <= nb; ++j) {
                    if (j > 0) mbar_wait(v_full, vn++ & 1u, abort, a.err);
                    const uint32_t ks = kn & 1u;      // K's buffer
                    const uint64_t kdj = kd + (ks * SM::kTile >> 4);
    #pragma unroll 1
                    for (uint32_t t2 = 0; t2 < nt; ++t2) {
                        if (j > 0) {
                            mbar_wait(p_full + t2, pn[t2]++ & 1u, abort, a.err);
                            tc_fence_after();
    #pragma unroll
                            for (int i = 0; i < (int)kTlKeys / 16; ++i)
                                umma_f16_ts_if(is0, tmem + kTmO + t2 * DH, tmem + kTmS + t2 * kTlKeys + i * 8,
                                               vd + (uint64_t)(i * (2048 >> 4)), idesc_o, (j == 1 && i == 0) ? 0u : 1u);
                            if (j == nb) umma_commit_if(is0, o_full + t2);
                            if (t2 + 1 == nt) umma_commit_if(is0, v_empty);
                        }
                        if (j < nb) {
                            if (t2 == 0) mbar_wait(k_full + ks, kn >> 1 & 1u, abort, a.err);
                            if (j == 0) mbar_wait(q_full + t2, qn[t2]++ & 1u, abort, a.err);
                            tc_fence_after();
    #pragma unroll
                            for (int i = 0; i < DH / 16; ++i) {
                                const uint32_t at = ((uint32_t)(i / 4) * SM::kChunk + (i % 4) * 32) >> 4;
                                umma_f16_ss_if(is0, tmem + kTmS + t2 * kTlKeys, qd + (t2 * SM::kTile >> 4) + at, kdj + at,
                                               idesc_s, i > 0 ? 1u : 0u);
                            }
                            umma_commit_if(is0, s_full + t2);
                        }
                    }
                    if (j < nb) umma_commit_if(is0, k_empty + ks), ++kn;
                }
                u += nb;
                if (u < end) tile_next(k, a);
            }
            // tensor memory may only be freed once every issued MMA has completed
            umma_commit_if(is0, mdone);
            if (is0) drain_wait(mdone, 0);
        }
    } else if (warp < 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTlRegsOther));
        // ---------------- codes -> fp16: lane has key row 32 (warp - 4) + lane ----------------
        const uint32_t row = (warp - 4) * 32 + lane, grp = row >> 4;
        uint32_t n = 0;
        TileCursor k = k0;
        auto convert = [&](const uint8_t *src, uint8_t *dst, bool keep) {
            // 16 codes: piece p of the row in the ring's swizzle; 32 bytes of fp16: pieces 2 p, 2 p + 1 of a 64-column chunk
#pragma unroll
            for (int q = 0; q < DH / 64; ++q) {
                uint4 x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t p = q * 4 + i;
                    x[i] = lds16(smem_u32(src) + row * DH + (DH == 128 ? (p ^ (row & 7)) : (p ^ (row >> 1 & 3))) * 16);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t w[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
                    uint32_t h[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (FP8) {
                            h[2 * i] = e4m3x2_to_h2(w[i] & 0xFFFFu), h[2 * i + 1] = e4m3x2_to_h2(w[i] >> 16);
                        } else {
                            const uint32_t y = w[i] ^ 0x80808080u;
                            h[2 * i] = hsub2(__byte_perm(y, 0x64646464u, 0x4140), kMagicVal);
                            h[2 * i + 1] = hsub2(__byte_perm(y, 0x64646464u, 0x4342), kMagicVal);
                        }
                    }
                    if (!keep)
#pragma unroll
                        for (int i = 0; i < 8; ++i) h[i] = 0;
                    uint8_t *to = dst + q * SM::kChunk + row * 128;
                    *reinterpret_cast<uint4 *>(to + (((2 * j) ^ (row & 7)) * 16)) = make_uint4(h[0], h[1], h[2], h[3]);
                    *reinterpret_cast<uint4 *>(to + (((2 * j + 1) ^ (row & 7)) * 16)) = make_uint4(h[4], h[5], h[6], h[7]);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
        };
        // K of block n + 1 goes before V of block n: K has two buffers, so it is ready while the matrix unit is at block n
        auto keys = [&](uint32_t i) {
            const uint32_t st = i & 1;
            mbar_wait(c_full + st, i >> 1 & 1, abort, a.err);
            const float4 info = *reinterpret_cast<const float4 *>(sm + SM::kInfo + (st * 8 + grp) * 16);
            const bool ok = info.z != 0.f;
            if (i >= 2) mbar_wait(k_empty + st, (i >> 1 & 1) ^ 1u, abort, a.err);
            if ((lane & 15) == 0) {
                const float vs = ok ? fmaxf(info.y, 0x1p-80f) : 1.f;
                // the first factor > 0: a masked score of -infinity stays that
                *reinterpret_cast<float4 *>(sm + SM::kGroup + ((i & 3) * 8 + grp) * 16) =
                    make_float4(fmaxf(ok ? info.x * a.sl2 : 0.f, 0x1p-100f), ok ? __log2f(vs) : -INFINITY, __frcp_rn(vs), 0.f);
            }
            convert(sm + SM::kRing + st * 2 * SM::kCodes, sm + SM::kK + st * SM::kTile, ok);
            if (lane == 0) mbar_arrive(k_full + st);
        };
        if (begin < end) keys(0);
        for (u64 u = begin; u < end; ++u, ++n) {
            const uint32_t st = n & 1;
            if (u + 1 < end) keys(n + 1);
            const bool ok = reinterpret_cast<const float4 *>(sm + SM::kInfo + (st * 8 + grp) * 16)->z != 0.f;
            if (n > 0) mbar_wait(v_empty, (n - 1) & 1u, abort, a.err);
            // rows that are no keys can hold anything; their weights are 0
            convert(sm + SM::kRing + (st * 2 + 1) * SM::kCodes, sm + SM::kV, ok && (int)(k.b * kTlKeys + row) < k.lim_hi);
            if (lane == 0) mbar_arrive(v_full), mbar_arrive(c_empty + st);
            if (u + 1 < end && ++k.b == k.blocks) tile_next(k, a);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTlRegs));
        // ---------------- softmax and output ----------------
        const uint32_t t2 = (warp - 8) >> 3, half = (warp - 8) >> 2 & 1, quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t st = t - 256;                                                              // of 512 softmax threads
        constexpr uint32_t kHalfKeys = kTlKeys / 2, kHalfCols = DH / 2;
        const uint32_t lane_base = tmem + (quarter * 32u << 16);
        const uint32_t s_addr = lane_base + kTmS + t2 * kTlKeys, o_addr = lane_base + kTmO + t2 * DH + half * kHalfCols;
        float *row_max = reinterpret_cast<float *>(sm + SM::kRowMax) + t2 * 256 + row;            // [2][128] of the tile: the halves' maxima
        float *row_sum = reinterpret_cast<float *>(sm + SM::kQ + t2 * SM::kTile) + row;           // over Q at an item's end
        uint32_t n = 0, sn = 0, on = 0;      // blocks of the run, blocks of this tile, items of this tile
        TileCursor k = k0;
        auto all_sync = [&]() { asm volatile("bar.sync 1, 512;" ::: "memory"); };
        auto tile_sync = [&]() { asm volatile("bar.sync %0, 256;" ::"r"(2 + t2) : "memory"); };
        for (u64 u = begin; u < end;) {
            const uint32_t b0 = k.b, nb = (uint32_t)min((u64)(k.blocks - k.b), end - u), rr = t2 * kTlRows + row;
            const bool live = k.nrows > t2 * kTlRows, mine = rr < k.nrows;      // the tile's, this row's
            const uint32_t qi = (k.row0 + rr) / a.G, gi = (k.row0 + rr) - qi * a.G;
            const int ctx = (int)k.v.ctx;
            const int lim = mine ? min(max(k.v.base + (int)qi + 1, 0), ctx) : k.lim_hi;
            const int lim_lo = min(max(k.v.base + (int)((k.row0 + t2 * kTlRows) / a.G) + 1, 0), ctx);
            float m = -INFINITY, l = 0.f;
            if (live) {
                // Q rows -> swizzled operand, whole rows by neighbouring lanes (the tile's score products of the item before
                // have completed). This warp has 16 of its quarter's rows.
                const size_t own = mine ? (size_t)(k.v.qs + qi) * a.ldq + ((size_t)k.kvh * a.G + gi) * DH : ~(size_t)0;
                constexpr int kPieces = DH / 8, kRowsPer = 32 / kPieces;
                const uint32_t piece = lane % kPieces;
                uint4 x[16 / kRowsPer];      // all loads before the first store
#pragma unroll
                for (int i = 0; i < 16 / kRowsPer; ++i) {
                    const size_t at = __shfl_sync(0xffffffffu, own, half * 16 + i * kRowsPer + lane / kPieces);
                    x[i] = make_uint4(0, 0, 0, 0);
                    if (at == ~(size_t)0) continue;
                    const __half *qp = a.q + at + piece * 8;
                    if (a.vec) {
                        x[i] = *reinterpret_cast<const uint4 *>(qp);
                    } else {
                        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
                        for (int e = 0; e < 8; ++e) w[e >> 1] |= (uint32_t)__half_as_ushort(qp[e]) << (16 * (e & 1));
                        x[i] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 16 / kRowsPer; ++i) {
                    const uint32_t r = quarter * 32 + half * 16 + i * kRowsPer + lane / kPieces;
                    *reinterpret_cast<uint4 *>(sm + SM::kQ + t2 * SM::kTile + (piece >> 3) * SM::kChunk + r * 128 +
                                               (((piece & 7) ^ (r & 7)) * 16)) =
                        make_uint4(x[i].x ^ a.flip, x[i].y ^ a.flip, x[i].z ^ a.flip, x[i].w ^ a.flip);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full + t2);
            }
            for (uint32_t j = 0; j < nb; ++j, ++n) {
                if (!live) continue;
                const int key0 = (int)((b0 + j) * kTlKeys + half * kHalfKeys);
                const float4 *grp = reinterpret_cast<const float4 *>(sm + SM::kGroup + (n & 3) * 128 + half * 64);
                mbar_wait(s_full + t2, sn++ & 1u, abort, a.err);      // and P V of the block before is complete
                tc_fence_after();
                float sc[kHalfKeys];
                {
                    uint32_t v0[32], v1[32];   // two loads in flight, one wait
                    tmem_ld_32x32b_x32(s_addr + half * kHalfKeys, v0);
                    tmem_ld_32x32b_x32(s_addr + half * kHalfKeys + 32, v1);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) sc[i] = __uint_as_float(v0[i]), sc[32 + i] = __uint_as_float(v1[i]);
                }
                if (key0 + (int)kHalfKeys > lim_lo) {
#pragma unroll
                    for (int i = 0; i < (int)kHalfKeys; ++i)
                        if (key0 + i >= lim) sc[i] = -INFINITY;
                }
                // 16 keys share their scales (>= 0): the largest exponent comes from the largest score
                float mb = -INFINITY;
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const float4 gr = grp[h];
                    const float *x = sc + 16 * h;
                    const float a0 = max3(x[0], x[1], x[2]), a1 = max3(x[3], x[4], x[5]), a2 = max3(x[6], x[7], x[8]);
                    const float a3 = max3(x[9], x[10], x[11]), a4 = max3(x[12], x[13], x[14]);
                    mb = fmaxf(mb, fmaf(max3(max3(a0, a1, a2), fmaxf(a3, a4), x[15]), gr.x, gr.y));
                }
                row_max[half * 128] = mb;
                tile_sync();      // both halves' maxima are there, and both hold their scores: P may go over S
                mb = fmaxf(mb, row_max[(half ^ 1) * 128]);
                // the maximum only moves when a weight would pass 2^8 (exact room in fp16); O is rescaled then
                float alpha = 1.f;
                const bool raise = mb > m + 8.f;
                if (raise) {
                    alpha = fast_exp2(m - mb);
                    l *= alpha;
                    m = mb;
                }
                if (j > 0 && __any_sync(0xffffffffu, raise)) {
#pragma unroll 1
                    for (int c = 0; c < (int)kHalfCols / 16; ++c) {
                        uint32_t v[16];
                        tmem_ld_32x32b_x16(o_addr + c * 16, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
                        tmem_st_32x32b_x16(o_addr + c * 16, v);
                    }
                }
                const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t packed[16];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float4 gr = grp[2 * c + h];
                        const float y = gr.y - ms;
                        float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float p0 = fast_exp2(fmaf(sc[32 * c + 16 * h + 2 * i], gr.x, y));
                            const float p1 = fast_exp2(fmaf(sc[32 * c + 16 * h + 2 * i + 1], gr.x, y));
                            s4[(2 * i) & 3] += p0, s4[(2 * i + 1) & 3] += p1;
                            packed[8 * h + i] = pack_h2(p0, p1);
                        }
                        l = fmaf((s4[0] + s4[1]) + (s4[2] + s4[3]), gr.z, l);
                    }
                    tmem_st_32x32b_x16(s_addr + half * (kHalfKeys / 2) + 16 * c, packed);
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + t2);
                // the other half has read row_max before it arrives at the next block's tile_sync, and that one writes after
                // s_full, which follows both halves' arrivals here
            }
            // ---- the item's end: O / l, or partial sums of an item that other CTAs share ----
            if (live) {
                mbar_wait(o_full + t2, on++ & 1u, abort, a.err);
                tc_fence_after();
                row_sum[half * 128] = l;
                tile_sync();
                l = row_sum[0] + row_sum[128];
                if (l == 0.f && mine) l = no_weight(a, k.v, k.kvh, k.row0 + rr, DH, b0 * kTlKeys);
                tile_sync();      // read before the next item's Q goes there
            }
            const bool whole = b0 == 0 && nb == k.blocks;
            const uint32_t slot = 2 * blockIdx.x + (b0 == 0 ? 1 : 0);
            constexpr size_t kSlot = (size_t)kTlItem * (DH + 2);
            float *po = a.part + slot * kSlot, *pm = po + kTlItem * DH, *pl = pm + kTlItem;      // [DH][256], [256], [256]
            __half *op = a.o + (size_t)(k.v.qs + qi) * a.ldo + ((size_t)k.kvh * a.G + gi) * DH + half * kHalfCols;
            auto write_out = [&](const float (&y)[16], int c, float inv) {
                if (a.vec_o) {
#pragma unroll
                    for (int q = 0; q < 2; ++q)
                        *reinterpret_cast<uint4 *>(op + c * 16 + q * 8) =
                            make_uint4(pack_h2(y[8 * q] * inv, y[8 * q + 1] * inv), pack_h2(y[8 * q + 2] * inv, y[8 * q + 3] * inv),
                                       pack_h2(y[8 * q + 4] * inv, y[8 * q + 5] * inv),
                                       pack_h2(y[8 * q + 6] * inv, y[8 * q + 7] * inv));
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) op[c * 16 + i] = __float2half_rn(y[i] * inv);
                }
            };
            if (live) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 2
                for (int c = 0; c < (int)kHalfCols / 16; ++c) {
                    uint32_t v[16];
                    float y[16];
                    tmem_ld_32x32b_x16(o_addr + c * 16, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 16; ++i) y[i] = __uint_as_float(v[i]);
                    if (mine) {
                        if (whole) {
                            write_out(y, c, inv);
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; ++i) po[(size_t)(half * kHalfCols + c * 16 + i) * kTlItem + rr] = y[i];
                        }
                    }
                }
                tc_fence_before();
                if (mine && !whole && half == 0) pm[rr] = m, pl[rr] = l;
            }
            if (!whole) {
                const u64 i0 = u - b0;      // the item's first unit: its CTA counts the arrivals
                const uint32_t c0 = (uint32_t)(i0 / per), c1 = (uint32_t)((i0 + k.blocks - 1) / per);
                all_sync();
                if (st == 0) {
                    const uint32_t before = atom_add_acq_rel_gpu(a.counters + c0, 1u);
                    mi.flag = before == c1 - c0;
                    if (mi.flag) a.counters[c0] = 0;      // for the next call
                }
                all_sync();
                if (mi.flag && mine) {
                    const uint32_t parts = c1 - c0 + 1;
                    auto part = [&](uint32_t i) { return a.part + (size_t)(2 * (c0 + i) + (i == 0)) * kSlot; };
                    float mt = -INFINITY, lt = 0.f;
#pragma unroll 4
                    for (uint32_t i = 0; i < parts; ++i) mt = fmaxf(mt, __ldcg(part(i) + kTlItem * DH + rr));
#pragma unroll 4
                    for (uint32_t i = 0; i < parts; ++i) {
                        const float mi2 = __ldcg(part(i) + kTlItem * DH + rr);
                        const float li = __ldcg(part(i) + kTlItem * DH + kTlItem + rr);
                        lt = fmaf(li, mi2 == -INFINITY ? 0.f : fast_exp2(mi2 - mt), lt);
                    }
                    const float inv = lt == 0.f ? 0.f : 1.f / lt;
                    float f[4];      // factors of the first parts; more are rare
#pragma unroll
                    for (uint32_t p = 0; p < 4; ++p) {
                        const float mp = p < parts ? __ldcg(part(p) + kTlItem * DH + rr) : -INFINITY;
                        f[p] = mp == -INFINITY ? 0.f : fast_exp2(mp - mt);
                    }
#pragma unroll 2
                    for (int c = 0; c < (int)kHalfCols / 16; ++c) {
                        float y[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) y[i] = 0.f;
                        const size_t at = (size_t)(half * kHalfCols + c * 16) * kTlItem + rr;
#pragma unroll
                        for (uint32_t p = 0; p < 4; ++p) {
                            if (p >= parts) continue;
                            const float *src = part(p) + at;
#pragma unroll
                            for (int i = 0; i < 16; ++i) y[i] = fmaf(__ldcg(src + i * kTlItem), f[p], y[i]);
                        }
                        for (uint32_t p = 4; p < parts; ++p) {
                            const float mp = __ldcg(part(p) + kTlItem * DH + rr);
                            const float fp = mp == -INFINITY ? 0.f : fast_exp2(mp - mt);
                            const float *src = part(p) + at;
#pragma unroll
                            for (int i = 0; i < 16; ++i) y[i] = fmaf(__ldcg(src + i * kTlItem), fp, y[i]);
                        }
                        write_out(y, c, inv);
                    }
                }
            }
            u += nb;
            if (u < end) tile_next(k, a);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

constexpr size_t kCounterBytes = 16384;
constexpr uint32_t kMaxSms = 160;         // the grid is cut there, so that the workspace is
// Token numbers are int in the kernels, and they run ahead of a request's last token by up to 32 units of 256 when page ids are
// read, by a block of a tile, and by its new rows in a row's limit.
constexpr uint64_t kMaxTokens = (1ull << 31) - (1u << 14);

template <int DH, int NT, int NW, bool FP8>
cudaError_t launch_rows(KvArgs &a, const CUtensorMap &mkv, const CUtensorMap &mv, int sms, cudaStream_t st) {
    constexpr uint32_t kPerSm = (NT == 1 ? 16 : DH == 64 ? 12 : 8) / NW;
    static_assert(kMaxSms * kPerSm * 4 <= kCounterBytes &&
                      kCounterBytes + (size_t)2 * kPerSm * kMaxSms * 8 * NT * (DH + 2) * 4 <= SH_CUDA_KV8_WS_BYTES,
                  "workspace: a counter and two partial items per CTA");
    static_assert(kPerSm * (RowsSmem<DH, NT, NW>::kBytes + 1024) <= 228 * 1024, "shared memory of the CTAs of an SM");
    const cudaError_t e = sh::allow_smem<k_attn_kv8_rows<DH, NT, NW, FP8>>(RowsSmem<DH, NT, NW>::kBytes);
    if (e != cudaSuccess) return e;
    return sh::launch_pdl(k_attn_kv8_rows<DH, NT, NW, FP8>, dim3(sms * kPerSm), dim3(NW * 32), RowsSmem<DH, NT, NW>::kBytes, st,
                          mkv, mv, a);
}

template <int DH, bool FP8>
cudaError_t launch_tiles(KvArgs &a, const CUtensorMap &mk, const CUtensorMap &mv, int sms, cudaStream_t st) {
    static_assert(kCounterBytes + (size_t)2 * kMaxSms * kTlItem * (DH + 2) * 4 <= SH_CUDA_KV8_WS_BYTES,
                  "workspace: two partial items per CTA");
    constexpr auto kernel = k_attn_kv8_tiles<DH, FP8>;
    // the kernel hands registers from warp to warp: it has to start with as many as it ends with
    static_assert(512 * kTlRegs + (kTlThreads - 512) * kTlRegsOther <= kTlThreads * 80, "registers");
    static std::atomic<bool> enough[sh::kMaxDevices];
    std::atomic<bool> &ok = enough[sh::current_device() % sh::kMaxDevices];
    cudaError_t e = sh::allow_smem<kernel>(TilesSmem<DH>::kBytes);
    if (e != cudaSuccess) return e;
    if (!ok.load(std::memory_order_relaxed)) {
        cudaFuncAttributes at;
        e = cudaFuncGetAttributes(&at, kernel);
        if (e != cudaSuccess) return e;
        if (at.numRegs < 80) return cudaErrorInvalidDeviceFunction;
        ok.store(true, std::memory_order_relaxed);
    }
    return sh::launch_pdl(kernel, dim3(sms), dim3(kTlThreads), TilesSmem<DH>::kBytes, st, mk, mv, a);
}

// K or V codes as [pages, heads * page, dh] bytes: boxes of 16 tokens of one page and head
bool kv_map(CUtensorMap *m, uint64_t base, const sh_cuda_kv8_t *c) {
    sh::PFN_encodeTiled enc = sh::encode_tiled();
    if (!enc) return false;
    cuuint64_t dims[3] = {c->dh, (cuuint64_t)c->heads * c->page, c->pages};
    cuuint64_t strides[2] = {c->dh, c->page_stride};
    cuuint32_t box[3] = {c->dh, 16, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, (void *)base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               c->dh == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// K and V codes as [2, pages, heads * page, dh] bytes, the lower array first (one of them where both are the same array):
// boxes of 16 tokens of one page and head, of K and V at once; where pages allow it of the 32 tokens that a step takes.
// Arrays further apart than a map's stride can be (2^40 bytes: two allocators may use address ranges 2^46 apart) get a map each.
bool kv_pair_map(CUtensorMap *m, CUtensorMap *mv, const sh_cuda_kv8_t *c, KvArgs &a) {
    sh::PFN_encodeTiled enc = sh::encode_tiled();
    if (!enc) return false;
    const uint64_t lo = c->k < c->v ? c->k : c->v, hi = c->k < c->v ? c->v : c->k;
    const bool apart = hi - lo >= (1ull << 40);
    const uint32_t step = 2048 / c->dh, rows = step < c->page ? step : c->page, arrays = lo == hi ? 1 : 2;
    a.boxes = step / rows, a.box_bytes = arrays * rows * c->dh, a.box_step = a.boxes == 1 ? 16 * c->dh : 2048;
    a.k_at = c->k <= c->v || apart ? 0 : rows * c->dh, a.v_at = c->k < c->v || apart ? rows * c->dh : 0;
    a.apart = apart ? rows * c->dh : 0;
    auto map = [&](CUtensorMap *to, uint64_t base, uint32_t n) {
        cuuint64_t dims[4] = {c->dh, (cuuint64_t)c->heads * c->page, c->pages, n};
        cuuint64_t strides[3] = {c->dh, c->page_stride, n == 2 ? hi - lo : c->page_stride};
        cuuint32_t box[4] = {c->dh, rows, 1, n};
        cuuint32_t estr[4] = {1, 1, 1, 1};
        return enc(to, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, (void *)base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   c->dh == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    };
    return apart ? map(m, c->k, 1) && map(mv, c->v, 1) : map(m, lo, arrays);
}

}  // namespace

extern "C" {

int sh_cuda_attention_kv8(uint64_t q, uint64_t o, const sh_cuda_kv8_t *c, uint64_t table, uint32_t ld_table,
                          uint64_t lens, uint64_t q_start, uint32_t R, uint32_t T, uint32_t max_q, uint32_t H,
                          uint32_t ldq, uint32_t ldo, float scale, uint64_t ws, size_t ws_bytes) {
    const int bad = sh::kv8_check(c, "sh_cuda_attention_kv8");
    if (bad) return bad;
    if (H == 0 || H % c->heads || (uint64_t)H * c->dh > ldq || (uint64_t)H * c->dh > ldo ||
        (uint64_t)T * H >= (1ull << 31) || ld_table == 0 || T + (uint64_t)ld_table * c->page > kMaxTokens ||
        !(fabsf(scale) < INFINITY)) {
        sh::set_error(-1, "[sh_cuda_attention_kv8] need H a multiple of the cache's %u heads, ldq, ldo >= H dh, T H < 2^31, "
                      "T + ld_table page <= 2^31 - 2^14, a finite scale (H=%u ldq=%u ldo=%u T=%u ld_table=%u)", c->heads, H,
                      ldq, ldo, T, ld_table);
        return -1;
    }
    if (!ws || !sh::aligned16(ws) || ws_bytes < SH_CUDA_KV8_WS_BYTES) {
        sh::set_error(-1, "[sh_cuda_attention_kv8] workspace null, not 16-byte aligned, or less than %u bytes",
                      SH_CUDA_KV8_WS_BYTES);
        return -1;
    }
    if (R == 0 || T == 0) return 0;
    if (!q || !o || !table || !lens || !q_start || ((q | o) & 1) || !sh::words_ok(table, lens, q_start)) {
        sh::set_error(-1, "[sh_cuda_attention_kv8] a null or misaligned array");
        return -1;
    }
    const sh::DeviceState &s = sh::state();
    KvArgs a = {};
    a.q = (const __half *)q, a.o = (__half *)o;
    a.k = (const uint8_t *)c->k, a.v = (const uint8_t *)c->v;
    a.ks = (const float *)c->k_scale, a.vs = (const float *)c->v_scale;
    a.table = (const int *)table, a.lens = (const int *)lens, a.q_start = (const int *)q_start;
    a.page_stride = c->page_stride;
    a.ld_table = ld_table, a.R = R, a.T = T, a.G = H / c->heads, a.heads = c->heads, a.pages = c->pages;
    a.page_shift = sh::kv8_shift(c->page), a.ldq = ldq, a.ldo = ldo, a.sl2 = scale * 1.4426950408889634f;
    a.vec = sh::aligned16(q) && ldq % 8 == 0 && (o & 3) == 0 && ldo % 2 == 0;
    a.vec_o = sh::aligned16(o) && ldo % 8 == 0;
    a.counters = (uint32_t *)ws, a.part = (float *)(ws + kCounterBytes), a.err = s.dev_err;
    const int sms = s.num_sms < (int)kMaxSms ? s.num_sms : (int)kMaxSms;
    const bool fp8 = c->fmt == SH_FP8, wide = (uint64_t)max_q * a.G > 8;
    const bool tall = (uint64_t)max_q * a.G > 64;
    CUtensorMap mk, mv = {};
    if (tall ? !kv_map(&mk, c->k, c) || !kv_map(&mv, c->v, c) : !kv_pair_map(&mk, &mv, c, a)) {
        sh::set_error(-1, "[sh_cuda_attention_kv8] no tensor map for the cache (page_stride=%llu)",
                      (unsigned long long)c->page_stride);
        return -1;
    }
    cudaError_t e;
    // Eight warps per CTA (two CTAs per SM) where items are fewer than SMs and many CTAs share one: half as many partial sums
    // to join. Four warps (four CTAs) where a CTA walks several items: the others go on while one ends an item. 32 heads over 8
    // of 128, eight warps beside four: 131072 tokens of one request (8 items) 57 us and 64; up to 8192 tokens of 4 requests 19.5
    // and 21.7, of 8 (64 items) 27.7 and 28.6, of 16 (128) 40.5 and 40.3, of 19 (152) 48.8 and 43.9, of 64 123 and 115.
    const bool few = (uint64_t)R * c->heads < (uint64_t)sms;
#define SH_KV8(dh, nt, n) \
    (fp8 ? launch_rows<dh, nt, n, true>(a, mk, mv, sms, s.stream) : launch_rows<dh, nt, n, false>(a, mk, mv, sms, s.stream))
    // The kernel above takes a tile of 16 rows after the other, this one 256 at once. 16 requests of up to 8192 tokens, heads of 128:
    // 48 rows 106 us there and 127 here, 64 rows 136 and 128, 96 rows 179 and 131; 32 of up to 4000, heads of 64: 60 rows 56 and
    // 66, 72 rows 70 and 66; 4 of up to 8192: 96 rows 59 and 63, 128 rows 75 and 71; a single one is level from about 200 rows on.
    if (tall) {
        a.flip = scale < 0.f ? 0x80008000u : 0u;
        a.sl2 = fabsf(a.sl2);
        auto launch = c->dh == 64 ? (fp8 ? launch_tiles<64, true> : launch_tiles<64, false>)
                                  : (fp8 ? launch_tiles<128, true> : launch_tiles<128, false>);
        e = launch(a, mk, mv, sms, s.stream);
    } else if (c->dh == 64) e = wide ? SH_KV8(64, 2, 4) : few ? SH_KV8(64, 1, 8) : SH_KV8(64, 1, 4);
    else e = wide ? SH_KV8(128, 2, 4) : few ? SH_KV8(128, 1, 8) : SH_KV8(128, 1, 4);
#undef SH_KV8
    return sh::cuda_ok(e, "sh_cuda_attention_kv8") ? 0 : -1;
}

}  // extern "C"
