// Products of a few rows with 4-bit weights (sh_cuda_gemv_w4): Z[M, N] = X[M, K] W[K, N], W[k, n] = s (code - zero) with one
// scale and zero point per output column and group of 32, 64 or 128 k.
//
//     z[m, n] = sum_g s[n, g] sum_{k in g} (code[n, k] - zero[n, g]) x[m, k]
//
// Bound by the weights' bytes (half a byte per element, read once), and close behind by the instructions that turn codes
// into operands, so there are two forms of the inner product, both exact but for fp32 sums:
//   fp16   code - zero is a small integer, exact in fp16: the 16-row operand of the matrix instruction (16 columns of W x
//          16 k), 8 rows of X its columns, two or four times for more. 9 instructions turn a word into 8 operands (fp16
//          patterns 1024 + c and 1024 + 16 c, then one subtraction or FMA).
//   int8   for a single row and many columns: every finite fp16 value is an integer times 2^-24 below 2^41, i.e. six signed
//          base-256 digits. The codes are int8 operands as they are (3 instructions per 8), the digits of X are six of the
//          instruction's eight columns, of which a single row would leave seven empty, and the int32 sums of a group are
//          exact. The zero point enters as -zero sum(digits). A 16 x 128 step takes 4 matrix instructions and 24 others, not
//          8 and 72, but the digits take longer to lay out, so that it pays from about three tiles per SM on (K 4096, group
//          128, beside fp16: 2 tiles 6.1 and 5.5 us, 3 tiles 7.5 and 7.0, 3.5 tiles 7.9 and 8.2, 6 tiles 10.6 and 11.5, 49152
//          columns 23.9 and 30; K 2048 and 8192 cross between 3 and 4 tiles as well).
//          Infinities and NaN have no digits; outputs of such a row get those terms one by one.
//
// One CTA per SM: X is laid out in shared memory once, then groups of 8 warps walk tiles of 16 columns of W, each warp an
// eighth of K. A warp has its own ring of stages, filled by TMA boxes of 16 columns x 128 bytes with 128-byte swizzle (one
// instruction per step; per-lane copies cost the L1 one tag look-up per column instead, which bound an earlier
// form), without a barrier between warps. A lane reads the codes it needs as they lie: the order of k inside the matrix
// instruction is free when both operands agree. A tile's scales and zero points come as rows of 16 bytes, one tile
// ahead. When the columns alone do not fill the GPU, the CTAs of a cluster share K. All partial sums meet in shared
// memory in a fixed order.
#include "sh_internal.cuh"

namespace {

constexpr uint32_t kUnit = 256;   // k per step of a warp
constexpr uint32_t kMaxK = 1u << 18;   // one row of X over the CTAs of the largest cluster

struct W4Args {
    const __half *x, *scales, *bias, *res;
    const uint8_t *codes, *zeros;
    __half *z;
    uint32_t M, N, K, ldx, ldw, ldz, ldr, vec;
    uint32_t staged;      // a tile's scales and zero points can be copied whole
    int *err;
};

__device__ __forceinline__ void w4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t w4_sub(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t w4_fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
// (a & b) | c in one instruction (written in C, the two constants make it two)
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
// codes 0 .. 7 of a word minus the zero point, as the pairs (0, 4), (1, 5), (2, 6), (3, 7)
__device__ __forceinline__ void w4_word(uint32_t w, uint32_t zlo, uint32_t zhi, uint32_t (&h)[4]) {
    constexpr uint32_t kSixteenth = 0x2C002C00u;
    const uint32_t v = w >> 8;
    h[0] = w4_sub(and_or(w, 0x000F000Fu, 0x64006400u), zlo);
    h[1] = w4_fma(and_or(w, 0x00F000F0u, 0x64006400u), kSixteenth, zhi);
    h[2] = w4_sub(and_or(v, 0x000F000Fu, 0x64006400u), zlo);
    h[3] = w4_fma(and_or(v, 0x00F000F0u, 0x64006400u), kSixteenth, zhi);
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}
// N words from shared memory in one instruction (N 1, 2 or 4)
template <int N>
__device__ __forceinline__ void load_shared(uint32_t (&w)[N], uint32_t at) {
    if constexpr (N == 1) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(at) : "memory");
    else if constexpr (N == 2) asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
    else
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
}

// In each half of a step (128 k), word i of lane column c holds 8 codes from k = 32 c + 8 i (group 128), 64 (i / 2) + 16 c
// + 8 (i % 2) (group 64) or 32 i + 8 c (group 32): all lanes of a matrix instruction are in one group.
// Row g of the matrix instruction is row tile_row(g) of the tile, row g + 8 the one 8 further: the two rows that a quarter
// of a warp reads at once then lie in different halves of the 128-byte swizzle.
__device__ __forceinline__ uint32_t tile_row(uint32_t g) { return (g >> 1) | (g & 1) << 2; }

constexpr uint32_t kGroupWarps = 8, kGroupThreads = 256, kStage = 16 * kUnit / 2;
constexpr int kDigits = 6;
constexpr uint32_t kRows = 16;      // columns of W per tile

// x 2^24 as six signed base-256 digits: bytes of value + 0x808080808080, each less 128
__device__ __forceinline__ void digits_of(uint32_t h, uint32_t &lo, uint32_t &hi) {
    const uint32_t e = (h >> 10) & 31u;
    const uint32_t m = (h & 1023u) | (e ? 1024u : 0u), sh = e ? e - 1 : 0;
    unsigned long long v = (unsigned long long)m << sh;
    if (e == 31) v = 0;
    v = 0x808080808080ull + ((h & 0x8000u) ? 0ull - v : v);
    lo = (uint32_t)v ^ 0x80808080u;
    hi = (uint32_t)(v >> 32) ^ 0x8080u;
}

__device__ __forceinline__ void w4_imma(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// integer below 2^22 in magnitude -> float, without the conversion unit
__device__ __forceinline__ float small_to_float(int v) { return __int_as_float(v + 0x4B400000) - 12582912.f; }

struct W4Layout {     // offsets into shared memory
    uint32_t red, part, zero, flag, bars, sc, sc_bytes, xs, x, bytes;
};
// nt: groups of 8 columns of the matrix instruction; steps: of one CTA; gu: quantisation groups per step;
// groups: of the scales kept; iters: tiles of one group of warps whose sums are kept
__host__ __device__ inline W4Layout w4_layout(uint32_t ng, uint32_t d, uint32_t nt, uint32_t gu, bool digits,
                                              bool zeros, uint32_t steps, uint32_t m, uint32_t groups, uint32_t iters) {
    W4Layout l;
    uint32_t at = ng * kGroupWarps * d * kStage;
    l.red = at, at += (nt == 1 ? 2 : 1) * ng * kGroupWarps * 8 * nt * 16 * 4;
    l.part = at, at += ng * iters * 16 * m * 4;
    l.zero = at, at += 64;
    l.flag = at, at += 16;
    l.bars = at, at += ng * (kGroupWarps * d + 2) * 8 + 16;            // and the abort flag
    l.sc_bytes = 16 * groups * (zeros ? 3 : 2);
    l.sc = at, at += 2 * ng * l.sc_bytes;
    l.xs = at, at += digits ? steps * gu * 8 * 4 : 0;
    l.x = at, at += steps * (digits ? 4 * kDigits * 64 : 8 * m * 64);
    l.bytes = at + 1024;       // the ring starts on a multiple of 1024
    return l;
}

// INT: digits (M == 1); NT: groups of 8 columns of the matrix instruction; NG: groups of 8 warps; D: stages; Z: zero points
// given
template <int G, bool INT, int NT, int NG, int D, bool Z>
__global__ void __launch_bounds__(NG * kGroupThreads, 1)
    k_gemv_w4(const __grid_constant__ CUtensorMap mw, W4Args a, uint32_t splits, uint32_t tiles, uint32_t iters) {
    constexpr uint32_t kThreads = NG * kGroupThreads, kCols = 8 * NT;
    constexpr int GU = kUnit / G;                                  // quantisation groups per step
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5, g = lane >> 2, c = lane & 3;
    const uint32_t grp = warp / kGroupWarps, gw = warp % kGroupWarps, gt = t % kGroupThreads;
    const uint32_t units = (a.K + kUnit - 1) / kUnit, groups = a.K / G;
    const uint32_t parts = splits * kGroupWarps, part = blockIdx.y * kGroupWarps + gw;
    auto border = [&](uint32_t p) { return (uint32_t)((uint64_t)units * p / parts); };
    const uint32_t u0 = border(part), nu = border(part + 1) - u0;                    // steps of this warp per tile
    const uint32_t x0 = border(blockIdx.y * kGroupWarps), x1 = border((blockIdx.y + 1) * kGroupWarps);   // of this CTA
    const uint32_t xcols = INT ? kDigits * a.M : a.M;
    const W4Layout L = w4_layout(NG, D, NT, GU, INT, Z, (units + splits - 1) / splits + 1, a.M, a.staged ? groups : 0,
                                 iters);
    // tiles of this group: the first ones of all SMs before any SM's second ones
    const uint32_t tile0 = grp * gridDim.x + blockIdx.x, tile_step = NG * gridDim.x;

    uint64_t *full = reinterpret_cast<uint64_t *>(smem + L.bars) + warp * D;
    uint64_t *sc_full = reinterpret_cast<uint64_t *>(smem + L.bars) + NG * kGroupWarps * D + grp * 2;
    volatile int *abort = reinterpret_cast<volatile int *>(smem + L.bars + NG * (kGroupWarps * D + 2) * 8);
    if (lane == 0) {
#pragma unroll
        for (int d = 0; d < D; ++d) mbar_init(full + d, 1);
        if (gw == 0) mbar_init(sc_full, 1), mbar_init(sc_full + 1, 1);
    }
    if (t == 0) *abort = 0, prefetch_tmap(&mw);
    fence_mbar_init();
    fence_proxy_async_smem();
    __syncwarp();
    pdl_launch_dependents();
    pdl_wait();

    // ---- the stream of this warp's steps, D ahead ----------------------------------------------------------------------
    uint8_t *ring = smem + warp * (D * kStage);
    uint32_t p_tile = nu ? tile0 : tiles, p_left = nu, p_slot = 0;
    auto issue = [&]() {
        if (p_tile >= tiles) return;
        if (lane == 0) {
            mbar_arrive_expect_tx(full + p_slot, kStage);
            tma_load_2d(ring + p_slot * kStage, &mw, full + p_slot, (int)((u0 + nu - p_left) * (kUnit / 2)),
                        (int)(p_tile * kRows));
        }
        p_slot = p_slot + 1 == D ? 0 : p_slot + 1;
        if (--p_left == 0) p_left = nu, p_tile += tile_step;
    };
#pragma unroll
    for (int d = 0; d < D; ++d) issue();

    // ---- scales and zero points of a tile, one tile ahead: its rows lie together. A last tile of
    // fewer rows, and arrays that are too long or not 16-byte aligned, are read where they lie.
    const uint32_t sc0 = smem_u32(smem) + L.sc + grp * 2 * L.sc_bytes;
    auto staged = [&](uint32_t tile) { return a.staged && tile * kRows + kRows <= a.N; };
    auto fetch_scales = [&](uint32_t tile, uint32_t turn) {
        if (gt == 0 && tile < tiles && staged(tile)) {
            mbar_arrive_expect_tx(sc_full + turn, L.sc_bytes);
            bulk_load(sc0 + turn * L.sc_bytes, a.scales + (size_t)tile * kRows * groups, 2 * kRows * groups, sc_full + turn);
            if (Z)
                bulk_load(sc0 + turn * L.sc_bytes + 2 * kRows * groups, a.zeros + (size_t)tile * kRows * groups, kRows * groups,
                          sc_full + turn);
        }
    };
    fetch_scales(tile0, 0);
    fetch_scales(tile0 + tile_step, 1);

    // ---- X in the order of the operands ------------------------------------------------------------------------------
    uint4 *s_x = reinterpret_cast<uint4 *>(smem + L.x);
    int *s_xs = reinterpret_cast<int *>(smem + L.xs);
    int *s_flag = reinterpret_cast<int *>(smem + L.flag);      // INT: the row has infinities or NaN
    if (t == 0) *s_flag = 0;
    if (t < 16) reinterpret_cast<uint32_t *>(smem + L.zero)[t] = 0;
    if (INT)
        for (uint32_t i = t; i < (x1 - x0) * GU * kCols; i += kThreads) s_xs[i] = 0;
    __syncthreads();
    const uint32_t per_row = (x1 - x0) * 32;      // pieces of 8 neighbouring k in this CTA's steps
    constexpr uint32_t kBatch = INT ? 1 : 4;      // pieces per thread in flight
    for (uint32_t p0 = t; p0 < per_row * a.M; p0 += kBatch * kThreads) {
        uint32_t xs[kBatch][4];
#pragma unroll
        for (uint32_t q = 0; q < kBatch; ++q) {
            const uint32_t p = p0 + q * kThreads, m = p / per_row, at = x0 * kUnit + (p - m * per_row) * 8;
            uint32_t (&x)[4] = xs[q];
            x[0] = x[1] = x[2] = x[3] = 0;
            if (p < per_row * a.M && at < a.K) {
                const __half *xp = a.x + (size_t)m * a.ldx + at;
                if (a.vec) {
                    const uint4 v = __ldcg(reinterpret_cast<const uint4 *>(xp));      // once per CTA: past the L1
                    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e >> 1] |= (uint32_t)__half_as_ushort(xp[e]) << (16 * (e & 1));
                }
            }
        }
#pragma unroll
        for (uint32_t q = 0; q < kBatch; ++q) {
            const uint32_t p = p0 + q * kThreads, m = p / per_row, i = p - m * per_row;
            if (p >= per_row * a.M) continue;
            // word ii of column cc in half u of the CTA's steps
            const uint32_t u = i >> 4, j = i & 15;
            const uint32_t cc = G == 128 ? j >> 2 : G == 64 ? (j >> 1) & 3 : j & 3;
            const uint32_t ii = G == 128 ? j & 3 : G == 64 ? (j >> 3) * 2 + (j & 1) : j >> 2;
            const uint32_t (&x)[4] = xs[q];
            if (!INT) {
                // pairs (0, 4), (1, 5), (2, 6), (3, 7) as w4_word's; [half][word][row][c]
                s_x[((u * 4 + ii) * a.M + m) * 4 + cc] =
                    make_uint4(__byte_perm(x[0], x[2], 0x5410), __byte_perm(x[0], x[2], 0x7632),
                               __byte_perm(x[1], x[3], 0x5410), __byte_perm(x[1], x[3], 0x7632));
            } else {
                // digits of k 0, 2, 4, 6 and of k 1, 3, 5, 7; [half][word pair][column][c][word of the pair]
                bool special = false;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    special |= (x[e] & 0x7C00u) == 0x7C00u || (x[e] & 0x7C000000u) == 0x7C000000u;
                if (special) *s_flag = 1;
                uint32_t d[2][kDigits];
#pragma unroll
                for (int odd = 0; odd < 2; ++odd) {
                    uint32_t lo[4], hi[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) digits_of(odd ? x[e] >> 16 : x[e] & 0xFFFFu, lo[e], hi[e]);
                    const uint32_t p0 = __byte_perm(lo[0], lo[1], 0x5140), p1 = __byte_perm(lo[2], lo[3], 0x5140);
                    const uint32_t p2 = __byte_perm(lo[0], lo[1], 0x7362), p3 = __byte_perm(lo[2], lo[3], 0x7362);
                    const uint32_t p4 = __byte_perm(hi[0], hi[1], 0x5140), p5 = __byte_perm(hi[2], hi[3], 0x5140);
                    d[odd][0] = __byte_perm(p0, p1, 0x5410), d[odd][1] = __byte_perm(p0, p1, 0x7632);
                    d[odd][2] = __byte_perm(p2, p3, 0x5410), d[odd][3] = __byte_perm(p2, p3, 0x7632);
                    d[odd][4] = __byte_perm(p4, p5, 0x5410), d[odd][5] = __byte_perm(p4, p5, 0x7632);
                }
                const uint32_t grp_q = G == 128 ? 0 : G == 64 ? ii >> 1 : ii;
#pragma unroll
                for (int k = 0; k < kDigits; ++k) {
                    uint2 *dst = reinterpret_cast<uint2 *>(s_x + ((u * 2 + (ii >> 1)) * kDigits + k) * 4 + cc) + (ii & 1);
                    *dst = make_uint2(d[0][k], d[1][k]);
                    const int sum = __dp4a((int)d[0][k], 0x01010101, __dp4a((int)d[1][k], 0x01010101, 0));
                    if (sum) atomicAdd(s_xs + (u * (GU / 2) + grp_q) * kCols + k, sum);
                }
            }
        }
    }
    __syncthreads();

    // this lane's operand column of X; the zero line where X has none
    constexpr uint32_t kPieces = INT ? 4 : 8;        // 16-byte pieces of a step per lane
    uint32_t bx[NT], bstep[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const bool has = nt * 8 + g < xcols;
        bx[nt] = smem_u32(smem) + (has ? L.x + (((u0 - x0) * kPieces * xcols + nt * 8 + g) * 4 + c) * 16 : L.zero);
        bstep[nt] = has ? xcols * 64 : 0;
    }
    float *s_red0 = reinterpret_cast<float *>(smem + L.red) + grp * ((NT == 1 ? 2 : 1) * kGroupWarps * kCols * kRows);
    // INT: the quad's columns are digits of one value, and only their sum goes through shared memory
    const float weight = __int_as_float((127 - 24 + 16 * (int)min(c, 2u)) << 23);
    float *s_part = reinterpret_cast<float *>(smem + L.part) + grp * iters * kRows * a.M;
    auto group_sync = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(grp + 1), "n"(kGroupThreads) : "memory"); };
    auto finish = [&](float v, uint32_t m, uint32_t n, bool special, float bias, float res) {
        if (INT && special)
            for (uint32_t k = 0; k < a.K; ++k) {
                const float x = __half2float(a.x[(size_t)m * a.ldx + k]);
                if (!(fabsf(x) < INFINITY)) {
                    const uint32_t code = a.codes[(size_t)n * a.ldw + k / 2] >> (4 * (k & 1)) & 15u;
                    const uint32_t zero = Z ? a.zeros[(size_t)n * groups + k / G] & 15u : 8u;
                    v = fmaf(((float)code - (float)zero) * __half2float(a.scales[(size_t)n * groups + k / G]), x, v);
                }
            }
        v += bias;
        v += res;
        a.z[(size_t)m * a.ldz + n] = __float2half_rn(v);
    };

    auto bias_of = [&](uint32_t n) { return a.bias ? __half2float(a.bias[n]) : 0.f; };
    auto res_of = [&](uint32_t m, uint32_t n) { return a.res ? __half2float(a.res[(size_t)m * a.ldr + n]) : 0.f; };
    // The outputs of a thread in each tile: one, or two sixteen rows apart. A single row's sixteen go to the warps in turn.
    constexpr int kOut = NT > 2 ? 2 : 1;
    const uint32_t om = INT ? 0 : gt / kRows, orow = gt % kRows;

    const uint32_t swz = tile_row(g), w_at = smem_u32(ring) + swz * 128;
    uint32_t slot = 0, phase = 0, iter = 0;
    for (uint32_t tile = tile0; tile < tiles; tile += tile_step, ++iter) {
        const uint32_t turn = iter & 1;
        float acc[NT][4];
        uint32_t bat[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f, bat[nt] = bx[nt];
        const int *xs = s_xs + (u0 - x0) * GU * kCols + 2 * c;
        // what the output adds is on its way while the products are taken
        const uint32_t on = tile * kRows + orow;
        bool mine[kOut], writes[kOut];
        float bias[kOut], res[kOut];
#pragma unroll
        for (int e = 0; e < kOut; ++e) {
            mine[e] = INT ? gw == (iter & 7) && lane < kRows : om + 16 * e < a.M;
            writes[e] = mine[e] && on < a.N && splits == 1;
            bias[e] = writes[e] ? bias_of(on) : 0.f, res[e] = writes[e] ? res_of(om + 16 * e, on) : 0.f;
        }
        const bool in_smem = staged(tile);
        const uint32_t sat = sc0 + turn * L.sc_bytes + 2 * (swz * groups + u0 * GU);
        const uint32_t zat = sc0 + turn * L.sc_bytes + 2 * kRows * groups + swz * groups + u0 * GU;
        if (in_smem && !mbar_try_wait(sc_full + turn, iter >> 1 & 1)) mbar_wait(sc_full + turn, iter >> 1 & 1, abort, a.err);
#pragma unroll 1
        for (uint32_t u = 0; u < nu; ++u, xs += GU * kCols) {
            if (!mbar_try_wait(full + slot, phase)) mbar_wait(full + slot, phase, abort, a.err);
            const uint32_t at = w_at + slot * kStage;
            slot = slot + 1 == D ? 0 : slot + 1;
            phase ^= slot == 0;
            // scales and zero points of the step's groups; 0 past K, where codes and operands of X are zeros too
            float s[2][GU];       // rows swz, swz + 8 of the tile
            uint32_t z[2][GU];
            if (in_smem) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint32_t h[GU / 2], y[(GU + 3) / 4];
                    load_shared<GU / 2>(h, sat + e * 16 * groups + u * 2 * GU);
                    if (Z) {
                        const uint32_t at_z = zat + e * 8 * groups + u * GU;
                        if (GU == 2) asm volatile("ld.shared.u16 %0, [%1];" : "=r"(y[0]) : "r"(at_z) : "memory");
                        else load_shared<(GU + 3) / 4>(y, at_z);
                    }
#pragma unroll
                    for (int q = 0; q < GU; ++q) {
                        s[e][q] = __half2float(__ushort_as_half((uint16_t)(h[q / 2] >> (16 * (q & 1)))));
                        z[e][q] = Z ? y[q / 4] >> (8 * (q & 3)) & 15u : 8u;
                    }
                }
            } else {
                const uint32_t q0 = (u0 + u) * GU;
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int q = 0; q < GU; ++q) {
                        const size_t i = (size_t)min(tile * kRows + swz + 8 * e, a.N - 1) * groups + min(q0 + q, groups - 1);
                        s[e][q] = q0 + q < groups ? __half2float(a.scales[i]) : 0.f;
                        z[e][q] = Z ? a.zeros[i] & 15u : 8u;
                    }
            }
            constexpr int kPer = 4 / (GU / 2);        // words per quantisation group
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t w[2][4];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    // 16-byte piece p of row r lies at piece p ^ (r % 8): the row's part of the address is in `at`
                    const uint32_t row = at + e * 1024;
                    if (G == 128) {
                        load_shared<4>(w[e], row + ((half * 4 + c) ^ swz) * 16);
                    } else if (G == 64) {
#pragma unroll
                        for (uint32_t q = 0; q < 2; ++q) {
                            uint32_t v[2];
                            load_shared<2>(v, row + ((half * 4 + 2 * q + (c >> 1)) ^ swz) * 16 + (c & 1) * 8);
                            w[e][2 * q] = v[0], w[e][2 * q + 1] = v[1];
                        }
                    } else {
#pragma unroll
                        for (uint32_t q = 0; q < 4; ++q) {
                            uint32_t v[1];
                            load_shared<1>(v, row + ((half * 4 + q) ^ swz) * 16 + c * 4);
                            w[e][q] = v[0];
                        }
                    }
                }
                int gi[4];        // sums of a quantisation group: INT
                float gf[NT][4];  // or fp16
                uint32_t b[NT][4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int q = half * (GU / 2) + i / kPer;
                    const int z0 = (int)z[0][q], z1 = (int)z[1][q];
                    if (i % kPer == 0) {
                        if (INT) {
                            const int2 y = *reinterpret_cast<const int2 *>(xs + q * kCols);
                            gi[0] = -z0 * y.x, gi[1] = -z0 * y.y, gi[2] = -z1 * y.x, gi[3] = -z1 * y.y;
                        } else {
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) gf[nt][0] = gf[nt][1] = gf[nt][2] = gf[nt][3] = 0.f;
                        }
                    }
                    if (!INT || i % 2 == 0)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            load_shared<4>(b[nt], bat[nt]);
                            bat[nt] += bstep[nt];
                        }
                    if (INT) {
                        const uint32_t a0 = w[0][i] & 0x0F0F0F0Fu, a2 = (w[0][i] >> 4) & 0x0F0F0F0Fu;
                        const uint32_t a1 = w[1][i] & 0x0F0F0F0Fu, a3 = (w[1][i] >> 4) & 0x0F0F0F0Fu;
                        w4_imma(gi, a0, a1, a2, a3, b[0][i % 2 * 2], b[0][i % 2 * 2 + 1]);
                    } else {
                        uint32_t h0[4], h1[4];
                        const uint32_t y0 = (uint32_t)z0 * 0x00010001u, y1 = (uint32_t)z1 * 0x00010001u;
                        w4_word(w[0][i], 0x64006400u | y0, 0xD400D400u | y0 << 4, h0);
                        w4_word(w[1][i], 0x64006400u | y1, 0xD400D400u | y1 << 4, h1);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            w4_mma(gf[nt], h0[0], h1[0], h0[1], h1[1], b[nt][0], b[nt][1]);
                            w4_mma(gf[nt], h0[2], h1[2], h0[3], h1[3], b[nt][2], b[nt][3]);
                        }
                    }
                    if (i % kPer == kPer - 1) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                acc[nt][e] = fmaf(INT ? small_to_float(gi[e]) : gf[nt][e], s[e >> 1][q], acc[nt][e]);
                    }
                }
            }
            __syncwarp();
            issue();      // into the stage just read
        }

        // ---- partial sums of the K parts, in their order. With two buffers one is written again two tiles later, behind the
        // barrier of the tile between, which no warp passes before all have read it; one buffer takes a second barrier. -----
        float *s_red = s_red0 + (NT == 1 ? turn : 0) * (kGroupWarps * kCols * kRows);
        if (INT) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float v = c < 3 ? fmaf(acc[0][2 * e + 1], 256.f, acc[0][2 * e]) * weight : 0.f;
                v += __shfl_xor_sync(0xffffffffu, v, 1);
                v += __shfl_xor_sync(0xffffffffu, v, 2);
                if (c == 0) s_red[gw * kRows + swz + 8 * e] = v;
            }
        } else {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    s_red[(gw * kCols + nt * 8 + 2 * c + (e & 1)) * kRows + swz + 8 * (e >> 1)] = acc[nt][e];
        }
        fence_proxy_async_smem();      // this tile's scales have been read: their buffer is copied into again
        group_sync();
        fetch_scales(tile + 2 * tile_step, turn);
#pragma unroll
        for (int e = 0; e < kOut; ++e) {
            const uint32_t m = om + 16 * e;
            float v = 0.f;
            if (mine[e]) {
#pragma unroll
                for (uint32_t w = 0; w < kGroupWarps; ++w) v += s_red[INT ? w * kRows + orow : (w * kCols + m) * kRows + orow];
            }
            if (splits > 1) {
                if (mine[e]) s_part[(iter * a.M + m) * kRows + orow] = v;
            } else if (writes[e]) {
                finish(v, m, on, *s_flag, bias[e], res[e]);
            }
        }
        if (NT > 1) group_sync();
    }
    if (*abort)      // a copy did not arrive in time: give those in flight as long again
    {
        for (int d = 0; d < D; ++d) drain_wait(full + d, phase ^ (d < (int)slot));
        for (uint32_t i = iter > 2 ? iter - 2 : 0; a.staged && i < iter; ++i) drain_wait(sc_full + (i & 1), i >> 1 & 1);
    }
    if (splits > 1) {
        cluster_sync_all();
        iter = 0;
        for (uint32_t tile = tile0; tile < tiles; tile += tile_step, ++iter)
            for (uint32_t i = blockIdx.y * kGroupThreads + gt; i < kRows * a.M; i += splits * kGroupThreads) {
                const uint32_t m = i / kRows, n = tile * kRows + i % kRows;
                if (n >= a.N) continue;
                const uint32_t at = smem_u32(s_part + iter * kRows * a.M + i), fat = smem_u32(s_flag);
                float v = 0.f;
                int special = 0;
                for (uint32_t k = 0; k < splits; ++k) {
                    float y;
                    int f;
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(y) : "r"(mapa_shared(at, k)) : "memory");
                    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(f) : "r"(mapa_shared(fat, k)) : "memory");
                    v += y;
                    special |= f;
                }
                finish(v, m, n, special != 0, bias_of(n), res_of(m, n));
            }
        cluster_sync_all();      // the other CTAs have read this one's sums
    }
}

// the codes as [N, K / 2] bytes: 16 columns of W x 128 bytes per box, zeros past N and K
bool w4_map(CUtensorMap *m, uint64_t codes, uint32_t N, uint32_t K, uint32_t ldw) {
    sh::PFN_encodeTiled enc = sh::encode_tiled();
    if (!enc) return false;
    cuuint64_t dims[2] = {K / 2, N};
    cuuint64_t strides[1] = {ldw};
    cuuint32_t box[2] = {kUnit / 2, 16};
    cuuint32_t estr[2] = {1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void *)codes, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
           CUDA_SUCCESS;
}

constexpr size_t kSmemMax = 227 * 1024, kMaxScales = 64 * 1024;

// Clusters of s CTAs (one per SM) of a kernel that run at once: the GPU's SMs come in groups that a cluster does not cross, so
// there are fewer than num_sms / s of them (33 of 4, not 37), and one more would be a second wave. Asked once per kernel and
// device; when the runtime gives no answer the next call asks again.
template <auto Kernel>
uint32_t w4_clusters(uint32_t threads, uint32_t s, uint32_t sms) {
    if (s == 1) return sms;
    static std::atomic<uint32_t> known[sh::kMaxDevices][9];      // s is 2, 4 or 8
    std::atomic<uint32_t> &k = known[sh::current_device() % sh::kMaxDevices][s];
    const uint32_t n = k.load(std::memory_order_relaxed);
    if (n) return n;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1, s), cfg.blockDim = dim3(threads), cfg.dynamicSmemBytes = kSmemMax;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1, attr[0].val.clusterDim.y = s, attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    int got = 0;
    if (cudaOccupancyMaxActiveClusters(&got, Kernel, &cfg) != cudaSuccess || got <= 0) {
        cudaGetLastError();
        return sms / s;
    }
    const uint32_t most = (uint32_t)got < sms / s ? (uint32_t)got : sms / s;
    k.store(most, std::memory_order_relaxed);
    return most;
}

template <int G, bool INT, int NT, int NG, int D>
cudaError_t w4_try(W4Args a, const CUtensorMap &mw, int sms, cudaStream_t st, bool &fits, uint32_t most = 8) {
    const uint32_t tiles = (a.N + 15) / 16, units = (a.K + kUnit - 1) / kUnit;
    uint32_t s = 1, room, iters;
    size_t smem;
    // Scales copied whole, the tile's before they are needed: 16 rows of 14336 x 4096, group 128, 19.4 us, 21.1 read where they lie.
    // At long K and group 128 their room costs X further pieces: 8 rows of 8192 x 28672 110 us, 63 without.
    // K parts over a cluster while the columns alone leave SMs idle and every warp keeps a step, or until X fits
    a.staged = (((uint64_t)a.scales | (uint64_t)a.zeros) & 15) == 0 && a.K % kUnit == 0 && a.K / G * 96 <= kMaxScales / NG;
    auto kernel = a.zeros ? k_gemv_w4<G, INT, NT, NG, D, true> : k_gemv_w4<G, INT, NT, NG, D, false>;
    const cudaError_t e = a.zeros ? sh::allow_smem<k_gemv_w4<G, INT, NT, NG, D, true>>(kSmemMax)
                                  : sh::allow_smem<k_gemv_w4<G, INT, NT, NG, D, false>>(kSmemMax);
    if (e != cudaSuccess) return e;
    for (;; s *= 2) {
        room = a.zeros ? w4_clusters<k_gemv_w4<G, INT, NT, NG, D, true>>(NG * kGroupThreads, s, (uint32_t)sms)
                       : w4_clusters<k_gemv_w4<G, INT, NT, NG, D, false>>(NG * kGroupThreads, s, (uint32_t)sms);
        const uint32_t ctas = tiles < room ? tiles : room;
        iters = s > 1 ? (tiles + ctas * NG - 1) / (ctas * NG) : 0;      // sums kept for the cluster
        smem = w4_layout(NG, D, NT, kUnit / G, INT, a.zeros != nullptr, (units + s - 1) / s + 1, a.M,
                         a.staged ? a.K / G : 0, iters).bytes;
        if (s == most || !((tiles * s * 2 <= (uint32_t)sms && units >= kGroupWarps * s * 2) || smem > kSmemMax)) break;
    }
    fits = smem <= kSmemMax;
    if (!fits) return cudaSuccess;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles < room ? tiles : room, s);
    cfg.blockDim = dim3(NG * kGroupThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = sh::pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1, attr[1].val.clusterDim.y = s, attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = s > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, mw, a, s, tiles, iters);
}

// Rows of X go in one piece, or in pieces of at most 16 and fewer when they do not fit beside each other (eight for 32
// rows of 8192 x 28672 in groups of 128). A second piece finds the weights in L2 unless they are larger than that.
template <int G>
cudaError_t w4_run(W4Args a, const CUtensorMap &mw, int sms, cudaStream_t st, bool &fits) {
    cudaError_t e = cudaSuccess;
    fits = false;
    const uint32_t tiles = (a.N + 15) / 16;
    if (a.M == 1 && tiles >= 3u * sms) e = w4_try<G, true, 1, 3, 2>(a, mw, sms, st, fits);
    if (!fits && e == cudaSuccess && a.M <= 8) e = w4_try<G, false, 1, 3, 2>(a, mw, sms, st, fits);
    if (e == cudaSuccess && a.M > 8 && a.M <= 16) e = w4_try<G, false, 2, 2, 2>(a, mw, sms, st, fits);
    // all of up to 32 rows where X then needs no more than two parts of K (20 rows of 9000 x 2048 13.3 us, 16.3 in two pieces;
    // with four parts 32 rows of 4096 x 4096 take 20.4 us, 19.3 in two pieces)
    if (e == cudaSuccess && a.M > 16) e = w4_try<G, false, 4, 2, 2>(a, mw, sms, st, fits, 2);
    // long K: one group of warps, whose scales take less shared memory
    if (!fits && e == cudaSuccess && a.M == 1) e = w4_try<G, false, 1, 1, 3>(a, mw, sms, st, fits);
    if (fits || e != cudaSuccess || a.M == 1) return e;
    const uint32_t first = a.M > 16 ? 16 : a.M > 8 ? 8 : a.M / 2, M = a.M;
    a.M = first;
    e = w4_run<G>(a, mw, sms, st, fits);
    if (e != cudaSuccess || !fits) return e;
    a.x += (size_t)first * a.ldx, a.z += (size_t)first * a.ldz;
    if (a.res) a.res += (size_t)first * a.ldr;
    a.M = M - first;
    return w4_run<G>(a, mw, sms, st, fits);
}

}  // namespace

extern "C" {

int sh_cuda_gemv_w4(uint64_t x, uint64_t codes, uint64_t scales, uint64_t zeros, uint64_t z, uint32_t M, uint32_t N,
                    uint32_t K, uint32_t ldx, uint32_t ldw, uint32_t ldz, uint32_t group, uint64_t bias,
                    uint64_t residual, uint32_t ldr, uint32_t flags) {
    if (flags & ~(SH_EPI_BIAS | SH_EPI_RESIDUAL)) {
        sh::set_error(-1, "[sh_cuda_gemv_w4] flags 0x%x: only SH_EPI_BIAS and SH_EPI_RESIDUAL", flags);
        return -1;
    }
    if (M == 0 || N == 0) return 0;
    if (M > 32 || (group != 32 && group != 64 && group != 128) || K == 0 || K > kMaxK || K % group || ldx < K || ldz < N ||
        (uint64_t)ldw * 2 < K || ldw % 16 || N >= (1u << 31) - 64) {
        sh::set_error(-1, "[sh_cuda_gemv_w4] need M <= 32, group 32, 64 or 128, K %% group == 0, K <= 262144, ldx >= K, ldz >= N, "
                      "ldw >= K / 2, ldw %% 16 == 0 (M=%u N=%u K=%u group=%u ldx=%u ldw=%u ldz=%u)", M, N, K, group, ldx, ldw,
                      ldz);
        return -1;
    }
    if (!x || !codes || !scales || !z || !sh::aligned16(codes) || ((x | scales | z) & 1) ||
        ((flags & SH_EPI_BIAS) && (!bias || (bias & 1))) ||
        ((flags & SH_EPI_RESIDUAL) && (!residual || (residual & 1) || ldr < N))) {
        sh::set_error(-1, "[sh_cuda_gemv_w4] a null or misaligned operand, or ldr < N");
        return -1;
    }
    W4Args a = {};
    a.x = (const __half *)x, a.codes = (const uint8_t *)codes, a.scales = (const __half *)scales;
    a.zeros = (const uint8_t *)zeros, a.z = (__half *)z;
    a.bias = flags & SH_EPI_BIAS ? (const __half *)bias : nullptr;
    a.res = flags & SH_EPI_RESIDUAL ? (const __half *)residual : nullptr;
    a.M = M, a.N = N, a.K = K, a.ldx = ldx, a.ldw = ldw, a.ldz = ldz, a.ldr = ldr;
    a.vec = sh::aligned16(x) && ldx % 8 == 0;
    const sh::DeviceState &s = sh::state();
    a.err = s.dev_err;
    CUtensorMap mw;
    if (!w4_map(&mw, codes, N, K, ldw)) {
        sh::set_error(-1, "[sh_cuda_gemv_w4] no tensor map for the codes (N=%u K=%u ldw=%u)", N, K, ldw);
        return -1;
    }
    bool fits = true;
    const cudaError_t e = group == 128 ? w4_run<128>(a, mw, s.num_sms, s.stream, fits)
                          : group == 64 ? w4_run<64>(a, mw, s.num_sms, s.stream, fits)
                                        : w4_run<32>(a, mw, s.num_sms, s.stream, fits);
    if (!sh::cuda_ok(e, "sh_cuda_gemv_w4")) return -1;
    if (!fits) {
        sh::set_error(-1, "[sh_cuda_gemv_w4] K=%u: one row of X does not fit in shared memory", K);
        return -1;
    }
    return 0;
}

}  // extern "C"
