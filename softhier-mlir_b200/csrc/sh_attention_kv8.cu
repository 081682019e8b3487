// Attention over the paged 8-bit K / V cache (sh_cuda_attention_kv8): new rows of a batch of requests against all of
// their cached tokens, grouped-query heads, causal among the new rows.
//
// With x_j = scale log2(e) ks_j (q . kcode_j) and w_j = 2^(x_j + log2 vs_j - m), m the running maximum of the exponent,
//     o = (sum_j w_j vcode_j) / (sum_j w_j / vs_j)
// so the value scales ride in the exponent: w_j stays in fp16's range whatever the scales are, and the codes themselves
// (int8 and e4m3 are exact in fp16) are the operands of the second product. The first product is exact up to its
// fp32 sums; w_j is rounded to fp16 (2^-11 relative, as the outputs are), its sum is taken in fp32 before that.
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
    uint32_t min_units;
    float sl2;            // scale * log2(e)
    uint32_t vec;         // q rows take 16-byte loads, o rows 4-byte stores
    uint32_t *counters;   // arrivals per CTA whose last item goes on in others, zero between calls
    float *part;
    int *err;
};

// A request as the kernels see it: lengths that no index leaves the arrays with, whatever the device arrays hold.
struct ReqView {
    uint32_t qs, nq, ctx;
    int base;             // tokens before its first new row (< 0: the first rows have none)
};
__device__ __forceinline__ ReqView req_view(const KvArgs &a, uint32_t r) {
    ReqView v;
    const int s = a.q_start[r], e = a.q_start[r + 1], len = a.lens[r];
    const int s0 = min(max(s, 0), (int)a.T), e0 = min(max(e, s0), (int)a.T);
    v.qs = (uint32_t)s0;
    v.nq = (uint32_t)(e0 - s0);
    v.ctx = min((uint32_t)max(len, 0), a.ld_table << a.page_shift);
    v.base = (int)v.ctx - max(e - s, 0) + (s0 - s);
    return v;
}

__device__ __forceinline__ uint4 ldg16(const void *p) {   // streamed once: past L1
    uint4 r;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}
__device__ __forceinline__ uint2 ldg8(const void *p) {
    uint2 r;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
    return r;
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
// int8: code + 128 in the low byte of the fp16 pattern 0x6400 is 1152 + code, exactly; 1152 comes off again
constexpr uint32_t kMagic = 0x64806480u, kMagicVal = 0x64806480u;   // fp16 1152 = 0x6480 as well

// the four codes of a word as two fp16 pairs: int8 (0, 2), (1, 3); e4m3 (0, 1), (2, 3)
template <bool FP8>
__device__ __forceinline__ void word_to_h2(uint32_t w, uint32_t &p, uint32_t &q) {
    if (FP8) {
        p = e4m3x2_to_h2(w & 0xFFFFu);
        q = e4m3x2_to_h2(w >> 16);
    } else {
        p = hsub2((w & 0x00FF00FFu) ^ kMagic, kMagicVal);
        q = hsub2(((w >> 8) & 0x00FF00FFu) ^ kMagic, kMagicVal);
    }
}
// byte B of two words as an fp16 pair (lo from a, hi from b)
template <bool FP8, int B>
__device__ __forceinline__ uint32_t byte_pair(uint32_t a, uint32_t b) {
    if (FP8) return e4m3x2_to_h2(__byte_perm(a, b, B | (4 + B) << 4));
    return hsub2((__byte_perm(a, b, B | B << 4 | (4 + B) << 8 | (4 + B) << 12) & 0x00FF00FFu) ^ kMagic, kMagicVal);
}

// ================================================================================================================
// Few rows per request (single tokens, drafts). The K / V bytes bound it, so each is read once per tile of up to
// 8 NT (query row, query head) pairs of one kv head, straight into the registers of the warp that uses it.
// Both products keep the 8-bit side as the 16-row operand of the matrix instruction and the rows as its 8 columns:
//     S^T (16 tokens x 8 rows) = K (16 x dh) Q^T,     O^T (16 dims x 8 rows) += V^T (16 x 16 tokens) W^T
// so a group of up to 8 query heads fills the instruction. Its index along the contracted side may be permuted freely when
// both operands agree: a lane takes 16 neighbouring columns of its K rows, and 4 tokens of V with dh / 8 neighbouring
// columns, so every load is 16 bytes (8 for V at dh = 64) and a quarter-warp covers whole 32-byte sectors. W^T comes from
// S^T by an 8 x 8 transpose in registers.
//
// Work is split evenly whatever the lengths are: the units (request, kv head, row tile, 64 tokens), in this order, are dealt
// to the CTAs in equal contiguous runs, which every CTA works out from the lengths by itself. An item (request, head, tile)
// that spans CTAs leaves partial sums in the workspace, at most two per CTA; the CTA that arrives last joins them in
// the order of the CTAs, so results do not depend on timing.
// ================================================================================================================
constexpr uint32_t kWarps = 4, kThreads = kWarps * 32, kKeys = 16 * kWarps;   // keys per unit

template <int DH, int NT, bool FP8>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 4 : 3) k_attn_kv8_rows(KvArgs a) {
    constexpr uint32_t RT = 8 * NT;                 // rows of a tile
    constexpr int KC = DH / 64;                     // 16-byte pieces of a K row per lane
    constexpr int VB = DH / 8;                      // V columns per lane
    constexpr int VW = VB / 4;                      // as words
    __shared__ float s_o[kWarps][RT][DH];
    __shared__ float s_m[kWarps][RT], s_l[kWarps][RT];
    __shared__ unsigned long long s_part[kWarps];
    __shared__ unsigned long long s_off;
    __shared__ uint32_t s_r, s_flag;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5, g = lane >> 2, c = lane & 3;
    const uint32_t page1 = (1u << a.page_shift) - 1;

    // ---- this CTA's run of units ------------------------------------------------------------------------------------
    typedef unsigned long long u64;
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
    for (uint32_t w = 0; w < kWarps; ++w) {
        if (w < warp) incl += s_part[w];
        total += s_part[w];
    }
    u64 per = (total + gridDim.x - 1) / gridDim.x;
    if (per < a.min_units) per = a.min_units;
    const u64 begin = per * blockIdx.x, end = min(total, begin + per);
    if (begin >= end) return;
    if (begin >= incl - sum && begin < incl) {
        u64 off = begin - (incl - sum);
        for (uint32_t r = r0; r < r1; ++r) {
            const ReqView v = req_view(a, r);
            const uint32_t tiles = (v.nq * a.G + RT - 1) / RT, blocks = max(1u, (v.ctx + kKeys - 1) / kKeys);
            const u64 n = (u64)a.heads * tiles * blocks;
            if (off < n) {
                s_r = r, s_off = off;
                break;
            }
            off -= n;
        }
    }
    __syncthreads();
    uint32_t r = s_r;
    u64 off = s_off;

    for (u64 u = begin; u < end;) {
        const ReqView v = req_view(a, r);
        const uint32_t tiles = (v.nq * a.G + RT - 1) / RT, blocks = max(1u, (v.ctx + kKeys - 1) / kKeys);
        const u64 units = (u64)a.heads * tiles * blocks;
        if (off >= units) {      // on to the next request (one without new rows has no units)
            off -= units;
            ++r;
            continue;
        }
        const uint32_t item = (uint32_t)(off / blocks), b0 = (uint32_t)(off - (u64)item * blocks);
        const uint32_t kvh = item / tiles, tile = item - kvh * tiles;
        const uint32_t b1 = (uint32_t)min((u64)blocks, (u64)b0 + (end - u));
        const uint32_t row0 = tile * RT, nrows = min(RT, v.nq * a.G - row0);
        // keys of the tile's first and last row
        const int ctx = (int)v.ctx;
        const int lim_lo = min(max(v.base + (int)(row0 / a.G) + 1, 0), ctx);
        const int lim_hi = min(max(v.base + (int)((row0 + nrows - 1) / a.G) + 1, 0), ctx);
        const uint32_t be = min(b1, (uint32_t)(lim_hi + kKeys - 1) / kKeys);

        // ---- Q as the column operand: lane (g, c) holds columns 16 c .. of row 8 nt + g ------------------------------
        uint32_t qf[NT][KC * 4][2];
        int lim[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const uint32_t n = nt * 8 + g;
            const uint32_t rr = row0 + n, qi = rr / a.G, gi = rr - qi * a.G;
            const __half *qp = a.q + (size_t)(v.qs + qi) * a.ldq + ((size_t)kvh * a.G + gi) * DH + c * 16;
#pragma unroll
            for (int j = 0; j < KC; ++j) {
                uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                if (n < nrows) {
                    if (a.vec) {
                        *reinterpret_cast<uint4 *>(w) = *reinterpret_cast<const uint4 *>(qp + j * 64);
                        *reinterpret_cast<uint4 *>(w + 4) = *reinterpret_cast<const uint4 *>(qp + j * 64 + 8);
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            w[e >> 1] |= (uint32_t)__half_as_ushort(qp[j * 64 + e]) << (16 * (e & 1));
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // columns 4 i .. 4 i + 3 in the order word_to_h2 gives K's
                    qf[nt][j * 4 + i][0] = FP8 ? w[2 * i] : __byte_perm(w[2 * i], w[2 * i + 1], 0x5410);
                    qf[nt][j * 4 + i][1] = FP8 ? w[2 * i + 1] : __byte_perm(w[2 * i], w[2 * i + 1], 0x7632);
                }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t m = nt * 8 + 2 * c + e;
                lim[nt][e] = m < nrows ? min(max(v.base + (int)((row0 + m) / a.G) + 1, 0), ctx) : lim_hi;
            }
        }

        float o[DH / 16][NT][4];
        float m[NT][2], l[NT][2];
#pragma unroll
        for (int i = 0; i < DH / 16; ++i)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][nt][e] = 0.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) m[nt][0] = m[nt][1] = -INFINITY, l[nt][0] = l[nt][1] = 0.f;

        const int *row_table = a.table + (size_t)r * a.ld_table;
        const size_t head_tok = (size_t)kvh << a.page_shift;
        // page of this warp's 16 tokens of block b; -1: none of them is a key, or the table is wrong
        auto page_of = [&](uint32_t b) -> int {
            const uint32_t tok = b * kKeys + warp * 16;
            if (b >= be || (int)tok >= lim_hi) return -1;
            const int pid = row_table[tok >> a.page_shift];
            if ((uint32_t)pid < a.pages) return pid;
            atomicCAS(a.err, 0, (int)sh::kErrBadArgs);
            return -1;
        };
        auto tile_off = [&](int pid, uint32_t b) {
            const uint32_t in = (b * kKeys + warp * 16) & page1;
            return (size_t)(uint32_t)pid * a.page_stride + (head_tok + in) * DH;
        };
        uint4 kr[2][KC];
        uint32_t vr[4][VW];
        float ks = 0.f, vs = 0.f;
        auto load_k = [&](int pid, uint32_t b) {
            const uint8_t *p = a.k + tile_off(pid, b) + g * DH + c * 16;
#pragma unroll
            for (int j = 0; j < KC; ++j) {
                kr[0][j] = ldg16(p + j * 64);
                kr[1][j] = ldg16(p + 8 * DH + j * 64);
            }
        };
        auto load_v = [&](int pid, uint32_t b) {
            const uint8_t *p = a.v + tile_off(pid, b) + g * VB;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t tok = 2 * c + (e & 1) + 8 * (e >> 1);
                if (VW == 4) {
                    const uint4 x = ldg16(p + tok * DH);
                    vr[e][0] = x.x, vr[e][1] = x.y, vr[e][VW - 2] = x.z, vr[e][VW - 1] = x.w;
                } else {
                    const uint2 x = ldg8(p + tok * DH);
                    vr[e][0] = x.x, vr[e][1] = x.y;
                }
            }
        };
        int pid = page_of(b0), pid_next = page_of(b0 + 1);
        if (pid >= 0) {
            ks = a.ks[(size_t)pid * a.heads + kvh];
            vs = a.vs[(size_t)pid * a.heads + kvh];
            load_k(pid, b0);
            load_v(pid, b0);
        }
        for (uint32_t b = b0; b < be; ++b) {
            const int pid_2 = page_of(b + 2);
            const bool act = pid >= 0;
            float s[NT][4];
            if (act) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
                for (int j = 0; j < KC; ++j) {
                    const uint32_t *ka = reinterpret_cast<const uint32_t *>(&kr[0][j]);
                    const uint32_t *kb = reinterpret_cast<const uint32_t *>(&kr[1][j]);
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
            }
            const float ksl = ks * a.sl2, vcl = fmaxf(vs, 0x1p-80f);
            float ks_n = 0.f, vs_n = 0.f;
            if (pid_next >= 0) {
                ks_n = a.ks[(size_t)pid_next * a.heads + kvh];
                vs_n = a.vs[(size_t)pid_next * a.heads + kvh];
                load_k(pid_next, b + 1);
            }
            if (act) {
                const float lvs = __log2f(vcl), rvs = __frcp_rn(vcl);
                const int tok0 = (int)(b * kKeys + warp * 16);
                bool raise = false;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float x = fmaf(s[nt][e], ksl, lvs);
                        if (tok0 + 16 > lim_lo && tok0 + (int)g + 8 * (e >> 1) >= lim[nt][e & 1]) x = -INFINITY;
                        s[nt][e] = x;
                        raise |= x > m[nt][e & 1] + 8.f;
                    }
                // the maximum only moves when a weight would pass 2^8 (exact room in fp16), which is rare after the start
                if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float x = fmaxf(s[nt][e], s[nt][e + 2]);
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                            const float now = fmaxf(m[nt][e], x);
                            const float f = now == -INFINITY ? 1.f : fast_exp2(m[nt][e] - now);
                            m[nt][e] = now;
                            l[nt][e] *= f;
#pragma unroll
                            for (int i = 0; i < DH / 16; ++i) o[i][nt][e] *= f, o[i][nt][e + 2] *= f;
                        }
                }
                uint32_t w0[NT], w1[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float mm = m[nt][e & 1];
                        w[e] = fast_exp2(s[nt][e] - (mm == -INFINITY ? 0.f : mm));
                        l[nt][e & 1] = fmaf(w[e], rvs, l[nt][e & 1]);
                    }
                    w0[nt] = movmatrix(pack_h2(w[0], w[1]));
                    w1[nt] = movmatrix(pack_h2(w[2], w[3]));
                }
                if (tok0 + 16 > ctx) {      // rows past the last token can hold anything
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (tok0 + (int)(2 * c + (e & 1) + 8 * (e >> 1)) >= ctx)
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
                    }
                }
            }
            if (pid_next >= 0) load_v(pid_next, b + 1);
            pid = pid_next, pid_next = pid_2;
            ks = ks_n, vs = vs_n;
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
                if (g == 0) s_m[warp][n] = m[nt][e], s_l[warp][n] = x;
#pragma unroll
                for (int i = 0; i < DH / 16; ++i)
                    *reinterpret_cast<float2 *>(&s_o[warp][n][g * VB + 2 * i]) = make_float2(o[i][nt][e], o[i][nt][e + 2]);
            }
        __syncthreads();
        const bool whole = b0 == 0 && b1 == blocks;
        const uint32_t slot = 2 * blockIdx.x + (b0 == 0 ? 1 : 0);
        float *po = a.part + (size_t)slot * RT * (DH + 2), *pm = po + RT * DH, *pl = pm + RT;
        for (uint32_t e = t; e < nrows * (DH / 2); e += kThreads) {
            const uint32_t n = e / (DH / 2), d = 2 * (e - n * (DH / 2));
            float mx = -INFINITY;
#pragma unroll
            for (uint32_t w = 0; w < kWarps; ++w) mx = fmaxf(mx, s_m[w][n]);
            float x = 0.f, y = 0.f, ll = 0.f;
#pragma unroll
            for (uint32_t w = 0; w < kWarps; ++w) {
                const float f = s_m[w][n] == -INFINITY ? 0.f : fast_exp2(s_m[w][n] - mx);
                const float2 p = *reinterpret_cast<const float2 *>(&s_o[w][n][d]);
                x = fmaf(p.x, f, x);
                y = fmaf(p.y, f, y);
                ll = fmaf(s_l[w][n], f, ll);
            }
            if (whole) {
                const float inv = ll == 0.f ? 0.f : 1.f / ll;
                const uint32_t rr = row0 + n, qi = rr / a.G, gi = rr - qi * a.G;
                __half *op = a.o + (size_t)(v.qs + qi) * a.ldo + ((size_t)kvh * a.G + gi) * DH + d;
                if (a.vec) *reinterpret_cast<__half2 *>(op) = __floats2half2_rn(x * inv, y * inv);
                else op[0] = __float2half_rn(x * inv), op[1] = __float2half_rn(y * inv);
            } else {
                *reinterpret_cast<float2 *>(po + n * DH + d) = make_float2(x, y);
                if (d == 0) pm[n] = mx, pl[n] = ll;
            }
        }
        if (!whole) {
            // the item's CTAs: c0 holds its first unit and counts the arrivals
            const u64 u0 = u - b0;
            const uint32_t c0 = (uint32_t)(u0 / per), c1 = (uint32_t)((u0 + blocks - 1) / per);
            __threadfence();
            __syncthreads();
            if (t == 0) {
                const uint32_t before = atom_add_acq_rel_gpu(a.counters + c0, 1u);
                s_flag = before == c1 - c0;
                if (s_flag) a.counters[c0] = 0;      // for the next call
            }
            __syncthreads();
            if (s_flag) {
                __threadfence();
                for (uint32_t e = t; e < nrows * (DH / 4); e += kThreads) {
                    const uint32_t n = e / (DH / 4), d = 4 * (e - n * (DH / 4));
                    const size_t stride = 2 * RT * (DH + 2);
                    const float *first = a.part + (size_t)(2 * c0 + 1) * RT * (DH + 2);
                    const float *rest = a.part + (size_t)(2 * c0) * RT * (DH + 2);
                    float mx = __ldcg(first + RT * DH + n);
                    for (uint32_t k = 1; k <= c1 - c0; ++k) mx = fmaxf(mx, __ldcg(rest + k * stride + RT * DH + n));
                    float ll = 0.f;
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                    for (uint32_t k = 0; k <= c1 - c0; ++k) {
                        const float *p = k ? rest + k * stride : first;
                        const float mk = __ldcg(p + RT * DH + n);
                        const float f = mk == -INFINITY ? 0.f : fast_exp2(mk - mx);
                        const float4 y = __ldcg(reinterpret_cast<const float4 *>(p + n * DH + d));
                        ll = fmaf(__ldcg(p + RT * DH + RT + n), f, ll);
                        x.x = fmaf(y.x, f, x.x), x.y = fmaf(y.y, f, x.y);
                        x.z = fmaf(y.z, f, x.z), x.w = fmaf(y.w, f, x.w);
                    }
                    const float inv = ll == 0.f ? 0.f : 1.f / ll;
                    const uint32_t rr = row0 + n, qi = rr / a.G, gi = rr - qi * a.G;
                    __half *op = a.o + (size_t)(v.qs + qi) * a.ldo + ((size_t)kvh * a.G + gi) * DH + d;
                    const float z[4] = {x.x * inv, x.y * inv, x.z * inv, x.w * inv};
                    if (a.vec) {
                        reinterpret_cast<__half2 *>(op)[0] = __floats2half2_rn(z[0], z[1]);
                        reinterpret_cast<__half2 *>(op)[1] = __floats2half2_rn(z[2], z[3]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) op[i] = __float2half_rn(z[i]);
                    }
                }
            }
        }
        u += b1 - b0;
        off += b1 - b0;
    }
}

constexpr size_t kCounterBytes = 16384;
constexpr uint32_t kMaxSms = 160;         // the grid is cut there, so that the workspace is

template <int DH, int NT, bool FP8>
cudaError_t launch_rows(KvArgs &a, int sms, cudaStream_t st) {
    constexpr uint32_t kPerSm = NT == 1 ? 4 : 3;
    static_assert(kMaxSms * kPerSm * 4 <= kCounterBytes &&
                      kCounterBytes + (size_t)2 * kPerSm * kMaxSms * 8 * NT * (DH + 2) * 4 <= SH_CUDA_KV8_WS_BYTES,
                  "workspace: a counter and two partial items per CTA");
    const uint32_t grid = (uint32_t)sms * kPerSm;
    return sh::launch_pdl(k_attn_kv8_rows<DH, NT, FP8>, dim3(grid), dim3(kThreads), 0, st, a);
}

}  // namespace

extern "C" {

int sh_cuda_attention_kv8(uint64_t q, uint64_t o, const sh_cuda_kv8_t *c, uint64_t table, uint32_t ld_table,
                          uint64_t lens, uint64_t q_start, uint32_t R, uint32_t T, uint32_t max_q, uint32_t H,
                          uint32_t ldq, uint32_t ldo, float scale, uint64_t ws, size_t ws_bytes) {
    const int bad = sh::kv8_check(c, "sh_cuda_attention_kv8");
    if (bad) return bad;
    if (H == 0 || H % c->heads || (uint64_t)H * c->dh > ldq || (uint64_t)H * c->dh > ldo ||
        (uint64_t)T * H >= (1ull << 31) || ld_table == 0 || ld_table >= (1u << 31) / c->page || !(fabsf(scale) < INFINITY)) {
        sh::set_error(-1, "[sh_cuda_attention_kv8] need H a multiple of the cache's %u heads, ldq, ldo >= H dh, T H and "
                      "ld_table page < 2^31, a finite scale (H=%u ldq=%u ldo=%u T=%u ld_table=%u)", c->heads, H, ldq, ldo,
                      T, ld_table);
        return -1;
    }
    if (!ws || !sh::aligned16(ws) || ws_bytes < SH_CUDA_KV8_WS_BYTES) {
        sh::set_error(-1, "[sh_cuda_attention_kv8] workspace null, not 16-byte aligned, or less than %u bytes",
                      SH_CUDA_KV8_WS_BYTES);
        return -1;
    }
    if (R == 0 || T == 0) return 0;
    if (!q || !o || !table || !lens || !q_start || ((q | o) & 1)) {
        sh::set_error(-1, "[sh_cuda_attention_kv8] null array, or odd q / o");
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
    a.min_units = 2;
    a.vec = sh::aligned16(q) && ldq % 8 == 0 && (o & 3) == 0 && ldo % 2 == 0;
    a.counters = (uint32_t *)ws, a.part = (float *)(ws + kCounterBytes), a.err = s.dev_err;
    const int sms = s.num_sms < (int)kMaxSms ? s.num_sms : (int)kMaxSms;
    const bool fp8 = c->fmt == SH_FP8, wide = (uint64_t)max_q * a.G > 8;
    cudaError_t e;
#define SH_KV8(dh, nt) (fp8 ? launch_rows<dh, nt, true>(a, sms, s.stream) : launch_rows<dh, nt, false>(a, sms, s.stream))
    if (c->dh == 64) e = wide ? SH_KV8(64, 2) : SH_KV8(64, 1);
    else e = wide ? SH_KV8(128, 2) : SH_KV8(128, 1);
#undef SH_KV8
    return sh::cuda_ok(e, "sh_cuda_attention_kv8") ? 0 : -1;
}

}  // extern "C"
