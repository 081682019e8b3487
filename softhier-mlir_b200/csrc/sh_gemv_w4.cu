// Products of a few rows with 4-bit weights (sh_cuda_gemv_w4): Z[M, N] = X[M, K] W[K, N], W[k, n] = s (code - zero) with one
// scale and zero point per output column and group of 32, 64 or 128 k.
//
//     z[m, n] = sum_g s[n, g] sum_{k in g} (code[n, k] - zero[n, g]) x[m, k]
// code - zero is a small integer, exact in fp16, and is the 16-row operand of the tensor-core instruction (16 columns
// of W x 16 k) with up to 8 rows of X as its columns; the inner sum runs in its fp32 accumulator and is multiplied by the
// scale once per group. Nothing is rounded before Z.
//
// Bound by the weights' bytes (half a byte per element, read once). A lane loads the codes that it needs itself, 16
// bytes of a column of W at a time: the order of k inside the instruction is free when both operands agree, so the
// codes stay in their plain layout. Two warps' worth of ALU work per byte is what is left beside the loads: 9
// instructions turn a word into 8 fp16 operands (fp16 patterns 1024 + c and 1024 + 16 c, then one subtraction or FMA).
// The K range is split over the warps of a CTA and the CTAs of a cluster, whose partial sums meet in shared memory in a
// fixed order, so that all SMs have loads in flight when N alone would not fill them.
#include "sh_internal.cuh"

namespace {

constexpr uint32_t kW4Warps = 8, kW4Threads = 32 * kW4Warps, kUnit = 128;   // k per step of a warp

struct W4Args {
    const __half *x, *scales, *bias, *res;
    const uint8_t *codes, *zeros;
    __half *z;
    uint32_t M, N, K, ldx, ldw, ldz, ldr, vec;
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
// codes 0 .. 7 of a word minus the zero point, as the pairs (0, 4), (1, 5), (2, 6), (3, 7)
__device__ __forceinline__ void w4_word(uint32_t w, uint32_t zlo, uint32_t zhi, uint32_t (&h)[4]) {
    constexpr uint32_t kSixteenth = 0x2C002C00u;
    const uint32_t v = w >> 8;
    h[0] = w4_sub((w & 0x000F000Fu) | 0x64006400u, zlo);
    h[1] = w4_fma((w & 0x00F000F0u) | 0x64006400u, kSixteenth, zhi);
    h[2] = w4_sub((v & 0x000F000Fu) | 0x64006400u, zlo);
    h[3] = w4_fma((v & 0x00F000F0u) | 0x64006400u, kSixteenth, zhi);
}

// The words of one step of a lane: words[i] holds 8 codes at k offset word_k(i) of the step.
template <int G>
__device__ __forceinline__ uint32_t word_k(uint32_t c, uint32_t i) {
    return G == 128 ? c * 32 + i * 8 : G == 64 ? (i >> 1) * 64 + c * 16 + (i & 1) * 8 : i * 32 + c * 8;
}
template <int G>
__device__ __forceinline__ void load_words(uint32_t (&w)[4], const uint8_t *row, uint32_t c, uint32_t groups_left) {
    if (G == 128) {
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(row + c * 16));
    } else if (G == 64) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            w[2 * i] = w[2 * i + 1] = 0;
            if ((uint32_t)i < groups_left)
                asm volatile("ld.global.nc.v2.u32 {%0, %1}, [%2];" : "=r"(w[2 * i]), "=r"(w[2 * i + 1])
                             : "l"(row + i * 32 + c * 8));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = 0;
            if ((uint32_t)i < groups_left)
                asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(w[i]) : "l"(row + i * 16 + c * 4));
        }
    }
}

template <int G, int NT, int RW, int WR>
__global__ void __launch_bounds__(kW4Threads, 2) k_gemv_w4(W4Args a, uint32_t splits) {
    constexpr uint32_t WK = kW4Warps / WR, kRows = 16 * RW * WR;   // columns of W per CTA
    constexpr int GU = kUnit / G;                                  // groups per step
    __shared__ float s_red[WK][kRows][NT * 8];
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5, g = lane >> 2, c = lane & 3;
    const uint32_t wr = warp % WR, wk = warp / WR;
    const uint32_t n0 = blockIdx.x * kRows + wr * 16 * RW;
    const uint32_t units = (a.K + kUnit - 1) / kUnit, groups = a.K / G;
    const uint32_t part = blockIdx.y * WK + wk, parts = splits * WK;
    const uint32_t u0 = (uint32_t)((uint64_t)units * part / parts), u1 = (uint32_t)((uint64_t)units * (part + 1) / parts);

    const uint8_t *row[RW][2];
    size_t srow[RW][2];
#pragma unroll
    for (int i = 0; i < RW; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t n = min(n0 + i * 16 + g + 8 * e, a.N - 1);   // columns past the end repeat the last one
            row[i][e] = a.codes + (size_t)n * a.ldw;
            srow[i][e] = (size_t)n * groups;
        }
    float acc[RW][NT][4];
#pragma unroll
    for (int i = 0; i < RW; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[i][nt][0] = acc[i][nt][1] = acc[i][nt][2] = acc[i][nt][3] = 0.f;

    struct Step {
        uint32_t w[RW][2][4];
        __half s[RW][2][GU];
        uint8_t z[RW][2][GU];
    };
    auto load = [&](Step &st, uint32_t u) {
        const uint32_t left = groups - u * GU;
#pragma unroll
        for (int i = 0; i < RW; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                load_words<G>(st.w[i][e], row[i][e] + (size_t)u * (kUnit / 2), c, left);
#pragma unroll
                for (int q = 0; q < GU; ++q) {
                    const bool in = GU == 1 || (uint32_t)q < left;
                    st.s[i][e][q] = in ? __ldg(a.scales + srow[i][e] + u * GU + q) : __half(0.f);
                    st.z[i][e][q] = in && a.zeros ? __ldg(a.zeros + srow[i][e] + u * GU + q) : (uint8_t)8;
                }
            }
    };
    auto compute = [&](const Step &st, uint32_t u) {
        const uint32_t left = groups - u * GU;
        float ga[RW][NT][4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            constexpr int kPer = 4 / GU;        // words per group
            const uint32_t q = i / kPer;
            if (i % kPer == 0) {
#pragma unroll
                for (int r = 0; r < RW; ++r)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) ga[r][nt][0] = ga[r][nt][1] = ga[r][nt][2] = ga[r][nt][3] = 0.f;
            }
            uint32_t b[NT][4];      // x in the order of w4_word's pairs
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const uint32_t m = nt * 8 + g;
                uint32_t x[4] = {0, 0, 0, 0};
                if (m < a.M && (GU == 1 || q < left)) {
                    const __half *xp = a.x + (size_t)m * a.ldx + (size_t)u * kUnit + word_k<G>(c, i);
                    if (a.vec) {
                        const uint4 v = __ldg(reinterpret_cast<const uint4 *>(xp));
                        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e >> 1] |= (uint32_t)__half_as_ushort(xp[e]) << (16 * (e & 1));
                    }
                }
                b[nt][0] = __byte_perm(x[0], x[2], 0x5410), b[nt][1] = __byte_perm(x[0], x[2], 0x7632);
                b[nt][2] = __byte_perm(x[1], x[3], 0x5410), b[nt][3] = __byte_perm(x[1], x[3], 0x7632);
            }
#pragma unroll
            for (int r = 0; r < RW; ++r) {
                uint32_t h0[4], h1[4];
                const uint32_t z0 = (st.z[r][0][q] & 15u) * 0x00010001u, z1 = (st.z[r][1][q] & 15u) * 0x00010001u;
                w4_word(st.w[r][0][i], 0x64006400u | z0, 0xD400D400u | z0 << 4, h0);
                w4_word(st.w[r][1][i], 0x64006400u | z1, 0xD400D400u | z1 << 4, h1);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    w4_mma(ga[r][nt], h0[0], h1[0], h0[1], h1[1], b[nt][0], b[nt][1]);
                    w4_mma(ga[r][nt], h0[2], h1[2], h0[3], h1[3], b[nt][2], b[nt][3]);
                }
            }
            if (i % kPer == kPer - 1) {
#pragma unroll
                for (int r = 0; r < RW; ++r) {
                    const float s0 = __half2float(st.s[r][0][q]), s1 = __half2float(st.s[r][1][q]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        acc[r][nt][0] = fmaf(ga[r][nt][0], s0, acc[r][nt][0]);
                        acc[r][nt][1] = fmaf(ga[r][nt][1], s0, acc[r][nt][1]);
                        acc[r][nt][2] = fmaf(ga[r][nt][2], s1, acc[r][nt][2]);
                        acc[r][nt][3] = fmaf(ga[r][nt][3], s1, acc[r][nt][3]);
                    }
                }
            }
        }
    };
    // the next step's words are in flight while this one's are used
    Step cur, nxt;
    if (u0 < u1) load(cur, u0);
    for (uint32_t u = u0; u < u1; ++u) {
        if (u + 1 < u1) load(nxt, u + 1);
        compute(cur, u);
        cur = nxt;
    }

    // ---- partial sums of the K parts, in their order -------------------------------------------------------------
#pragma unroll
    for (int r = 0; r < RW; ++r)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                s_red[wk][wr * 16 * RW + r * 16 + g + 8 * (e >> 1)][nt * 8 + 2 * c + (e & 1)] = acc[r][nt][e];
    __syncthreads();
    for (uint32_t i = t; i < kRows * NT * 8; i += kW4Threads) {
        float *p = &s_red[0][0][0] + i;
        float v = p[0];
#pragma unroll
        for (uint32_t w = 1; w < WK; ++w) v += p[w * kRows * NT * 8];
        p[0] = v;
    }
    if (splits > 1) cluster_sync_all();
    else __syncthreads();
    for (uint32_t i = blockIdx.y * kW4Threads + t; i < kRows * NT * 8; i += splits * kW4Threads) {
        const uint32_t m = i / kRows, rl = i - m * kRows, n = blockIdx.x * kRows + rl;
        if (m >= a.M || n >= a.N) continue;
        const float *p = &s_red[0][rl][m];
        float v = 0.f;
        if (splits > 1) {
            const uint32_t at = smem_u32(p);
            for (uint32_t k = 0; k < splits; ++k) {
                float y;
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(y) : "r"(mapa_shared(at, k)) : "memory");
                v += y;
            }
        } else {
            v = *p;
        }
        if (a.bias) v += __half2float(a.bias[n]);
        if (a.res) v += __half2float(a.res[(size_t)m * a.ldr + n]);
        a.z[(size_t)m * a.ldz + n] = __float2half_rn(v);
    }
    if (splits > 1) cluster_sync_all();      // the other CTAs have read this one's sums
}

template <int G, int NT, int RW, int WR>
cudaError_t w4_launch(const W4Args &a, uint32_t splits, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((a.N + 16 * RW * WR - 1) / (16 * RW * WR), splits);
    cfg.blockDim = dim3(kW4Threads);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1, attr[0].val.clusterDim.y = splits, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = sh::pdl_enabled() ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, k_gemv_w4<G, NT, RW, WR>, a, splits);
}

template <int G>
cudaError_t w4_pick(const W4Args &a, int sms, cudaStream_t st) {
    const uint32_t nt = (a.M + 7) / 8;
    // K parts over the CTAs of a cluster until about two CTAs per SM have work of at least two steps per warp
    auto split = [&](uint32_t rows, uint32_t wk) {
        const uint32_t blocks = (a.N + rows - 1) / rows, units = (a.K + kUnit - 1) / kUnit;
        uint32_t s = 1;
        while (s < 8 && blocks * s < 2u * sms && units >= 2 * wk * 2 * s) s *= 2;
        return s;
    };
    if (nt == 1) return w4_launch<G, 1, 1, 2>(a, split(32, 4), st);
    if (nt == 2) return w4_launch<G, 2, 2, 2>(a, split(64, 4), st);
    return w4_launch<G, 4, 2, 2>(a, split(64, 4), st);
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
    if (M > 32 || (group != 32 && group != 64 && group != 128) || K == 0 || K % group || ldx < K || ldz < N ||
        (uint64_t)ldw * 2 < K || ldw % 16 || N >= (1u << 31) - 64) {
        sh::set_error(-1, "[sh_cuda_gemv_w4] need M <= 32, group 32, 64 or 128, K %% group == 0, ldw %% 16 == 0 (M=%u N=%u K=%u "
                      "group=%u ldx=%u ldw=%u ldz=%u)", M, N, K, group, ldx, ldw, ldz);
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
    const cudaError_t e = group == 128 ? w4_pick<128>(a, s.num_sms, s.stream)
                          : group == 64 ? w4_pick<64>(a, s.num_sms, s.stream)
                                        : w4_pick<32>(a, s.num_sms, s.stream);
    return sh::cuda_ok(e, "sh_cuda_gemv_w4") ? 0 : -1;
}

}  // extern "C"
