/* sh_ops_cuda.h -- extensions of libsh_ops_cuda.so beyond the reference header (runtime/sh_ops.h).
 *
 * They have no counterpart in the reference: they expose what a GPU backend needs and a RISC-V cluster did not
 * (caller-owned device memory, streams, asynchronous error state) and the fused / batched forms of the hot-path
 * ops that the encoder driver uses (GEMM epilogues, residual + LayerNorm, attention over a batch of sequences).
 * All pointers are device pointers passed as uint64_t, sizes and leading dimensions are in elements, like the
 * reference ABI.
 */
#ifndef SH_OPS_CUDA_H
#define SH_OPS_CUDA_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- runtime ------------------------------------------------------------------------------------------------
 * Bind caller-owned device memory (e.g. a torch tensor's data_ptr) as the HBM arena of the current device;
 * the library never frees it. Returns 0, or -1 when base is NULL / not 256-byte aligned. */
int      sh_cuda_set_arena(void *base, size_t bytes);
void    *sh_cuda_arena_base(void);
size_t   sh_cuda_arena_bytes(void);
/* All ops of the calling thread's current device are enqueued on this stream (a cudaStream_t; NULL = the
 * legacy default stream). */
int      sh_cuda_set_stream(void *stream);
void    *sh_cuda_get_stream(void);
int      sh_cuda_synchronize(void);                 /* stream sync; returns the cudaError_t code */
int      sh_cuda_last_error(void);                  /* first error recorded since the previous call, then cleared */
const char *sh_cuda_last_error_string(void);        /* text of that error ("" when none) */
int      sh_cuda_device_error(void);                /* syncs, returns and clears the kernels' error word (1 = a
                                                       bounded wait gave up) */
int      sh_cuda_num_sms(void);
float    sh_cuda_timer_last_ms(void);               /* the period the last sh_timer_end printed */
uint32_t sh_cuda_abi_version(void);                 /* 1 */

/* ---- GEMM with fused epilogue ---------------------------------------------------------------------------------
 * Z[M,N] = epi(X[M,K] . W[K,N]) with fp32 accumulation, fp16 out. `flags`:
 *   SH_EPI_ACCUMULATE  t = acc + Z_old           (sh_gemm_cfg.accumulate)
 *   SH_EPI_BIAS        t = t + bias[col]         (bias: 1 x N fp16)
 *   SH_EPI_GELU        t = gelu_tanh(t)          (after the bias)
 *   SH_EPI_RESIDUAL    t = t + R[row, col]       (R: M x N fp16, leading dim ldr)
 *   SH_EPI_F32_OUT     Z is fp32 (ldz in fp32 elements; SH_EPI_ACCUMULATE then reads fp32 Z)
 *   SH_EPI_ACC_F32_IN  t = t + R32[row, col] with R32 an fp32 matrix passed as `residual` (leading dim ldr);
 *                      not combined with SH_EPI_RESIDUAL. Together with SH_EPI_F32_OUT this carries a K-split
 *                      product in fp32 across calls (the SUMMA panels) and rounds it to fp16 once.
 *   SH_GEMM_SIMT       use the CUDA-core fallback kernel (tests)
 * splits: 0 = library choice of split-K, 1 = none, n = K split n ways (partials reduced in a fixed order).
 * Returns 0 or -1 (reason printed). */
#define SH_EPI_ACCUMULATE 0x1u
#define SH_EPI_BIAS       0x2u
#define SH_EPI_GELU       0x4u
#define SH_EPI_RESIDUAL   0x8u
#define SH_EPI_F32_OUT    0x10u
#define SH_EPI_ACC_F32_IN 0x20u
#define SH_GEMM_SIMT      0x100u
int sh_cuda_gemm(uint64_t x, uint64_t w, uint64_t z, uint32_t M, uint32_t N, uint32_t K, uint32_t ldx, uint32_t ldw,
                 uint32_t ldz, uint64_t bias, uint64_t residual, uint32_t ldr, uint32_t flags, uint32_t splits);

/* ---- the GEMM planner as a query ---------------------------------------------------------------------------------
 * No counterpart in the reference. The kernel and tiling sh_cuda_gemm picks for 16-byte-aligned operands of an
 * M x N x K product with `splits` as in sh_cuda_gemm, on a GPU with `num_sms` SMs (0: the current device's; any
 * other value makes no CUDA call, so the query runs without a GPU):
 *   kernel      0 CUDA-core fallback (K == 0), 1 single-CTA tcgen05 (128 x bn tiles), 2 two-CTA tcgen05 (256 x bn)
 *   k_blocks    64-deep K blocks; splits: K pieces per tile (split-K, single-CTA kernel only)
 *   units       work units of the launch: tiles x splits, or for kernel 2 whole tiles below full_units and
 *               256-column slices of the remaining tiles past it (a short last wave of 256 x 512 tiles)
 *   grid        CTAs launched
 * Returns 0, or -1 when out is NULL. */
typedef struct sh_cuda_gemm_plan_t {
    uint32_t kernel, bn, tiles_m, tiles_n, k_blocks, splits, full_units, units, grid;
} sh_cuda_gemm_plan_t;
int sh_cuda_gemm_plan(uint32_t M, uint32_t N, uint32_t K, uint32_t splits, uint32_t num_sms,
                      sh_cuda_gemm_plan_t *out);

/* ---- GEMM with LayerNorm folded in, and row statistics out ----------------------------------------------------------
 * No counterpart in the reference: the library form of "layernorm -> gemm" (frontend/siglip.py:136-162) without
 * materialising the normalised rows. With W' = diag(gamma) W, colsum = 1^T W' (fp32, 1 x N) and
 * d = beta W + bias (fp16, 1 x N, passed as `bias` with SH_EPI_BIAS),
 *     layernorm(X) W + bias = rstd_r (X W' - mean_r colsum) + d,
 * so the GEMM reads raw X. Flags (in addition to sh_cuda_gemm's):
 *   SH_EPI_LN_IN     t = rstd_r (acc - mean_r colsum[col]) first; mean_r / rstd_r (eps `ln_eps`) come from
 *                    `ln_stats`: K / 64 (sum, sum of squares) fp32 pairs per row, K % 64 == 0
 *   SH_EPI_STATS_OUT write N / 64 (sum, sum of squares) fp32 pairs per row of the final outputs (before fp16
 *                    rounding) to `stats_out`, N % 64 == 0: the next GEMM's ln_stats
 * No split-K; 16-byte aligned operands. Returns 0 or -1 (reason printed). */
#define SH_EPI_LN_IN      0x40u
#define SH_EPI_STATS_OUT  0x80u
int sh_cuda_gemm_ln(uint64_t x, uint64_t w, uint64_t z, uint32_t M, uint32_t N, uint32_t K, uint32_t ldx,
                    uint32_t ldw, uint32_t ldz, uint64_t bias, uint64_t residual, uint32_t ldr, uint32_t flags,
                    uint64_t ln_stats, uint64_t ln_colsum, float ln_eps, uint64_t stats_out);
/* (sum, sum of squares) of every 64 columns of each row of X (cols % 64 == 0): the row statistics of a matrix no
 * GEMM produced (the encoder's input). Returns 0 or -1. */
int sh_cuda_row_stats(uint64_t x, uint32_t rows, uint32_t cols, uint32_t ld, uint64_t stats_out);
/* dst[r, c] = src[r, c] * gamma[r] in fp16 (W' = diag(gamma) W for sh_cuda_gemm_ln). Returns 0 or -1. */
int sh_cuda_scale_rows(uint64_t dst, uint64_t src, uint32_t rows, uint32_t cols, uint32_t ld_src, uint32_t ld_dst,
                       uint64_t gamma);

/* ---- split-K GEMM without allocation -------------------------------------------------------------------------
 * No counterpart in the reference. The same computation, arguments and return codes as sh_cuda_gemm, for callers
 * that cannot let the library call cudaMalloc (a host whose own pool owns all device memory, or a loop that cannot
 * take cudaMalloc's implicit device synchronisation). Split-K partial tiles and arrival counters live in one fixed
 * 8 MiB array compiled into the library (held on every GPU that loads it until exit) instead of a growable
 * workspace; a call needing more (tiles x splits x 128 x BN x 4 bytes of partials, or more than 4096 tiles) returns
 * -2. The first call on a device looks the array up with cudaGetSymbolAddress and should come before any stream
 * capture. Calls share the array: calls that overlap on the GPU race and must be serialised by the caller. */
int sh_cuda_gemm_splitk_noalloc(uint64_t x, uint64_t w, uint64_t z, uint32_t M, uint32_t N, uint32_t K, uint32_t ldx,
                                uint32_t ldw, uint32_t ldz, uint64_t bias, uint64_t residual, uint32_t ldr,
                                uint32_t flags, uint32_t splits);

/* ---- fused residual add + LayerNorm ---------------------------------------------------------------------------
 * h = a + b (stored, fp16), y = layernorm(h) * gamma + beta, both rows x cols with leading dim ld. */
void sh_cuda_add_layernorm(uint64_t h, uint64_t y, uint64_t a, uint64_t b, uint64_t gamma, uint64_t beta,
                           uint32_t rows, uint32_t cols, uint32_t ld, float eps);

/* ---- attention over a batch of sequences ------------------------------------------------------------------------
 * B sequences of S rows stacked along the rows of q/k/v/o (sequence b = rows [b S, (b+1) S)); otherwise
 * sh_attention. Returns 0 or -1. */
int sh_cuda_attention_batched(uint64_t q, uint64_t k, uint64_t v, uint64_t o, uint32_t S, uint32_t D, uint32_t H,
                              uint32_t ldq, uint32_t ldk, uint32_t ldv, uint32_t ldo, float scale, uint32_t B);

/* ---- decoding: paged 8-bit K / V cache and 4-bit weights ------------------------------------------------------------
 * No counterpart in the reference (its attention reads whole fp16 K / V matrices, runtime/sh_ops.h:109-127, 277-304, and
 * its GEMMs fp16 weights). One decode step of a batch of requests is
 *     sh_cuda_gemv_w4 (Q|K|V) -> sh_rope -> sh_cuda_kv_tables -> sh_cuda_kv8_append -> sh_cuda_attention_kv8
 *     -> sh_cuda_gemv_w4 (output projection), ...
 * all on the library stream, with every length on the device, so that a step can be captured into a graph and replayed.
 *
 * The cache holds `pages` pages of `page` tokens. The codes of page p, head h, token t, column d are the bytes
 *     k[p * page_stride + (h * page + t) * dh + d], v[the same]
 * and stand for code * k_scale[p * heads + h] (v_scale for v): one fp32 scale, >= 0, per page and head.
 *   fmt    SH_INT8 (two's complement) or SH_FP8 (e4m3: 4 exponent bits, bias 7; the NaN codes 0x7F, 0xFF stay unused)
 *   page   16, 32, 64 or 128;  dh  64 or 128;  pages * page < 2^31
 *   page_stride  bytes from page to page, a multiple of 16, >= heads * page * dh (more when K and V pages alternate in
 *                one allocation)
 *   k, v   16-byte aligned; k_scale, v_scale 4-byte aligned
 * The struct is read during the call only. */
typedef struct sh_cuda_kv8_t {
    uint64_t k, v, k_scale, v_scale, page_stride;
    uint32_t pages, page, heads, dh, fmt;
} sh_cuda_kv8_t;

/* Block tables and slot maps of one step from the requests' lengths. For R <= 8192 requests (int32 arrays on the
 * device): lens[r] tokens are in the cache and add[r] follow in this step (0: none; < 0: the request has ended).
 * table[r * ld_table + b] is the page of tokens [b page, (b + 1) page) of request r, ring[pages] the free pages in the
 * order of their use: `count` entries from index `head` on, modulo pages, with pool = {head, count, ..}, eight words.
 *   - A request that needs new pages takes them from the ring's head, requests in order. Requests whose blocks would
 *     pass ld_table, and all from the first one on that the ring cannot serve whole, are put off: they keep their
 *     length and get no slots (requests that need no new page are served all the same).
 *   - A request that has ended gives its pages to the ring's tail (its table row is left as it was) and has length 0
 *     afterwards; pages given back can be taken from the next call on.
 * Writes: the new entries of table and ring; lens_out[R]; q_start[R + 1], the first row of each request's new tokens;
 * for row i < t_cap slots[i] = page * (tokens per page) + offset and pos[i] = the token's position in its request (the
 * row of a RoPE table), or slot -1 for the rows of put-off requests, and slot -1, pos 0 for rows past the last token;
 * pool_out = {head, count, number of requests put off, ..}. lens_out may be lens and pool_out may be pool (a running
 * pool); with other addresses a call can be repeated. lens[r] + add[r] and the sum of all add > 0 stay below 2^31; rows
 * from t_cap on get table entries but no slot. R == 0 writes nothing. Words 3..6 of pool_out are left alone, word 7 belongs to the
 * library: zero before the first call. Returns 0 or -1 (reason printed). */
int sh_cuda_kv_tables(uint64_t lens, uint64_t add, uint32_t R, uint32_t page, uint64_t table, uint32_t ld_table,
                      uint64_t ring, uint32_t pages, uint64_t pool, uint64_t pool_out, uint64_t lens_out,
                      uint64_t q_start, uint64_t slots, uint64_t pos, uint32_t t_cap);

/* The rows k[T, heads * dh], v[T, heads * dh] (fp16, leading dims ldk, ldv) into the cache at slots[T] (int32; < 0: no
 * row). Tokens of one page follow one another with rising slots, as sh_cuda_kv_tables lays them out; rows of a page
 * before the first new one are its older tokens, rows after the last new one are left as they were. Per page and head
 *     s' = max(s if there are older tokens, up8(max |x| / qmax)),  code = round(x / s'),  qmax = 127 or 448,
 * rounding to nearest even, up8 = the next value with 8 significant bits (no quotient then lies within rounding error
 * of a border between two codes without lying on it, so every correct division gives the same codes); when s' > s
 * the older codes become round(code s / s'). +-infinity counts as +-65504, NaN as 0. A slot past the cache, or one
 * that does not rise within its page, is not written and raises the device error word (2); a page whose tokens
 * do not follow one another is left with unspecified codes. Returns 0, -1, or -3 for fmt. */
int sh_cuda_kv8_append(const sh_cuda_kv8_t *cache, uint64_t k, uint64_t v, uint32_t T, uint32_t ldk, uint32_t ldv,
                       uint64_t slots);

/* Attention of the new rows of R requests over the cache: row q_start[r] + i of q (i < q_start[r + 1] - q_start[r] = n)
 * is a query of request r, which has lens[r] tokens in the cache, these n last, and attends its tokens
 * j <= lens[r] - n + i; query head h reads head h / (H / heads) of the cache. o = softmax(scale q k^T) v in the rows of q,
 * fp16 (leading dims ldq, ldo); a row without any token gives zeros, an infinity or a NaN in a row of q NaN in its head
 * (where the row has a token); rows of o outside [q_start[0], q_start[R]) and past T are left as they were. The rows of a
 * request that was put off are not in the cache: they attend its tokens as if they were its last ones, and their outputs are to
 * be ignored. One token per request, a few drafted ones, and whole prompt chunks are all served, in any mixture. q holds T rows;
 * max_q, the most rows of one request, picks the kernel for all of them: a wrong value costs time. With max_q * H / heads > 64
 * the softmax weights are rounded to fp16 (2^-11 of each, next to the same rounding of the output), else only the output is,
 * so a row's last bits depend on the side that max_q is on. ws: ws_bytes >= SH_CUDA_KV8_WS_BYTES of device memory, 16-byte aligned, zeroed once before its first use,
 * for the calls of one stream at a time (a graph that may run beside other calls has its own). A table entry outside the
 * cache, or a length past ld_table * page, raises the device error word (2) and those tokens are left out. T * H < 2^31 and
 * T + ld_table * page <= 2^31 - 2^14. Returns 0, -1, or -3 for fmt. */
#define SH_CUDA_KV8_WS_BYTES (48u << 20)
int sh_cuda_attention_kv8(uint64_t q, uint64_t o, const sh_cuda_kv8_t *cache, uint64_t table, uint32_t ld_table,
                          uint64_t lens, uint64_t q_start, uint32_t R, uint32_t T, uint32_t max_q, uint32_t H,
                          uint32_t ldq, uint32_t ldo, float scale, uint64_t ws, size_t ws_bytes);

/* Z[M, N] = epi(X[M, K] . W[K, N]) for 1 <= M <= 32 rows and 4-bit weights: row n of `codes` (ldw bytes, a multiple of 16,
 * >= K / 2; 16-byte aligned) holds the codes of column n of W, k = 2 i in the low and k = 2 i + 1 in the high half of
 * byte i, and W[k, n] = scales[n, k / group] * (code - zeros[n, k / group]): fp16 scales and uint8 zero points (0..15)
 * of K / group columns, zeros == 0 meaning 8 everywhere. group 32, 64 or 128, K % group == 0, K <= 262144. X, Z fp16 with
 * leading dims ldx, ldz; fp32 accumulation in a fixed order. flags: SH_EPI_BIAS and SH_EPI_RESIDUAL as in sh_cuda_gemm
 * (Z may be the residual, not X). Returns 0 or -1 (reason printed). */
int sh_cuda_gemv_w4(uint64_t x, uint64_t codes, uint64_t scales, uint64_t zeros, uint64_t z, uint32_t M, uint32_t N,
                    uint32_t K, uint32_t ldx, uint32_t ldw, uint32_t ldz, uint32_t group, uint64_t bias,
                    uint64_t residual, uint32_t ldr, uint32_t flags);

/* ---- synthetic inputs -------------------------------------------------------------------------------------------
 * N(mean, std) fp16 from the LCG of sh_test_fill_fp16: per element two draws d0, d1, u = (d + 0.5) / 2^24 and
 * Box-Muller z = sqrt(-2 ln u0) cos(2 pi u1), with ln and cos evaluated as fixed series of correctly rounded fp32
 * operations (no library math, no FMA contraction), so every implementation of the definition gives the same bits.
 * sh_cuda_fill_normal_fp16 fills device memory on the library stream; sh_cuda_host_fill_normal_fp16 fills host
 * memory (fp16 codes) on the calling CPU thread and needs no GPU. */
void sh_cuda_fill_normal_fp16(uint64_t a, uint32_t rows, uint32_t cols, uint32_t ld, uint32_t seed, float mean,
                              float stdev);
void sh_cuda_host_fill_normal_fp16(uint16_t *dst, uint32_t rows, uint32_t cols, uint32_t ld, uint32_t seed,
                                   float mean, float stdev);

/* ---- LCG sub-block fill (2-D block-distributed inputs) -----------------------------------------------------------
 * Fill rows x cols (leading dim ld) with elements [row0 .., col0 ..] of the global gcols-wide matrix that
 * sh_test_fill_fp16(.., seed, lo, hi, scale) would produce: every rank generates exactly its own block. */
void sh_cuda_fill_lcg_block(uint64_t a, uint32_t rows, uint32_t cols, uint32_t ld, uint32_t seed, int lo, int hi,
                            float scale, uint64_t row0, uint64_t col0, uint64_t gcols);

/* ---- HBM preload images -------------------------------------------------------------------------------------------
 * No counterpart in the reference's C runtime (its simulator loads the image at reset): the ELF32 images of
 * softhier_mlir/sim/preload.py (one PT_LOAD segment per array, physical address hbm_base + HBM offset, hbm_base
 * 0xC0000000 there) copied into the arena at sh_hbm_addr(offset) with synchronous copies; bytes between a
 * segment's file size and memory size are zeroed. Returns the number of segments, -1 (bad file) or -2 (a segment
 * outside the arena). sh_preload_elf_segments only lists the segments (offsets, memory sizes; no GPU needed) and
 * returns their count. */
int sh_cuda_preload_elf(const char *path, uint64_t hbm_base);
int sh_preload_elf_segments(const char *path, uint64_t hbm_base, uint64_t *offsets, uint64_t *sizes,
                            uint32_t max_segments);

/* ---- peer memory for the multi-GPU SUMMA --------------------------------------------------------------------------
 * Device buffers that other processes of the node can map (CUDA IPC), and asynchronous 2-D copies between any two
 * device addresses of the node (copy engines over NVLink when source and destination are on different GPUs). */
void *sh_cuda_ipc_alloc(size_t bytes);                     /* cudaMalloc'd, exportable; NULL on failure */
int   sh_cuda_ipc_free(void *p);
int   sh_cuda_ipc_handle(void *p, void *handle64);          /* 64-byte handle of a sh_cuda_ipc_alloc buffer */
void *sh_cuda_ipc_open(const void *handle64);               /* map a peer's buffer into this process */
int   sh_cuda_ipc_close(void *p);
int   sh_cuda_copy2d(uint64_t dst, size_t dpitch, uint64_t src, size_t spitch, size_t width_bytes, size_t rows,
                     void *stream);

#ifdef __cplusplus
}
#endif
#endif /* SH_OPS_CUDA_H */
