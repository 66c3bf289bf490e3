/*
 * cutie.h — C ABI of the B200 (sm_100a) residual-add + RMSNorm + FP8 (e4m3)
 * activation-quantization path.
 *
 * Every entry point is destination-passing: the caller owns and preallocates
 * all device buffers, nothing is allocated inside, and the work is enqueued
 * asynchronously on the caller's CUDA stream (`stream` is a cudaStream_t; NULL
 * means the legacy default stream) on the calling thread's current device.
 * No C++ exception crosses this boundary: every function returns a status code
 * (CUTIE_OK == 0) and, on failure, a message readable through
 * cutie_last_error() on the same thread.
 *
 * Reference interfaces replaced (paths within the S1ro1/thingy project):
 *   cutie_rms_norm_fp8          <- RMSNorm.__call__ / rms_norm_kernel
 *                                  (src/cutie/rms_norm/rms_norm.py:50-311),
 *                                  compiled and bound through cute.compile at
 *                                  src/cutie/rms_norm/bench.py:278-301, and the
 *                                  functional reference it must agree with,
 *                                  residual_rms_norm_fp8_reference
 *                                  (src/cutie/rms_norm/bench.py:83-100).
 *   cutie_per_token_cast_to_fp8 <- per_token_cast_to_fp8_triton /
 *                                  _per_token_fp8_kernel
 *                                  (src/cutie/vendor/prime_rl/fp8_utils.py:21-89),
 *                                  the op behind the custom op
 *                                  cutie::per_token_fp8_quant
 *                                  (src/cutie/rms_norm/bench.py:68-80).
 *   cutie_rms_norm              <- rms_norm / rms_norm_on_stream
 *                                  (src/cutie/rms_norm/rms_norm.py:11-33, fp32)
 *                                  and rms_norm_reference
 *                                  (src/cutie/rms_norm/bench.py:58-65, bf16).
 */
#ifndef CUTIE_H_
#define CUTIE_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define CUTIE_ABI_VERSION 1

#if defined(__GNUC__)
#define CUTIE_API __attribute__((visibility("default")))
#else
#define CUTIE_API
#endif

/* ---- status codes ------------------------------------------------------- */
enum cutie_status {
  CUTIE_OK = 0,
  CUTIE_ERR_INVALID_ARGUMENT = -1, /* bad shape, null pointer, bad enum      */
  CUTIE_ERR_UNSUPPORTED = -2,      /* valid request this build cannot serve  */
  CUTIE_ERR_ALIGNMENT = -3,        /* pointer / leading dim not 16-B aligned */
  CUTIE_ERR_CUDA = -4,             /* a CUDA runtime call failed             */
};

/* ---- quantization granularity (who shares one scale) -------------------- */
enum cutie_quant_mode {
  CUTIE_QUANT_NONE = 0,  /* no FP8 output (plain RMSNorm)                    */
  CUTIE_QUANT_TOKEN = 1, /* one scale per row (group = H)                    */
  CUTIE_QUANT_GROUP = 2, /* one scale per `group_size` contiguous elements   */
};

/* ---- how a scale is encoded --------------------------------------------- */
enum cutie_scale_fmt {
  CUTIE_SCALE_FP32 = 0,      /* fp32 s = max(amax/448, 1e-4)                 */
  CUTIE_SCALE_FP32_POW2 = 1, /* fp32 s = 2^ceil(log2(max(amax/448, 1e-4)))   */
                             /* (the reference's use_ue8m0=True rule)        */
  CUTIE_SCALE_E8M0 = 2,      /* one byte: biased exponent of the POW2 scale  */
};

/* ---- where scale (row m, group g) lives --------------------------------- */
enum cutie_scale_layout {
  CUTIE_LAYOUT_ROW_MAJOR = 0,   /* scale[m * ld_scale + g], ld >= n_groups   */
  CUTIE_LAYOUT_COL_MAJOR = 1,   /* scale[g * ld_scale + m], ld >= M          */
  CUTIE_LAYOUT_MX_SWIZZLED = 2, /* Blackwell block-scaled-GEMM layout:       */
  /* 128x4 tiles of 512 bytes, tile (m/128, g/4) at ((m/128)*ceil(G/4)+g/4)*512,
   * inside a tile (m%32)*16 + ((m%128)/32)*4 + g%4. Rows are padded to a
   * multiple of 128 and groups to a multiple of 4; padding bytes are written
   * as 0. Requires CUTIE_SCALE_E8M0. ld_scale is ignored.                   */
  CUTIE_LAYOUT_COL_MAJOR_PACKED = 3, /* e8m0 exponents packed four to a     */
  /* little-endian 32-bit word along the groups, words M-major: scale (m, g) is
   * byte g%4 of word (g/4)*ld_scale + m, i.e. byte offset
   * (g/4)*4*ld_scale + 4*m + g%4 (the packed UE8M0 scale tensor that
   * DeepGEMM-style SM100 FP8 GEMMs take: int32 [M, ceil(G/4)], stride
   * (1, ld_scale)). ld_scale counts words, >= M; 0 means M rounded up to a
   * multiple of 4 (16-byte aligned columns). Bytes of groups past the last
   * one in the final word are not written. Requires CUTIE_SCALE_E8M0.
   * No counterpart in the reference, which writes fp32 row-major scales.  */
};

/* ---- element types for cutie_rms_norm ----------------------------------- */
enum cutie_dtype {
  CUTIE_DTYPE_BF16 = 0,
  CUTIE_DTYPE_F32 = 1,
  CUTIE_DTYPE_F16 = 2, /* moe rows and optimizer only */
};

/*
 * Fused [residual add] -> RMSNorm -> [FP8 e4m3 quantization].
 *
 *   r   = bf16(x + residual)                (or r = x when residual is NULL)
 *   inv = 1 / RN(sqrt(RN(sum(r^2) / H) + eps))            (fp32 statistics)
 *   n   = bf16( bf16(r * inv) * weight )    (cast before the weight multiply)
 *   per group: amax = max|n|, s = max(amax / 448, 1e-4) [, rounded up to 2^k]
 *   q   = e4m3_rne(RN(n / s))
 *
 * x, residual, weight, residual_out, normalized_out: bf16. q: e4m3 bytes.
 * M >= 0 rows, H > 0 columns, H % 8 == 0; in CUTIE_QUANT_GROUP mode
 * group_size is 32, 64 or 128 and the last group of a row may be partial
 * (n_groups = ceil(H / group_size)). Leading dimensions are in elements; every
 * row must start 16-byte aligned. residual_out / normalized_out may be NULL
 * (not written); residual_out requires residual. q and scale may be NULL only
 * when quant_mode == CUTIE_QUANT_NONE. ld_scale == 0 selects the dense leading
 * dimension (n_groups for row-major, M for column-major).
 * threads_per_row: 0 picks the launch shape; otherwise a multiple of 32 in
 * [32, 1024] that must cover the row with at most 8 16-byte vectors a thread.
 */
CUTIE_API int cutie_rms_norm_fp8(const void* x, int64_t ldx,
                       const void* residual, int64_t ldr,
                       const void* weight, float eps,
                       int64_t M, int64_t H,
                       int quant_mode, int group_size,
                       int scale_fmt, int scale_layout, int64_t ld_scale,
                       void* q, int64_t ldq, void* scale,
                       void* residual_out, int64_t ldro,
                       void* normalized_out, int64_t ldn,
                       int threads_per_row, void* stream);

/*
 * Quantization alone: bf16 x [M, H] -> e4m3 q [M, H] + scales, one scale per
 * (row, group). Same scale rules, formats and layouts as above; group_size 0
 * means one scale per row. Mirrors per_token_cast_to_fp8_triton(x, use_ue8m0,
 * gran_k) (src/cutie/vendor/prime_rl/fp8_utils.py:63-89), whose defaults are
 * group_size 128, CUTIE_SCALE_FP32 (use_ue8m0=False) or CUTIE_SCALE_FP32_POW2
 * (use_ue8m0=True), row-major [M, ceil(H/128)] scales.
 */
CUTIE_API int cutie_per_token_cast_to_fp8(const void* x, int64_t ldx,
                                int64_t M, int64_t H, int group_size,
                                int scale_fmt, int scale_layout,
                                int64_t ld_scale,
                                void* q, int64_t ldq, void* scale,
                                int threads_per_row, void* stream);

/*
 * Standalone RMSNorm, out = f(x) [M, H].
 *   dtype == CUTIE_DTYPE_BF16: out = bf16(bf16(x * inv) * w), inv as above
 *     (rms_norm_reference, src/cutie/rms_norm/bench.py:58-65).
 *   dtype == CUTIE_DTYPE_F32:  out = RN(RN(x / RN(sqrt(RN(mean(RN(x^2))) + eps))) * w)
 *     (rms_norm, src/cutie/rms_norm/rms_norm.py:11-20).
 * x, weight and out share `dtype`. H % 8 == 0 (bf16) or H % 4 == 0 (f32).
 */
CUTIE_API int cutie_rms_norm(const void* x, int64_t ldx, const void* weight, float eps,
                   int64_t M, int64_t H, int dtype,
                   void* out, int64_t ldo, int threads_per_row, void* stream);

/*
 * Backward of cutie_rms_norm_fp8 (bf16, with or without a residual). The
 * reference has no backward pass (src/cutie/rms_norm/bench.py is forward
 * only); these are the gradients torch autograd gives its PyTorch forward
 * (bench.py:58-65 and the residual add of bench.py:97), op for op in fp32:
 *   inv = the forward's inv_rms of r;  dt = bf16(dn * w);  b = sum(dt * r)
 *   dx  = bf16(bf16(dt * inv + ((-0.5 * b) * inv^3 / H) * (2 * r)) + dro)
 *   dw  = bf16(sum over rows of bf16(dn * bf16(r * inv)))
 * d_normalized (dn): bf16 [M, H] gradient of the normalized output;
 * r: bf16 [M, H], the forward's RMSNorm input (x + residual, i.e.
 * residual_out, or x); d_residual_out (dro): gradient of residual_out, or
 * NULL; dx: bf16 [M, H], the gradient of x and of residual; d_weight: bf16
 * [H] or NULL. The weight gradient is summed per CTA into `workspace` (fp32,
 * at least cutie_rms_norm_backward_workspace(M, H) bytes, 16-byte aligned,
 * caller-owned, contents need not be initialised) and reduced over CTAs in a
 * fixed order, so it is deterministic. quant_mode CUTIE_QUANT_GROUP with
 * group_size 128 also writes dx as FP8 codes q + scales (formats and layouts
 * as in cutie_rms_norm_fp8); CUTIE_QUANT_NONE writes none. H % 8 == 0,
 * H <= 32768. Asynchronous on `stream`; nothing is allocated.
 */
CUTIE_API int cutie_rms_norm_backward(const void* d_normalized, int64_t ldd,
                                      const void* r, int64_t ldr, const void* weight,
                                      const void* d_residual_out, int64_t lddr,
                                      float eps, int64_t M, int64_t H,
                                      void* dx, int64_t lddx, void* d_weight,
                                      void* workspace, size_t workspace_bytes,
                                      int quant_mode, int group_size, int scale_fmt,
                                      int scale_layout, int64_t ld_scale,
                                      void* q, int64_t ldq, void* scale, void* stream);

/* Workspace bytes cutie_rms_norm_backward needs for d_weight on the current
 * device (one fp32 row of H partial sums per CTA of its grid). */
CUTIE_API size_t cutie_rms_norm_backward_workspace(int64_t M, int64_t H);

/*
 * cutie_rms_norm_backward without a workspace argument: it allocates nothing
 * and needs no device memory from the caller beyond inputs and outputs. It
 * has no counterpart in the reference. It is for callers that cannot
 * allocate device memory: code that runs where a cudaMalloc is not allowed
 * or must not happen (inside an allocator's or a framework's callbacks, a
 * plug-in whose host owns every device buffer, a memory pool that must not
 * grow), or that cannot hold a workspace between calls.
 *
 * The partial sums of d_weight go to a device array of the library instead:
 * 2^20 floats (4 MiB), present on every GPU that loads the library until the
 * process exits. Its CTAs are capped so that their rows of H partial sums
 * fit (2^20 / H CTAs, e.g. 146 at H = 7168), so d_weight is summed in a
 * different grouping than cutie_rms_norm_backward's (the same bound on the
 * error; dx, q and scale are identical). The cap costs time where it is
 * below the regular grid: measured on a B200 (residual gradient, 1x128 FP8
 * copy of dx) 210.6 against 183.4 us at 16384 x 7168 (146 CTAs), 122.8
 * against 116.6 us at 16384 x 4096, 881 against 236 us at 2048 x 32768
 * (32 CTAs). Sizes: as cutie_rms_norm_backward
 * (H <= 32768, which always fits the array); a larger H is refused with
 * CUTIE_ERR_UNSUPPORTED. Every row of the array that a call reads was
 * written by that call, so nothing needs clearing between calls.
 *
 * Every call resolves the array's device address in the calling thread's
 * current context (cudaGetSymbolAddress; nothing is cached, so the address
 * stays right after cudaDeviceReset or under another driver context). The
 * first call in a context also loads the library's device code there: make
 * that first call before any stream capture. All calls on a device share the
 * one array, so calls that may run at the same time on the GPU (other
 * streams, other host threads) race on it and give wrong d_weight: order
 * them on one stream.
 */
CUTIE_API int cutie_rms_norm_backward_noalloc(const void* d_normalized, int64_t ldd,
                                              const void* r, int64_t ldr, const void* weight,
                                              const void* d_residual_out, int64_t lddr,
                                              float eps, int64_t M, int64_t H,
                                              void* dx, int64_t lddx, void* d_weight,
                                              int quant_mode, int group_size, int scale_fmt,
                                              int scale_layout, int64_t ld_scale,
                                              void* q, int64_t ldq, void* scale, void* stream);

/*
 * MXFP8 block-scaled GEMM on the tensor cores, the consumer of this path's
 * 1x32 codes and swizzled e8m0 scales (no counterpart in the reference, whose
 * bench stops before the GEMM, src/cutie/rms_norm/bench.py:4-7):
 *   D[m, n] = bf16( sum_k A[m, k] 2^(sA[m, k/32] - 127) * B[n, k] 2^(sB[n, k/32] - 127) )
 * with fp32 accumulation. a: e4m3 [M, K] (K contiguous, lda bytes between
 * rows), a_scale: its e8m0 scales in CUTIE_LAYOUT_MX_SWIZZLED for [M, K/32]
 * (rows padded to 128, as cutie_rms_norm_fp8 writes them); b: e4m3 [N, K]
 * (ldb) with b_scale likewise for [N, K/32]; d: bf16 [M, N] (ldd elements).
 * N and K multiples of 128, any M >= 0; a, b, d rows and both scale buffers
 * 16-byte aligned. Asynchronous on `stream`; nothing is allocated.
 */
CUTIE_API int cutie_gemm_mxfp8(const void* a, int64_t lda, const void* a_scale,
                               const void* b, int64_t ldb, const void* b_scale,
                               void* d, int64_t ldd, int64_t M, int64_t N, int64_t K,
                               void* stream);

/*
 * RMSNorm -> MXFP8 quantization -> block-scaled GEMM in ONE kernel: the
 * norm-and-quantize step becomes the GEMM's A-operand prologue, so the FP8
 * codes and scales of the activation never leave the chip (no counterpart in
 * the reference; it composes rms_norm_reference, src/cutie/rms_norm/bench.py:
 * 58-65, the 1x32 UE8M0 quantizer rule of src/cutie/vendor/prime_rl/
 * fp8_utils.py:50-57 with gran_k 32, and the GEMM its output feeds):
 *   A = cutie_rms_norm_fp8(x, weight, eps, group 32, e8m0, swizzled) codes,
 *   D[m, n] = bf16( sum_k A[m, k] 2^(sA[m, k/32] - 127) * b[n, k] 2^(sB[n, k/32] - 127) )
 * x: bf16 [M, K] (ldx elements, 16-byte aligned rows), weight: bf16 [K];
 * b / b_scale / d as cutie_gemm_mxfp8. q / q_scale: both NULL, or an e4m3
 * [M, K] buffer (ldq bytes) and a swizzled e8m0 scale buffer that receive A
 * and its scales as cutie_rms_norm_fp8 would write them (for a backward pass
 * that keeps the quantized activation). N and K multiples of 128,
 * K <= 65536. The CTAs that share 128 rows of x run as a thread-block cluster
 * (8, 4, 2 or 1 CTAs along N, the largest that divides N / 128) and quantize
 * each A tile once between them. Asynchronous on `stream`; nothing is
 * allocated.
 */
CUTIE_API int cutie_rms_norm_mxfp8_gemm(const void* x, int64_t ldx, const void* weight,
                                        float eps, const void* b, int64_t ldb,
                                        const void* b_scale, void* d, int64_t ldd, int64_t M,
                                        int64_t N, int64_t K, void* q, int64_t ldq,
                                        void* q_scale, void* stream);

/*
 * Cast of a bf16 matrix x [M, H] (ldx elements between rows) to e4m3 in both
 * orientations, reading x once:
 *   s = max(amax / 448, 1e-4), rounded up to a power of two for
 *   CUTIE_SCALE_FP32_POW2; q = e4m3(x / s)
 * the rule of cutie_per_token_cast_to_fp8 (src/cutie/vendor/prime_rl/
 * fp8_utils.py:50-57), over
 *   CUTIE_TILE_BLOCK: 128 x 128 blocks (weights). s: fp32 [ceil(M/128),
 *     ceil(H/128)], lds elements between rows. qt / st (both NULL, or both
 *     given): the codes [H, M] of x's transpose and its scales
 *     [ceil(H/128), ceil(M/128)].
 *   CUTIE_TILE_TWO_WAY: 1 x 128 groups of the rows for q, 128 x 1 groups of
 *     the columns for qt (activations and gradients; qt and st are required).
 *     Scales are group-major: s element (row, g) at g * lds + row, st element
 *     (column, g) at g * ldst + column. CUTIE_SCALE_GRADIENT added to
 *     scale_fmt: a group with amax < 1e-4 has s = max(amax / 448, 2^-92). At
 *     the scale 1e-4 the codes of |x| < 9.8e-8 are all zero, and gradients are
 *     often smaller than that (2^-92 is the least scale for which the division
 *     stays correctly rounded; the codes of |x| < 2^-102 are zero).
 * Ragged last blocks and groups are reduced over their valid elements. H is a
 * multiple of 8, M >= 0 any; x rows 16-byte, q and qt rows 8-byte aligned
 * (16-byte for cutie_fp8_block_gemm). A group with an infinity gets an
 * infinite scale and NaN codes; a NaN gives a NaN code and does not count for
 * its group's scale. Asynchronous on `stream`; nothing is allocated.
 */
enum {
  CUTIE_TILE_BLOCK = 0,
  CUTIE_TILE_TWO_WAY = 1,
  CUTIE_TILE_BLOCK_F32 = 8, /* CUTIE_TILE_BLOCK of an fp32 x, rounded to bf16 first */
};
enum {
  CUTIE_SCALE_GRADIENT = 16, /* added to scale_fmt, CUTIE_TILE_TWO_WAY only  */
};
CUTIE_API int cutie_cast_fp8_tiles(const void* x, int64_t ldx, int64_t M, int64_t H,
                                   int tile_kind, int scale_fmt, void* q, int64_t ldq, void* s,
                                   int64_t lds, void* qt, int64_t ldqt, void* st, int64_t ldst,
                                   void* stream);

/*
 * FP8 product with a scale for each block of 128:
 *   D[m, n] = sum_kb sA[m, kb] sB[n, kb] sum_{k in block kb} a[m, k] b[n, k]
 * a: e4m3 [M, K] (lda bytes between rows), a_scale: fp32, element (m, kb) at
 * m * sa_row + kb * sa_kb (row- or group-major, as the quantizers write it).
 * b: e4m3 [N, K] (ldb), b_scale: element (n, kb) at (n / 128) * sb_row +
 * kb * sb_kb for 128 x 128 blocks (b_rows = 0), at n * sb_row + kb * sb_kb
 * for 1 x 128 groups (b_rows = 1). d: [M, N], ldd elements between rows, bf16
 * or fp32 (d_dtype: CUTIE_DTYPE_*); accumulate (fp32 only): D += the product.
 * The sum of a 128-wide block is made on the tensor cores in fp32, the sum
 * over blocks in fp32 registers, one rounding to bf16 at the end. M, N and K
 * may be any size >= 0 (K = 0: zeros, or D unchanged); a and b rows 16-byte
 * aligned (lda and ldb multiples of 16). Asynchronous on `stream`; nothing is
 * allocated.
 */
CUTIE_API int cutie_fp8_block_gemm(const void* a, int64_t lda, const void* a_scale,
                                   int64_t sa_row, int64_t sa_kb, const void* b, int64_t ldb,
                                   const void* b_scale, int64_t sb_row, int64_t sb_kb,
                                   int b_rows, void* d, int64_t ldd, int d_dtype, int accumulate,
                                   int64_t M, int64_t N, int64_t K, void* stream);

/*
 * The two-way cast (CUTIE_TILE_TWO_WAY) of rows sorted by expert
 * (cutie_moe_sort with align a multiple of 128): rows whose source is -1 count as
 * zeros, whatever x holds there; all codes and scales are written. R is a multiple
 * of 128.
 */
CUTIE_API int cutie_cast_fp8_sorted(const void* x, int64_t ldx, int64_t R, int64_t H,
                                    const void* sources, int scale_fmt, void* q, int64_t ldq,
                                    void* s, int64_t lds, void* qt, int64_t ldqt, void* st,
                                    int64_t ldst, void* stream);

/*
 * The experts' products on sorted rows: for each expert e, rows offsets[e] to
 * offsets[e + 1] of
 *   D = dequant(A) dequant(B[e])^T
 * and zeros in padding, the rows of e from offsets[e] + counts[e] on, and in
 * the rows before the first expert's and behind the last's. A: e4m3 [R, K] (lda), fp32
 * scales of 1 x 128 groups, element (r, kb) at r * sa_row + kb * sa_kb. B:
 * e4m3 [E, N, K], row n of expert e at e * b_expert + n * ldb, fp32 scales of
 * 128 x 128 blocks at e * sb_expert + nb * sb_row + kb * sb_kb. D: bf16 or fp32
 * [R, N] (ldd). offsets: int32 [E + 1] on the GPU, multiples of 128 that do
 * not decrease, the last at most R (cutie_moe_sort, align 128); counts: int32
 * [E] likewise, or NULL: no padding; E <= 512, R a multiple of 128. Rows of A and B and b_expert on 16-byte, rows of D on
 * 32-byte boundaries, N a multiple of 16 (fp32: 8). With B's strides exchanged
 * the same call is the input gradient. Sums as in cutie_fp8_block_gemm.
 */
CUTIE_API int cutie_fp8_grouped_gemm(const void* a, int64_t lda, const void* a_scale,
                                     int64_t sa_row, int64_t sa_kb, const void* b, int64_t ldb,
                                     int64_t b_expert, const void* b_scale, int64_t sb_row,
                                     int64_t sb_kb, int64_t sb_expert, const void* offsets, const void* counts,
                                     int64_t E, void* d, int64_t ldd, int d_dtype, int64_t R,
                                     int64_t N, int64_t K, void* stream);

/*
 * The experts' weight gradients: D[e] = the product of A and B^T over the
 * columns offsets[e] to offsets[e + 1], zero for an expert without rows.
 * A: e4m3 [N, R], B: e4m3 [K, R], both with fp32 scales of 1 x 128 groups
 * (the transposes that cutie_cast_fp8_sorted makes of the gradient and of the
 * input). D: bf16 or fp32 [E, N, K], element (e, n, k) at e * d_expert + n *
 * ldd + k. Otherwise as above, with K in the place of N.
 */
CUTIE_API int cutie_fp8_grouped_wgrad(const void* a, int64_t lda, const void* a_scale,
                                      int64_t sa_row, int64_t sa_kb, const void* b, int64_t ldb,
                                      const void* b_scale, int64_t sb_row, int64_t sb_kb,
                                      const void* offsets, int64_t E, void* d, int64_t ldd,
                                      int64_t d_expert, int d_dtype, int64_t R, int64_t N,
                                      int64_t K, void* stream);

/*
 * A whole mixture-of-experts layer for few tokens in one kernel:
 *   logits = x router^T (fp32 sums of bf16 products); scores = softmax or
 *   sigmoid of the logits; each token takes the top_k experts of the largest
 *   logits (with a bias: of the largest score + bias), ties to the lowest
 *   index, NaN last; weights w = the chosen scores, divided by their sum if
 *   renormalize, times routed_scale (all NaN under softmax if any of the
 *   token's logits is)
 *   g, u = dequant(q) dequant(w13[e])^T; h = silu(g) u (fp32);
 *   (qh, sh) = the 1 x 128 cast of h: s = max(amax / 448, 1e-4), e4m3(h / s)
 *   out[t] = bf16( sum_j w[t, j] dequant(qh) dequant(w2[e_j])^T )
 * x: bf16 [T, H] (ldx), the router's input; q: e4m3 [T, H] (ldq bytes) with
 * fp32 scales of 1 x 128 groups, element (t, g) at t * sq_row + g * sq_kb: x
 * quantized, as cutie_rms_norm_fp8 writes both (normalized_out, q and scale).
 * router: bf16 [E, H]; bias: fp32 [E] or NULL. w13: e4m3 [E, 2 I, H], rows
 * 0..I-1 of an expert its gate, I..2I-1 its up projection, w2: e4m3
 * [E, H, I]; w13_scale [E, 2 I / 128, H / 128] and w2_scale [E, H / 128,
 * I / 128]: fp32, 128 x 128 blocks, all contiguous (cutie_cast_fp8_tiles).
 * out: bf16 [T, H] (ldo). topk_ids (int32) and topk_weights (fp32), [T,
 * top_k], receive the choices; either may be NULL.
 * 0 <= T <= 64, 1 <= E <= 512, 1 <= top_k <= min(E, 16), H and I multiples
 * of 128; rows of x, out 16-byte, of q 16-byte aligned.
 * workspace: cutie_moe_fp8_workspace(T, E, top_k, H, I) bytes of device
 * memory, 256-byte aligned, whose first 8 bytes are zero before its first
 * use; the kernel leaves them ready for the next call, of any sizes, on the
 * same device. Calls that may overlap on the GPU need workspaces of their
 * own. The kernel is a cooperative launch over the whole device. Asynchronous
 * on `stream`; nothing is allocated.
 */
enum cutie_moe_scoring {
  CUTIE_SCORE_SOFTMAX = 0,
  CUTIE_SCORE_SIGMOID = 1,
};
CUTIE_API size_t cutie_moe_fp8_workspace(int64_t T, int64_t E, int64_t top_k, int64_t H, int64_t I);
CUTIE_API int cutie_moe_fp8(const void* x, int64_t ldx, const void* q, int64_t ldq,
                            const void* q_scale, int64_t sq_row, int64_t sq_kb,
                            const void* router, const void* bias, const void* w13,
                            const void* w13_scale, const void* w2, const void* w2_scale,
                            int64_t T, int64_t E, int64_t top_k, int64_t H, int64_t I,
                            int scoring, int renormalize, float routed_scale, void* out,
                            int64_t ldo, void* topk_ids, void* topk_weights, void* workspace,
                            size_t workspace_bytes, void* stream);

/*
 * Tokens sorted by expert: the plan by which rows go to experts and back.
 * ids: int32 or int64 (wide) [T, k], contiguous: the experts that each token
 * takes; an id outside [0, E) is an absent choice (dropped, or another rank's).
 * Choices are sorted by expert, those of one expert in the order t k + j;
 * every expert's rows begin at a multiple of `align` (fp8 products: 128).
 *   sources[r]      = t k + j of sorted row r, -1 in padding       int32 [R]
 *   positions[t, j] = its sorted row, -1 where absent              int32 [T, k]
 *   offsets[e]      = where expert e's rows begin; offsets[E] ends int32 [E + 1]
 *   counts[e]       = its rows, without padding                    int32 [E]
 * R >= cutie_moe_plan_rows(T, k, E, align), the most rows that any ids need;
 * sources behind offsets[E] are -1. 1 <= E <= 512, 1 <= align <= 65536, k >= 1,
 * T k <= 2^30, R < 2^31. workspace: cutie_moe_sort_workspace(T, k, E) bytes, 4-byte
 * aligned (0: NULL will do). Asynchronous on `stream`; nothing is allocated.
 */
CUTIE_API int64_t cutie_moe_plan_rows(int64_t T, int64_t k, int64_t E, int64_t align);
CUTIE_API size_t cutie_moe_sort_workspace(int64_t T, int64_t k, int64_t E);
CUTIE_API int cutie_moe_sort(const void* ids, int wide, int64_t T, int64_t k, int64_t E,
                             int64_t align, void* sources, int64_t R, void* positions,
                             void* offsets, void* counts, void* workspace,
                             size_t workspace_bytes, void* stream);

/*
 * Rows to their experts: out[r] = x[sources[r] / k], zeros where sources[r]
 * is -1. x: [T, H], out: [R, H] of elements of element_bytes (1, 2, 4; codes
 * and scales too), leading dimensions in elements. The gradient of it is
 * cutie_moe_combine without weights.
 */
CUTIE_API int cutie_moe_permute(const void* x, int64_t ldx, int element_bytes, int64_t T,
                                int64_t H, int64_t k, const void* positions, const void* sources,
                                int64_t R, void* out, int64_t ldo, void* stream);

/*
 * Rows back to their tokens: out[t] = sum_j weights[t, j] rows[positions[t, j]],
 * absent choices left out; weights: fp32 [T, k] or NULL (all one). rows: [R, H],
 * out: [T, H], dtype CUTIE_DTYPE_*; sums in fp32 in the order of j, rounded once.
 */
CUTIE_API int cutie_moe_combine(const void* rows, int64_t ldr, int dtype, const void* weights,
                                const void* positions, int64_t T, int64_t k, int64_t H,
                                int64_t R, void* out, int64_t ldo, void* stream);

/*
 * Its gradients: d_rows[positions[t, j]] = weights[t, j] d_out[t], zeros where
 * sources[r] is -1; d_weights[t, j] = <d_out[t], rows[positions[t, j]]> in fp32,
 * 0 for absent choices. Either of d_rows and d_weights may be NULL; rows may be
 * NULL without d_weights.
 */
CUTIE_API int cutie_moe_combine_backward(const void* d_out, int64_t ldd, const void* rows,
                                         int64_t ldr, int dtype, const void* weights,
                                         const void* positions, const void* sources, int64_t T,
                                         int64_t k, int64_t H, int64_t R, void* d_rows,
                                         int64_t lddr, void* d_weights, void* stream);

/*
 * One step of AdamW over `count` tensors in as few launches as their table
 * needs (480 tensors each). For every element, in fp32, rounded operation by
 * operation (with codes only the states are, the update to a few 2^-24):
 *   g' = g grad_scale;  m' = b1 m + (1 - b1) g';  v' = b2 v + (1 - b2) (g' g')
 *   p' = p (1 - lr decay) - (lr / (1 - b1^step)) (m' / (sqrt(v') / sqrt(1 - b2^step) + eps))
 * params, grads, exp_avg, exp_avg_sq: host arrays of device pointers to sizes[i]
 * contiguous elements; param_dtype and grad_dtype: CUTIE_DTYPE_*, the same, or
 * fp32 gradients, or bf16 gradients of fp32 parameters. Without scales
 * (avg_scale, sq_scale NULL) the states are fp32; with them exp_avg holds e4m3
 * codes of m, exp_avg_sq of sqrt(v), and the scales fp32 values a group of 128
 * elements of a tensor (the last group may be shorter), max(amax / 448, 2^-92).
 * Codes are rounded up or down at random, the nearer the likelier, by a hash of
 * (seed, step, the tensor's index in the list, the element): the same inputs
 * give the same bits. An infinite gradient makes its group's codes NaN.
 * step >= 1, or step_ptr: an int64 on the GPU (read when the kernel runs, so a
 * captured call may count); lr, or lr_ptr: an fp32 on the GPU. grad_scale: an fp32
 * on the GPU or NULL. Any alignment of elements; 16-byte aligned tensors (codes
 * 8) are faster. No tensor may overlap another. Asynchronous on `stream`.
 */
CUTIE_API int cutie_adamw(int64_t count, void* const* params, int param_dtype,
                          const void* const* grads, int grad_dtype, void* const* exp_avg,
                          void* const* avg_scale, void* const* exp_avg_sq, void* const* sq_scale,
                          const int64_t* sizes, int64_t step, const void* step_ptr, double lr,
                          const void* lr_ptr, double beta1, double beta2, double eps,
                          double weight_decay, const void* grad_scale, uint64_t seed,
                          void* stream);

/*
 * Device-side status of this library's kernels on the current device: 0 when
 * no kernel has hit a failure since the last clear; otherwise the first error
 * code recorded (1 = a bulk-copy wait ran out: a row never arrived in shared
 * memory within ~2 s and the kernel stopped early, leaving outputs
 * incomplete, see cutie_set_wait_limit; 2 = a kernel was launched with a
 * shared-memory ring depth it does not hold and wrote nothing). Synchronises with the device; `clear` != 0
 * resets the word.
 * A negative return is a CUDA failure (see cutie_last_error()).
 */
CUTIE_API int cutie_device_error(int clear);

/*
 * Limit, in SM clock cycles, on every wait that the kernels launched later
 * by the calling thread make for their own bulk copies and exchanges
 * (cutie_gemm_mxfp8's keep the default). The default, about 2 s, bounds a copy
 * that never lands. A wait that runs out stops the kernel early with device
 * error 1 (cutie_device_error); the kernel first lets the copies it issued
 * land, so the GPU stays usable.
 * cycles == 0 restores the default; cycles < 0 makes every wait that would
 * have to block give up at once, which exercises that failure path with
 * valid inputs (the outputs of such a launch are incomplete). Affects this
 * thread only; returns the previous limit. No counterpart in the reference,
 * whose kernels have no waits that can run out.
 */
CUTIE_API int64_t cutie_set_wait_limit(int64_t cycles);

/* Message of the last failing call on this thread ("" if none). */
CUTIE_API const char* cutie_last_error(void);

/* CUTIE_ABI_VERSION of the loaded library. */
CUTIE_API int cutie_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* CUTIE_H_ */
