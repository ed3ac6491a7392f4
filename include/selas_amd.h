/*
 * selas_amd.h - C ABI of the MI355X (gfx950) NF4 hot path.
 *
 * One shared library, libselas_amd.so, built by hipcc from selas_amd/csrc/.
 * Every entry point:
 *   - takes plain device pointers, element counts and strides (in elements,
 *     not bytes), never a framework type;
 *   - launches asynchronously on the HIP stream passed as `stream` (a
 *     hipStream_t; pass the caller's current stream so that stream-ordered
 *     buffer reuse stays correct) and never synchronises the device;
 *   - allocates nothing and frees nothing: outputs and scratch memory are
 *     caller-owned (a tiled linear whose launch splits its last round of tiles
 *     over K takes a workspace argument, sized by selas_linear_workspace_bytes,
 *     and selas_attention_split one sized by selas_attention_workspace_bytes);
 *   - returns SELAS_OK or an error code and never throws; the message of the
 *     last error on the calling thread is returned by selas_last_error().
 *
 * Data formats follow the reference codec (selas/codecs.py:1-16, 58-63,
 * 86-119): NF4 weights are `packed` uint8 [numel/2] (element 2i in the high
 * nibble of byte i), `absmax` fp32 [numel/blocksize] over the flattened
 * tensor, and a 16-entry fp32 codebook passed by value from host memory
 * (the tensor's meta["code"]); int8_row weights are `q` int8 in the weight's
 * shape and `scale` fp32, one per row.
 *
 * Kernels, tile shapes and K splits are chosen from shapes, dtypes and pointer
 * alignment (and the GPU's CU count) only, never from streams, earlier calls or
 * allocation results, and use no atomics, so equal inputs give equal bits on
 * every call and every stream.
 */
#ifndef SELAS_AMD_H
#define SELAS_AMD_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Return codes. */
#define SELAS_OK 0
#define SELAS_EINVAL 1       /* invalid argument (sizes, dtypes, nulls): ValueError in the reference */
#define SELAS_EUNSUPPORTED 2 /* valid, but outside what a fused kernel covers: caller falls back */
#define SELAS_EHIP 3         /* HIP runtime or launch error */

/* Element types (the `dtype` arguments). */
#define SELAS_F32 0
#define SELAS_F16 1
#define SELAS_BF16 2
/* Integer types of selas_rope's positions. */
#define SELAS_I32 3
#define SELAS_I64 4

/* Weight codecs (the `codec` argument of selas_linear_workspace_bytes). */
#define SELAS_CODEC_NF4 0
#define SELAS_CODEC_INT8_ROW 1

/* Message of the last failed call on this thread ("" if none). */
const char *selas_last_error(void);

/* ABI version of this header (bumped on any new or changed signature). */
int selas_abi_version(void);

/* ------------------------------------------------------------------ codec */

/*
 * NF4 decode: out[2i]   = dtype(code[packed[i] >> 4] * absmax[i / (blocksize/2)])
 *             out[2i+1] = dtype(code[packed[i] & 15] * absmax[i / (blocksize/2)])
 * The fp32 product is rounded once, to nearest even, to out_dtype; the bits
 * equal the reference decode for every input except NaN payloads.
 * Replaces nf4_dequant / nf4_dequant_torch (selas/codecs.py:178-199, 260-266)
 * and the Triton kernel (codecs.py:207-228).
 */
int selas_nf4_dequant(const uint8_t *packed, const float *absmax, int64_t n_bytes, int64_t blocksize,
                      const float code[16], void *out, int out_dtype, void *stream);

/*
 * NF4 encode of an fp32 tensor of n elements (n % blocksize == 0, blocksize
 * even): absmax[b] = max |w| over block b; each element divided by the block's
 * absmax (1 where absmax is 0) is mapped to the number of codebook midpoints
 * (code[i]+code[i+1])/2 that are not >= it (ties go to the lower code), and
 * two codes are packed per byte, first element high.
 * Replaces encode_nf4 (selas/codecs.py:99-119).
 */
int selas_nf4_encode(const float *w, int64_t n, int64_t blocksize, const float code[16], uint8_t *packed,
                     float *absmax, void *stream);

/*
 * selas_nf4_encode of a tensor of dtype w_dtype (the exact conversion to fp32
 * is part of the kernel). 16-bit tensors need blocksize 64, 16-byte alignment
 * and a codebook whose midpoints ascend in (-1, 1), at most one in each of the 64
 * buckets [b, b + 1) of 31.999 m + 32 and none but 0 within 2e-6 of an edge of its
 * bucket (otherwise SELAS_EUNSUPPORTED: convert to fp32 first).
 */
int selas_nf4_encode_typed(const void *w, int w_dtype, int64_t n, int64_t blocksize, const float code[16],
                           uint8_t *packed, float *absmax, void *stream);

/*
 * int8_row decode of a weight of `rows` rows of `cols` elements (q int8
 * [rows, cols], scale fp32 [rows]):
 *   out[r, c] = dtype(float(q[r, c]) * float(dtype(scale[r])))
 * i.e. q.to(dtype) * scale.to(dtype) computed in dtype; for bf16 and fp16 the
 * product is exact in fp32 and rounded once. Bit-identical to the reference
 * decode (selas/codecs.py:273-277) except NaN payloads.
 */
int selas_int8_row_dequant(const int8_t *q, const float *scale, int64_t rows, int64_t cols, void *out,
                           int out_dtype, void *stream);

/*
 * int8_row encode of an fp32 weight [rows, cols]: scale[r] = max |w[r, :]| / 127
 * (1 where that max is not positive), q[r, c] = clamp(round_half_even(w[r, c] /
 * scale[r]), -127, 127), with IEEE fp32 division.
 * Replaces encode_int8_row (selas/codecs.py:86-96).
 */
int selas_int8_row_encode(const float *w, int64_t rows, int64_t cols, int8_t *q, float *scale, void *stream);

/*
 * selas_int8_row_encode of a weight of dtype w_dtype (the exact conversion to
 * fp32 is part of the kernel). 16-bit weights need 16-byte alignment and cols a
 * multiple of 8, at most 16384 (otherwise SELAS_EUNSUPPORTED: convert first).
 */
int selas_int8_row_encode_typed(const void *w, int w_dtype, int64_t rows, int64_t cols, int8_t *q, float *scale,
                                void *stream);

/* ------------------------------------------------------------ linear */

/*
 * Quantized linear forward y = x W^T + bias with W an NF4 [N, K] weight:
 *   x     [M, K]  dtype, row stride ldx (K contiguous)
 *   bias  [N]     dtype or NULL
 *   y     [M, N]  dtype, row stride ldy
 * dtype is SELAS_BF16 (fp32 accumulation, one rounding of acc + bias).
 * M > 32 runs a tiled MFMA GEMM with the dequantization fused into the operand
 * load; its operand is the reference's decoded weight bf16(code*absmax) bit for
 * bit. M <= 32 runs a skinny dequant-GEMM that multiplies x by the codes and
 * scales the fp32 block sums by absmax (for K = 1024, 2048, 3072 in fp16 after
 * an exact power-of-two rescale of parts of each row of x, by one kernel for M <= 2
 * and another up to 32; otherwise in bf16 with codes split into two bf16 terms); it
 * agrees with the decoded-weight product to the rounding of the decoded weight. A
 * row's bits do not depend on the other rows; they may differ in the last bit
 * between M <= 2, M <= 32 and the tiled GEMM. Every output of the tiled GEMM sums K in
 * one order, whatever M and the tile height, except where a launch splits its
 * last round of tiles over K (long K and a last round of few tiles, e.g.
 * M 6144, N 3072, K 15360): those tiles' K ranges are summed in fp32 by a
 * second kernel, in a fixed order, from fp32 partial tiles kept in `workspace`
 * (device memory of workspace_bytes >= selas_linear_workspace_bytes for this
 * shape, 16-byte aligned, not read or written by anything else until the
 * launch has run; NULL and 0 where that size is 0, otherwise SELAS_EINVAL).
 * Whether and how a launch splits depends on M, N, K and the CU count only.
 * Returns SELAS_EUNSUPPORTED
 * when the shape or layout is outside the fused kernels (blocksize != 64,
 * K % 64 != 0, misaligned rows, dtype other than bf16); the caller then
 * decodes with selas_nf4_dequant and uses a library GEMM.
 * Replaces UnitView.linear for NF4 weights (selas/store.py:289-293):
 * decode (codecs.py:269-280) followed by F.linear.
 */
int selas_nf4_linear(const void *x, int64_t M, int64_t K, int64_t ldx, const uint8_t *packed,
                     const float *absmax, int64_t blocksize, const float code[16], int64_t N,
                     const void *bias, void *y, int64_t ldy, int dtype, void *workspace, int64_t workspace_bytes,
                     void *stream);

/* At most this many linears per selas_nf4_linear_batched call. */
#define SELAS_MAX_BATCHED_LINEARS 4

/* One quantized linear of a batched launch (host-memory array element); the
 * first fields mean what the arguments of selas_nf4_linear mean.
 * gelu_cols (0 = none) makes the last gelu_cols output columns
 * y2[m, j] = bf16(gelu_tanh(bf16(x W^T + b)[m, N - gelu_cols + j])) instead, with
 * row stride ldy2: the GELU that follows the block's MLP input linears
 * (flux.py:194-200), applied to the rounded output exactly as a separate GELU
 * kernel would. N - gelu_cols must be a multiple of 256; with gelu_cols = N, y
 * is not written and may be NULL. */
typedef struct selas_nf4_gemm_problem {
  const void *x;
  int64_t M, K, ldx;
  const uint8_t *packed;
  const float *absmax;
  int64_t N;
  const void *bias;
  void *y;
  int64_t ldy;
  void *y2;
  int64_t ldy2, gelu_cols;
} selas_nf4_gemm_problem;

/*
 * Up to SELAS_MAX_BATCHED_LINEARS independent quantized linears (each its own
 * x, weight, bias and y; all M > 32) in one launch of the tiled GEMM: the
 * tiles of all problems share the GPU, so a small problem fills the CUs a
 * large one leaves idle in its last round. Each y has the bits
 * selas_nf4_linear gives for that problem alone, except in tiles that the
 * batch's launch splits over K (the plan, like the workspace it needs, depends
 * on all the problems' shapes: e.g. 4096- and 2048-token problems of
 * K 12288 together leave a last round of few tiles that neither leaves alone).
 * workspace / workspace_bytes as for selas_nf4_linear, sized by
 * selas_linear_workspace_bytes over the same problems. Returns SELAS_EUNSUPPORTED,
 * launching nothing, when any problem is outside the tiled GEMM (M <= 32 or
 * any reason selas_nf4_linear would give); the caller then runs them one by one.
 * No counterpart in the reference: it replaces consecutive UnitView.linear
 * calls on independent inputs, e.g. the image and text streams of FLUX's
 * double block (selas/models/flux.py:300-324).
 */
int selas_nf4_linear_batched(const selas_nf4_gemm_problem *problems, int64_t count, int64_t blocksize,
                             const float code[16], int dtype, void *workspace, int64_t workspace_bytes,
                             void *stream);

/*
 * Bytes of device workspace that selas_nf4_linear (count 1) or
 * selas_nf4_linear_batched (codec SELAS_CODEC_NF4), or their int8_row twins
 * (SELAS_CODEC_INT8_ROW), need for these problems on the current device:
 * 0 unless the launch splits its last round of tiles over K, then
 * split tiles x K ranges x 256 KiB (at most the CU count x 256 KiB, 64 MiB on
 * MI355X). Reads only M, K and N of each problem (the other fields may be
 * NULL); problems with M = 0 are skipped, and M <= 32 gives 0 (skinny kernels).
 * No counterpart in the reference: selas's decode-then-F.linear needs no
 * scratch beyond the decoded weight (selas/store.py:289-293).
 */
int selas_linear_workspace_bytes(const selas_nf4_gemm_problem *problems, int64_t count, int codec,
                                 int64_t *bytes);

/*
 * Rows and columns of the output tiles that the same launch runs in (0 and 0 where a
 * skinny kernel takes it); the arguments as for selas_linear_workspace_bytes. It says
 * which kernel a size runs, for measurements and tests; the bits do not depend on it.
 * No counterpart in the reference.
 */
int selas_linear_tile(const selas_nf4_gemm_problem *problems, int64_t count, int codec, int64_t *rows,
                      int64_t *cols);

/*
 * Quantized linear forward y = x W^T + bias with W an int8_row [N, K] weight
 * (q int8 [N, K] row-major, 16-byte aligned; scale fp32 [N]); x, bias, y and
 * dtype as for selas_nf4_linear.
 * M > 32 runs the tiled MFMA GEMM of selas_nf4_linear with the int8 operand
 * bf16(q * bf16(scale)), the reference's decoded weight bit for bit. M <= 32
 * runs a skinny kernel (for K = 1024, 2048, 3072 the streaming kernel of
 * selas_int8_row_linear_grouped) that multiplies x by q exactly and scales the fp32 row
 * sums by bf16(scale): it agrees with the decoded-weight product to the bf16
 * rounding of the decoded weight. workspace / workspace_bytes as for
 * selas_nf4_linear (selas_linear_workspace_bytes with SELAS_CODEC_INT8_ROW).
 * Returns SELAS_EUNSUPPORTED for K % 64 != 0,
 * misaligned rows or a dtype other than bf16 (the caller then decodes with
 * selas_int8_row_dequant and uses a library GEMM).
 * Replaces UnitView.linear for int8_row weights (selas/store.py:289-293):
 * decode (codecs.py:273-277) followed by F.linear.
 */
int selas_int8_row_linear(const void *x, int64_t M, int64_t K, int64_t ldx, const int8_t *q, const float *scale,
                          int64_t N, const void *bias, void *y, int64_t ldy, int dtype, void *workspace,
                          int64_t workspace_bytes, void *stream);

/*
 * selas_nf4_linear_batched for int8_row weights: in each problem `packed`
 * holds q and `absmax` the row scales; gelu_cols, y2 and the workspace as
 * there (selas_linear_workspace_bytes with SELAS_CODEC_INT8_ROW).
 * No counterpart in the reference (see selas_nf4_linear_batched).
 */
int selas_int8_row_linear_batched(const selas_nf4_gemm_problem *problems, int64_t count, int dtype, void *workspace,
                                  int64_t workspace_bytes, void *stream);


/*
 * One NF4 weight of a grouped skinny linear (device-memory array element).
 * packed/absmax as for selas_nf4_linear, bias [n] bf16 or NULL, y [M, n] bf16
 * with row stride ldy. The layout is fixed: 4 pointers then 2 int64.
 */
typedef struct selas_nf4_gemv_desc {
  const uint8_t *packed;
  const float *absmax;
  const void *bias;
  void *y;
  int64_t n;
  int64_t ldy;
} selas_nf4_gemv_desc;

/*
 * `count` quantized linears that share one input x [M, K] (M <= 32, K = 1024,
 * 2048 or 3072, blocksize 64, bf16, at most 1023 weights, 16-byte aligned codes
 * and x rows, x spanning under 4 GiB), computed by one launch: y_i = x W_i^T + b_i.
 * `descs` is a device array of `count` descriptors and total_n the sum of
 * their n (it sizes the launch). Each output has the bits selas_nf4_linear
 * gives for that weight alone.
 * Replaces the per-unit loop of FluxRunner.modulations (selas/models/flux.py:
 * 428-445), which calls UnitView.linear once per modulation weight with the
 * same silu(vec) input.
 */
int selas_nf4_linear_grouped(const void *x, int64_t M, int64_t K, int64_t ldx, const selas_nf4_gemv_desc *descs,
                             int64_t count, int64_t total_n, int64_t blocksize, const float code[16], int dtype,
                             void *stream);

/* At most this many weights per selas_nf4_linear_grouped_static call. */
#define SELAS_STATIC_MAX_WEIGHTS 1023
/* At most this many streams per GPU call selas_nf4_linear_grouped_static. */
#define SELAS_STATIC_MAX_STREAMS 8

/*
 * selas_nf4_linear_grouped that allocates nothing and needs no device memory of
 * the caller's beyond x, the weights, biases and outputs: `descs` is an array
 * of `count` descriptors in HOST memory (read during the call only), and the
 * sum of their n is computed here. The library stages the descriptors in
 * device tables of its own: SELAS_STATIC_MAX_STREAMS tables of
 * SELAS_STATIC_MAX_WEIGHTS * 48 bytes (392,832 bytes in all) per GPU, held until
 * the process ends. Each stream that calls on a GPU gets its own table, at its
 * first call; a call from a further stream returns SELAS_EUNSUPPORTED, and
 * count above SELAS_STATIC_MAX_WEIGHTS is rejected with SELAS_EINVAL. A call
 * rewrites its stream's table before its kernels read it, and enqueues both
 * under that table's lock: calls on one stream are ordered (also from several
 * host threads), and calls on different streams use different tables. A
 * stream handle that is destroyed and handed out again keeps the old table, so
 * the destroyed stream's calls must have finished. Each output has the bits
 * selas_nf4_linear_grouped (and selas_nf4_linear) gives for that weight.
 * No counterpart in the reference. It is for callers that cannot allocate
 * device memory: code under HIP graph capture, serving loops with a fixed
 * memory budget, harnesses that forbid hipMalloc.
 */
int selas_nf4_linear_grouped_static(const void *x, int64_t M, int64_t K, int64_t ldx, const selas_nf4_gemv_desc *descs,
                                    int64_t count, int64_t blocksize, const float code[16], int dtype, void *stream);

/*
 * selas_nf4_linear_grouped for int8_row weights (M <= 32, K = 1024, 2048 or
 * 3072, bf16, 16-byte aligned x rows, x spanning under 4 GiB): in each
 * descriptor `packed` holds q [n, K] (16-byte aligned) and
 * `absmax` the n row scales. Each output has the bits selas_int8_row_linear
 * gives for that weight alone (the same kernel serves M <= 32 there).
 * Replaces the per-weight UnitView.linear calls of FluxRunner.modulations
 * (selas/models/flux.py:428-445) for int8_row weights.
 */
int selas_int8_row_linear_grouped(const void *x, int64_t M, int64_t K, int64_t ldx, const selas_nf4_gemv_desc *descs,
                                  int64_t count, int64_t total_n, int dtype, void *stream);

/* ------------------------------------------------------------ segments
 *
 * The memory-bound code between the block linears (selas/models/flux.py:
 * 164-200). Tensors are [B, L, D] with D contiguous; `sb`/`sl` are the batch
 * and row strides in elements. Per-batch vectors (shift, scale, gate) are
 * [B, D] with batch stride `mod_sb`. Outputs are contiguous. All math is fp32.
 */

/* out = dtype(LayerNorm(x; no affine, eps 1e-6) * (1 + scale) + shift).
 * Replaces _mod_in (flux.py:164-166) with _ln (flux.py:146-147). */
int selas_mod_in(const float *x, int64_t B, int64_t L, int64_t D, int64_t x_sb, int64_t x_sl,
                 const float *shift, const float *scale, int64_t mod_sb, void *out, int out_dtype,
                 void *stream);

/* out = x + g * float(y), y clamped to +-65504 first when guard != 0.
 * Replaces _gated_add (flux.py:169-171) with _res (flux.py:141-143). */
int selas_gated_add(const float *x, int64_t B, int64_t L, int64_t D, int64_t x_sb, int64_t x_sl,
                    const float *g, int64_t g_sb, const void *y, int y_dtype, int64_t y_sb, int64_t y_sl,
                    int guard, float *out, void *stream);

/* x_out = x + g * float(y) as above, and h = mod_in(x_out, shift, scale) in one pass.
 * Replaces _gated_add_mod (flux.py:174-176). */
int selas_gated_add_mod(const float *x, int64_t B, int64_t L, int64_t D, int64_t x_sb, int64_t x_sl,
                        const float *g, int64_t g_sb, const void *y, int y_dtype, int64_t y_sb, int64_t y_sl,
                        int guard, const float *shift, const float *scale, int64_t mod_sb, float *x_out,
                        void *h, int h_dtype, void *stream);

/* Single-stream attention prep: qkv [B, L, 3*H*Dh] (channel = which*H*Dh + h*Dh + d,
 * strides qkv_sb, qkv_sl) -> q, k = dtype(RoPE(RMSNorm(.) * scale)), v = copy,
 * each [B, H, L, Dh] contiguous. RMSNorm eps 1e-6 over Dh in fp32; RoPE rotates
 * interleaved pairs with cos/sin [L, Dh/2] fp32. Dh must be even and at most 128.
 * Replaces _qkv_single (flux.py:188-191) with _heads, qk_rms, apply_rope (117-132). */
int selas_qkv_single(const void *qkv, int64_t B, int64_t L, int64_t H, int64_t Dh, int64_t qkv_sb,
                     int64_t qkv_sl, const float *q_scale, const float *k_scale, const float *cos,
                     const float *sin, void *q, void *k, void *v, int dtype, void *stream);

/* Double-stream attention prep: text qkv [B, Lt, 3HDh] and image qkv [B, Li, 3HDh],
 * each normalised with its own q/k scales, joined text-first along L, RoPE with
 * cos/sin [Lt+Li, Dh/2]; q, k, v [B, H, Lt+Li, Dh] contiguous.
 * Replaces _qkv_double (flux.py:179-185). */
int selas_qkv_double(const void *tqkv, int64_t t_sb, int64_t t_sl, int64_t Lt, const void *iqkv, int64_t i_sb,
                     int64_t i_sl, int64_t Li, int64_t B, int64_t H, int64_t Dh, const float *tq_scale,
                     const float *tk_scale, const float *iq_scale, const float *ik_scale, const float *cos,
                     const float *sin, void *q, void *k, void *v, int dtype, void *stream);

/* out = gelu_tanh(h) for rows x cols (row stride ld), out contiguous.
 * Replaces _gelu (flux.py:194-195). */
int selas_gelu(const void *h, int64_t rows, int64_t cols, int64_t ld, void *out, int dtype, void *stream);

/* out[r] = concat(attn[r] (Da), gelu_tanh(mlp[r]) (Dm)), out [rows, Da+Dm] contiguous.
 * Replaces _attn_mlp (flux.py:198-200). */
int selas_attn_mlp(const void *attn, int64_t rows, int64_t Da, int64_t lda, const void *mlp, int64_t Dm,
                   int64_t ldm, void *out, int dtype, void *stream);

/* ------------------------------------------------------------ attention
 *
 * The block attention (selas/models/flux.py:135-138): SDPA over q, k, v
 * [B, H, L, Dh] followed by transpose(1, 2).reshape(B, L, H*Dh).
 */

/*
 * out[b, l, h*Dh + d] = sum_j softmax_j(q[b,h,l,:] . k[b,h,j,:] / sqrt(Dh)) v[b,h,j,d]
 * with q, k [B, H, L, Dh] contiguous, the values given transposed as vt
 * [B, H, Dh, Lp] (selas_transpose_heads; Lp = L rounded up to a multiple of 64,
 * the columns past L zero), out [B, L, H*Dh] with row stride ldo
 * (>= H*Dh; e.g. the first columns of the [attention | GELU(mlp)] input of the
 * single block's second linear, flux.py:198-200). bf16 in
 * and out; scores, softmax and sums in fp32, the probabilities rounded to bf16
 * for the second product (as the flash backends of torch's SDPA do). Takes
 * Dh = 128 and any L; otherwise SELAS_EUNSUPPORTED (the caller runs SDPA).
 * Replaces _attention (flux.py:135-138).
 */
int selas_attention(const void *q, const void *k, const void *vt, int64_t B, int64_t H, int64_t L, int64_t Dh,
                    void *out, int64_t ldo, int dtype, void *stream);

/*
 * selas_attention with the values as v [B, H, L, Dh] in place of v^T: the
 * kernel transposes them on their way to the matrix cores. Same bits. At most
 * 65535 heads. out may not overlap q, k or v.
 */
int selas_attention_v(const void *q, const void *k, const void *v, int64_t B, int64_t H, int64_t L, int64_t Dh,
                      void *out, int64_t ldo, int dtype, void *stream);

/*
 * selas_attention_v where the 256-query items of an image leave a last round of
 * few, and most CUs idle: those items run as ranges of keys on the idle CUs, their
 * fp32 partial outputs are kept in `workspace` (device memory, 16-byte aligned, at
 * least selas_attention_workspace_bytes) and added in key order. The choice depends
 * on H, L and the CU count only, so an image has the same bits in every batch; the
 * size is B times an image's. With a size of 0 the call is selas_attention_v, bit
 * for bit. A workspace that is missing or too small is SELAS_EINVAL, with nothing
 * launched.
 */
int selas_attention_split(const void *q, const void *k, const void *v, int64_t B, int64_t H, int64_t L, int64_t Dh,
                          void *out, int64_t ldo, int dtype, void *workspace, int64_t workspace_bytes, void *stream);
int selas_attention_workspace_bytes(int64_t B, int64_t H, int64_t L, int64_t *bytes);

/*
 * vt[i, d, l] = v[i, l, d] for BH heads of [L, Dh] (bf16, Dh = 128), with vt rows
 * of Lp = L rounded up to a multiple of 64 tokens and vt[i, d, l] = 0 for l >= L:
 * the value layout selas_attention reads. No counterpart in the reference.
 */
int selas_transpose_heads(const void *v, int64_t BH, int64_t L, int64_t Dh, void *vt, int dtype, void *stream);

/* ------------------------------------------------------------ rotary positions */

/* At most this many tensors per selas_rope call, and position axes. */
#define SELAS_ROPE_MAX_PARTS 3
#define SELAS_ROPE_MAX_AXES 4

/* One tensor of a selas_rope call (host-memory array element): x and y are
 * [B, heads, L, Dh] with unit channel stride and any batch, head and row strides
 * (elements). scale: the RMS norm's scale [Dh] fp32, NULL for no norm. rotate 0
 * leaves the angles out (the values, which are laid out along with q and k). */
typedef struct selas_rope_part {
  const void *x;
  int64_t x_sb, x_sh, x_sl;
  void *y;
  int64_t y_sb, y_sh, y_sl;
  const float *scale;
  int64_t heads;
  int64_t rotate;
} selas_rope_part;

/*
 * Rotary positions with several axes, taken from the positions themselves:
 *   z = x, or x / sqrt(mean(x^2) + 1e-6) * scale over a head's Dh channels;
 *   pair j of axis a turns by pos[b, l, a] * theta^(-2j / axis_dim[a]):
 *   (z0, z1) -> (z0 cos - z1 sin, z0 sin + z1 cos), by the negative angle when
 *   inverse != 0 (the rotation's gradient; no part may then have a scale).
 * The pairs of the axes follow each other; with R = sum(axis_dim) pair i is
 * channels (2i, 2i + 1), or (i, i + R/2) when halves != 0, and channels from R on
 * are not rotated. ids is [B, L, axes] (fp32, SELAS_I32 or SELAS_I64, unit last
 * stride; ids_sb 0 where the images share their positions). Each axis_dim is
 * even, R <= Dh. Angles are formed and reduced in fp64, the rest is fp32 and
 * rounded once. dtype is the tensors' type. y may be x (same address and strides);
 * otherwise no y may overlap an x or another y. Dh <= 256 where the tensors can be read
 * in vectors of 4 elements (strides, Dh, R and, with halves, R/2 multiples of 4, addresses
 * of 16 bytes in fp32 and of 8 otherwise), Dh <= 128 elsewhere (SELAS_EUNSUPPORTED).
 * Next to selas_qkv_single and selas_qkv_double, which take cos/sin tables that a
 * batch shares. Restates qk_rms, apply_rope and rope_tables (flux.py:106-126).
 */
int selas_rope(const selas_rope_part *parts, int64_t count, int64_t B, int64_t L, int64_t Dh, const void *ids,
               int ids_dtype, int64_t ids_sb, int64_t ids_sl, int64_t axes, const int64_t *axis_dim, double theta,
               int halves, int inverse, int dtype, void *stream);

/* ------------------------------------------------------------ raw linear */

/* Activations of selas_raw_linear. */
#define SELAS_ACT_NONE 0
#define SELAS_ACT_GELU 1 /* tanh approximation */
#define SELAS_ACT_SILU 2

/* One linear of a selas_raw_linear call (host-memory array element):
 *   y[b, l, n] = residual[b, l, n] + gate[b, n] * act(sum_k x[b, l, k] w[n, k] + bias[n])
 * with act(..) clamped to the fp16 range (+-65504, NaN passes through) where guard != 0,
 * as selas_gated_add clamps the linear's output. Unit column strides, batch strides *_sb
 * and row strides *_sl in elements, and the rows of w ldw elements apart. bias, gate and residual may be NULL. The
 * dtypes of bias, gate, residual and y are each SELAS_F32 or the call's dtype.
 * y may be the residual (same address, strides and dtype) and overlap nothing else. */
typedef struct selas_raw_linear_problem {
  const void *x;
  int64_t x_sb, x_sl;
  const void *w;
  int64_t ldw;
  const void *bias;
  const void *gate;
  int64_t gate_sb;
  const void *residual;
  int64_t r_sb, r_sl;
  void *y;
  int64_t y_sb, y_sl;
  int64_t B, L, N, K;
  int bias_dtype, gate_dtype, residual_dtype, y_dtype, act, guard;
} selas_raw_linear_problem;

/*
 * Up to SELAS_MAX_BATCHED_LINEARS independent linears with unquantized weights,
 * x and w in dtype (bf16 or fp16, otherwise SELAS_EUNSUPPORTED), fp32 accumulation
 * and epilogue, one rounding at the end. K may be 0 (act(bias) remains). With more than
 * 32 rows and 64 columns, min(256, rows) rows of K elements of each operand, K rounded up to 64, must take less
 * than 2^31 - 4096 bytes (K to 4,194,240 at 256 rows; otherwise SELAS_EUNSUPPORTED).
 * workspace: device memory of at least selas_raw_linear_workspace_bytes for
 * these problems, 16-byte aligned, not used by anything else until the call has
 * run; NULL and 0 where that size is 0, otherwise SELAS_EINVAL. The kernels, tiles
 * and K ranges depend on the problems' shapes, strides, alignment and the CU count
 * only, so equal calls give equal bits.
 * Next to selas_nf4_linear_batched, for the raw codec's weights: UnitView.linear
 * (selas/store.py:289-293) with the activation (flux.py:150-151, 194-195) and the
 * gated residual add (flux.py:169-171) that follow it.
 */
int selas_raw_linear(const selas_raw_linear_problem *problems, int64_t count, int dtype, void *workspace,
                     int64_t workspace_bytes, void *stream);
int selas_raw_linear_workspace_bytes(const selas_raw_linear_problem *problems, int64_t count, int dtype,
                                     int64_t *bytes);

/*
 * Rows of x and of w per output tile of that launch, and its K ranges per tile (0, 0, 0 where
 * no problem is tiled: at most 32 rows, or 64 columns). It says which kernel a size runs, for
 * measurements and tests.
 */
int selas_raw_linear_tile(const selas_raw_linear_problem *problems, int64_t count, int dtype, int64_t *rows,
                          int64_t *cols, int64_t *ranges);

/* ------------------------------------------------------------ attention of the text side */

/* One call of selas_text_attention (host memory): q [B, H, Lq, Dh], k and v [B, Hk, Lk, Dh] with unit channel stride and
 * any batch, head and row strides (*_sb, *_sh, *_sl, elements; that of an axis of one element is not looked at, but not
 * negative), H a multiple of Hk; query head h reads key head h / (H / Hk). out is [B, Lq, H*Dh] (o_sb, o_sl); lse
 * [B, H, Lq] fp32, contiguous, or NULL.
 * Key j of image b exists where j < lengths[b] (NULL: all Lk; values outside 0 .. Lk count as the nearer end) and
 * mask[b * mask_sb + j] != 0 (NULL: all). start[b], or start0 where start is NULL, is the position of the image's first
 * query among the keys' positions 0 .. Lk - 1: with causal != 0 query i sees the keys j <= start + i.
 * table [buckets, H] (row stride table_sl, type table_dtype) is the learned bias, or NULL. Its buckets are those of
 * selas_relative_buckets. Finite entries beyond +-2^17 count as +-2^17, one of -inf leaves its keys no weight. */
typedef struct selas_text_attention_problem {
  const void *q;
  int64_t q_sb, q_sh, q_sl;
  const void *k;
  int64_t k_sb, k_sh, k_sl;
  const void *v;
  int64_t v_sb, v_sh, v_sl;
  void *out;
  int64_t o_sb, o_sl;
  float *lse;
  const int32_t *lengths;
  const uint8_t *mask;
  int64_t mask_sb;
  const int32_t *start;
  int64_t start0;
  const void *table;
  int64_t table_sl;
  int64_t B, H, Hk, Lq, Lk, Dh, buckets, max_distance;
  double scale;
  int table_dtype, bidirectional, causal, reserved; /* reserved: 0 */
} selas_text_attention_problem;

/*
 * s_ij = scale * q_i . k_j + table[bucket(j - (start + i)), h];  out_i = sum_j softmax_j(s_ij) v_j over the keys
 * that query i sees; lse_i = log(sum_j exp(s_ij)). A query that sees no key gets zeros and an lse of -inf. What
 * keys and values that no query sees hold (NaN, infinities) does not reach a result. dtype (bf16 or fp16, otherwise SELAS_EUNSUPPORTED)
 * is that of q, k, v and out; scores, maxima and sums are fp32, the probabilities are rounded to dtype for the second product.
 * Takes Dh a multiple of 8 up to 128, addresses of 16 bytes and strides of 8 elements (out: 8 bytes and 4 elements), row
 * strides up to 2^23 elements, and what its launches hold (each under 2^32 threads: 2^23 images times key heads of few
 * queries, 2^24 tiles of 128 queries); otherwise SELAS_EUNSUPPORTED. scale is in 1e-10 .. 1e10. out and lse overlap nothing.
 * workspace: at least selas_text_attention_workspace_bytes, 16-byte aligned, not used by anything else until the call has
 * run; NULL and 0 where that size is 0. Kernels and the split of the keys depend on the sizes, on which of lengths, mask and
 * table are given and on the CU count only, so equal calls give equal bits.
 * Next to selas_attention, for the attention of the text encoders (selas/models/t5.py:66, clip.py:34) and of image tokens
 * to an encoder's states. */
int selas_text_attention(const selas_text_attention_problem *problem, int dtype, void *workspace, int64_t workspace_bytes,
                         void *stream);
int selas_text_attention_workspace_bytes(const selas_text_attention_problem *problem, int dtype, int64_t *bytes);

/*
 * The gradients of that call for grad, the gradient of out ([B, Lq, H*Dh], g_sb, g_sl): problem is the forward call's, with
 * the out and lse that it wrote (out may be a copy at other strides). dq [B, H, Lq, Dh], dk and dv [B, Hk, Lk, Dh] are
 * contiguous, in dtype; dtable [buckets, H] contiguous, in table_dtype (unused where table is NULL). Keys that are not seen
 * have gradients of 0, and so have queries that see none; what those hold, or their rows of grad, reaches nothing. grad's
 * address and strides are as q's (the batch stride always), dq, dk and dv 8-byte aligned. dk and dv are summed over the query
 * heads that share a key head, dtable over everything, in fp32 and in one order: no atomics. workspace as in
 * selas_text_attention, of selas_text_attention_backward_workspace_bytes. */
int selas_text_attention_backward(const selas_text_attention_problem *problem, const void *grad, int64_t g_sb, int64_t g_sl,
                                  void *dq, void *dk, void *dv, void *dtable, int dtype, void *workspace,
                                  int64_t workspace_bytes, void *stream);
int selas_text_attention_backward_workspace_bytes(const selas_text_attention_problem *problem, int dtype, int64_t *bytes);

/*
 * The buckets of one direction: bucket t begins at distance edges[t] (edges[0] = 0, ascending), as many as *count says (at
 * most 128; edges has room for them). With n buckets a direction (all of them, or half when bidirectional != 0), e = n / 2
 * and m = max_distance: distance a is in bucket a if a < e, else in e + floor((n - e) log(a / e) / log(m / e)), at most
 * n - 1, in exact arithmetic (a distance on a border belongs to the bucket that begins there). Keys after the query have the
 * buckets from n on when bidirectional != 0, bucket 0 otherwise. n is 2 to 128, e < m <= 512 (above: SELAS_EUNSUPPORTED). */
int selas_relative_buckets(int64_t buckets, int64_t max_distance, int bidirectional, int32_t *edges, int64_t *count);

#ifdef __cplusplus
}
#endif

#endif /* SELAS_AMD_H */
