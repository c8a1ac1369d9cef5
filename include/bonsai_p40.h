// bonsai_p40.h -- C ABI of the MI355X (gfx950) PQ2_0 matmul path.
//
// Drop-in for the reference header include/bonsai_p40.h of
// boetti-dev/p40-kernel: every declaration of that header is kept with the
// same name, argument order, argument meaning and return-code convention, so
// C++ host code written against it links against libbonsai_p40.so unchanged.
// Where the reference's host and device code disagree, the reference name
// keeps what the reference LIBRARY does when it reads memory (the FWHT's
// 1024-entry signs), and its rounding follows the host code (below).
// The library is written for AMD CDNA4 (gfx950) in HIP; `bonsai_stream` is a
// hipStream_t (NULL = the default stream).
//
// Conventions shared by every entry point (reference: gemv_p40.cu:200-219,
// gemm_p40.cu:143-154, gemv_repack_p40.cu:196-220, elementwise_p40.cu:75-80):
//   * all pointers are device pointers owned by the caller; nothing is
//     allocated and nothing synchronises -- work is enqueued on `stream`;
//   * return 1 for invalid arguments, 0 for an empty no-op, otherwise the
//     hipError_t of the launch (so 0 = enqueued).  Callers test `!= 0`;
//   * a NULL device pointer that the requested work would read or write is an
//     invalid argument (1, nothing launched), where the reference launches
//     anyway; optional pointers (signs, norm weights, status) may be NULL.
//     The empty no-ops (n_out <= 0, n_tok <= 0, ...) still return 0 first, as
//     in the reference;
//   * block_pq2_0 = 34 bytes (fp16 d, 32 bytes of 2-bit codes, element j in
//     byte j/4 at bits 2(j%4), value (code-1)*d); block_q8_1 = 36 bytes (fp16
//     d, int16 sum s stored as raw bits, 32 int8 in the PQ2_0-native permuted
//     order: position j holds element 16(j>>4) + 4(j&3) + ((j>>2)&3));
//   * Q8_1 buffers must be 4-byte aligned.  PQ2_0 weights need only the
//     2-byte alignment of the format; 16-byte aligned weights with
//     n_in % 1024 == 0 take the streaming fast path.
//   * rounding follows the reference HOST code (src/pq2_0.h:99-126,
//     src/p40_common.h:82-114): q = lroundf(x/d) (ties away from zero) and the
//     fp16 scale rounds ties away from zero, so Q8_1 bytes equal the host's.
#pragma once

#include <cstdint>
#include <cstddef>

#ifdef __cplusplus
extern "C" {
#endif

// Opaque stream handle (a hipStream_t), reference include/bonsai_p40.h:16.
typedef void * bonsai_stream;

// --- decode (batch = 1) matrix-vector -------------------------------------
// y[n_out] = W[n_out, n_in] . x with x already in permuted Q8_1 (xq).
// Replaces include/bonsai_p40.h:21-22 (src/kernels/gemv_p40.cu:210-219).
// Errors: 1 if n_in <= 0 or n_in % 128 != 0 or xq is not 4-byte aligned;
// 0 (no-op) if n_out <= 0; then 1 if n_out >= 2^30 or n_in / 128 > 2^24.
int bonsai_p40_gemv(const void * W, const void * xq, float * y,
                    int64_t n_out, int64_t n_in, bonsai_stream stream);

// Quantise n floats to permuted Q8_1 (n/32 blocks of 36 bytes).
// Replaces include/bonsai_p40.h:25 (src/kernels/gemv_p40.cu:200-208).
// Errors: 1 if n <= 0 or n % 32 != 0.
int bonsai_p40_quant_activations(const float * x, void * out, int64_t n, bonsai_stream stream);

// --- prefill (batch > 1) ----------------------------------------------------
// Y[n_out, n_tok] (row-major, Y[r*n_tok + t]) = W . X, X in permuted Q8_1,
// chunk-major: block (c, t) at index c*n_tok + t (src/kernels/gemm_p40.cu:75).
// Replaces include/bonsai_p40.h:29-30 (src/kernels/gemm_p40.cu:143-154).
// n_tok == 1 runs the decode GEMV; 2 tokens the streaming kernel with
// per-token activation planes; 3..8 the block-diagonal 16x16x64 int8 MFMA
// kernel, except 4 tokens on 1024-, 5120- and 6144-column rows and 3 on
// 1024- and 6144-column rows, which take the 4x4x4 int8 MFMA streaming
// kernel; 9..16 the streamed 16x16x32 int8 MFMA kernel, or f16-MFMA 80x16
// tiles that read s as it does on matrices of more than 64 rows a CU where
// rounds of 80 rows a CU, rounded up, are no more than n_out in rounds of 64
// (n_in % 1024 == 0, n_in >= 5120, 16-byte aligned W); larger n_tok the
// f16-MFMA tile GEMMs: small tiles with K split over a workgroup's waves where
// larger ones would leave CUs idle, for all tokens or those past the whole
// larger tiles (n_in % 1024 == 0, 16-byte aligned W), else 128- to 256-row
// tiles (other alignments: 64-bit-offset MFMA kernels).  The GEMV, the streamed small-batch kernels and the 80x16 tiles
// subtract each Q8_1 block's stored sum s as the reference does
// (src/pq2_0.h:169); the GEMMs for more than 16 tokens and the kernels for
// other alignments multiply (code - 1) by q directly and do not read s.  The
// two agree for blocks whose s is the sum of their q, which holds for every
// block this library's or the reference's quantiser writes.
// The kernels add in different orders, each within fp32 rounding of the sum:
// the last bits of a token's column may depend on n_tok, on the token's place
// in the call and on n_out (so on how a prompt is chunked or a matrix sharded
// by rows); the same call gives the same bytes every time.  A block scale that
// is infinite gives infinities and NaN, and which of them depends on the
// kernel.
// Errors: 1 if n_in <= 0 or n_in % 128 != 0, Xq is not 4-byte or W not 2-byte
// aligned, or n_out, n_tok or n_in / 128 is too large for the launch; 0
// (no-op) if n_out <= 0 or n_tok <= 0.
int bonsai_p40_gemm(const void * W, const void * Xq, float * Y,
                    int64_t n_out, int64_t n_in, int64_t n_tok, bonsai_stream stream);

// bonsai_p40_gemm with a caller workspace (an addition; the reference has no
// counterpart): where the long-prompt kernel runs (the rows bonsai_p40_gemm
// gives its 256- or 160-row tiles) on a matrix of 8192 rows or more, Xq is
// first converted once into the workspace (each q byte as f16, each d as
// fp32: both exact), and the tiles take the activation from there by DMA
// instead of converting it per tile; elsewhere it runs bonsai_p40_gemm.
// Y is bit-identical to bonsai_p40_gemm's.  workspace: 16-byte aligned,
// bonsai_p40_gemm_workspace_bytes(n_in, n_tok) bytes; NULL (any ws_bytes)
// runs bonsai_p40_gemm.  The workspace is scratch for the call (stream-
// ordered: calls that share one must be ordered on one stream).  Errors: those
// of bonsai_p40_gemm, and 1 if workspace is not 16-byte aligned or ws_bytes is
// smaller than the size the call needs.
int bonsai_p40_gemm_ws(const void * W, const void * Xq, float * Y, int64_t n_out, int64_t n_in,
                       int64_t n_tok, void * workspace, int64_t ws_bytes, bonsai_stream stream);
// Workspace bytes bonsai_p40_gemm_ws needs (n_tok * n_in / 32 * 68); 0 where
// it needs none (n_in or n_tok <= 0, or the converted activation would not
// be addressable with 32-bit offsets: 2 GiB and more, the call then runs
// bonsai_p40_gemm whatever the workspace).
int64_t bonsai_p40_gemm_workspace_bytes(int64_t n_in, int64_t n_tok);

// --- aligned repacked layout ------------------------------------------------
// Size-neutral row: d[nb] fp16, then 4 planes of nb 8-byte code units; unit
// u = plane*nb + block at byte 2*nb + 8u (src/pq2_0_repack.h:46-57).
// src and dst must not overlap.  Errors: 1 if n_in % 128 != 0, n_out <= 0 or
// n_in/128 is not a positive multiple of 8.
// Replaces include/bonsai_p40.h:35 (src/kernels/gemv_repack_p40.cu:196-207).
int bonsai_p40_repack(const void * src, void * dst, int64_t n_out, int64_t n_in, bonsai_stream stream);
// y = W_repacked . x for fp32 x (quantised to Q8_1 inside the kernel).
// Replaces include/bonsai_p40.h:36-37 (src/kernels/gemv_repack_p40.cu:209-220).
// Errors: as bonsai_p40_repack, plus 1 if W is not 8-byte aligned (its 8-byte
// code units are read whole) or, on widths without the streaming kernel, the
// quantised activation (n_in/32 * 40 bytes) does not fit the 160 KiB LDS of a
// workgroup.
int bonsai_p40_gemv_repack(const void * W, const float * x, float * y,
                           int64_t n_out, int64_t n_in, bonsai_stream stream);

// --- transforms -----------------------------------------------------------------
// In-place normalised Sylvester-Hadamard transform in blocks of 1024.  signs
// (optional, NULL = all +1) has 1024 entries, used by EVERY block: the meaning
// of the reference device kernel (elementwise_p40.cu:17-41, signs[i] with
// i < 1024), so a buffer sized for the reference library is never read past.
// Stage order h = 1..512 as the host, so the result is bit-identical to the
// host fwht_blocks() given that vector tiled to length n.  Errors: 1 if
// n <= 0 or n % 1024 != 0.  Replaces include/bonsai_p40.h:41
// (elementwise_p40.cu:75-80).
int bonsai_p40_fwht(float * x, const float * signs, int64_t n, bonsai_stream stream);

// Not on the PQ2_0 matmul path; kept so the reference's symbol set links.
// rmsnorm: y = x * (1/sqrt(mean(x^2) + eps)) * w per row (src/ops.h:13-22).
int bonsai_p40_rmsnorm(const float * x, const float * w, float * y,
                       int64_t n_rows, int64_t n, float eps, bonsai_stream stream);
// gdn_step / attn are outside this library's scope: they return 2
// ("not implemented") without touching memory.
int bonsai_p40_gdn_step(float * state, const float * q, const float * k, const float * v,
                        const float * g, const float * beta, float * out,
                        int n_k_heads, int n_v_heads, int K, int V, bonsai_stream stream);
int bonsai_p40_attn(const float * q, const float * k, const float * v, float * out,
                    int n_tok, int n_head, int n_head_kv, int head_dim, float scale,
                    bonsai_stream stream);

// --- additions (no counterpart in the reference header) -------------------------
// Every addition that takes `signs` reads a length-n vector (block b uses
// signs[1024 b ..]), the host form of src/fwht.h:38-42.

// bonsai_p40_fwht with the host's length-n signs (block b uses
// signs[1024 b .. 1024 b + 1023]): bit-identical to fwht_blocks(x, signs, n).
// Errors as bonsai_p40_fwht.
int bonsai_p40_fwht_signs_n(float * x, const float * signs, int64_t n, bonsai_stream stream);

// Fused decode pre-pass: xq = Q8_1(FWHT(signs .* x)) for one token of n floats
// (x is not modified).  One launch in place of bonsai_p40_fwht followed by
// bonsai_p40_quant_activations (elementwise_p40.cu:17-41 + gemv_p40.cu:168-196),
// bit-identical to the host fwht_blocks + quantize_row_q8_1(permute = true).
// Errors: 1 if n <= 0 or n % 1024 != 0.
int bonsai_p40_fwht_quant(const float * x, const float * signs, void * xq, int64_t n,
                          bonsai_stream stream);

// Batched pre-pass for the GEMM: X is [n_tok][n] fp32 (token rows); each token
// is optionally rotated (rotate != 0: FWHT with signs, n % 1024 == 0) and
// quantised on its own, written chunk-major (block (c, t) at c*n_tok + t) --
// the Xq layout bonsai_p40_gemm consumes, which the reference API has no
// producer for.  Errors: 1 if n <= 0, n % 32 != 0 (n % 1024 with rotate),
// n_tok <= 0 or n_tok > 65535 (one grid row per token), n * n_tok > 2^40, X or
// Xq is NULL, Xq is not 4-byte aligned, or signs is given without rotate.
int bonsai_p40_quant_tokens(const float * X, const float * signs, void * Xq, int64_t n,
                            int64_t n_tok, int rotate, bonsai_stream stream);

// Layer-input pre-pass: Xq = Q8_1(FWHT(signs .* RMSNorm(x, w, eps))) for n_tok
// token rows of n floats, one launch in place of bonsai_p40_rmsnorm followed by
// bonsai_p40_fwht and bonsai_p40_quant_activations (elementwise_p40.cu:17-41,
// 48-88 + gemv_p40.cu:168-196; RMSNorm as src/ops.h:13-22).  The sum of squares
// is accumulated in fp64 in one order shared by every normalising entry point
// (whatever n_tok), so the scale can differ from the reference's sequential
// fp32 sum by that sum's rounding; the rest is bit-identical to the
// host FWHT and quantiser.  Output chunk-major (block (c, t) at c*n_tok + t: the
// GEMM's Xq; for n_tok == 1 the GEMV's xq).  x, w and signs are [n_tok][n], [n]
// and [n] (signs may be NULL).  Errors: 1 if n <= 0, n % 1024 != 0, x or w is
// NULL, or xq is not 4-byte aligned; 0 (no-op) if n_tok <= 0.
int bonsai_p40_rmsnorm_fwht_quant(const float * x, const float * w, const float * signs, void * xq,
                                  int64_t n, int64_t n_tok, float eps, bonsai_stream stream);

// FFN glue of the decode chain: xq = Q8_1(FWHT(signs .* (silu(gate) * up)))
// with silu(g) = g / (1 + exp(-g)) (src/ops.h:27-31), one launch.
// Errors: 1 if n <= 0 or n % 1024 != 0.
int bonsai_p40_swiglu_fwht_quant(const float * gate, const float * up, const float * signs,
                                 void * xq, int64_t n, bonsai_stream stream);

// Fused decode GEMV from the fp32 activation: y = W . Q8_1(FWHT(signs .* x)),
// one launch in place of bonsai_p40_fwht_quant followed by bonsai_p40_gemv
// (the reference runs them as two kernels: elementwise_p40.cu:75-80 +
// gemv_p40.cu:200-219).  Every workgroup rotates and quantises x into its own
// LDS with the pre-pass's device code, so the Q8_1 bytes are the host's; on
// the model widths (n_in/128 in {8, 40, 48, 80, 96, 136}) with 16-byte
// aligned W, x and signs, y is bit-identical to the two-call sequence.  x is
// not modified; signs may be NULL.  Errors: 1 if n_in <= 0, n_in % 1024 != 0,
// x is NULL, or (other widths) the Q8_1 activation, 36 bytes per 32 columns,
// does not fit in a workgroup's LDS less 1 KiB (n_in > 144384 with MI355X's
// 160 KiB); 0 (no-op) if n_out <= 0.
int bonsai_p40_fwht_gemv(const void * W, const float * x, const float * signs, float * y,
                         int64_t n_out, int64_t n_in, bonsai_stream stream);

// Decode GEMV from an fp32 activation that is already in the weights' basis:
// y = W . Q8_1(x), one launch in place of bonsai_p40_quant_activations
// followed by bonsai_p40_gemv -- the reference's ggml hook sequence
// (integrations/prismml/bonsai-p40.diff:283-291), which needs a Q8_1 scratch
// buffer; this needs none.  Every workgroup quantises x into its own LDS with
// the quantiser's device code (host rounding); on the model widths with
// 16-byte aligned W and x, y is bit-identical to the two-call sequence.
// Errors: 1 if n_in <= 0, n_in % 1024 != 0, x is NULL, or (other widths) the
// Q8_1 activation does not fit in a workgroup's LDS less 1 KiB (n_in > 144384
// with MI355X's 160 KiB); 0 (no-op) if n_out <= 0.
int bonsai_p40_quant_gemv(const void * W, const float * x, float * y, int64_t n_out, int64_t n_in,
                          bonsai_stream stream);

// Grouped decode GEMV: y[m] = W[m] . xq for the n_mat (1..4) matrices that
// multiply one activation (q, k and v; gate and up), in one launch over the
// concatenated rows (the reference launches one GEMV per matrix,
// gemv_p40.cu:210-219).  W, y and n_out are host arrays of n_mat entries;
// every W[m] has n_in columns.  y[m] is bit-identical to bonsai_p40_gemv on
// W[m] alone.  Errors: as bonsai_p40_gemv, plus 1 if n_mat is outside 1..4,
// an array is NULL or a matrix has more than 2^30 - 1 rows; matrices with
// n_out[m] <= 0 are skipped (0 if all are).
int bonsai_p40_gemv_group(const void * const * W, float * const * y, const int64_t * n_out, int n_mat,
                          const void * xq, int64_t n_in, bonsai_stream stream);

// Grouped form of bonsai_p40_fwht_gemv: y[m] = W[m] . Q8_1(FWHT(signs .* x)),
// one rotation per workgroup for the whole group; y[m] is bit-identical to
// bonsai_p40_fwht_gemv on W[m] alone.  Errors: as bonsai_p40_fwht_gemv and
// bonsai_p40_gemv_group.
int bonsai_p40_fwht_gemv_group(const void * const * W, float * const * y, const int64_t * n_out, int n_mat,
                               const float * x, const float * signs, int64_t n_in, bonsai_stream stream);

// Layer-input grouped decode GEMV: y[m] = W[m] . Q8_1(FWHT(signs .* RMSNorm(x,
// norm_w, eps))) for the n_mat (1..4) matrices that read one normalised layer
// input (q/k/v after the attention norm, gate/up after the FFN norm), in one
// launch in place of bonsai_p40_rmsnorm + bonsai_p40_fwht +
// bonsai_p40_quant_activations + one bonsai_p40_gemv per matrix
// (elementwise_p40.cu:48-88, 17-41 + gemv_p40.cu:168-219).  Every workgroup
// normalises, rotates and quantises x into its own LDS; the sum of squares is
// fp64, added in the one order every normalising entry point uses, so y[m]
// equals bonsai_p40_rmsnorm_fwht_quant followed by bonsai_p40_gemv_group.  x and norm_w have n_in floats; signs may be NULL.
// Errors: as bonsai_p40_fwht_gemv_group, plus 1 if norm_w is NULL.
int bonsai_p40_rmsnorm_fwht_gemv_group(const void * const * W, float * const * y, const int64_t * n_out,
                                       int n_mat, const float * x, const float * norm_w, const float * signs,
                                       int64_t n_in, float eps, bonsai_stream stream);

// FFN gate/up with its SwiGLU glue in one launch (src/ops.h:27-31 after the
// gate and up GEMVs):  hq = Q8_1(FWHT(h_signs .* silu(Wg . a) * (Wu . a)))
// with a = Q8_1(FWHT(x_signs .* RMSNorm(x, norm_w, eps))) (norm_w NULL: no
// RMSNorm).  In place of bonsai_p40_rmsnorm_fwht_gemv_group on {Wg, Wu}
// followed by bonsai_p40_swiglu_fwht_quant (the reference runs rmsnorm, fwht,
// quant_activations, two gemv and the glue as separate kernels); hq is the
// same bytes, ready for the down projection's bonsai_p40_gemv.  Wg and Wu are
// n_ff x n_embd PQ2_0; x, norm_w, x_signs have n_embd floats, h_signs n_ff
// (signs may be NULL); hq has n_ff/32 Q8_1 blocks.
// workspace: BONSAI_P40_FFN_WORKSPACE_BYTES(n_ff) device bytes, 16-byte
// aligned, ZERO-FILLED before its first use.  Its first
// BONSAI_P40_FFN_SYNC_BYTES are flags, then 2 n_ff words through which the
// gate and up rows pass from the workgroups that compute them to the one that
// finishes their 1024-block; a completed call leaves all of it zero again
// (do not modify it between calls).  Calls that may run at the same time
// need their own workspaces.  status (device, may be NULL): the kernel adds 1
// for each internal wait that gave up (it then leaves hq partly unwritten and
// the workspace must be zero-filled again).  On widths without the one-launch
// kernel the call runs the grouped GEMV and the glue as two launches and the
// rows stay in the workspace as plain fp32.  Errors: 1 if a pointer is NULL
// or misaligned, n_ff or n_embd <= 0 or not a multiple of 1024.
#define BONSAI_P40_FFN_SYNC_BYTES 256
#define BONSAI_P40_FFN_WORKSPACE_BYTES(n_ff) (BONSAI_P40_FFN_SYNC_BYTES + 8 * (int64_t)(n_ff))
int bonsai_p40_ffn_gate_up_swiglu(const void * Wg, const void * Wu, const float * x, const float * norm_w,
                                  const float * x_signs, const float * h_signs, void * hq, int64_t n_ff,
                                  int64_t n_embd, float eps, void * workspace, uint32_t * status,
                                  bonsai_stream stream);

// bonsai_p40_ffn_gate_up_swiglu without a workspace argument, for callers
// that cannot allocate device memory (code under HIP graph capture, tight
// serving loops, harnesses that forbid allocation).  No counterpart in the
// reference.  The workspace is a static device array inside the library of
// BONSAI_P40_FFN_WORKSPACE_BYTES(BONSAI_P40_FFN_NOALLOC_MAX_NFF) bytes (~512
// KiB), one per GPU for the life of the process; the call allocates nothing
// (two kernel launches: a check that repairs the array after a wait that gave
// up, then the fused launch).  Every call
// on one GPU shares that array, so calls that overlap on one GPU (different
// streams, different host threads) race and must not be issued.  Errors: as
// bonsai_p40_ffn_gate_up_swiglu, plus 1 if n_ff > BONSAI_P40_FFN_NOALLOC_MAX_NFF;
// the hipError_t of the one-time symbol lookup if it fails.
#define BONSAI_P40_FFN_NOALLOC_MAX_NFF 65536
int bonsai_p40_ffn_gate_up_swiglu_noalloc(const void * Wg, const void * Wu, const float * x,
                                          const float * norm_w, const float * x_signs, const float * h_signs,
                                          void * hq, int64_t n_ff, int64_t n_embd, float eps, uint32_t * status,
                                          bonsai_stream stream);

// Reference ternary weight quantiser: n fp32 weights (n % 128 == 0, rows of a
// matrix back to back) -> n/128 block_pq2_0 with d = amax rounded to fp16
// half away from zero and code = clamp(lroundf(x / amax) + 1, 0, 3); bytes
// equal quantize_row_pq2_0 (src/pq2_0.h:74-90) for finite inputs.  A
// load-time transform; the reference has it only on the host.  Errors: 1 if
// n <= 0, n % 128 != 0, a pointer is NULL, x is not 4-byte or w not 2-byte
// aligned.
int bonsai_p40_quantize_pq2_0(const float * x, void * w, int64_t n, bonsai_stream stream);
// Its inverse: y = (code - 1) * d for n weights (src/pq2_0.h:62-71), exact.
// Errors as bonsai_p40_quantize_pq2_0.
int bonsai_p40_dequantize_pq2_0(const void * w, float * y, int64_t n, bonsai_stream stream);

// ---------------------------------------------------------------------------
// Decode chain: a sequence of dependent decode steps run by ONE persistent
// launch (no counterpart in the reference, whose host launches every matmul
// and glue op separately; each step computes exactly what the entry point
// named beside its kind computes).  One workgroup per CU; between two steps
// every workgroup waits at a grid-wide barrier (flag words in the workspace,
// bounded polling), and while it waits its waves already stream the first
// weight units of the next GEMV step into LDS.  A step's input may be an
// earlier step's output.
//   BONSAI_P40_CHAIN_Q8:     y[m] = W[m] . x, x the permuted Q8_1 of n_in
//                            values (bonsai_p40_gemv_group);
//   BONSAI_P40_CHAIN_FWHT:   x fp32: bonsai_p40_fwht_gemv_group (signs NULL or
//                            length n_in);
//   BONSAI_P40_CHAIN_RMSNORM_FWHT: x fp32: bonsai_p40_rmsnorm_fwht_gemv_group
//                            with norm_w and eps;
//   BONSAI_P40_CHAIN_SWIGLU: no matrix: q_out = Q8_1(FWHT(signs .* swiglu(x,
//                            x2))) over n_in values (bonsai_p40_swiglu_fwht_quant).
// Widths: FWHT / RMSNORM_FWHT n_in in {5120, 6144}; Q8 n_in in {5120, 6144,
// 17408}; SWIGLU n_in % 1024 == 0.  Up to 4 matrices per step (16-byte
// aligned, < 2 GiB each); x, x2, norm_w and signs 16-byte aligned, x of Q8
// steps and q_out 4-byte aligned.
#define BONSAI_P40_CHAIN_Q8 0
#define BONSAI_P40_CHAIN_FWHT 1
#define BONSAI_P40_CHAIN_RMSNORM_FWHT 2
#define BONSAI_P40_CHAIN_SWIGLU 3
typedef struct bonsai_p40_chain_step {
    int kind;
    int n_mat;                  // 1..4 (0 for SWIGLU)
    const void * W[4];
    float * y[4];
    int64_t n_out[4];
    int64_t n_in;
    const void * x;             // input (Q8_1 bytes or fp32; SWIGLU: gate rows)
    const float * x2;           // SWIGLU: up rows
    const float * norm_w;       // RMSNORM_FWHT: n_in weights
    const float * signs;        // NULL or n_in values of +-1
    void * q_out;               // SWIGLU: Q8_1 output (n_in/32 blocks)
    float eps;                  // RMSNORM_FWHT
} bonsai_p40_chain_step;
// Bytes of device memory a plan of n_steps steps needs.
int64_t bonsai_p40_chain_plan_bytes(int n_steps);
// Checks every step and writes the device form of the chain into plan (device
// memory of bonsai_p40_chain_plan_bytes bytes) with a blocking copy: a set-up
// call, made once per chain and device, before any launch that uses the plan
// (and outside stream capture).  Errors: 1 if a step is invalid (nothing is
// written), else the copy's hipError_t.
int bonsai_p40_chain_plan(const bonsai_p40_chain_step * steps, int n_steps, void * plan);
// Workspace of bonsai_p40_chain_run: one flag word per workgroup and, in its
// last word, the abort word.  Zero-fill it once before its first use and
// then leave it alone: every completed launch leaves it ready for the next.
// Launches that may run at the same time need their own workspaces.
#define BONSAI_P40_CHAIN_WORKSPACE_BYTES 4096
// Runs a planned chain on the device it was planned on.  status (device, may
// be NULL): incremented for every barrier wait that gave up (the chain's
// workgroups could not all be resident, e.g. beside another kernel); the
// first give-up sets the workspace's abort word, on which every workgroup
// leaves at its next barrier or poll, so a failed launch ends within about
// one wait bound.  The outputs of such a launch are not valid and the
// workspace must be zero-filled again: a launch that finds the abort word
// set adds 1 to status and does nothing.  Errors: 1 on bad arguments, else
// the launch's hipError_t.
int bonsai_p40_chain_run(const void * plan, int n_steps, void * workspace, uint32_t * status,
                         bonsai_stream stream);

// ---------------------------------------------------------------------------
// The token mixers between a layer's projections (no counterpart in the
// reference header but bonsai_p40_attn and bonsai_p40_gdn_step, whose dense
// caches and single steps they take the place of).  Each takes one struct,
// which the call copies: it may be changed or freed when the call returns.
// Metadata (lengths, positions, slots, page tables) is read on the device, so a
// captured graph may be replayed after it changed; a value out of range never
// leaves the buffers named here, and what it stands for is stated.  Element
// types:
#define BONSAI_P40_F32 0
#define BONSAI_P40_F16 1
#define BONSAI_P40_BF16 2
#define BONSAI_P40_Q8 3                 // pages only
// Pages of a key/value cache: page p holds, for each of n_kv_head heads,
// page_size (a power of two) rows of head_dim elements; element e of slot i of
// head h at p * page_stride + (h * page_size + i) * head_dim + e (elements;
// page_stride a multiple of 8, n_kv_head * page_size * head_dim at least).
// 16-byte aligned; keys and values in buffers of their own.
//   Q8 pages: a row is head_dim signed bytes n and one fp32 scale d, and stands for d * n
// (rounded once to fp32).  The bytes of slot i of head h of page p are at p * page_stride
// + (h * page_size + i) * head_dim, its scale, fp32, at p * page_stride + n_kv_head * page_size *
// head_dim + 4 * (h * page_size + i): page_stride is in bytes, a multiple of 16 and
// n_kv_head * page_size * (head_dim + 4) at least.  A page is one piece, to be copied as one.
// A row x is written as d = max |x| / 127, n = x * (127 / max |x|) rounded to the nearest
// whole number, ties to even, in fp32: d * n is off by 0.50002 d at most.  A row whose
// largest magnitude is below 2^-112 is written as 0, and one that holds a value that is
// not finite with d = NaN, so that all of it is (one that holds the largest fp32 number reads back as
// infinity there: 127 d is beyond it).  What is read may hold any n in -128 .. 127; keys and
// values that attention sees are to have |d| of 2^80 at most, as rows up to 2^87 have.

// RMSNorm of every query and key head, position rotation, and the append of
// keys and values to the pages, in one launch:
//   y = x / sqrt(mean(x^2) + eps) * w      (q_norm, k_norm: head_dim weights; NULL: y = x)
//   a = pos[t] * inv_freq[i] (radians, in fp64), (y_i, y_j) -> (y_i cos a - y_j sin a,
//   y_j cos a + y_i sin a) for i < n_rot / 2, j = i + n_rot / 2, or with interleaved != 0
//   the elements 2i and 2i + 1; elements from n_rot on pass.
// Element e of head h of token t of q at t * q_tok + h * q_head + e * q_el
// floats (k and v likewise).  Either the elements of a head are consecutive
// (q_el == 1: rows of a GEMV; a head's queries may be followed by its gates) or the
// tokens are (q_tok == 1: the feature-major Y of bonsai_p40_gemm, q_el = n_tok).
// q goes to q_out (q_type: fp32, f16 or bf16), token t at t * q_out_tok, heads
// one after another; k and v, rounded to kv_type (f16, bf16 or Q8), go to slot
// slots[t] = page * page_size + i.  A slot outside 0 .. n_pages * page_size - 1
// (-1: padding) is not written.  Slots of one call have to differ: what two
// tokens leave in one slot is a mix.  Where slots are not written, the pages
// stay as they were.  q_out and the pages overlap nothing that is read.
// Errors: 1 if head_dim is not 64, 128 or 256, n_rot is not a multiple of 8 in
// 0 .. head_dim, a type, page_size (1 .. 65536) or stride is not as stated (n_tok
// > 1 with neither stride 1, q_out_tok < n_head * head_dim or q_out rows not
// 16-byte aligned), n_head or n_kv_head is outside 1 .. 16384, n_tok is 2^25 or more, n_pages
// outside 0 .. 2^40, a pointer is NULL (pos and inv_freq may be where n_rot == 0) or
// misaligned; 0 (no-op) if n_tok <= 0.
typedef struct bonsai_p40_qk_norm_rope_args {
    const float * q, * k, * v;
    int64_t q_tok, q_head, q_el, k_tok, k_head, k_el, v_tok, v_head, v_el;
    int64_t n_tok;
    int n_head, n_kv_head, head_dim, n_rot, interleaved;
    float eps;
    const float * q_norm, * k_norm;
    const int32_t * pos;                // n_tok
    const double * inv_freq;            // n_rot / 2
    const int64_t * slots;              // n_tok
    void * q_out;
    int64_t q_out_tok;
    int q_type, kv_type;
    void * k_pages, * v_pages;
    int64_t n_pages, page_stride;
    int page_size;
} bonsai_p40_qk_norm_rope_args;
int bonsai_p40_qk_norm_rope(const bonsai_p40_qk_norm_rope_args * args, bonsai_stream stream);

// Causal attention of the new tokens of n_seq sequences over their pages, in
// which their own keys and values already are (bonsai_p40_qk_norm_rope):
//   out_t = sum_{j < p_t} softmax_j(scale q_t . k_j) v_j,   p_t = kv_len - n_new + t + 1
// for token t of the n_new = starts[s + 1] - starts[s] tokens of sequence s; 0
// where no key is seen.  n_head is a multiple of n_kv_head; query head h reads
// key/value head h / (n_head / n_kv_head).  Key j of sequence s is slot j %
// page_size of page table[s * table_stride + j / page_size].  A page outside
// 0 .. n_pages - 1 (-1: freed) holds no keys: they are not seen.  kv_len is cut to
// max_pages * page_size, starts, which does not fall (rows that two sequences claim
// are undefined), to 0 .. n_tok.  Rows of q and out before starts[0]
// and from starts[n_seq] on are not touched.  Keys and values that a token does
// not see never reach its output, whatever they hold.
// q and out: token t at t * q_tok and t * out_tok, heads one after another, of
// io_type: kv_type, or fp32 (Q8 pages: fp32, f16 or bf16); out overlaps nothing that is read.  Scores, softmax
// statistics and all sums are fp32.  io_type kv_type rounds each softmax weight once to
// it before the product with V (with f16 a weight below 2^-25 of its row's largest is
// off by up to 2^-36 of that one); fp32 keeps 22 bits of it or more (with f16 pages one
// below 2^-25 is off by up to 2^-47 of the largest).  A row whose largest scaled score is
// beyond 7e5 in magnitude has its scores rounded to fp32 (f16: and weights below
// 2^-14 off by up to 2^-25, fp32 rows 2^-36, of the largest).  A row all of whose seen scores are
// -inf is NaN, as 0 / 0 is; with fp32 rows so is one that sees a key that is not finite.
//   Q8 pages: a row of q is taken as whole numbers, an element off by at most 1.01 x 2^-15
// (fp32: 1.6 x 2^-23) of its largest one, if that is 2^-104 or more (else of 2^-104); a row with a value that is not
// finite gives NaN where it sees a key.  A weight times its value's
// d is rounded once to f16 (fp32: to 22 bits); one below 2^-25 of the row's largest such
// product, taken tile by tile of 32 keys, is off by up to 2^-36 (2^-47) of that, and any by 2^-136 / D
// (2^-147 / D) of it where the largest d that the row sees, D, is below 2^-100.
// max_kv: about the largest kv_len (0: unknown); it places the work, results hold for
// any.  workspace: bonsai_p40_attn_paged_workspace_bytes bytes (of the same
// args), 16-byte aligned, scratch for the call (stream-ordered; calls that may
// run at the same time, and graphs that may, need their own); NULL: few long
// sequences are not spread over the card.  The last bits depend on n_tok, n_seq,
// max_kv and on whether a workspace is given; the same call gives the same bytes.
// Errors: 1 if head_dim is not 64, 128 or 256, n_head (up to 65536) is no multiple
// of n_kv_head, io_type, kv_type, page_size (a power of two, 16 .. 65536) or a
// stride is not as stated (rows of q and out are 16-byte aligned), a Q8 page is 2 GiB or more, scale is not
// finite and > 0, max_pages * page_size > 2^31 - 65536, n_pages is outside 0 .. 2^31 - 1,
// a pointer is NULL or misaligned, the workspace is too small, or there are 2^24 / n_head tokens and
// sequences or more; 0 (no-op) if n_tok <= 0 or n_seq <= 0.
typedef struct bonsai_p40_attn_paged_args {
    const void * q;
    void * out;
    int64_t q_tok, out_tok;
    int64_t n_tok;
    int n_seq, n_head, n_kv_head, head_dim;
    int io_type, kv_type;
    float scale;
    const void * k_pages, * v_pages;
    int64_t n_pages, page_stride;
    int page_size, max_pages;
    const int32_t * table;              // n_seq rows of max_pages
    int64_t table_stride;
    const int32_t * starts;             // n_seq + 1
    const int32_t * kv_len;             // n_seq
    int64_t max_kv;
    void * workspace;
    int64_t workspace_bytes;
} bonsai_p40_attn_paged_args;
int bonsai_p40_attn_paged(const bonsai_p40_attn_paged_args * args, bonsai_stream stream);
// The pointers of args are not looked at; 0 where the call needs none or args
// are invalid.
int64_t bonsai_p40_attn_paged_workspace_bytes(const bonsai_p40_attn_paged_args * args);

// The same for a batch whose sequences, group by group, begin with the same keys (a
// system prompt, a document, several samples of one prompt), which are read once for all
// rows of the group: group g is sequences groups[g] .. groups[g + 1] - 1, and its first
// shared[g] keys (cut to 0 .. max_pages * page_size) are those of table[groups[g]].  A token of its
// sequence s sees all of them, and then keys shared[g] .. p_t - 1 of table[s], whose
// places are the same as in attn_paged (key j: slot j % page_size of page table[s *
// table_stride + j / page_size]): where the rows of a group have the same pages for the shared
// keys, or copies of them, and shared[g] <= kv_len - n_new, the result is attn_paged's but for the last bits.
// shared[g] need not end a page; what table[s] has before it is not read for s > groups[g],
// except that the 16 keys that hold key shared[g] are.
// groups, which does not fall (sequences that two groups claim are undefined), is cut to
// 0 .. n_seq; a sequence of no group sees its own keys, from 0 on.  max_shared: about the largest of
// shared (0: unknown); as max_kv it places the work: that of the own keys for max_kv - max_shared of
// them, or max_kv where max_shared is 0.  Where a sequence has more, as it is of no group or behind a short prefix, give
// max_shared and the most own keys together as max_kv, though no sequence be so long.  groups and
// shared are device memory, as the other lengths are.
// The workspace (attn.workspace, bonsai_p40_attn_shared_workspace_bytes bytes) is
// needed: the sums of the shared keys and of the own ones meet there.
// Errors: 1 as attn_paged, and if n_group or max_shared is negative, groups, shared or the
// workspace is NULL or misaligned, or there are 2^24 / n_head tokens and groups or more.  n_group == 0 is
// attn_paged.
typedef struct bonsai_p40_attn_shared_args {
    bonsai_p40_attn_paged_args attn;
    const int32_t * groups;             // n_group + 1
    const int32_t * shared;             // n_group
    int64_t max_shared;
    int n_group;
} bonsai_p40_attn_shared_args;
int bonsai_p40_attn_shared(const bonsai_p40_attn_shared_args * args, bonsai_stream stream);
// The pointers of args are not looked at; 0 where args are invalid.
int64_t bonsai_p40_attn_shared_workspace_bytes(const bonsai_p40_attn_shared_args * args);

// Rows read back from the pages of a cache, for a program that hands them on or
// works on them itself: k_out and v_out, token t at t * k_tok and t * v_tok elements of
// out_type (fp32, f16 or bf16), heads one after another, become the key and the value
// of slot slots[t] (= page * page_size + i), rounded once to out_type (Q8: d * n to fp32
// before).  Where a slot is outside 0 .. n_pages * page_size - 1 the rows stay as they were; the same
// slot may be read twice.  The outputs overlap nothing that is read.
// Errors: 1 if head_dim is not 64, 128 or 256, n_kv_head is outside 1 .. 16384, a type,
// page_size (a power of two, 1 .. 65536) or stride is not as stated (k_tok and v_tok at least a row, rows
// 16-byte aligned), n_pages is outside 0 .. 2^40, a pointer is NULL or misaligned, or there are
// over 2^30 tokens or 2^34 elements of k; 0 (no-op) if n_tok <= 0 or n_pages == 0.
typedef struct bonsai_p40_kv_read_args {
    const void * k_pages, * v_pages;
    int64_t n_pages, page_stride;
    int page_size, n_kv_head, head_dim, kv_type;
    const int64_t * slots;              // n_tok
    int64_t n_tok;
    void * k_out, * v_out;
    int64_t k_tok, v_tok;
    int out_type;
} bonsai_p40_kv_read_args;
int bonsai_p40_kv_read(const bonsai_p40_kv_read_args * args, bonsai_stream stream);

// Gated delta rule over the new tokens of n_seq sequences (the linear-attention
// layers), with a state S of k_dim x v_dim fp32 for each value head.  Token by
// token, for value head h and its key head:
//   S <- exp(g_t) S;  u = beta_t (v_t - S^T k_t);  S <- S + k_t u^T;  out_t = scale S^T q_t
// q and k are first divided by sqrt(sum of squares + l2_eps) where l2_eps > 0, and
// taken as they are where it is 0.  Value head h reads key head h % n_k_head
// (tiled != 0) or h / (n_v_head / n_k_head).  Sequence s starts from state[i] and
// leaves state_out[i], i = slots[s] (NULL: s): [n_states][n_v_head][k_dim][v_dim].
// state_out may be state.  Slots of one call have to differ; a sequence whose
// slot is outside 0 .. n_states - 1 is passed over (its rows of out, too).  One
// without tokens copies its state.  starts does not fall (what two sequences claim
// is undefined) and is cut to 0 .. n_tok.  Other states, and rows of out before starts[0] and
// from starts[n_seq] on, are not touched.
// q, k, v, out: type fp32, f16 or bf16; token t at t * q_tok (k_tok, v_tok,
// out_tok) elements, heads one after another: slices of one row may be passed;
// out overlaps nothing that is read.
// g and beta: fp32, head h of token t at t * gate_tok + h; a g below -10000 counts as
// that (exp is 0 there).  All sums are fp32's.  In chunks the operands of the products
// (rows of keys and queries, columns of the state and of the chunk's values) have 22 bits
// down to 2^-18 of the largest of their row or column, and are off by up to 2^-40 of that
// below; token by token they are fp32.
// A value that is not finite reaches what it has a part in: one of q its own token, one
// of v or the state its column from there on, one of k, g (but -inf) or beta its head
// from there on, of its sequence; and in chunks the earlier tokens of its chunk, too.
// max_new: about the largest number of tokens of a sequence (0: unknown); it picks
// between token-by-token steps and chunks of 64 tokens, results hold for any.
// workspace: bonsai_p40_gdn_workspace_bytes bytes (of the same args), 16-byte
// aligned, scratch for the call (stream-ordered; calls that may run at the
// same time, and graphs that may, need their own); NULL: token by token.
// Errors: 1 if k_dim is not 64 or 128, v_dim is not a multiple of 16 up to 256,
// n_v_head (up to 65536) is no multiple of n_k_head, the type or a stride is not as
// stated (q_tok, k_tok, v_tok, out_tok and gate_tok at least a row; q, k and v rows
// 16-byte aligned, v_tok up to 2^22), scale or l2_eps is not finite or l2_eps is negative, a
// pointer is NULL or misaligned, the workspace is too small, or there are more
// than 2^27 / n_v_head tokens or 2^40 states, or 2^20 / n_v_head sequences or more; 0 (no-op)
// if n_seq <= 0.
typedef struct bonsai_p40_gdn_args {
    const void * q, * k, * v;
    void * out;
    int64_t q_tok, k_tok, v_tok, out_tok;
    const float * g, * beta;
    int64_t gate_tok;
    const float * state;
    float * state_out;
    int64_t n_states;
    const int32_t * slots;              // n_seq, or NULL
    const int32_t * starts;             // n_seq + 1
    int64_t n_tok;
    int n_seq, n_k_head, n_v_head, k_dim, v_dim;
    int type, tiled;
    float scale, l2_eps;
    int64_t max_new;
    void * workspace;
    int64_t workspace_bytes;
} bonsai_p40_gdn_args;
int bonsai_p40_gdn(const bonsai_p40_gdn_args * args, bonsai_stream stream);
// The pointers of args are not looked at; 0 where the call needs none or args
// are invalid.
int64_t bonsai_p40_gdn_workspace_bytes(const bonsai_p40_gdn_args * args);

// Test hook: out[r * (n_in/32) + c] = the int32 chunk dot sum_k (code-1)*q of
// row r, chunk c, computed by the same device code path as bonsai_p40_gemv
// (the value of src/pq2_0.h:149-177 before scaling).  Errors as bonsai_p40_gemv.
int bonsai_p40_chunk_dots(const void * W, const void * xq, int32_t * out,
                          int64_t n_out, int64_t n_in, bonsai_stream stream);

// Tuning hook: the library reads its BONSAI_* environment variables (kernel
// variant selectors used by tests and sweeps) once per process, at the first
// call that needs one; this re-reads them after a caller changed them.
// Thread-safe; launches already enqueued keep the variants they were given.
// Returns 0.
int bonsai_p40_reload_tuning(void);

// Measurement helper: a streaming read of `bytes` (16-byte aligned, multiple
// of 16) with `blocks` workgroups of 256 lanes -- the achievable-HBM-bandwidth
// ceiling the GEMV is compared with (the role of the reference's
// tools/bwtest.cu).  `out` needs `blocks` words; it is written only in a
// practically impossible case.  Errors: 1 on bad sizes or alignment.
int bonsai_p40_stream_read(const void * buf, int64_t bytes, uint32_t * out, int blocks,
                           bonsai_stream stream);

// Measurement helper: MFMA peak probe.  `blocks` workgroups of 4 waves, each
// wave issuing iters * 4 independent back-to-back MFMAs of one kind (0 = int8
// v_mfma_i32_16x16x64_i8, 32768 ops each; 1 = f16 v_mfma_f32_16x16x32_f16,
// 16384 ops each).  clk (2 * blocks words) receives, per workgroup, the
// shader-clock and real-time (hipDeviceAttributeWallClockRate) deltas of its
// first wave's loop, from which the clock the MFMAs ran at follows.  sink
// needs `blocks` words.  Errors: 1 on bad arguments.
int bonsai_p40_mfma_probe(int kind, int blocks, int iters, uint64_t * clk, uint32_t * sink,
                          bonsai_stream stream);

// Measurement helper: does the VALU work while the matrix core does?
// `blocks` workgroups of 4 waves; per iteration each wave issues 4 independent
// v_mfma_f32_16x16x32_f16 (mode 0 or 2) and nf x 16 independent fp32 FMAs
// (mode 1 or 2).  Time modes 0, 1 and 2 with events: mode 2 near the larger
// of the other two means overlap, near their sum means the two pipes take
// turns.  Mode 3 is the prefill GEMM's chunk step alone (4 MFMAs with a zero
// accumulator input, then 16 FMAs folding their results into accumulators;
// nf unused): the floor of the GEMM's per-chunk cost without operand staging,
// LDS reads and barriers.  sink needs `blocks` words.  Errors: 1 on bad
// arguments.
int bonsai_p40_overlap_probe(int mode, int nf, int blocks, int iters, uint32_t * sink, bonsai_stream stream);

// Measurement helper: the decode GEMV's weight stream alone -- the unit
// LDS-DMA schedule bonsai_p40_gemv runs for an n_out x n_in PQ2_0 matrix
// (n_in 5120 or 17408; same units, grid, wave numbering, ring depth, issue
// rounds and waits), with no activation and no arithmetic: the floor the
// GEMV's own addressing puts under it (the role of the reference's
// tools/bwtest.cu:70-90).  W 4-byte aligned, under 2 GiB; sink needs one word
// per CU and is written only in a practically impossible case.  Errors: 1 on
// other widths, bad sizes or alignment.
int bonsai_p40_unit_dma_probe(const void * W, int64_t n_out, int64_t n_in, uint32_t * sink,
                              bonsai_stream stream);

// Measurement: one empty kernel (`blocks` workgroups of `threads` threads,
// 1..1024); replayed back to back it gives the cost of a launch that waits for
// the one before it -- the floor under every kernel of a decode chain.
// Errors: 1 on bad arguments.
int bonsai_p40_launch_probe(int blocks, int threads, uint32_t * sink, bonsai_stream stream);

#ifdef __cplusplus
}
#endif
