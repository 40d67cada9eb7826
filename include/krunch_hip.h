/*
 * krunch_hip.h — C ABI of libkrunch_hip.so, the MI355X (gfx950) engine for
 * krunch's batched RWKV-4 compress/decompress path.
 *
 * Conventions (all entry points):
 *   - device pointers and plain sizes only; `stream` is a hipStream_t (NULL =
 *     the default stream); launches are asynchronous, nothing synchronises
 *     unless stated;
 *   - return 0 on success, a negative code on failure; kr_last_error() gives
 *     the message (thread-local);
 *   - the caller owns every buffer; coder states and RNN states are mutated
 *     in place (as the reference's ops do, krunch_ac/cuda/main.cpp:111-130);
 *   - fp16 tensors are passed as uint16_t bit patterns;
 *   - cdf_precision is log2 of the CDF total (24 in the reference,
 *     krunch_ac/cdf.py:18-19; range_coder.cuh:19-20).
 *
 * Each declaration names the reference interface it replaces.
 */
#ifndef KRUNCH_HIP_H
#define KRUNCH_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---------------------------------------------------------------- errors */
const char* kr_last_error(void);
int kr_abi_version(void);

/* ------------------------------------------------------------ range coder
 * Coder state: 4 x uint32 per stream, {low, high, pending, bit_offset} for
 * encoding and {low, high, value, bit_offset} for decoding
 * (range_coder.cuh:24-40). Encoders start from {0, 0xFFFFFFFF, 0, 0} and OR
 * bits into a zero-filled output buffer; out_cap bounds every write (an
 * overflow sets *err_flag, which may be NULL). Decoders read zero bits past
 * the end of a stream: in_len bounds the whole input buffer, byte_limits
 * (nullable) each stream's own length. base_byte_offsets (nullable where
 * noted) gives each stream's first byte.
 */

/* replaces krunch_ac_cuda.encode_step (main.cpp encode_step; encode_kernel.cu:53-101):
 * N rows of one stream, full CDF rows of cdf_stride int32 entries. */
int kr_encode_step(const int32_t* cdf, int cdf_stride, const int32_t* symbols, int N,
                   uint8_t* output_buf, uint32_t out_cap, uint32_t* state, int cdf_precision,
                   uint32_t* err_flag, void* stream);

/* replaces krunch_ac_cuda.encode_finalize (encode_kernel.cu:106-119). */
int kr_encode_finalize(uint8_t* output_buf, uint32_t out_cap, uint32_t* state,
                       uint32_t* err_flag, void* stream);

/* replaces krunch_ac_cuda.encode_step_batched (encode_kernel.cu:148-197):
 * one symbol per stream, CDF rows [B, V+1]. */
int kr_encode_step_batched(const int32_t* cdfs, int V, const int32_t* symbols,
                           uint8_t* output_buf, uint32_t out_cap,
                           const int32_t* base_byte_offsets, uint32_t* states, int B,
                           int cdf_precision, uint32_t* err_flag, void* stream);

/* Fused-compress form of encode_step_batched over T steps: pairs[b*pair_stride+t]
 * = (cdf[sym], cdf[sym+1]) as produced by kr_softmax_cdf_pairs; stream b encodes
 * its first n_valid[b] rows (n_valid nullable = T). No reference counterpart: the
 * reference writes full [rows, V+1] CDFs and reads two entries per row
 * (cpp_path.py:499-500 + encode_kernel.cu:110-111). */
int kr_encode_pairs_batched(const uint32_t* pairs, int T, long long pair_stride,
                            const int32_t* n_valid, uint8_t* output_buf, uint32_t out_cap,
                            const int32_t* base_byte_offsets, uint32_t* states, int B,
                            int cdf_precision, uint32_t* err_flag, void* stream);

/* replaces krunch_ac_cuda.encode_finalize_batched (encode_kernel.cu:199-215);
 * base_byte_offsets nullable (all streams at offset 0 is then B = 1). */
int kr_encode_finalize_batched(uint8_t* output_buf, uint32_t out_cap,
                               const int32_t* base_byte_offsets, uint32_t* states, int B,
                               uint32_t* err_flag, void* stream);

/* replaces krunch_ac_cuda.decode_init_batched and, with B = 1 and NULL offsets,
 * decode_init (decode_kernel.cu:28-45,138-157). */
int kr_decode_init_batched(const uint8_t* input_buf, uint32_t in_len,
                           const int32_t* base_byte_offsets, const int32_t* byte_limits,
                           uint32_t* states, int B, void* stream);

/* replaces krunch_ac_cuda.decode_step_batched and, with B = 1, decode_step
 * (decode_kernel.cu:50-110,159-216): CDF rows [B, V+1] -> out_syms [B]. */
int kr_decode_step_batched(const int32_t* cdfs, int V, const uint8_t* input_buf,
                           uint32_t in_len, const int32_t* base_byte_offsets,
                           const int32_t* byte_limits, uint32_t* states, int32_t* out_syms,
                           int B, int cdf_precision, void* stream);

/* -------------------------------------------------------------------- CDF
 * One 1024-thread workgroup per row. V <= 65032 or V = 65536: a row is held
 * in registers as at most 512 leaves of numpy's pairwise summation, and
 * V in 65033..65535 needs 513 (KR_EUNSUPPORTED). Probabilities are
 * renormalised with numpy's float32 summation order, so results are
 * bit-identical to krunch_ac/cdf.py:22-74. Softmax of fp16 logits (row
 * stride ld elements): e = exp(x - max) with a fixed FMA-based routine,
 * q = e * (1 / sum e), then cdf.py on q.
 */

/* replaces krunch_ac.probs_to_cdf (cdf.py:22-74) / probs_to_cdf_gpu
 * (gpu_encode.py:22-48): float probs [N, ld] -> uint32 cdf [N, V+1]. */
int kr_probs_to_cdf(const float* probs, int N, int V, long long ld, uint32_t* cdf_out,
                    int cdf_precision, void* stream);

/* replaces krunch_ac_cuda.det_softmax_cdf (det_softmax_cdf.cu:62-195) and the
 * caller's cumsum (cpp_path.softmax_cdfs_per_row, :490-501): out [N, V+1] int32
 * holds the cumulative CDF (cumulative = 1) or 0 followed by the per-symbol
 * counts (cumulative = 0, the reference op's output). */
int kr_softmax_cdf(const uint16_t* logits, int N, int V, long long ld, int32_t* out,
                   int cumulative, int cdf_precision, void* stream);

/* The softmax probabilities q [N, V] fed to the CDF (test and inspection aid;
 * the reference's torch.softmax in inference.py:254 plays this role). */
int kr_softmax_probs(const uint16_t* logits, int N, int V, long long ld, float* probs,
                     void* stream);

/* Scores of tokens, for callers that want a text's cost or a model's next
 * tokens without a coder (no reference counterpart): per row of logits (fp16,
 * or fp32 with logits_f32; any row stride ld >= V; V <= 2^30, N <= 2^24), in nats,
 *   logprob[row]  = ln softmax(row)[tokens[row]]; 0 where tokens[row] = -1 (a
 *                   row without a token), NaN for any other id outside 0..V-1;
 *   entropy[row]  = -sum p ln p;
 *   top_logprob, top_token [N, n_top]: the n_top most likely tokens, largest
 *                   first, equal ones by lower id (n_top <= 32 and <= V; 0:
 *                   none, both pointers may be NULL).
 * A logit of -inf is a masked token: probability 0, never among the top ones
 * (missing ones are -1 with -inf). A row of only masked tokens has logprob
 * -inf and entropy 0; a row with a NaN or +inf has NaN everywhere and top
 * tokens -1. Sums are fp32 in an order that does not depend on N; ln of a row's
 * sum is within 2^-17 whatever V, and a row that keeps rising adds 2^-22 for each
 * time that a thread's running maximum does (V / 8192 times at most). These are
 * the softmax's own probabilities: the coder's integer CDF adds a floor of one
 * count per token and rounds to 2^-cdf_precision. */
int kr_token_scores(const void* logits, int logits_f32, int N, int V, long long ld,
                    const int32_t* tokens, float* logprob, float* entropy, int n_top,
                    float* top_logprob, int32_t* top_token, void* stream);

/* Cross entropy of a head in pieces of the vocabulary, without its logits (no
 * reference counterpart; beside kr_token_scores, which reads logits): x fp16
 * [N, C] and W fp16 [V, C] by row strides ldx, ldw (multiples of 8, below 2^21; x
 * and W 16-byte aligned; C a multiple of 64 up to 16384; N, V <= 2^24, N V <= 2^44):
 *   z = x W' (exact products, fp32 sums, not rounded to fp16 as logits are)
 *   lse[n]  = ln sum_v e^z[n][v];   loss[n] = lse[n] - z[n][targets[n]]
 * in nats; loss is 0 where targets[n] = -1 and NaN for any other id outside
 * 0..V-1; a row with a NaN or +inf in z is NaN. Sums are fp32; the order of a row's
 * depends on N and V (z itself does not). ws: kr_head_loss_workspace_bytes, 256-byte
 * aligned (at most 8 bytes for a row and 64 columns, of up to 65536 rows at a time).
 *
 * kr_head_loss_backward, from the same inputs, the lse of the forward call and
 * dloss fp32 [N]:
 *   dz[n][v] = dloss[n] (e^(z[n][v] - lse[n]) - [v = targets[n]])
 *   dx = dz W [N, C],  dW = dz' x [V, C], contiguous, 16-byte aligned, fp16 or
 * (out_f32) fp32; dx or dW may be NULL. Rows with target -1 or dloss 0 have no
 * gradient, whatever x, lse and dloss hold there; other ids outside 0..V-1 give
 * NaN. For fp16 outputs dz is rounded to fp16 on a scale where the largest finite
 * |dloss| is 2^14..2^15: by 2^-11 of each dz above 2^-28 of the largest |dloss|, by
 * 2^-39 of the largest |dloss| below; what that leaves of the target's dz is added
 * back, in dx and in dW. For fp32 outputs dz has a second such part: 2^-22 of each, and
 * products of twice the length. Sums are fp32 in an order that depends on the sizes and
 * the output type alone. N C and V C are at most 2^33. ws:
 * kr_head_loss_backward_workspace_bytes (dx, dw: which of them is wanted; enough for both
 * output types), 256-byte aligned: at most 176 MB of dz at once (256 columns at least), a
 * copy of x and fp32 partial sums. Outputs must not overlap inputs. */
size_t kr_head_loss_workspace_bytes(int N, int C, int V);
int kr_head_loss(const uint16_t* x, long long ldx, int N, int C, const uint16_t* W, long long ldw, int V,
                 const int32_t* targets, float* loss, float* lse, void* ws, size_t ws_bytes, void* stream);
size_t kr_head_loss_backward_workspace_bytes(int N, int C, int V, int dx, int dw);
int kr_head_loss_backward(const uint16_t* x, long long ldx, int N, int C, const uint16_t* W, long long ldw,
                          int V, const int32_t* targets, const float* lse, const float* dloss, int out_f32,
                          void* dx, void* dW, void* ws, size_t ws_bytes, void* stream);

/* Fused compress stage: per row only the interval of symbols[row],
 * pairs[row] = (cdf[sym], cdf[sym+1]) — replaces det_softmax_cdf + cumsum +
 * the coder's two reads (cpp_path.py:499-500, encode_kernel.cu:110-111). */
int kr_softmax_cdf_pairs(const uint16_t* logits, int N, int V, long long ld,
                         const int32_t* symbols, uint32_t* pairs, int cdf_precision,
                         void* stream);

/* Fused decompress stage for B streams (one row of logits each): CDF, search
 * for the decoder target, range decode; writes out_syms[b] and, if tokens is
 * given, tokens[b*tok_stride + tok_count[b]++]. Streams with
 * tok_count[b] >= n_tokens[b] are skipped (n_tokens nullable). Replaces
 * softmax_cdfs_per_row + decode_step_batched (inference.py:427-431). */
int kr_softmax_cdf_decode(const uint16_t* logits, int B, int V, long long ld,
                          const uint8_t* input_buf, uint32_t in_len,
                          const int32_t* base_byte_offsets, const int32_t* byte_limits,
                          uint32_t* states, int32_t* out_syms, int32_t* tokens,
                          long long tok_stride, int32_t* tok_count, const int32_t* n_tokens,
                          int cdf_precision, void* stream);

/* ------------------------------------------------------------ GEMM / model
 * Matrices of the model are stored transposed, [out, in] (K contiguous).
 * Every output element is reduced the same way whatever M or the kernel:
 * P_s = chain of v_mfma_f32_16x16x32_f16 over the 256-wide K slice s (from
 * zero), acc = P_0 + P_1 + ... added left to right in fp32; so a row's
 * result does not depend on how many rows share the call (K % 256 == 0).
 */

/* W [K, N] (row stride ldw) -> Wt [N, K] (row stride ldt), fp16. */
int kr_transpose_f16(const uint16_t* W, long long ldw, int K, int N, uint16_t* Wt,
                     long long ldt, void* stream);
/* The same with Wf, the fragment-packed copy of Wt (kr_pack_fragments below:
 * kr_fragment_bytes(N, K) bytes, 16-byte aligned), in the same launch;
 * K % 32 == 0. */
int kr_transpose_pack_f16(const uint16_t* W, long long ldw, int K, int N, uint16_t* Wt,
                          long long ldt, uint16_t* Wf, void* stream);

/* replaces krunch_ac_cuda.det_matmul (layer_cpp.cpp:728-822, det_matmul_tc*.cu):
 * out = epilogue(x [M,K] @ W) with W given as Wt [N, ldw]. epilogue: 0 fp32 out,
 * 1 fp16 out, 2 fp16 sigmoid, 3 fp16 relu^2, 4 fp16 res + acc, 5 fp16
 * res + gate * acc (res/gate [M, ldo] fp16, res may alias out). */
int kr_det_matmul(const uint16_t* x, int M, int K, const uint16_t* Wt, long long ldw, int N,
                  void* out, long long ldo, int epilogue, const uint16_t* res,
                  const uint16_t* gate, void* stream);

/* Fragment-packed copy of Wt [N, K] (row stride ld) for the small-M GEMM: each
 * 16-row x 32-column block is one contiguous 1 KB run in MFMA operand order
 * (no reference counterpart: the reference's WMMA kernels read row-major
 * weights, layer_cpp.cpp:206-290). Output holds kr_fragment_bytes(N, K) bytes,
 * rows padded to a multiple of 16 with zeros; K % 32 == 0. */
size_t kr_fragment_bytes(int N, int K);
int kr_pack_fragments(const uint16_t* Wt, long long ld, int N, int K, uint16_t* out,
                      void* stream);

/* kr_det_matmul on fragment-packed operands (the stepped decode's GEMM): xf is
 * x [M, K] packed by kr_pack_fragments (rows padded to 16), Wf is Wt [N, K]
 * packed; M <= 512, N < 16384. out_packed = 1 writes an fp16 result packed as
 * an [M, N] operand of the next product (elementwise fp16 epilogues only,
 * N % 32 == 0). Same bits as kr_det_matmul on the unpacked operands. */
int kr_det_matmul_packed(const uint16_t* xf, int M, int K, const uint16_t* Wf, int N, void* out,
                         long long ldo, int epilogue, const uint16_t* res, const uint16_t* gate,
                         int out_packed, void* stream);

/* Up to three kr_det_matmul_packed products sharing M and K in one launch of
 * the small-M kernel (independent outputs, same bits as separate calls): the
 * stepped layer runs its channel-mix R (sigmoid) and K (relu^2, packed
 * output) products this way. No reference counterpart: the reference runs
 * them as two matmuls (layer_cpp.cpp:623-628). M <= 512. */
typedef struct kr_packed_job {
    const uint16_t* xf;          /* x [M, K] fragment-packed */
    const uint16_t* Wf;          /* Wt [N, K] fragment-packed */
    int N;
    void* out;                   /* as kr_det_matmul_packed */
    long long ldo;
    int epilogue;
    const uint16_t* res;
    const uint16_t* gate;
    int out_packed;
} kr_packed_job;
int kr_det_matmul_packed_multi(const kr_packed_job* jobs, int n_jobs, int M, int K, void* stream);

/* w8a8 (the reference only sketches an int8 path,
 * docs/INT8_WEIGHTS_DESIGN.md): symmetric int8 with one fp32 scale per row,
 * amax = max|x|, s = amax / 127, inv = 127 / amax (both 1 when the row is
 * zero; IEEE float32 divides), q = the exact product x * inv rounded to the
 * nearest integer, ties to even (|q| <= 127).
 * Rows are tokens for activations and output channels (rows of Wt) for
 * weights. q is [M, K] row-major, or fragment-packed (packed = 1, rows padded
 * to 16, kr_quant_bytes) for the small-M GEMM; K % 64 == 0. */
size_t kr_quant_bytes(int M, int K, int packed);
int kr_quantize_rows(const uint16_t* x, long long ldx, int M, int K, int8_t* q, float* scales,
                     int packed, void* stream);

/* int8 GEMM: acc = sum_k xq[m,k] * wq[n,k] exactly in int32, value =
 * (float(acc) * sa[m]) * sw[n], then the epilogue of kr_det_matmul. packed = 1:
 * xq and wq fragment-packed (wq packed by kr_pack_fragments on its 16-bit
 * view, K/2 columns), M <= 512; packed = 0: both row-major [*, K];
 * packed = 2: as 1, but xq points to fp16 activations, fragment-packed
 * (kr_pack_fragments layout), which the product quantises per row on load
 * by the rule above (sa is not read and may be null) - for finite
 * activations, the same bits as kr_quantize_rows followed by packed = 1, in
 * one launch (the row maximum compares fp16 bit patterns, so a NaN in a row
 * gives that row a NaN scale, where kr_quantize_rows' fmaxf skips it). */
int kr_det_matmul_i8(const int8_t* xq, const float* sa, int M, int K, const int8_t* wq,
                     const float* sw, int N, void* out, long long ldo, int epilogue,
                     const uint16_t* res, const uint16_t* gate, int packed, void* stream);

/* w8a8 copy of one matrix (kr_quantize_rows on Wt: one scale per output channel). */
typedef struct kr_matrix_q8 {
    const int8_t* q;                      /* [N, K] row-major int8 (rows = output channels) */
    const int8_t* qf;                     /* the same fragment-packed (16-bit view, K/2 columns) */
    const float* scale;                   /* [N] */
} kr_matrix_q8;

typedef struct kr_layer_q8 {
    kr_matrix_q8 K, V, R, O, fK, fV, fR;
} kr_layer_q8;

/* 4-bit weights with group scales (no reference counterpart; beside w8a8, for
 * products over few rows, where the weights are most of what is read): integers
 * q in -8..7 and one fp16 scale per output and group of 32, 64 or 128 inputs,
 * weight = q * s. kr_quantize_w4 makes them from W [K, N] fp16 (element (k, n)
 * at W[k * ldk + n * ldn], so either orientation): s = fp16(max |w| / 7), q =
 * w / s to the nearest integer, ties to even, at most 7 in size, 0 where s is
 * 0; a group with an infinity or NaN gets a NaN scale. K % 32 == 0, K <= 2^20, any N.
 * q holds kr_w4_bytes(N, K) bytes, 16-byte aligned: blocks of 16 outputs x 128
 * inputs, 1 KB, outputs major; lane l of a block holds four 32-bit words, word
 * c the inputs 32 c + 8 (l / 16) + e of output l % 16 as nibbles q + 8, e = 0,
 * 2, 4, 6, 1, 3, 5, 7 from the low nibble up; outputs and inputs past N and K
 * are q = 0. scales is fp16 [ceil(K / group), N rounded up to 16], 8-byte
 * aligned, 0 past N. */
size_t kr_w4_bytes(int N, int K);
int kr_quantize_w4(const uint16_t* W, long long ldk, long long ldn, int N, int K, int group, void* q,
                   uint16_t* scales, void* stream);

/* out = epilogue(x [M, K] @ W) with W in 4 bits; epilogues, res and gate as
 * kr_det_matmul. x rows have stride ldx (a multiple of 8, x 16-byte aligned),
 * out rows any stride ldo >= N. Products q x are exact, their sums and the
 * scaling fp32: c_g = chain of v_mfma_f32_16x16x32_f16 over group g, acc =
 * fma(s_g, c_g, acc) over the groups in order from zero; so a row has the same
 * bits for any M. A NaN scale makes its output NaN; infinite scales are not
 * supported. With many rows the fp16 products are the faster ones: 768 x 50277 from
 * about 100 rows on at groups of 32, 190 at 64, 260 at 128. M <= 2^19. out must
 * not overlap x (out may be res). */
int kr_det_matmul_w4(const uint16_t* x, long long ldx, int M, int K, const void* q,
                     const uint16_t* scales, int group, int N, void* out, long long ldo, int epilogue,
                     const uint16_t* res, const uint16_t* gate, void* stream);

typedef struct kr_layer_weights {
    const void *ln1_w, *ln1_b;            /* fp16 [C] */
    const void *tm_k, *tm_v, *tm_r;       /* fp16 [C] */
    const float *decay;                   /* fp32 [C], w = -exp(time_decay_raw) */
    const float *first;                   /* fp32 [C], u = time_first */
    const void *Kt, *Vt, *Rt, *Ot;        /* fp16 [C, C] */
    const void *ln2_w, *ln2_b;            /* fp16 [C] */
    const void *ftm_k, *ftm_r;            /* fp16 [C] */
    const void *fKt;                      /* fp16 [F, C] */
    const void *fVt;                      /* fp16 [C, F] */
    const void *fRt;                      /* fp16 [C, C] */
    /* Fragment-packed copies of the seven matrices above (kr_pack_fragments),
     * read up to 512 rows (B*T) and, by the register-fed products, up to 1536
     * .. 2304 by width and codec; all NULL = use the row-major ones. */
    const void *Kf, *Vf, *Rf, *Of, *fKf, *fVf, *fRf;
    /* w8a8 codec: int8 copies of the seven matrices; the
     * layer then runs its GEMMs on int8 MFMA with per-token activation
     * quantisation. NULL = fp16 codec. The head stays fp16 either way. */
    const kr_layer_q8* q8;
} kr_layer_weights;

typedef struct kr_model_weights {
    int n_layer, C, F, V;                 /* C in {256,512,768,1024}, F % 64 == 0, V <= 65536 */
    const void* emb;                      /* fp16 [V, C] */
    const void *ln_out_w, *ln_out_b;      /* fp16 [C] */
    const void* headT;                    /* fp16 [V, C] */
    const kr_layer_weights* layers;       /* host array, n_layer entries */
    /* Fragment-packed copy of headT (kr_pack_fragments), read for C <= 768 by
     * the decode head (M <= 512 rows) and by the register-held rows above that;
     * NULL = the row-major head. */
    const void* headF;
} kr_model_weights;

/* w = -exp(raw) for the WKV decay (the rwkv loader's transform the reference
 * relies on, wkv_kernel.cu:41-45). */
int kr_prepare_decay(const float* raw, float* out, int n, void* stream);

/* RNN state of B streams for n_layer layers in one buffer; per layer
 * [att_xx fp16 | ffn_xx fp16 | aa | bb | pp fp32], each [B, C]
 * (cpp_path.fresh_state_batched, cpp_path.py:412-425). */
size_t kr_state_bytes(int n_layer, int B, int C);
/* att_xx = ffn_xx = aa = bb = 0, pp = -1e30 (fill kernel, graph-safe). */
int kr_state_init(void* state, int n_layer, int B, int C, void* stream);

/* Scratch needed by the layer stack for M = B*T rows. */
size_t kr_forward_workspace_bytes(long long M, int C, int F);

/* replaces krunch_ac_cuda.rwkv4_layer_step_cpp / _t1 (layer_cpp.cpp:294-637):
 * one layer over x [B*T, C] fp16 in place, state tensors [B, C] mutated. */
int kr_layer_step(const kr_layer_weights* L, int C, int F, void* x, int B, int T,
                  void* att_xx, float* aa, float* bb, float* pp, void* ffn_xx, void* ws,
                  size_t ws_bytes, void* stream);

/* kr_layer_step without a workspace argument, for callers that cannot
 * allocate device memory (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc). No counterpart in the reference. The
 * workspace is a static device array of KR_NOALLOC_SCRATCH_BYTES per GPU,
 * held until the process ends; nothing is allocated or freed. A call whose
 * kr_forward_workspace_bytes(B*T, C, F) exceeds it fails (KR_EINVAL): at
 * C = 768, F = 3072 that is B*T <= 1024 rows. Every call on one GPU shares
 * the array, so calls that overlap on one GPU (other streams or threads)
 * race; consecutive calls on one stream do not. Same kernels and bits as
 * kr_layer_step. */
#define KR_NOALLOC_SCRATCH_BYTES (32u << 20)
int kr_layer_step_noalloc(const kr_layer_weights* L, int C, int F, void* x, int B, int T,
                          void* att_xx, float* aa, float* bb, float* pp, void* ffn_xx,
                          void* stream);

/* Layer phase profiler; replaces the reference's KRUNCH_PHASE_PROFILE
 * profiler with read_phase_times / reset_phase_times (layer_cpp.cpp:111-157,
 * 825-836). When on, every kr_layer_step call (outside stream capture)
 * records HIP events between its phases on its stream, waits for the last one
 * and adds the elapsed milliseconds to running sums. The phases (this build's
 * kernel split; a fused launch leaves the phase it absorbed empty) are
 * kr_phase_name(0..kr_phase_count()-1): ln1_mix, kvr_matmul, wkv,
 * ow_matmul_residual, ln2_mix, ffn_rk_matmul, ffn_v_matmul_residual.
 * kr_phase_profile(1 / 0) turns it on / off and returns the previous state
 * (-1 only queries); KRUNCH_PHASE_PROFILE=1 turns it on at first use. */
int kr_phase_profile(int enable);
int kr_phase_count(void);
const char* kr_phase_name(int i);
int kr_read_phase_times(double* ms, int n, long long* call_count);
int kr_reset_phase_times(void);

/* Decode-step timing, the same profiler's role (layer_cpp.cpp:111-157) for
 * the stepped decode. kr_step_timing(p) with p = 3 (ow_matmul_residual),
 * 5 (ffn_rk_matmul) or 6 (ffn_v_matmul_residual) times that phase's product
 * in every layer of every later decode step (kr_decode_step, kr_decode_run,
 * graph or eager; at few streams phase 5's launch holds the LN2-mix too): each
 * of its waves stores its start and end on the GPU's
 * 100 MHz steady counter (a vector store per wave, also at every replay of a
 * captured graph), and in eager steps the launch goes through
 * hipExtLaunchKernel with two HIP events that take its dispatch's start and
 * end. Nothing else in the step changes. p = -1 turns it off; *previous
 * (nullable) receives the earlier setting. kr_step_timing_read waits for the
 * device and writes, for layers 0 .. n_read - 1 of the last timed step
 * (n_read = min(n, layers)), the launch's event duration (-1 for a graph
 * step) and its wave span (last wave end minus first wave start), in
 * microseconds; it fails if no timed step ran since the last reading. */
int kr_step_timing(int phase, int* previous);
int kr_step_timing_read(double* launch_us, double* span_us, int n, int* n_read);

/* replaces launch_krunch_wkv_forward (wkv_kernel.cu:75-92), fused with the
 * receptance: ry = fp16(r * fp16(y)); k, v fp32 [B*T, C], r/ry fp16. */
int kr_wkv(int B, int T, int C, const float* decay, const float* first, const float* k,
           const float* v, const uint16_t* r, float* aa, float* bb, float* pp, uint16_t* ry,
           void* stream);

/* WKV with heads (no reference counterpart; beside kr_wkv, for models whose
 * recurrence keeps a D x D matrix per head): r, k, v fp16 [B, T, H, D] by token
 * strides ldr, ldk, ldv (elements, multiples of 8; streams follow at T tokens),
 * state fp32 [B, H, D, D] (key channel major) updated in place, decay (w) and
 * first (u) fp32 [H], y fp16 by ldy:
 *   y_t = r_t (S + u k_t' v_t);  S <- e^w S + k_t' v_t
 * w above 0 counts as 0, -inf is no memory. D is 64 or 128. lens (nullable = T)
 * gives each stream's tokens, clamped to 0..T: its state stops there and its
 * later rows of y are zeros, whatever r, k, v hold there. chunked = 0: token by
 * token in fp32; T tokens in one call have the bits of T calls of one. chunked =
 * 1: 64 tokens at a time on the matrix units, for prompts: equal to that up to
 * rounding, and in an order that depends on B * H and T (the time axis is split
 * over workgroups where heads are few); rounding is 2^-22 of a value that enters
 * the matrix units (a state element, a weight r k' between two tokens, a decayed v)
 * and 2^-38 of the largest one of its value channel's state column, its
 * token's weights or its channel's v of the 64 tokens. A NaN or infinity of a token
 * then also reaches y of up to 63 tokens before it, and an infinite state
 * element makes y of its value channel infinite or NaN; other channels of the
 * state keep their values and their y. Calls of at most 8 tokens are the same
 * in both. y must not overlap r, k or v. ws: kr_wkv_heads_workspace_bytes
 * (chunked only, may be 0), 16-byte aligned, as r, k, v, state and y. */
size_t kr_wkv_heads_workspace_bytes(int B, int T, int H, int D);
int kr_wkv_heads(int B, int T, int H, int D, const uint16_t* r, long long ldr, const uint16_t* k,
                 long long ldk, const uint16_t* v, long long ldv, const float* decay,
                 const float* first, const int32_t* lens, float* state, uint16_t* y, long long ldy,
                 int chunked, void* ws, size_t ws_bytes, void* stream);

/* The gated delta rule (no reference counterpart; beside kr_wkv_heads, for models
 * whose keys replace what they had stored): q, k, v fp16 [B, T, H, D] by token strides
 * ldq, ldk, ldv (elements, multiples of 8; streams follow at T tokens), log_decay (g)
 * and beta fp32 [B, T, H] by token strides ldg, ldb, state fp32 [B, H, D, D] (key
 * channel major) updated in place, y fp16 by ldy:
 *   S <- e^g S;  u = beta (v_t - k_t S);  S <- S + k_t' u;  y_t = q_t S
 * g above 0 counts as 0, below -10000 (-inf too) is no memory. D is 64 or 128. lens
 * (nullable = T) gives each stream's tokens, clamped to 0..T: its state stops there and
 * its later rows of y are zeros, whatever the inputs hold there. chunked = 0: token by
 * token in fp32; T tokens in one call have the bits of T calls of one. chunked = 1:
 * 64 tokens at a time on the matrix units, for prompts: equal to that up to rounding
 * (2^-22 of a value that enters the matrix units: a state element, a weight between two
 * tokens, what a token writes; and 2^-38 of the largest one of its column or row), in
 * an order that depends on B * H and T (the time axis is split over workgroups where
 * heads are few); a NaN or infinity of a token then also reaches y of up to 63 tokens
 * before it. Calls of at most 8 tokens are the same in both. Keys of length 1 and beta in
 * 0..1 keep the recurrence stable; others are computed, too. y must not overlap q, k or
 * v. ws: kr_gated_delta_workspace_bytes (chunked only: 12 D D bytes for each head and
 * segment of a split, else 0), 16-byte aligned, as q, k, v, state and y. */
size_t kr_gated_delta_workspace_bytes(int B, int T, int H, int D);
int kr_gated_delta(int B, int T, int H, int D, const uint16_t* q, long long ldq, const uint16_t* k,
                   long long ldk, const uint16_t* v, long long ldv, const float* log_decay, long long ldg,
                   const float* beta, long long ldb, const int32_t* lens, float* state, uint16_t* y,
                   long long ldy, int chunked, void* ws, size_t ws_bytes, void* stream);

/* Gradients of kr_gated_delta (chunked): its inputs, with state as it was before the
 * call; dy fp16 [B, T, H, D] by ldy, and dstate fp32 [B, H, D, D], the gradient of the
 * state after the call (NULL: zeros). Writes dq, dk, dv fp16 [B, T, H, D], dlog_decay and
 * dbeta fp32 [B, T, H], all contiguous, and dstate0 fp32 [B, H, D, D], the gradient
 * of state. Tokens past lens have gradient 0, as a log_decay above 0 or below -10000
 * has. Values rounded as in the forward pass, sums fp32; dlog_decay is a difference of
 * sums over a chunk's tokens, so its error is relative to those, not to a small
 * gradient behind a strong decay. T <= 4194240. ws:
 * kr_gated_delta_backward_workspace_bytes (for each head and 64 tokens two states and two
 * rows of D fp32 values a token, 8 D (D + 64) bytes; for each head one state more, and
 * where the time axis is split five a segment, 20 D D bytes), 256-byte aligned; it must
 * not overlap anything, nor outputs the inputs. Everything but log_decay, beta, lens and
 * their gradients is 16-byte aligned. */
size_t kr_gated_delta_backward_workspace_bytes(int B, int T, int H, int D);
int kr_gated_delta_backward(int B, int T, int H, int D, const uint16_t* q, long long ldq, const uint16_t* k,
                            long long ldk, const uint16_t* v, long long ldv, const float* log_decay,
                            long long ldg, const float* beta, long long ldb, const int32_t* lens,
                            const float* state, const uint16_t* dy, long long ldy, const float* dstate,
                            uint16_t* dq, uint16_t* dk, uint16_t* dv, float* dlog_decay, float* dbeta,
                            float* dstate0, void* ws, size_t ws_bytes, void* stream);

/* All layers over x [B*T, C] (cpp_path.forward_packed_window's layer loop,
 * :155-160; forward_stepped_batched's with T = 1, :451-456). */
int kr_forward_layers(const kr_model_weights* m, void* x, int B, int T, void* state, void* ws,
                      size_t ws_bytes, void* stream);

/* x[row] = emb[ids[row]] (cpp_path.py:154,450). */
int kr_embed(const kr_model_weights* m, const int32_t* ids, int M, void* x, void* stream);

/* logits [M, ld] fp16 = LN_out(x) @ head (cpp_path.py:161-163); xn: [M, C] scratch
 * (x itself: LN_out in place).
 * The head has a reduction of its own: for every logit one chain of
 * v_mfma_f32_16x16x32_f16 over the whole K = C from zero, then fp16; the
 * same bits for any M, with or without headF (decode and compress agree). */
int kr_head_logits(const kr_model_weights* m, const void* x, int M, void* xn, void* logits,
                   long long ld, void* stream);
/* The same with xn (not x) holding M rounded up to 16 rows: the heads that read
 * fragment-packed rows, which kr_head_logits gives whole 16-row blocks only,
 * then take any M. */
int kr_head_logits_rows16(const kr_model_weights* m, const void* x, int M, void* xn, void* logits,
                          long long ld, void* stream);

/* One packed compress window for B streams x T tokens (rows b*T + t): embed,
 * layers, then per block of head_rows rows head logits -> softmax -> symbol
 * interval into pairs [B*T, 2]. Replaces the per-window body of
 * InferenceEngine._compress_chunk_cpp (inference.py:331-338). Encode the pairs
 * with kr_encode_pairs_batched. */
int kr_compress_window(const kr_model_weights* m, const int32_t* inputs, const int32_t* targets,
                       int B, int T, void* state, void* x, void* ws, size_t ws_bytes,
                       void* logits, long long ld, int head_rows, uint32_t* pairs,
                       int cdf_precision, void* stream);

/* One stepped decompress step for B streams: embed syms, layers (T = 1), head,
 * fused CDF + range decode; syms is read (previous tokens) and overwritten
 * (decoded tokens). Replaces one iteration of the loop in
 * _decompress_chunks_batched_cpp (inference.py:427-434). */
int kr_decode_step(const kr_model_weights* m, int B, void* state, int32_t* syms, void* x,
                   void* ws, size_t ws_bytes, void* logits, long long ld,
                   const uint8_t* input_buf, uint32_t in_len, const int32_t* base_byte_offsets,
                   const int32_t* byte_limits, uint32_t* ac_states, int32_t* tokens,
                   long long tok_stride, int32_t* tok_count, const int32_t* n_tokens,
                   int cdf_precision, void* stream);

/* n_steps decode steps. The B streams are split into n_groups groups of
 * ceil(B/n_groups) streams with independent workspaces (ws_bytes >=
 * kr_decode_workspace_bytes); with use_graph one step is captured into a HIP
 * graph whose groups are parallel branches, so their latency-bound kernels
 * overlap, and the graph is replayed n_steps times (the reference's graph
 * path, cpp_path.py:229-276). With one group, the graph's decode kernel also
 * runs layer 0's LN1-mix of each decoded symbol for the next step (a first-
 * step graph and a later-steps graph); the state, tokens and coder state it
 * leaves are those of the eager path (use_graph = 0), x and ws are scratch.
 * The graphs run on `stream`, which must not be capturing. Synchronous with
 * respect to the work it enqueues. */
size_t kr_decode_workspace_bytes(int B, int n_groups, int C, int F);
int kr_decode_run(const kr_model_weights* m, int B, void* state, int32_t* syms, void* x,
                  void* ws, size_t ws_bytes, void* logits, long long ld,
                  const uint8_t* input_buf, uint32_t in_len, const int32_t* base_byte_offsets,
                  const int32_t* byte_limits, uint32_t* ac_states, int32_t* tokens,
                  long long tok_stride, int32_t* tok_count, const int32_t* n_tokens,
                  int cdf_precision, int n_steps, int n_groups, int use_graph, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* KRUNCH_HIP_H */
