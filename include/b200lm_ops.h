/*
 * b200lm_ops.h — operator-level C ABI of libb200lm.so.
 *
 * The reference hides its operators inside compiled_model_.Run
 * (runtime/executor/llm_litert_compiled_model_executor.cc:271,407,522), so these
 * entry points have no one-to-one reference symbol; each names the step of
 * that opaque graph it stands for.  They exist for the operator parity tests
 * and for the attention / GEMM micro-benchmarks; those on device memory (the
 * decode attention without allocations and what follows it) are also for use in
 * a serving loop of one's own.  All pointers are HOST
 * memory unless a name says "dev"; the calls copy in, run the kernel, copy out.
 * Same status-code and error-string conventions as b200lm.h.
 */
#ifndef B200LM_OPS_H_
#define B200LM_OPS_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Host-only repacks of canonical int4 rows ([n][k/2] bytes, element 2j in the
 * low nibble) into the decode layout (16x64 mma tiles) and the tensor-core GEMM
 * layout (128-row x 64-k blocks).  out must hold n_pad*k/2 bytes, n_pad = n
 * rounded up to 16 (W4T) or 128 (W4G).  No GPU needed. */
int B200LmOps_RepackW4T(const uint8_t* packed, int64_t n, int64_t k, uint8_t* out, char** err);
int B200LmOps_RepackW4G(const uint8_t* packed, int64_t n, int64_t k, uint8_t* out, char** err);

/* Bit-exact unpack gate: uploads canonical rows, repacks, and has the GPU
 * expand the decode layout back to int8 [n][k] with the same device function
 * the GEMV uses to address its tiles. */
int B200LmOps_UnpackW4(int32_t device, const uint8_t* packed, int64_t n, int64_t k, int8_t* out, char** err);

/* Decode GEMV (the int4 fully-connected op at batch 1..4):
 * y[c][n] = scale[n] * sum_k W[n][k] x[c][k], x quantised to `nterms` int8 terms. */
int B200LmOps_GemvW4(int32_t device, const uint8_t* packed, const float* scale, int64_t n, int64_t k,
                     const float* x, int32_t ncols, int32_t nterms, int32_t kslices, float* y, char** err);

/* Prefill GEMM (the int4 fully-connected op over T tokens), bf16 activations:
 * mode B200LM_GEMM_CHECK or B200LM_GEMM_TCGEN05.  out is [T][n] fp32.
 * repeat > 1 re-runs the kernel and, when ms_out != NULL, returns the mean
 * device time per run in milliseconds (CUDA events). */
int B200LmOps_GemmW4(int32_t device, int32_t mode, const uint8_t* packed, const float* scale, int64_t n,
                     int64_t k, const float* a, int32_t t, int32_t ksplit, int32_t repeat, float* out,
                     float* ms_out, char** err);

/* Fused gate/up GEMM + GeGLU: out[T][ffn] = gelu_tanh(A Wg^T) * (A Wu^T). */
int B200LmOps_GemmGegluW4(int32_t device, int32_t mode, const uint8_t* gate_packed, const float* gate_scale,
                          const uint8_t* up_packed, const float* up_scale, int64_t ffn, int64_t k,
                          const float* a, int32_t t, float* out, char** err);

/* Attention against a paged cache built from k, v [S][hkv][hd] (fp32 host,
 * stored as fp32 or bf16 pages): queries q [T][hq][hd] at positions
 * qpos0 + i (or all at qpos0 + T - 1 ... see below), causal, optional window
 * (window <= 0: global).  No QK-norm, no RoPE (raw q/k, as the attention-only
 * micro-benchmark specifies).  nsplit > 1 runs the split-KV decode kernel plus
 * the log-sum-exp combine (T is then a batch of independent single-token
 * queries all at position S - 1); nsplit == 1 runs the prefill kernel.
 * kv_bf16: bit 0 = bf16 pages (else fp32); bit 1 (decode only) = every query
 * gets its own physical copy of the cache and its own page table, i.e. a
 * batch of independent sequences instead of queries sharing one cache; bit 2
 * (decode only) = the streaming kernel of the wide decode step
 * (csrc/decode_wide.cuh: K / V in blocks of 16 positions by bulk async copies
 * into a shared-memory ring) instead of the register-resident split kernel
 * (two keys in flight per warp). */
int B200LmOps_Attention(int32_t device, const float* q, const float* k, const float* v, int32_t t, int32_t s,
                        int32_t hq, int32_t hkv, int32_t hd, int32_t qpos0, int32_t window,
                        int32_t kv_bf16, int32_t nsplit, int32_t repeat, float* out, float* ms_out,
                        char** err);

/* Causal self-attention over s tokens on the tensor cores (the prefill flash
 * kernel of the executor: TMA-staged K/V tiles, tcgen05 MMA with TMEM
 * accumulators, GQA-packed query tiles).  q [s][hq][hd], k, v [s][hkv][hd] fp32
 * host, rounded to bf16 on the device; scores are q.k / sqrt(hd); window <= 0
 * means global.  hd must be 128 or 256.  The kernel shifts the softmax by a
 * constant bound on the scores instead of a running maximum; inputs whose
 * scores could exceed 40 are rejected with FailedPrecondition.  repeat > 1
 * re-runs the kernel and returns the mean device time in ms_out. */
int B200LmOps_AttentionPrefillTc(int32_t device, const float* q, const float* k, const float* v, int32_t s,
                                 int32_t hq, int32_t hkv, int32_t hd, int32_t window, int32_t repeat, float* out,
                                 float* ms_out, char** err);

/* Split-KV decode attention that allocates nothing.  It has no counterpart in
 * the reference.  It is for callers that may not allocate device memory when
 * they call in: code running inside another runtime's execution callback, a
 * serving loop that bans allocator calls once it is warm, or a process whose
 * GPU memory was handed out completely at start-up.  The ordinary entry point
 * above allocates scratch for the per-split partial results on every call;
 * this one keeps them (with the query positions and an error word) in one
 * fixed 8 MiB device array that is part of the library image (and 129 KiB of
 * counters beside it), so every GPU that loads the library holds those until
 * the process ends.
 *
 * All pointers are DEVICE memory owned by the caller:
 *   q_dev          [batch] rows of (hq + 2*hkv)*hd floats, the layout of a fused
 *                  QKV projection; only the first hq*hd floats of a row are read
 *   k_pages_dev,   paged cache [page][hkv][256][hd], fp32 or bf16 (kv_bf16),
 *   v_pages_dev    already holding positions 0 .. s-1
 *   page_table_dev [ceil(s/256)] physical page of each logical page
 *   out_dev        [batch][hq][hd] floats
 * Every query sits at position s-1 (causal; window <= 0 means global).  Work is
 * queued on `stream` (NULL: the default stream) and the call returns without
 * waiting.
 *
 * With all four data pointers on 16-byte boundaries the kernel of
 * csrc/attn_mma.cuh runs, or that of csrc/attn_tc.cuh for many queries over a
 * long bf16 cache; they read the cache once for the whole batch and pick their
 * own number of splits; nsplit then only enters the size check below.
 * Otherwise the split kernel of csrc/decode_ops.cuh runs with nsplit splits.
 *
 * Limits: batch <= 16368 and batch*hq*nsplit*(hd+2)*4 bytes <= 8 MiB - 64 KiB;
 * larger requests are rejected with InvalidArgument.  Pages of a bf16 cache
 * start within 32 TB of the first.  The first call on a
 * device looks up the array's address and sets a kernel attribute; make that
 * first call before starting any stream capture.  All calls on a device share
 * the array, which keeps what the last call left in it; two calls whose kernels
 * overlap on the GPU -- different streams, no ordering between them -- race on
 * it, which spoils the results of those calls and of no others.  The error word
 * is only written by a call that fails and stays until the status call below has
 * reported it.  The caller's current device is left as it was.  The per-device
 * set-up is done under a lock, so first calls from several threads are safe. */
int B200LmOps_AttentionDecodeStatic(int32_t device, const float* q_dev, const void* k_pages_dev,
                                    const void* v_pages_dev, const int32_t* page_table_dev, int32_t batch, int32_t s,
                                    int32_t hq, int32_t hkv, int32_t hd, int32_t window, int32_t kv_bf16,
                                    int32_t nsplit, float* out_dev, void* stream, char** err);

/* Which kernel a call of this shape with aligned pointers runs on `device`: how
 * many clusters of csrc/attn_tc.cuh share the keys of 128 query rows of a kv
 * head, or 0 where csrc/attn_mma.cuh takes the call.  For tests and tuning; does
 * the per-device set-up of the call above.  No counterpart in the reference. */
int B200LmOps_AttentionDecodeStaticClusters(int32_t device, int32_t batch, int32_t s, int32_t hq, int32_t hkv,
                                            int32_t hd, int32_t window, int32_t kv_bf16, int32_t* clusters,
                                            char** err);

/* Status of the work queued by B200LmOps_AttentionDecodeStatic on `stream`:
 * waits for the stream, then reads and clears the error word of the static
 * array (no allocation either).  Returns OK when no call since the last status
 * call failed, InvalidArgument when a query position lay outside the cache,
 * DeadlineExceeded when a bounded device-side wait gave up; *device_error
 * (optional) receives the raw word.  No counterpart in the reference. */
int B200LmOps_AttentionDecodeStaticStatus(int32_t device, void* stream, int32_t* device_error, char** err);

/* ---------------------------------------------------------------------------
 * Operators over caller-owned DEVICE memory: int4 products with group scales,
 * QK norm with rotation, and a cache held in 4 bits with the attention over it.
 * The reference has no counterpart.  Common to all of them:
 *   - arguments ending in _dev are device memory of `device`; arguments are
 *     checked on the host first, on failure nothing has been queued.  Work goes
 *     to `stream` (NULL: the default stream), the call returns without waiting,
 *     allocates nothing, keeps no state and may be captured into a CUDA graph
 *     (the first call of a kind on a device raises kernel attributes: make it
 *     before the capture).  The caller's current device is left as it was.
 *   - element types are B200LM_F32, B200LM_BF16, B200LM_F16; strides count
 *     elements.  Rows need no more alignment than their type's.  Inputs and
 *     outputs do not overlap unless said so.
 *   - status_dev (may be NULL) is a word of the caller's, zero at first, to which
 *     the kernels add what only they can see: a position or a length outside the
 *     cache, the page table or the rotation table, a page number outside the
 *     pool (of the pages that a token, or any row of a sequence, needs).  What
 *     such a token or sequence would have written stays as it was; the others
 *     are served.  B200LmOps_DeviceStatus reads the word. */
#define B200LM_F32 0
#define B200LM_BF16 1
#define B200LM_F16 2

/* Waits for `stream`, then reads and clears *status_dev.  OK when the word was
 * zero, InvalidArgument for a bad position, length or page, DeadlineExceeded when
 * a bounded device-side wait gave up; *device_error (optional) receives the word.
 * Not for a stream that is being captured.  Calls on other streams need words of
 * their own: what they add between the read and the clearing would be lost. */
int B200LmOps_DeviceStatus(int32_t device, void* stream, int32_t* status_dev, int32_t* device_error, char** err);

/* Weights of a grouped int4 product, laid out once on the host.  packed as above
 * ([n][k/2], two's complement, k even), scale and offset (NULL: none)
 * [n][ceil(k/group)] as 16-bit words, fp16 or bf16.  The image is made of strips
 * of 16 rows and, in a strip, blocks of 128 k; rows and k past the end are zero.
 * A block is two tiles of 64 k of the W4T layout (512 bytes each), then the scales
 * [8][128/group][2] of the rows g and g + 8, then the offsets likewise.
 * GemvW4GroupedBytes gives the image's size. */
int B200LmOps_GemvW4GroupedBytes(int64_t n, int64_t k, int32_t group, int32_t has_offset, int64_t* bytes, char** err);
int B200LmOps_RepackW4Grouped(const uint8_t* packed, const uint16_t* scale, const uint16_t* offset, int64_t n, int64_t k,
                              int32_t group, uint8_t* out, char** err);

/* y[c][r] = sum over the groups g of k of
 *   scale[r][g] * sum_{j in g} q[r][j] x[c][j]  +  offset[r][g] * sum_{j in g} x[c][j]
 * for ncols = 1 .. 8 columns x [ncols] rows of ldx, y [ncols] rows of ldy.  group is
 * 32, 64 or 128 (the last group may be shorter), scale_type B200LM_BF16 or _F16.
 * w_dev is the image above, on a 16-byte boundary.  Sums are in fp32, and x
 * enters exact to 2^-27 of the largest value of a block of 128 (2^-20 with more
 * than four columns of a 16-bit type), of 2^-117 where all of them are smaller; an
 * infinity or NaN in a column makes all of its outputs NaN. */
int B200LmOps_GemvW4Grouped(int32_t device, const void* w_dev, int32_t scale_type, int32_t has_offset, int64_t n, int64_t k,
                            int32_t group, const void* x_dev, int32_t x_type, int64_t ldx, int32_t ncols, void* y_dev,
                            int32_t y_type, int64_t ldy, void* stream, char** err);

/* RMSNorm of every query and key head (gains q_gain_dev, k_gain_dev [hd] fp32;
 * NULL: no norm) and the rotation of its first `rot` elements, element i paired
 * with i + rot/2, by row pos_dev[t] of cos_dev, sin_dev [rope_rows][rot/2] fp32.
 * qkv_dev holds `tokens` rows of qkv_stride elements, the layout of a fused QKV
 * projection: hq query heads, hkv key heads, hkv value heads.  Queries go to
 * q_out_dev [tokens] rows of q_stride, keys to k_out_dev rows of k_stride, in
 * qkv's type; they may be the rows' own places.  hd is 64, 128 or 256, rot a
 * multiple of 16 up to hd (0: no rotation; cos_dev and sin_dev are not read).
 * Norms hold over the whole range of the types (sums of squares beyond fp32's are
 * taken in fp64); a row of zeros with eps 0 gives NaN.
 * A token with a negative position is padding: its rows are left alone. */
int B200LmOps_QkNormRope(int32_t device, const void* qkv_dev, int32_t type, int64_t qkv_stride, int32_t tokens, int32_t hq,
                         int32_t hkv, int32_t hd, int32_t rot, const float* q_gain_dev, const float* k_gain_dev, float eps,
                         const float* cos_dev, const float* sin_dev, int32_t rope_rows, const int32_t* pos_dev,
                         void* q_out_dev, int64_t q_stride, void* k_out_dev, int64_t k_stride, int32_t* status_dev,
                         void* stream, char** err);

/* A paged cache in 4 bits.  For each page and kv head lie, in this order, the K
 * codes, K scales, V codes and V scales of 256 positions.  A row of hd elements is
 * cut into groups of 64 or 128; of each group are kept m = its lowest value,
 * s = (highest - lowest) / 15, both rounded to fp32 and then fp16 (lowest and
 * highest are held to -64000 .. 64000), and a code of 4 bits for each element,
 * c = rint((x - m) / s) held to 0 .. 15, which stands for s c + m.  A group with an
 * infinity or NaN stands for NaN.
 * Scales are [256][hd/group] pairs (s, m).  Codes lie in planes of 128 elements
 * (64 at hd 64), [plane][256] rows of 64 (32) bytes.  In a K row byte
 * w t + 4 j + i (t, i < 4; w = 16 or 8) holds the elements 32 j + 4 t + i (low
 * nibble) and 16 more (high).  In a V row byte b of unit g (8 units of 8 or 4
 * bytes) holds the elements 16 b + g and 8 more; where planes are 128 wide the
 * units of positions with bit 1 set lie four further, modulo eight.
 * page_table_dev [batch] rows of table_stride: physical page of each logical page
 * of 256 positions.  pages_dev on a 16-byte boundary. */
typedef struct B200LmKv4Cache {
  int32_t struct_size;           /* sizeof(B200LmKv4Cache) */
  int32_t batch;                 /* sequences (rows of the page table) */
  int32_t hkv, hd, group;
  int32_t reserved;              /* 0 */
  void* pages_dev;
  int64_t num_pages;
  const int32_t* page_table_dev;
  int64_t table_stride;          /* logical pages of a sequence */
} B200LmKv4Cache;

/* Bytes of one page: 512 * hkv * (hd/2 + 4 * hd/group). */
int B200LmOps_Kv4PageBytes(int32_t hkv, int32_t hd, int32_t group, int64_t* bytes, char** err);

/* QkNormRope whose keys, with the value heads of the rows, go into the cache: token
 * t is position pos_dev[t] of sequence seq_dev[t] (NULL: sequence t).  Norm and
 * rotation of the keys are computed in fp64 and rounded to fp32, so that codes do
 * not depend on the order of sums.  No two tokens of a call may share a position. */
int B200LmOps_QkNormRopeAppendKv4(int32_t device, const void* qkv_dev, int32_t type, int64_t qkv_stride, int32_t tokens,
                                  int32_t hq, int32_t hkv, int32_t hd, int32_t rot, const float* q_gain_dev,
                                  const float* k_gain_dev, float eps, const float* cos_dev, const float* sin_dev,
                                  int32_t rope_rows, const int32_t* pos_dev, void* q_out_dev, int64_t q_stride,
                                  const B200LmKv4Cache* cache, const int32_t* seq_dev, int32_t* status_dev, void* stream,
                                  char** err);

/* The values that cached positions stand for: rows pos_dev[t] of sequences
 * seq_dev[t] (NULL: sequence t), k_out_dev and v_out_dev [tokens][hkv][hd] of
 * out_type (either may be NULL).  Negative positions are padding. */
int B200LmOps_Kv4Read(int32_t device, const B200LmKv4Cache* cache, const int32_t* seq_dev, const int32_t* pos_dev,
                      int32_t tokens, int32_t out_type, void* k_out_dev, void* v_out_dev, int32_t* status_dev, void* stream,
                      char** err);

/* softmax(scale q K^T) V over the cache.  q_dev holds the query tokens of all
 * sequences one behind the other, `tokens` rows of q_stride elements with hq heads
 * of hd first; sequence b has the rows q_start_dev[b] .. q_start_dev[b + 1] - 1
 * (NULL: one row each), at most max_q of them.  kv_len_dev[b] positions of it are
 * cached, the query tokens being the last of them: token i of n sits at position
 * kv_len - n + i, sees the positions up to its own and, with window > 0, the last
 * `window` of those.  A row that sees none gives zeros.  kv_len_dev[b] is at most
 * max_kv, max_kv at most 256 * table_stride.  scale <= 0 means 1/sqrt(hd).  out_dev
 * is of q's type; rows behind the last sequence's are left as they were.
 *
 * Scores are sums of exact products in fp32.  A key's weight, times its scales,
 * enters the second product to 2^-22, or 2^-36 of the row's largest where that is
 * more.  bf16 calls with many rows of a kv head (16 and more, head sizes 128 and
 * 256) may run on a kernel that rounds weights and values to fp16 for the second
 * product, 2^-11 of each (weights 2^-36 of the row's largest where that is more).
 * A group that stands for NaN makes, in V, its own elements of the rows that see
 * the position NaN, in K all of those rows.
 *
 * workspace_dev (16-byte boundary) holds the partial results of sequences whose
 * keys are shared out; AttentionKv4Workspace says how many bytes calls up to the
 * given sizes may need (on 148 multiprocessors up to 5 MB for single tokens, 20 MB
 * for chunks).  Zero it once before its first use; every call leaves the part that has to be zero at zero.  It serves one
 * call at a time: calls, or replays of captured ones, that may overlap need
 * workspaces of their own. */
int B200LmOps_AttentionKv4Workspace(int32_t device, int32_t batch, int32_t hkv, int32_t hd, int32_t hq, int32_t max_q,
                                    int32_t max_kv, int64_t* bytes, char** err);
int B200LmOps_AttentionKv4(int32_t device, const B200LmKv4Cache* cache, const void* q_dev, int32_t q_type, int64_t q_stride,
                           const int32_t* kv_len_dev, const int32_t* q_start_dev, int32_t tokens, int32_t max_q,
                           int32_t max_kv, int32_t hq, int32_t window, float scale, void* out_dev, int64_t out_stride,
                           void* workspace_dev, int64_t workspace_bytes, int32_t* status_dev, void* stream, char** err);

#ifdef __cplusplus
}
#endif
#endif /* B200LM_OPS_H_ */
