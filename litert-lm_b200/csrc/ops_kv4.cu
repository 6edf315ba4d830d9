// Entry points of the QK norm with rotation, of the cache in 4 bits and of the attention over it (include/b200lm_ops.h).
#include "../../include/b200lm_ops.h"
#include "kv4_attn.cuh"
#include "kv4_rows.cuh"
#include "op_host.h"

#include <algorithm>

namespace b200lm {

static void check_heads(int hkv, int hd) {
  B2_CHECK(hkv > 0 && hkv <= 1024, kInvalidArgument, "hkv must be 1 .. 1024");
  B2_CHECK(hd == 64 || hd == 128 || hd == 256, kUnimplemented, "hd must be 64, 128 or 256");
}
static void check_group(int hd, int group) {
  B2_CHECK((group == 64 || group == 128) && group <= hd, kUnimplemented, "group must be 64 or 128 and at most hd");
}
static void check_query_heads(int hq) { B2_CHECK(hq > 0 && hq <= 4096, kInvalidArgument, "hq must be 1 .. 4096"); }
static void check_type(int type) { B2_CHECK(type >= kF32 && type <= kF16, kInvalidArgument, "unknown element type"); }
static void check_pointer(const void* p, size_t align, const char* name) {
  B2_CHECK(p, kInvalidArgument, std::string(name) + " is null");
  B2_CHECK((uintptr_t)p % align == 0, kInvalidArgument, std::string(name) + " is misaligned");
}
static void check_optional(const void* p, size_t align, const char* name) {
  if (p) check_pointer(p, align, name);
}

static Kv4Args cache_args(const B200LmKv4Cache* c) {
  B2_CHECK(c, kInvalidArgument, "cache is null");
  B2_CHECK(c->struct_size == (int32_t)sizeof(B200LmKv4Cache), kInvalidArgument, "cache: struct_size does not match this library");
  B2_CHECK(c->reserved == 0, kInvalidArgument, "cache: reserved must be 0");
  check_heads(c->hkv, c->hd);
  check_group(c->hd, c->group);
  B2_CHECK(c->batch > 0 && c->batch <= 65535, kInvalidArgument, "cache: batch must be 1 .. 65535");
  B2_CHECK(c->num_pages > 0 && c->num_pages <= 0x7FFFFFFF, kInvalidArgument, "cache: num_pages out of range");
  B2_CHECK(c->table_stride > 0 && c->table_stride <= 0x7FFFFFFF / kKv4Page, kInvalidArgument, "cache: table_stride out of range");
  check_pointer(c->pages_dev, 16, "cache: pages_dev");
  check_pointer(c->page_table_dev, 4, "cache: page_table_dev");
  Kv4Args k{};
  k.pages = reinterpret_cast<uint8_t*>(c->pages_dev);
  k.num_pages = c->num_pages;
  k.table = c->page_table_dev;
  k.table_stride = c->table_stride;
  k.batch = c->batch;
  k.hkv = c->hkv;
  k.d = Kv4Dims{c->hd, c->group};
  return k;
}

// Rows of a call, checked; the caller adds where keys go.
static RowArgs row_args(const void* qkv, int type, int64_t stride, int tokens, int hq, int hkv, int hd, int rot, const float* q_gain, const float* k_gain, float eps,
                        const float* cos, const float* sin, int rope_rows, const int* pos, void* q_out, int64_t q_stride, int* status) {
  check_type(type);
  check_heads(hkv, hd);
  check_query_heads(hq);
  B2_CHECK(tokens >= 0, kInvalidArgument, "tokens is negative");
  B2_CHECK(stride >= (int64_t)(hq + 2 * hkv) * hd && q_stride >= (int64_t)hq * hd, kInvalidArgument, "a row stride is shorter than its row");
  B2_CHECK(rot >= 0 && rot <= hd && rot % 16 == 0, kInvalidArgument, "rot must be a multiple of 16 up to hd");
  B2_CHECK(eps >= 0.f, kInvalidArgument, "eps must not be negative");
  check_pointer(qkv, elem_size(type), "qkv_dev");
  check_pointer(q_out, elem_size(type), "q_out_dev");
  check_pointer(pos, 4, "pos_dev");
  check_optional(q_gain, 4, "q_gain_dev");
  check_optional(k_gain, 4, "k_gain_dev");
  check_optional(status, 4, "status_dev");
  if (rot > 0) {
    check_pointer(cos, 4, "cos_dev");
    check_pointer(sin, 4, "sin_dev");
    B2_CHECK(rope_rows > 0, kInvalidArgument, "rope_rows must be positive");
  }
  RowArgs a{};
  a.qkv = qkv; a.stride = stride; a.type = type; a.tokens = tokens; a.hq = hq; a.hkv = hkv; a.rot = rot;
  a.q_gain = q_gain; a.k_gain = k_gain; a.eps = eps; a.cos = cos; a.sin = sin; a.rope_rows = rope_rows; a.pos = pos;
  a.q_out = q_out; a.q_stride = q_stride; a.status = status;
  return a;
}

template <int HD, int TYPE, int GROUP, int NP, bool VEC>
static void launch_rows_at(cudaStream_t st, const RowArgs& a) {
  const int n = NP * (256 / HD);
  const long long jobs = (long long)a.tokens * ((a.hq + n - 1) / n + (GROUP ? 2 : 1) * ((a.hkv + n - 1) / n));
  B2_CHECK(jobs <= 0x7FFFFFFF, kInvalidArgument, "too many tokens for one call");
  launch_pdl(qk_norm_rope_kernel<HD, TYPE, GROUP, NP, VEC>, dim3((unsigned)((jobs + 3) / 4)), dim3(128), 0, st, a);
}
template <int HD, int TYPE, int GROUP>
static void launch_rows_as(cudaStream_t st, const RowArgs& a, int sms) {
  const int esz = elem_size(a.type);
  const uintptr_t all = (uintptr_t)a.qkv | (uintptr_t)(a.stride * esz) | (uintptr_t)a.q_out | (uintptr_t)(a.q_stride * esz) | (uintptr_t)a.k_out | (uintptr_t)(a.k_stride * esz) |
                        (uintptr_t)a.q_gain | (uintptr_t)a.k_gain | (a.rot ? (uintptr_t)a.cos | (uintptr_t)a.sin : 0);
  // one pass a warp while that leaves room on the GPU (a token's chain of latencies), else four: rotation and gains are read less often
  if (all % 16 != 0) launch_rows_at<HD, TYPE, GROUP, 1, false>(st, a);
  else if ((long long)a.tokens * (a.hq + 2 * a.hkv) <= 16ll * sms) launch_rows_at<HD, TYPE, GROUP, 1, true>(st, a);
  else launch_rows_at<HD, TYPE, GROUP, 4, true>(st, a);
}
template <int HD, int GROUP>
static void launch_rows_type(cudaStream_t st, const RowArgs& a, int sms) {
  if (a.type == kF32) launch_rows_as<HD, kF32, GROUP>(st, a, sms);
  else if (a.type == kBf16) launch_rows_as<HD, kBf16, GROUP>(st, a, sms);
  else launch_rows_as<HD, kF16, GROUP>(st, a, sms);
}
// group 0: keys are written out.
static void launch_rows(cudaStream_t st, const RowArgs& a, int hd, int group, int sms) {
  if (hd == 64) group ? launch_rows_type<64, 64>(st, a, sms) : launch_rows_type<64, 0>(st, a, sms);
  else if (hd == 128) group == 64 ? launch_rows_type<128, 64>(st, a, sms) : group ? launch_rows_type<128, 128>(st, a, sms) : launch_rows_type<128, 0>(st, a, sms);
  else group == 64 ? launch_rows_type<256, 64>(st, a, sms) : group ? launch_rows_type<256, 128>(st, a, sms) : launch_rows_type<256, 0>(st, a, sms);
}

template <int HD, int GROUP, int TYPE>
static void launch_read_as(cudaStream_t st, const Kv4Args& kv, const int* seq, const int* pos, int tokens, void* k, void* v, int* status) {
  const int n = 256 / HD;
  const long long jobs = (long long)tokens * ((kv.hkv + n - 1) / n);
  B2_CHECK(jobs <= 0x7FFFFFFF, kInvalidArgument, "too many tokens for one call");
  const dim3 grid((unsigned)((jobs + 3) / 4));
  if (((uintptr_t)k | (uintptr_t)v) % 16 == 0) launch_pdl(kv4_read_kernel<HD, TYPE, GROUP, true>, grid, dim3(128), 0, st, kv, seq, pos, tokens, k, v, status);
  else launch_pdl(kv4_read_kernel<HD, TYPE, GROUP, false>, grid, dim3(128), 0, st, kv, seq, pos, tokens, k, v, status);
}
template <int HD, int GROUP>
static void launch_read(cudaStream_t st, int type, const Kv4Args& kv, const int* seq, const int* pos, int tokens, void* k, void* v, int* status) {
  if (type == kF32) launch_read_as<HD, GROUP, kF32>(st, kv, seq, pos, tokens, k, v, status);
  else if (type == kBf16) launch_read_as<HD, GROUP, kBf16>(st, kv, seq, pos, tokens, k, v, status);
  else launch_read_as<HD, GROUP, kF16>(st, kv, seq, pos, tokens, k, v, status);
}

void launch_kv4_attn_64(cudaStream_t st, const Kv4AttnArgs& a, int rb);
void launch_kv4_attn_128(cudaStream_t st, const Kv4AttnArgs& a, int rb);
void launch_kv4_attn_256(cudaStream_t st, const Kv4AttnArgs& a, int rb);

void launch_kv4_chunk(cudaStream_t st, const Kv4AttnArgs& a);

// How a call's keys are shared out.  A unit is a (sequence, kv head, row tile).
struct Kv4Plan {
  int rb, row_tiles, share, splits;
  int64_t units, bytes;
};
constexpr int kChunkRows = 16;             // fewer query rows of a kv head never pay for the tensor-core kernel

// The tensor-core kernel: one CTA an SM, tiles of 64 keys.
static Kv4Plan plan_chunk(int batch, int hkv, int hd, int hq, int max_q, int max_kv, int window, int sms) {
  Kv4Plan p;
  const long long rows = (long long)max_q * (hq / hkv);
  p.rb = 128;
  const long long tiles = (rows + 127) / 128;
  p.units = tiles * hkv * batch;
  B2_CHECK(tiles * hkv * 16 <= 0x7FFFFFFF, kInvalidArgument, "too many query rows for one call");
  p.row_tiles = (int)tiles;
  const int round = 64;
  const long long keys = (window > 0 ? std::min<long long>(max_kv, (long long)window + max_q) : max_kv) + round;
  long long best = std::min<long long>(std::max<long long>(1, sms / p.units), 16);      // one round of CTAs
  best = std::max<long long>(1, std::min(best, keys / (4 * round)));                    // of at least four tiles each
  p.share = (int)std::min<long long>((keys / best + round) / round * round, 1 << 30);
  p.splits = (int)((keys + p.share - 1) / p.share);
  p.bytes = kKaTickets * 4 + std::min<int64_t>(sms, p.units * 16) * 128 * (hd + 2) * 4;
  return p;
}
static Kv4Plan plan_attention(int batch, int hkv, int hd, int hq, int max_q, int max_kv, int window, int sms) {
  Kv4Plan p;
  const long long rows = (long long)max_q * (hq / hkv);
  p.rb = ka_rows(hd, rows);
  const long long tiles = (rows + p.rb - 1) / p.rb;
  p.units = tiles * hkv * batch;
  B2_CHECK(tiles * hkv <= 0x7FFFFFFF, kInvalidArgument, "too many query rows for one call");
  p.row_tiles = (int)tiles;
  // Shares for 2 CTAs an SM four times over, so that sequences of different lengths even out (64 of 300 .. 8192: 90 us against 129
  // with one share a CTA), but none shorter than four rounds of the CTA's warps where the GPU is full without (16 x 5 rows
  // over a window of 1024: 27 us against 32), as a share costs its set-up and its part of the join.
  const int round = (hd == 256 ? 16 : 32) * kKaWarps;
  const long long keys = (window > 0 ? std::min<long long>(max_kv, (long long)window + max_q) : max_kv) + 32;
  auto shares = [&](long long ctas) { return std::min<long long>(512, std::max<long long>(1, ctas * sms / p.units)); };
  auto length = [&](long long n) { return (keys / n + round) / round * round; };
  p.share = (int)std::min<long long>(std::max(length(shares(8)), std::min<long long>(4 * round, length(shares(2)))), 1 << 30);
  p.splits = (int)((keys + p.share - 1) / p.share);
  B2_CHECK(tiles * hkv * p.splits <= 0x7FFFFFFF, kInvalidArgument, "too many query rows for one call");
  // What a call up to these sizes may need: fewer units can have more shares, but all of them at most these.
  p.bytes = kKaTickets * 4 + std::min<int64_t>(512 * p.units, 8 * sms) * p.rb * (hd + 2) * 4;
  return p;
}

// Which of the two a call takes, by what they would cost in us.  Fitted to 16 .. 64 rows over 2048 and 4096 keys of 1, 16 and 64
// sequences: mma.sync grows with rows x keys (64 sequences x 4 kv heads x 16 rows x 4096 keys of 256: 289 us, 32 rows 565),
// the tensor-core kernel with tiles of 128 rows (265 and 268, and 26 us at the least, where 16 rows over 2048 keys take 13).
static bool chunk_pays(const Kv4Plan& few, const Kv4Plan& many, int hd, int max_kv, int window, int max_q, int sms) {
  const double keys = window > 0 ? std::min<double>(max_kv, (double)window + max_q) : max_kv;
  const double simple = 8 + 0.25e-6 * (double)few.units * keys * hd;
  const double tiles = (double)((many.units * many.splits + sms - 1) / sms) * many.share / 64;
  return (hd == 256 ? 20 + 1.85 * tiles : 14 + 0.9 * tiles) < simple;
}

}  // namespace b200lm

using namespace b200lm;

extern "C" int B200LmOps_DeviceStatus(int32_t device, void* stream, int32_t* status_dev, int32_t* device_error, char** err) {
  OP_TRY
  check_pointer(status_dev, 4, "status_dev");
  require_device(device);
  DeviceScope scope(device);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int word = 0;
  B2_CUDA(cudaMemcpyAsync(&word, status_dev, sizeof(int), cudaMemcpyDeviceToHost, st));
  B2_CUDA(cudaStreamSynchronize(st));
  if (device_error) *device_error = word;
  if (word != kDevOk) B2_CUDA(cudaMemsetAsync(status_dev, 0, sizeof(int), st));
  if (word == kDevBadPosition) throw Error{kInvalidArgument, "a position, length or page lay outside its table"};
  if (word == kDevBarrierTimeout) throw Error{kDeadlineExceeded, "a bounded device-side wait gave up"};
  if (word != kDevOk) throw Error{kInternal, "device error word " + std::to_string(word)};
  OP_END
}

extern "C" int B200LmOps_Kv4PageBytes(int32_t hkv, int32_t hd, int32_t group, int64_t* bytes, char** err) {
  OP_TRY
  B2_CHECK(bytes, kInvalidArgument, "null pointer");
  check_heads(hkv, hd);
  check_group(hd, group);
  *bytes = (int64_t)hkv * Kv4Dims{hd, group}.head_bytes();
  OP_END
}

extern "C" int B200LmOps_QkNormRope(int32_t device, const void* qkv_dev, int32_t type, int64_t qkv_stride, int32_t tokens, int32_t hq,
                                    int32_t hkv, int32_t hd, int32_t rot, const float* q_gain_dev, const float* k_gain_dev, float eps,
                                    const float* cos_dev, const float* sin_dev, int32_t rope_rows, const int32_t* pos_dev,
                                    void* q_out_dev, int64_t q_stride, void* k_out_dev, int64_t k_stride, int32_t* status_dev,
                                    void* stream, char** err) {
  OP_TRY
  RowArgs a = row_args(qkv_dev, type, qkv_stride, tokens, hq, hkv, hd, rot, q_gain_dev, k_gain_dev, eps, cos_dev, sin_dev, rope_rows, pos_dev, q_out_dev, q_stride, status_dev);
  check_pointer(k_out_dev, elem_size(type), "k_out_dev");
  B2_CHECK(k_stride >= (int64_t)hkv * hd, kInvalidArgument, "a row stride is shorter than its row");
  a.k_out = k_out_dev;
  a.k_stride = k_stride;
  require_device(device);
  if (tokens == 0) return kOk;
  DeviceScope scope(device);
  launch_rows(reinterpret_cast<cudaStream_t>(stream), a, hd, 0, device_sms(device));
  OP_END
}

extern "C" int B200LmOps_QkNormRopeAppendKv4(int32_t device, const void* qkv_dev, int32_t type, int64_t qkv_stride, int32_t tokens,
                                             int32_t hq, int32_t hkv, int32_t hd, int32_t rot, const float* q_gain_dev,
                                             const float* k_gain_dev, float eps, const float* cos_dev, const float* sin_dev,
                                             int32_t rope_rows, const int32_t* pos_dev, void* q_out_dev, int64_t q_stride,
                                             const B200LmKv4Cache* cache, const int32_t* seq_dev, int32_t* status_dev, void* stream,
                                             char** err) {
  OP_TRY
  RowArgs a = row_args(qkv_dev, type, qkv_stride, tokens, hq, hkv, hd, rot, q_gain_dev, k_gain_dev, eps, cos_dev, sin_dev, rope_rows, pos_dev, q_out_dev, q_stride, status_dev);
  a.kv = cache_args(cache);
  B2_CHECK(cache->hkv == hkv && cache->hd == hd, kInvalidArgument, "the cache's heads are not the rows'");
  check_optional(seq_dev, 4, "seq_dev");
  B2_CHECK(seq_dev || tokens <= cache->batch, kInvalidArgument, "more tokens than sequences: seq_dev says whose they are");
  a.seq = seq_dev;
  require_device(device);
  if (tokens == 0) return kOk;
  DeviceScope scope(device);
  launch_rows(reinterpret_cast<cudaStream_t>(stream), a, hd, cache->group, device_sms(device));
  OP_END
}

extern "C" int B200LmOps_Kv4Read(int32_t device, const B200LmKv4Cache* cache, const int32_t* seq_dev, const int32_t* pos_dev,
                                 int32_t tokens, int32_t out_type, void* k_out_dev, void* v_out_dev, int32_t* status_dev, void* stream,
                                 char** err) {
  OP_TRY
  const Kv4Args kv = cache_args(cache);
  check_type(out_type);
  B2_CHECK(tokens >= 0, kInvalidArgument, "tokens is negative");
  B2_CHECK(k_out_dev || v_out_dev, kInvalidArgument, "null pointer");
  check_optional(k_out_dev, elem_size(out_type), "k_out_dev");
  check_optional(v_out_dev, elem_size(out_type), "v_out_dev");
  check_optional(seq_dev, 4, "seq_dev");
  check_optional(status_dev, 4, "status_dev");
  check_pointer(pos_dev, 4, "pos_dev");
  B2_CHECK(seq_dev || tokens <= cache->batch, kInvalidArgument, "more tokens than sequences: seq_dev says whose they are");
  require_device(device);
  if (tokens == 0) return kOk;
  DeviceScope scope(device);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const auto read = kv.d.hd == 64 ? launch_read<64, 64> : kv.d.hd == 128 ? (kv.d.group == 64 ? launch_read<128, 64> : launch_read<128, 128>) : kv.d.group == 64 ? launch_read<256, 64> : launch_read<256, 128>;
  read(st, out_type, kv, seq_dev, pos_dev, tokens, k_out_dev, v_out_dev, status_dev);
  OP_END
}

static void check_attention(int batch, int hkv, int hd, int hq, int max_q, int max_kv) {
  check_heads(hkv, hd);
  check_query_heads(hq);
  B2_CHECK(batch > 0 && batch <= 65535, kInvalidArgument, "batch must be 1 .. 65535");
  B2_CHECK(hq % hkv == 0, kInvalidArgument, "hq must be a multiple of hkv");
  B2_CHECK((long long)max_q * (hq / hkv) <= (1 << 30), kInvalidArgument, "too many query rows for one call");
  B2_CHECK(max_q >= 1 && max_q <= (1 << 30) && max_kv >= 0 && max_kv <= (1 << 30), kInvalidArgument, "max_q must be 1 .. 2^30, max_kv 0 .. 2^30");
}

extern "C" int B200LmOps_AttentionKv4Workspace(int32_t device, int32_t batch, int32_t hkv, int32_t hd, int32_t hq, int32_t max_q,
                                               int32_t max_kv, int64_t* bytes, char** err) {
  OP_TRY
  B2_CHECK(bytes, kInvalidArgument, "null pointer");
  check_attention(batch, hkv, hd, hq, max_q, max_kv);
  require_device(device);
  DeviceScope scope(device);
  const int sms = device_sms(device);
  *bytes = plan_attention(batch, hkv, hd, hq, max_q, max_kv, 0, sms).bytes;
  if (hd >= 128 && (long long)max_q * (hq / hkv) >= kChunkRows) *bytes = std::max(*bytes, plan_chunk(batch, hkv, hd, hq, max_q, max_kv, 0, sms).bytes);
  OP_END
}

extern "C" int B200LmOps_AttentionKv4(int32_t device, const B200LmKv4Cache* cache, const void* q_dev, int32_t q_type, int64_t q_stride,
                                      const int32_t* kv_len_dev, const int32_t* q_start_dev, int32_t tokens, int32_t max_q,
                                      int32_t max_kv, int32_t hq, int32_t window, float scale, void* out_dev, int64_t out_stride,
                                      void* workspace_dev, int64_t workspace_bytes, int32_t* status_dev, void* stream, char** err) {
  OP_TRY
  Kv4AttnArgs a{};
  a.kv = cache_args(cache);
  check_attention(cache->batch, cache->hkv, cache->hd, hq, max_q, max_kv);
  check_type(q_type);
  B2_CHECK(tokens >= 0, kInvalidArgument, "tokens is negative");
  B2_CHECK(q_start_dev || (tokens == cache->batch && max_q == 1), kInvalidArgument, "without q_start_dev every sequence has one token: tokens = batch, max_q = 1");
  B2_CHECK(max_kv <= cache->table_stride * kKv4Page, kInvalidArgument, "max_kv is beyond the page table");
  B2_CHECK(q_stride >= (int64_t)hq * cache->hd && out_stride >= (int64_t)hq * cache->hd, kInvalidArgument, "a row stride is shorter than its row");
  check_pointer(q_dev, elem_size(q_type), "q_dev");
  check_pointer(out_dev, elem_size(q_type), "out_dev");
  check_pointer(kv_len_dev, 4, "kv_len_dev");
  check_optional(q_start_dev, 4, "q_start_dev");
  check_optional(status_dev, 4, "status_dev");
  check_optional(workspace_dev, 16, "workspace_dev");
  require_device(device);
  if (tokens == 0) return kOk;
  DeviceScope scope(device);
  if (window < 0 || window >= max_kv) window = 0;           // it hides nothing; and a position less a window stays within 32 bits
  a.q = q_dev; a.q_type = q_type; a.q_stride = q_stride; a.kv_len = kv_len_dev; a.q_start = q_start_dev;
  a.tokens = tokens; a.max_q = max_q; a.max_kv = max_kv; a.hq = hq; a.window = window;
  a.qscale = 1.4426950408889634f * (scale > 0.f ? scale : 1.f / sqrtf((float)cache->hd));
  a.out = out_dev; a.out_stride = out_stride; a.status = status_dev;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int sms = device_sms(device);
  Kv4Plan p = plan_attention(cache->batch, cache->hkv, cache->hd, hq, max_q, max_kv, window, sms);
  bool chunk = false;
  if (q_type == kBf16 && cache->hd >= 128 && (long long)max_q * (hq / cache->hkv) >= kChunkRows) {
    const Kv4Plan many = plan_chunk(cache->batch, cache->hkv, cache->hd, hq, max_q, max_kv, window, sms);
    chunk = chunk_pays(p, many, cache->hd, max_kv, window, max_q, sms);
    if (chunk) p = many;
  }
  B2_CHECK(p.splits == 1 || (workspace_dev && workspace_bytes >= p.bytes), kInvalidArgument,
           "the workspace is smaller than AttentionKv4Workspace says: " + std::to_string(p.bytes) + " bytes");
  a.row_tiles = p.row_tiles; a.share = p.share; a.splits = p.splits;
  a.tickets = reinterpret_cast<unsigned*>(workspace_dev);
  a.parts = reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(workspace_dev) + kKaTickets * 4);
  if (chunk) launch_kv4_chunk(st, a);
  else if (cache->hd == 64) launch_kv4_attn_64(st, a, p.rb);
  else if (cache->hd == 128) launch_kv4_attn_128(st, a, p.rb);
  else launch_kv4_attn_256(st, a, p.rb);
  OP_END
}
