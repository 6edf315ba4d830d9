// Rows of a fused QKV projection: RMSNorm of each query and key head with the rotation in the same pass, keys written out or,
// with the values, put into the cache in 4 bits; and the way back from there.
//
//   y = x / sqrt(mean x^2 + eps) * gain;   (y_i, y_{i + r/2}) -> (y_i c_i - y_{i + r/2} s_i, y_{i + r/2} c_i + y_i s_i)
//   m = fp16(low), s = fp16((high - low) / 15), code = rint((x - m) / s) held to 0 .. 15
//
// Every byte is read and written once.  What bounds it are issue slots and latencies of the rows' chains, behind them HBM: 8191
// rows of 8 and 4 heads of 256 in bf16 take 24.7 us = 4.4 TB/s (68 % of the copy rate); 2001 rows of 32 and 16 heads of 128 with
// their codes 29.1 us, where the bytes take 9 (300 instructions a pass of 256 elements; ALU 45 %, conversions 25 % busy; with
// registers for 24 warps an SM, unbounded a fifth more); reading them back 9.4 us = 3.9 TB/s; a single token 1.9 us.
//
// A lane holds eight neighbouring elements, so a pass of a warp takes 1, 2 or 4 heads (of 256, 128, 64); the other halves of the
// pairs lie at the same place of a lane rot / 16 further and come from there as they lay in memory.  A warp takes up to four
// passes over heads of one kind and token, asks for their rows at once and keeps gain and rotation multiplied in registers.
// Queries, and keys that are written out, are computed in fp32, heads whose squares leave that in fp64.  Keys that go into the cache are computed in fp64 and rounded to fp32 before their
// codes are decided: a code next to a border would otherwise depend on the order of the sum, and one step of a code is a
// fifteenth of the group's range.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"
#include "gemv_grouped.cuh"
#include "kv4.h"

namespace b200lm {

struct Kv4Args {
  uint8_t* pages;
  long long num_pages;
  const int* table;
  long long table_stride;
  int batch, hkv;
  Kv4Dims d;
};

struct RowArgs {
  const void* qkv;
  long long stride;
  int type, tokens, hq, hkv, rot;
  const float *q_gain, *k_gain;
  float eps;
  const float *cos, *sin;
  int rope_rows;
  const int* pos;
  void* q_out;
  long long q_stride;
  void* k_out;                 // null: keys and values go into the cache
  long long k_stride;
  const int* seq;
  Kv4Args kv;
  int* status;
};

__device__ __forceinline__ void set_status(int* status, int code) {
  if (status) atomicMax(status, code);
}

// W neighbouring elements of a row as they lie in memory: whole words where the row starts allow it (`vec`), else one by one.
template <int TYPE, int W>
struct RawRow {
  static constexpr int N = TYPE == kF32 ? W : W / 2;
  uint32_t u[N];
  __device__ __forceinline__ void load(const void* p, long long i, bool vec) {
    const char* a = reinterpret_cast<const char*>(p) + i * elem_size(TYPE);
    if (vec) {
      if constexpr (N >= 4) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
          const uint4 v = reinterpret_cast<const uint4*>(a)[j / 4];
          u[j] = v.x; u[j + 1] = v.y; u[j + 2] = v.z; u[j + 3] = v.w;
        }
      } else if constexpr (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(a);
        u[0] = v.x; u[1] = v.y;
      } else {
        u[0] = *reinterpret_cast<const uint32_t*>(a);
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if constexpr (TYPE == kF32) u[j] = reinterpret_cast<const uint32_t*>(a)[j];
        else u[j] = reinterpret_cast<const uint16_t*>(a)[2 * j] | (uint32_t)reinterpret_cast<const uint16_t*>(a)[2 * j + 1] << 16;
      }
    }
  }
  __device__ __forceinline__ void store(void* p, long long i, bool vec) const {
    char* a = reinterpret_cast<char*>(p) + i * elem_size(TYPE);
    if (vec) {
      if constexpr (N >= 4) {
#pragma unroll
        for (int j = 0; j < N; j += 4) reinterpret_cast<uint4*>(a)[j / 4] = make_uint4(u[j], u[j + 1], u[j + 2], u[j + 3]);
      } else if constexpr (N == 2) {
        *reinterpret_cast<uint2*>(a) = make_uint2(u[0], u[1]);
      } else {
        *reinterpret_cast<uint32_t*>(a) = u[0];
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if constexpr (TYPE == kF32) reinterpret_cast<uint32_t*>(a)[j] = u[j];
        else {
          reinterpret_cast<uint16_t*>(a)[2 * j] = (uint16_t)u[j];
          reinterpret_cast<uint16_t*>(a)[2 * j + 1] = (uint16_t)(u[j] >> 16);
        }
      }
    }
  }
  __device__ __forceinline__ void get(float (&x)[W]) const {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if constexpr (TYPE == kF32) x[j] = __uint_as_float(u[j]);
      else {
        const float2 f = gg_pair(u[j], TYPE == kBf16);
        x[2 * j] = f.x;
        x[2 * j + 1] = f.y;
      }
    }
  }
  __device__ __forceinline__ void put(const float (&x)[W]) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if constexpr (TYPE == kF32) u[j] = __float_as_uint(x[j]);
      else if constexpr (TYPE == kBf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
        u[j] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
        u[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
  }
};
template <int W>
__device__ __forceinline__ void row_load(const void* p, long long i, int type, float (&x)[W]) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p) + i * elem_size(type);
  auto as = [&](auto raw) {
    constexpr int bytes = 4 * decltype(raw)::N;
    raw.load(p, i, at % (bytes < 16 ? bytes : 16) == 0);
    raw.get(x);
  };
  if (type == kF32) as(RawRow<kF32, W>());
  else if (type == kBf16) as(RawRow<kBf16, W>());
  else as(RawRow<kF16, W>());
}

constexpr int kVec = 8;             // elements of a lane

// 1 / sqrt(m) to 2^-43 for every m: m = 4^k f with f in 1 .. 4, where fp32's root starts.
static __device__ __noinline__ double far_root(double m) {
  if (!(m > 0.0 && m < INFINITY)) return m == 0.0 ? INFINITY : m > 0.0 ? 0.0 : NAN;
  const int hi = __double2hiint(m), k = ((hi >> 20) - 1023) >> 1;
  const double f = __hiloint2double(hi - k * (1 << 21), __double2loint(m)), r = rsqrtf((float)f);
  return r * (1.5 - 0.5 * f * r * r) * __hiloint2double((1023 - k) << 20, 0);
}
__device__ __forceinline__ double inverse_root(double m) {
  // inside fp32's range, 2^-120 .. 2^120, without the detour
  if ((uint32_t)(__double2hiint(m) - ((1023 - 120) << 20)) >= 240u << 20) return far_root(m);
  const double r = rsqrtf((float)m);
  return r * (1.5 - 0.5 * m * r * r);
}
// What fp32 can root: outside, the squares of a row leave it (or all of them are zero).
__device__ __forceinline__ bool far_from_one(float mean) { return !(mean >= 0x1p-100f && mean <= 0x1p100f); }

// Norm and rotation of the elements x that this lane holds of a head, `other` being those of the lane with the other halves of the
// pairs: y = inv (x ca + other sb), ca = gain * cos, sb = +- the other's gain * sin.  True where that has to be done in fp64.
template <typename T, int HD>
__device__ __forceinline__ bool norm_rotate(const float (&x)[kVec], const float (&other)[kVec], bool norm, float eps, const T (&ca)[kVec], const T (&sb)[kVec], bool rotates, T (&y)[kVec]) {
  T inv = 1;
  bool far = false;
  if (norm) {
    T sum = 0;
#pragma unroll
    for (int j = 0; j < kVec; ++j) sum += (T)x[j] * (T)x[j];
#pragma unroll
    for (int o = HD / kVec / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const T mean = sum * (T)(1.0 / HD);
    if constexpr (sizeof(T) == 8) {
      inv = inverse_root(mean + (T)eps);
    } else {
      inv = rsqrtf(mean + eps);
      far = far_from_one(mean);
    }
  }
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    y[j] = (T)x[j] * ca[j];
    if (rotates) y[j] += (T)other[j] * sb[j];
    y[j] *= inv;
  }
  return far;
}

// What fp64 says where fp32 leaves it open; kept out of the loops, which it would push out of the instruction cache.
static __device__ __noinline__ float step64(float low, float high) { return (float)(((double)high - (double)low) / 15.0); }
static __device__ __noinline__ uint32_t code64(float x, float m, float s) { return s == 0.f ? 0u : (uint32_t)fmin(fmax(rint(((double)x - (double)m) / (double)s), 0.0), 15.0); }

// Codes, a byte each, of this lane's elements, GL lanes being a group; returns the pair (s, m) as fp16 bits.
template <int GL>
__device__ __forceinline__ uint32_t quantise(const float (&x)[kVec], uint32_t (&word)[2]) {
  float low = x[0], high = x[0];
  bool nan = x[0] != x[0];
#pragma unroll
  for (int j = 1; j < kVec; ++j) {
    low = fminf(low, x[j]);
    high = fmaxf(high, x[j]);
    nan = nan || x[j] != x[j];
  }
  if (nan) high = INFINITY;                                // the comparisons pass a NaN over
#pragma unroll
  for (int o = 1; o < GL; o <<= 1) {
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
  }
  const bool bad = !isfinite(low) || !isfinite(high);
  constexpr float top = 64000.f;                           // with every rounding, m + 15 s stays inside fp16's range
  low = fminf(fmaxf(low, -top), top);
  high = fminf(fmaxf(high, -top), top);
  const __half m = __float2half_rn(low);
  // (high - low) / 15 in fp32 is off by at most 2^-22 of itself: where that could lead to another fp16 number, fp64 decides
  const float step = (high - low) * (1.f / 15.f);
  __half s = __float2half_rn(step);
  if (!bad && (__half_as_ushort(__float2half_rn(step * (1.f - 3e-7f))) != __half_as_ushort(__float2half_rn(step * (1.f + 3e-7f)))))
    s = __float2half_rn(step64(low, high));
  const float mf = __half2float(m), sf = __half2float(s), inv = sf > 0.f ? __fdividef(1.f, sf) : 0.f;
  constexpr float whole = 12582912.f;                      // 1.5 * 2^23: adding it rounds, and leaves a code in the lowest byte
  float r[kVec], near = 0.f;
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    const float from = x[j] - mf;
    r[j] = fmaf(from, inv, whole);
    near = fmaxf(near, fabsf(fmaf(from, inv, whole - r[j])));
    r[j] = fminf(fmaxf(r[j], whole), whole + 15.f);
  }
  // the quotient, three roundings off, is off by at most 2^-21 of 16: nearer to a border than 1e-5 fp64 decides.  (Far outside
  // 0 .. 15, where fp16 could not tell m from its neighbours, it is held to the range either way.)
  if (near > 0.5f - 1e-5f && !bad) {
#pragma unroll 1
    for (int j = 0; j < kVec; ++j) {
      float v = x[0];
#pragma unroll
      for (int i = 1; i < kVec; ++i) v = i == j ? x[i] : v;
      const float c = whole + (float)code64(v, mf, sf);
#pragma unroll
      for (int i = 0; i < kVec; ++i) r[i] = i == j ? c : r[i];
    }
  }
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const uint32_t lo = __byte_perm(__float_as_uint(r[4 * q]), __float_as_uint(r[4 * q + 1]), 0x0040), hi = __byte_perm(__float_as_uint(r[4 * q + 2]), __float_as_uint(r[4 * q + 3]), 0x0040);
    word[q] = bad ? 0u : __byte_perm(lo, hi, 0x5410);
  }
  return bad ? 0x7E007E00u : (uint32_t)__half_as_ushort(s) | (uint32_t)__half_as_ushort(m) << 16;     // NaN, NaN
}

// Places of the element e0 = 8 i in a K or V row whose planes lie one behind the other: K has the bytes of its neighbours in two
// words a quarter of a plane's row apart, V has them in the same byte of eight units (`place` of the first four, of the others).
template <int HD>
__host__ __device__ __forceinline__ constexpr uint32_t k_place(uint32_t e0) {
  constexpr uint32_t PL = HD < 128 ? HD : 128, ROW = PL / 2;
  return e0 / PL * ROW + e0 % 16 / 4 * (ROW / 4) + e0 % PL / 32 * 4;
}
template <int HD>
__host__ __device__ __forceinline__ constexpr uint32_t v_place(uint32_t slot, uint32_t e0, uint32_t q) {
  constexpr uint32_t PL = HD < 128 ? HD : 128, ROW = PL / 2;
  return e0 / PL * ROW + (4 * q ^ (PL == 128 ? 4 * (slot >> 1 & 1) : 0)) * (ROW / 8) + e0 % PL / 16;
}

// These are the layout's own places (kv4.h), for every element.
template <int HD>
constexpr bool places_agree() {
  constexpr int PL = HD < 128 ? HD : 128, ROW = PL / 2;
  const Kv4Dims d{HD, 64};
  for (int slot = 0; slot < 4; ++slot)
    for (int e = 0; e < HD; ++e) {
      const int behind = ((e / PL) * kKv4Page + slot) * ROW - e / PL * ROW, e0 = e & ~7, j = e & 7;      // planes one behind the other
      if (d.k_byte(slot, e) - behind != (int)k_place<HD>(e0 & ~16) + j / 4 * (ROW / 4) + j % 4 || d.k_high(e) != ((e0 & 16) != 0)) return false;
      if (d.v_byte(slot, e) - behind != (int)v_place<HD>(slot, e0, j / 4) + j % 4 * (ROW / 8) || d.v_high(e) != ((e0 & 8) != 0)) return false;
    }
  return true;
}
static_assert(places_agree<64>() && places_agree<128>() && places_agree<256>(), "the layout of the cache");

// Writes the codes of the warp's rows, those of lane / (HD / 8) = `sub`; `stage` is the warp's own.  Of K a lane has the bytes of whole
// words (elements 16 apart share a byte, four neighbours a word).  Of V, neighbours lie in different units: the rows are put
// together in shared memory first.
template <int HD>
__device__ __forceinline__ void put_codes(uint8_t* codes, uint32_t slot, bool is_v, bool active, uint32_t lane, uint32_t (&word)[2], uint8_t* stage) {
  constexpr uint32_t PL = HD < 128 ? HD : 128, ROW = PL / 2, LH = HD / kVec;
  const uint32_t e0 = lane % LH * kVec, apart = is_v ? 1 : 2;
#pragma unroll
  for (int q = 0; q < 2; ++q) word[q] |= __shfl_down_sync(0xffffffffu, word[q], apart) << 4;
  if (!is_v) {
    if ((e0 & 16) || !active) return;
    uint8_t* at = codes + slot * ROW + e0 / PL * (kKv4Page - 1) * ROW + k_place<HD>(e0);
    *reinterpret_cast<uint32_t*>(at) = word[0];
    *reinterpret_cast<uint32_t*>(at + ROW / 4) = word[1];
    return;
  }
  __syncwarp();                                                      // the rows before have been taken away
  if (!(e0 & 8)) {
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int j = 0; j < 4; ++j) stage[lane / LH * (HD / 2) + v_place<HD>(slot, e0, q) + j * (ROW / 8)] = (uint8_t)(word[q] >> (8 * j));
  }
  __syncwarp();
  const uint32_t at = lane % LH * 4;                                 // a row has HD / 2 = 4 LH bytes
  if (active) *reinterpret_cast<uint32_t*>(codes + (at / ROW * kKv4Page + slot) * ROW + at % ROW) = *reinterpret_cast<const uint32_t*>(stage + lane * 4);
}

// Physical page of (sequence, position), or null (and the status set) where there is none.
__device__ __forceinline__ uint8_t* kv4_page(const Kv4Args& kv, int seq, int pos, int* status) {
  if (seq < 0 || seq >= kv.batch || pos / kKv4Page >= kv.table_stride) { set_status(status, kDevBadPosition); return nullptr; }
  const int page = kv.table[seq * kv.table_stride + pos / kKv4Page];
  if (page < 0 || page >= kv.num_pages) { set_status(status, kDevBadPosition); return nullptr; }
  return kv.pages + (long long)page * kv.hkv * kv.d.head_bytes();
}

template <bool VEC>
__device__ __forceinline__ void table_row(const float* p, long long i, float (&x)[kVec]) {
  RawRow<kF32, kVec> r;
  r.load(p, i, VEC);
  r.get(x);
}

// What a warp has to do: NP passes of 256 / HD heads of one kind and token.
template <int HD, int NP, bool APPEND>
struct RowJob {
  static constexpr int LH = HD / kVec, HP = 32 / LH, NH = NP * HP;     // lanes of a head, heads of a pass, of a warp
  int tok, heads, passes, mine;                                        // mine: this lane's first head; those behind the last compute the last one's and write nothing
  bool is_q, is_v;
  long long row;                                                       // of qkv, at this lane's elements of head 0
  __device__ __forceinline__ explicit RowJob(const RowArgs& a) {
    const int lane = threadIdx.x & 31;
    // a token's jobs: query heads, key heads, value heads
    const int jq = (a.hq + NH - 1) / NH, jk = (a.hkv + NH - 1) / NH;
    const uint32_t per = jq + (APPEND ? 2 : 1) * jk, job = blockIdx.x * 4 + (threadIdx.x >> 5);
    tok = (int)(job / per);
    const int part = (int)(job - tok * per);
    is_q = part < jq;
    is_v = APPEND && part >= jq + jk;
    heads = is_q ? a.hq : a.hkv;
    const int h0 = (is_q ? part : is_v ? part - jq - jk : part - jq) * NH;
    passes = min(NP, (heads - h0 + HP - 1) / HP);
    mine = h0 + lane / LH;
    row = tok * a.stride + (is_q ? 0 : is_v ? a.hq + a.hkv : a.hq) * HD + lane % LH * kVec;
  }
};

// The heads of a warp whose squares leave fp32 (a bit for each pass, by lane), once more in fp64 from memory, where they are as they were.
// It finds out by itself what the warp's job is, so that nothing of that stays in registers for it (the loops of the others lost a fifth
// to that: 24.7 us -> 29.0 for 8191 rows).
template <int HD, int TYPE, int NP, bool APPEND, bool VEC>
static __device__ __noinline__ void far_heads(const RowArgs* args, uint32_t far) {
  using Job = RowJob<HD, NP, APPEND>;
  const RowArgs& a = *args;
  const Job w(a);
  const int lane = threadIdx.x & 31, e0 = lane % Job::LH * kVec, half = a.rot / 2;
  const bool rotates = e0 < a.rot, first = e0 < half;
  const int other_lane = lane + (rotates ? (first ? half / kVec : -(half / kVec)) : 0);
  const float* gain = (w.is_q ? a.q_gain : a.k_gain) + e0;
  const long long turn = (long long)a.pos[w.tok] * half + e0 - (first ? 0 : half);
  void* out = w.is_q ? a.q_out : a.k_out;
  const long long at = w.tok * (w.is_q ? a.q_stride : a.k_stride) + e0;
#pragma unroll 1
  for (int i = 0; i < w.passes; ++i) {
    if (!__any_sync(0xffffffffu, far >> i & 1)) continue;
    const int head = w.mine + i * Job::HP;
    RawRow<TYPE, kVec> raw;
    raw.load(a.qkv, w.row + min(head, w.heads - 1) * HD, VEC);
    float x[kVec];
    raw.get(x);
    double sum = 0;
#pragma unroll
    for (int j = 0; j < kVec; ++j) sum += (double)x[j] * x[j];
#pragma unroll
    for (int o = Job::LH / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const double inv = inverse_root(sum * (1.0 / HD) + (double)a.eps);
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const double v = (double)x[j] * gain[j], other = __shfl_sync(0xffffffffu, v, other_lane);
      x[j] = (float)((rotates ? v * a.cos[turn + j] + (first ? -other : other) * a.sin[turn + j] : v) * inv);
    }
    raw.put(x);
    if ((far >> i & 1) && head < w.heads) raw.store(out, at + head * HD, VEC);
  }
}

// GROUP 0: keys are written out, else keys and values go into the cache.
// VEC: all rows and tables start on 16-byte boundaries.
template <int HD, int TYPE, int GROUP, int NP, bool VEC>
__global__ void __launch_bounds__(128, GROUP ? 6 : 1) qk_norm_rope_kernel(const __grid_constant__ RowArgs a) {
  constexpr int LH = HD / kVec, HP = 32 / LH;                           // lanes of a head, heads of a pass
  constexpr bool APPEND = GROUP > 0;
  __shared__ __align__(16) uint8_t stage[4][APPEND ? 128 : 16];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, e0 = lane % LH * kVec;
  const RowJob<HD, NP, APPEND> job(a);
  const int tok = job.tok, heads = job.heads, passes = job.passes, mine = job.mine;
  const bool is_q = job.is_q, is_v = job.is_v;
  if (tok >= a.tokens) return;
  RawRow<TYPE, kVec> raw[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i)
    if (i < passes) raw[i].load(a.qkv, job.row + min(mine + i * HP, heads - 1) * HD, VEC);
  const int pos = a.pos[tok];
  if (pos < 0) return;
  if (a.rot > 0 && pos >= a.rope_rows) { set_status(a.status, kDevBadPosition); return; }
  uint8_t* page = nullptr;
  if constexpr (APPEND) {
    page = kv4_page(a.kv, a.seq ? a.seq[tok] : tok, pos, a.status);
    if (!page) return;
  }
  const int half = a.rot / 2, slot = pos % kKv4Page;
  const bool rotates = e0 < a.rot && !is_v, first = e0 < half;
  const int other_lane = lane + (rotates ? (first ? half / kVec : -(half / kVec)) : 0);
  const bool norm = (is_q ? a.q_gain : a.k_gain) != nullptr && !is_v;
  float ca[kVec], sb[kVec], gain[kVec];
#pragma unroll
  for (int j = 0; j < kVec; ++j) ca[j] = gain[j] = 1.f, sb[j] = 0.f;
  if (norm) table_row<VEC>(is_q ? a.q_gain : a.k_gain, e0, gain);
  if (rotates) {
    const long long i = (long long)pos * half + e0 - (first ? 0 : half);
    table_row<VEC>(a.cos, i, ca);
    table_row<VEC>(a.sin, i, sb);
  }
  auto next = [&]() {                                                // an appending kernel's loops stand once: unrolled, they miss the instruction cache
#pragma unroll
    for (int i = 0; i + 1 < NP; ++i) raw[i] = raw[i + 1];
  };
  auto normed = [&](auto one, auto&& done) {                          // one: a number of the type that norm and rotation are computed in
    using T = decltype(one);
    constexpr int kUnroll = APPEND ? 1 : NP;
    T c[kVec], s[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const float other_gain = __shfl_sync(0xffffffffu, gain[j], other_lane);
      c[j] = (T)ca[j] * (T)gain[j];
      s[j] = (T)(first ? -sb[j] : sb[j]) * (T)other_gain;
    }
#pragma unroll kUnroll
    for (int i = 0; i < NP; ++i) {
      if (i >= passes) break;
      RawRow<TYPE, kVec> fellow;
#pragma unroll
      for (int j = 0; j < RawRow<TYPE, kVec>::N; ++j) fellow.u[j] = __shfl_sync(0xffffffffu, raw[0].u[j], other_lane);
      float x[kVec], f[kVec];
      raw[0].get(x);
      fellow.get(f);
      T y[kVec];
      const bool far = norm_rotate<T, HD>(x, f, norm, a.eps, c, s, rotates, y);
#pragma unroll
      for (int j = 0; j < kVec; ++j) x[j] = (float)y[j];
      done(i, x, far);
      next();
    }
  };
  if (is_q || !APPEND) {
    void* out = is_q ? a.q_out : a.k_out;
    const long long at = tok * (is_q ? a.q_stride : a.k_stride) + e0;
    uint32_t left = 0;
    normed(1.f, [&](int i, const float (&x)[kVec], bool far) {
      RawRow<TYPE, kVec> y;
      y.put(x);
      if (mine + i * HP < heads && !far) y.store(out, at + (mine + i * HP) * HD, VEC);
      left |= (uint32_t)far << i;
    });
    if (__any_sync(0xffffffffu, left != 0)) far_heads<HD, TYPE, NP, APPEND, VEC>(&a, left);
  }
  if constexpr (APPEND) {
    constexpr Kv4Dims d{HD, GROUP};
    constexpr int GL = GROUP / kVec;
    auto put = [&](int i, const float (&x)[kVec], bool) {
      const int h = mine + i * HP;
      uint8_t* head = page + (long long)h * d.head_bytes();
      uint32_t word[2];
      const uint32_t pair = quantise<GL>(x, word);
      put_codes<HD>(head + (is_v ? d.v_codes() : d.k_codes()), slot, is_v, h < heads, lane, word, stage[threadIdx.x >> 5]);
      if (lane % GL == 0 && h < heads) reinterpret_cast<uint32_t*>(head + (is_v ? d.v_scales() : d.k_scales()))[slot * d.groups() + lane % LH / GL] = pair;
    };
    if (is_v) {
#pragma unroll 1
      for (int i = 0; i < passes; ++i) {
        float x[kVec];
        raw[0].get(x);
        put(i, x, false);
        next();
      }
    } else if (!is_q) {
      normed(1.0, put);
    }
  }
}

// 256 / HD kv heads of a token a warp, K and V of each.
template <int HD, int TYPE, int GROUP, bool VEC>
__global__ void __launch_bounds__(128) kv4_read_kernel(const Kv4Args kv, const int* seq, const int* pos, int tokens, void* k_out, void* v_out, int* status) {
  constexpr uint32_t PL = HD < 128 ? HD : 128, ROW = PL / 2;
  constexpr int LH = HD / kVec, HP = 32 / LH;
  constexpr Kv4Dims d{HD, GROUP};
  __shared__ __align__(16) uint8_t stage[4][128];
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t lane = threadIdx.x & 31, e0 = lane % LH * kVec, per = (kv.hkv + HP - 1) / HP, job = blockIdx.x * 4 + (threadIdx.x >> 5);
  const int tok = (int)(job / per), h = (int)(job - tok * per) * HP + lane / LH;
  if (tok >= tokens) return;
  const int p = pos[tok];
  if (p < 0) return;
  const uint8_t* page = kv4_page(kv, seq ? seq[tok] : tok, p, status);
  if (!page) return;
  const uint32_t slot = p % kKv4Page, at = lane % LH * 4;
  const uint8_t* head = page + (long long)min(h, kv.hkv - 1) * d.head_bytes();
  const uint8_t* k = head + d.k_codes() + slot * ROW + e0 / PL * (kKv4Page - 1) * ROW + k_place<HD>(e0 & ~16u);
  uint32_t kw[2] = {*reinterpret_cast<const uint32_t*>(k), *reinterpret_cast<const uint32_t*>(k + ROW / 4)};
  uint8_t* row = stage[threadIdx.x >> 5] + lane / LH * (HD / 2);
  *reinterpret_cast<uint32_t*>(row + at) = *reinterpret_cast<const uint32_t*>(head + d.v_codes() + (at / ROW * kKv4Page + slot) * ROW + at % ROW);
  const uint32_t ks = reinterpret_cast<const uint32_t*>(head + d.k_scales())[slot * d.groups() + e0 / GROUP];
  const uint32_t vs = reinterpret_cast<const uint32_t*>(head + d.v_scales())[slot * d.groups() + e0 / GROUP];
  __syncwarp();
  if (h >= kv.hkv) return;
  auto write = [&](void* out, uint32_t pair, const uint32_t (&word)[2], uint32_t shift) {
    const float2 sm = __half22float2(*reinterpret_cast<const __half2*>(&pair));
    float x[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) x[j] = fmaf(sm.x, (float)(word[j / 4] >> (8 * (j % 4) + shift) & 15u), sm.y);
    RawRow<TYPE, kVec> y;
    y.put(x);
    y.store(out, ((long long)tok * kv.hkv + h) * HD + e0, VEC);
  };
  if (k_out) write(k_out, ks, kw, e0 & 16 ? 4 : 0);
  if (v_out) {                                             // neighbours lie in different units: a byte of each
    uint32_t word[2] = {};
#pragma unroll
    for (int j = 0; j < kVec; ++j) word[j / 4] |= (uint32_t)row[v_place<HD>(slot, e0, j / 4) + j % 4 * (ROW / 8)] << (8 * (j % 4));
    write(v_out, vs, word, e0 & 8 ? 4 : 0);
  }
}

}  // namespace b200lm
