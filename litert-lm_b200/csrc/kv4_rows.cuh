// Rows of a fused QKV projection: RMSNorm of each query and key head with the rotation in the same pass, keys written out or,
// with the values, put into the cache in 4 bits; and the way back from there.
//
//   y = x / sqrt(mean x^2 + eps) * gain;   (y_i, y_{i + r/2}) -> (y_i c_i - y_{i + r/2} s_i, y_{i + r/2} c_i + y_i s_i)
//   m = fp16(low), s = fp16((high - low) / 15), code = rint((x - m) / s) held to 0 .. 15
//
// Every byte is read and written once: what bounds it is HBM for many tokens, one chain of latencies (row, two warp sums,
// table row) for a few.  A warp takes up to four heads of one kind and token, asks for their rows at once and keeps gain and
// rotation multiplied in registers; a lane holds hd / 32 neighbouring elements, so that the other half of a pair lies at the
// same place of a lane rot / hd * 16 further and comes from there as it lay in memory.
// Queries are computed in fp32.  Keys that go into the cache are computed in fp64 and rounded to fp32 before their
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
  bool vec, vec_q, vec_k;      // rows of qkv, q_out, k_out start on 16-byte boundaries
  int* status;
};

__device__ __forceinline__ void set_status(int* status, int code) {
  if (status) atomicMax(status, code);
}

// V neighbouring elements of a row as they lie in memory: whole words where the row starts allow it (`vec`), else one by one.
template <int TYPE, int V>
struct RawRow {
  static constexpr int N = TYPE == kF32 ? V : V / 2;
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
  __device__ __forceinline__ void get(float (&x)[V]) const {
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
  __device__ __forceinline__ void put(const float (&x)[V]) {
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
template <int V>
__device__ __forceinline__ void row_load(const void* p, long long i, int type, float (&x)[V]) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p) + i * elem_size(type);
  auto as = [&](auto raw) {
    constexpr int bytes = 4 * decltype(raw)::N;
    raw.load(p, i, at % (bytes < 16 ? bytes : 16) == 0);
    raw.get(x);
  };
  if (type == kF32) as(RawRow<kF32, V>());
  else if (type == kBf16) as(RawRow<kBf16, V>());
  else as(RawRow<kF16, V>());
}

// Norm and rotation of the V elements x that this lane holds of a head, `other` being those of the lane with the other halves of the
// pairs: y = inv (x ca + other sb), ca = gain * cos, sb = +- the other's gain * sin.
template <typename T, int V>
__device__ __forceinline__ void norm_rotate(const float (&x)[V], const float (&other)[V], bool norm, float eps, const T (&ca)[V], const T (&sb)[V], bool rotates, T (&y)[V]) {
  constexpr int HD = 32 * V;
  T inv = 1;
  if (norm) {
    T sum = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) sum += (T)x[j] * (T)x[j];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const T mean = sum * (T)(1.0 / HD) + (T)eps;
    inv = rsqrtf((float)mean);
    if constexpr (sizeof(T) == 8) inv = inv * (1.5 - 0.5 * mean * inv * inv);      // 2^-22 -> 2^-43
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    y[j] = (T)x[j] * ca[j];
    if (rotates) y[j] += (T)other[j] * sb[j];
    y[j] *= inv;
  }
}

// Codes of the group that this lane's V elements lie in (GL lanes of it); returns the pair (s, m) as fp16 bits.
template <int V, int GL>
__device__ __forceinline__ uint32_t quantise(const float (&x)[V], uint32_t (&code)[V]) {
  float low = x[0], high = x[0];
  bool nan = x[0] != x[0];
#pragma unroll
  for (int j = 1; j < V; ++j) {
    low = fminf(low, x[j]);
    high = fmaxf(high, x[j]);
    nan = nan || x[j] != x[j];
  }
  if (nan) high = INFINITY;                                // the comparisons pass a NaN over
  if constexpr (GL == 32) {                                // one instruction for the whole warp
    asm volatile("redux.sync.min.f32 %0, %0, 0xffffffff;" : "+f"(low));
    asm volatile("redux.sync.max.f32 %0, %0, 0xffffffff;" : "+f"(high));
  } else {
#pragma unroll
    for (int o = 1; o < GL; o <<= 1) {
      low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
      high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
    }
  }
  const bool bad = !isfinite(low) || !isfinite(high);
  constexpr float top = 65504.f;                           // fp16's largest
  const __half m = __float2half_rn(fminf(fmaxf(low, -top), top));
  const __half s = __float2half_rn(fminf((float)(((double)high - (double)low) / 15.0), top));
  const float mf = __half2float(m), sf = __half2float(s), inv = sf > 0.f ? 1.f / sf : 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    // three roundings leave a code below 16 off by at most 3 * 2^-24 * 16 = 3e-6: nearer to a border than that fp64 decides
    const float c = (x[j] - mf) * inv, whole = rintf(c);
    float decided = whole;
    if (fabsf(fabsf(c - whole) - 0.5f) < 1e-5f && sf > 0.f) decided = (float)rint(((double)x[j] - (double)mf) / (double)sf);
    code[j] = bad ? 0u : (uint32_t)fminf(fmaxf(decided, 0.f), 15.f);
  }
  if (bad) return 0x7E007E00u;                             // NaN, NaN
  return (uint32_t)__half_as_ushort(s) | (uint32_t)__half_as_ushort(m) << 16;
}

// Byte of element e0 + j (e0 = lane V) of a V row whose planes lie one behind the other.
template <int V>
__device__ __forceinline__ int v_place(int slot, int e0, int j) {
  constexpr int PL = V >= 4 ? 128 : 64, ROW = PL / 2;
  const int turn = PL == 128 ? 4 * (slot >> 1 & 1) : 0;
  return e0 / PL * ROW + ((e0 + j) % 8 ^ turn) * (ROW / 8) + e0 % PL / 16;
}

// Writes a row's codes; `stage` is the warp's own.  Of K a lane has the bytes of whole words (elements 16 apart share a byte, four
// neighbours a word).  Of V, neighbours lie in different units: the row is put together in shared memory first.
template <int V>
__device__ __forceinline__ void put_codes(uint8_t* codes, const Kv4Dims& d, int slot, bool is_v, int lane, const uint32_t (&code)[V], uint8_t* stage) {
  const int e0 = lane * V, apart = (is_v ? 8 : 16) / V;
  uint32_t byte[V];
#pragma unroll
  for (int j = 0; j < V; ++j) byte[j] = code[j] | __shfl_down_sync(0xffffffffu, code[j], apart) << 4;
  if (!is_v) {
    if (d.k_high(e0)) return;
    if constexpr (V == 2) {
      *reinterpret_cast<uint16_t*>(codes + d.k_byte(slot, e0)) = (uint16_t)(byte[0] | byte[1] << 8);
    } else {
#pragma unroll
      for (int j = 0; j < V; j += 4)
        *reinterpret_cast<uint32_t*>(codes + d.k_byte(slot, e0 + j)) = byte[j] | byte[j + 1] << 8 | byte[j + 2] << 16 | byte[j + 3] << 24;
    }
    return;
  }
  constexpr int ROW = V >= 4 ? 64 : 32, HALF = 16 * V;               // bytes of a plane's row, of all planes'
  __syncwarp();                                                      // the row before has been taken away
  if (!d.v_high(e0)) {
#pragma unroll
    for (int j = 0; j < V; ++j) stage[v_place<V>(slot, e0, j)] = (uint8_t)byte[j];
  }
  __syncwarp();
  if (lane * 4 < HALF) *reinterpret_cast<uint32_t*>(codes + (lane * 4 / ROW * kKv4Page + slot) * ROW + lane * 4 % ROW) = *reinterpret_cast<const uint32_t*>(stage + lane * 4);
}

// Physical page of (sequence, position), or null (and the status set) where there is none.
__device__ __forceinline__ uint8_t* kv4_page(const Kv4Args& kv, int seq, int pos, int* status) {
  if (seq < 0 || seq >= kv.batch || pos / kKv4Page >= kv.table_stride) { set_status(status, kDevBadPosition); return nullptr; }
  const int page = kv.table[seq * kv.table_stride + pos / kKv4Page];
  if (page < 0 || page >= kv.num_pages) { set_status(status, kDevBadPosition); return nullptr; }
  return kv.pages + (long long)page * kv.hkv * kv.d.head_bytes();
}

// NH heads of one kind and token a warp; GROUP 0: keys are written out, else keys and values go into the cache.
template <int HD, int TYPE, int GROUP, int NH>
__global__ void __launch_bounds__(128) qk_norm_rope_kernel(const RowArgs a) {
  constexpr int V = HD / 32;
  constexpr bool APPEND = GROUP > 0;
  __shared__ __align__(16) uint8_t stage[4][APPEND ? HD / 2 : 16];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  // a token's jobs: query heads, key heads, value heads
  const int jq = (a.hq + NH - 1) / NH, jk = (a.hkv + NH - 1) / NH;
  const uint32_t per = jq + (APPEND ? 2 : 1) * jk, job = blockIdx.x * 4 + (threadIdx.x >> 5);
  const int tok = (int)(job / per), part = (int)(job - tok * per);
  if (tok >= a.tokens) return;
  const bool is_q = part < jq, is_v = APPEND && part >= jq + jk;
  const int h0 = (is_q ? part : is_v ? part - jq - jk : part - jq) * NH, hn = min(NH, (is_q ? a.hq : a.hkv) - h0), e0 = lane * V;
  const long long row = tok * a.stride + ((is_q ? 0 : is_v ? a.hq + a.hkv : a.hq) + h0) * HD + e0;
  RawRow<TYPE, V> raw[NH];
#pragma unroll
  for (int i = 0; i < NH; ++i)
    if (i < hn) raw[i].load(a.qkv, row + i * HD, a.vec);
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
  const int other_lane = lane + (rotates ? (first ? half / V : -(half / V)) : 0);
  const bool norm = (is_q ? a.q_gain : a.k_gain) != nullptr && !is_v;
  float ca[V], sb[V], gain[V];
#pragma unroll
  for (int j = 0; j < V; ++j) ca[j] = gain[j] = 1.f, sb[j] = 0.f;
  if (norm) row_load<V>(is_q ? a.q_gain : a.k_gain, e0, kF32, gain);
  if (rotates) {
    const long long i = (long long)pos * half + e0 - (first ? 0 : half);
    row_load<V>(a.cos, i, kF32, ca);
    row_load<V>(a.sin, i, kF32, sb);
  }
  auto heads = [&](auto one, auto&& done) {                          // one: a number of the type that norm and rotation are computed in
    using T = decltype(one);
    T c[V], s[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float other_gain = __shfl_sync(0xffffffffu, gain[j], other_lane);
      c[j] = (T)ca[j] * (T)gain[j];
      s[j] = (T)(first ? -sb[j] : sb[j]) * (T)other_gain;
    }
#pragma unroll
    for (int i = 0; i < NH; ++i) {
      if (i >= hn) break;
      RawRow<TYPE, V> fellow;
#pragma unroll
      for (int j = 0; j < RawRow<TYPE, V>::N; ++j) fellow.u[j] = __shfl_sync(0xffffffffu, raw[i].u[j], other_lane);
      float x[V], f[V];
      raw[i].get(x);
      fellow.get(f);
      T y[V];
      norm_rotate<T, V>(x, f, norm, a.eps, c, s, rotates, y);
#pragma unroll
      for (int j = 0; j < V; ++j) x[j] = (float)y[j];
      done(i, x);
    }
  };
  if (is_q || !APPEND) {
    void* out = is_q ? a.q_out : a.k_out;
    const long long at = tok * (is_q ? a.q_stride : a.k_stride) + h0 * HD + e0;
    const bool vec = is_q ? a.vec_q : a.vec_k;
    heads(1.f, [&](int i, const float (&x)[V]) {
      RawRow<TYPE, V> y;
      y.put(x);
      y.store(out, at + i * HD, vec);
    });
  }
  if constexpr (APPEND) {
    constexpr Kv4Dims d{HD, GROUP};
    constexpr int gl = GROUP / V;
    auto put = [&](int i, const float (&x)[V]) {
      uint8_t* head = page + (long long)(h0 + i) * d.head_bytes();
      uint32_t code[V];
      const uint32_t pair = quantise<V, gl>(x, code);
      put_codes<V>(head + (is_v ? d.v_codes() : d.k_codes()), d, slot, is_v, lane, code, stage[threadIdx.x >> 5]);
      if (lane % gl == 0) reinterpret_cast<uint32_t*>(head + (is_v ? d.v_scales() : d.k_scales()))[slot * d.groups() + lane / gl] = pair;
    };
    if (is_v) {
#pragma unroll
      for (int i = 0; i < NH; ++i) {
        if (i >= hn) break;
        float x[V];
        raw[i].get(x);
        put(i, x);
      }
    } else if (!is_q) {
      heads(1.0, put);
    }
  }
}

// A warp per (token, kv head, K or V); a lane reads the bytes of V elements and their fellows.
template <int HD, int TYPE, int GROUP>
__global__ void __launch_bounds__(128) kv4_read_kernel(const Kv4Args kv, const int* __restrict__ seq, const int* __restrict__ pos, int tokens, void* k_out, void* v_out, bool vec, int* status) {
  constexpr int V = HD / 32;
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, sides = (k_out != nullptr) + (v_out != nullptr);
  const uint32_t per = sides * kv.hkv, job = blockIdx.x * 4 + (threadIdx.x >> 5);
  const int tok = (int)(job / per), part = (int)(job - tok * per), h = sides == 2 ? part >> 1 : part;
  if (tok >= tokens) return;
  const bool is_v = k_out == nullptr || (sides == 2 && (part & 1));
  const int p = pos[tok];
  if (p < 0) return;
  const uint8_t* page = kv4_page(kv, seq ? seq[tok] : tok, p, status);
  if (!page) return;
  constexpr Kv4Dims d{HD, GROUP};
  const uint8_t* head = page + (long long)h * d.head_bytes();
  const uint8_t* codes = head + (is_v ? d.v_codes() : d.k_codes());
  const int slot = p % kKv4Page, e0 = lane * V;
  const uint32_t pair = reinterpret_cast<const uint32_t*>(head + (is_v ? d.v_scales() : d.k_scales()))[slot * d.groups() + e0 / d.group];
  const float2 sm = __half22float2(*reinterpret_cast<const __half2*>(&pair));
  // the row's bytes come in words; V's neighbours lie in different units and are picked from shared memory
  constexpr int ROW = V >= 4 ? 64 : 32;
  __shared__ __align__(16) uint8_t stage[4][HD / 2];
  uint8_t* row = stage[threadIdx.x >> 5];
  if (lane * 8 < HD) reinterpret_cast<uint32_t*>(row)[lane] = *reinterpret_cast<const uint32_t*>(codes + (lane * 4 / ROW * kKv4Page + slot) * ROW + lane * 4 % ROW);
  __syncwarp();
  float x[V];
  const int k_at = e0 / (2 * ROW) * ROW + e0 % 16 / 4 * (ROW / 4) + e0 % (2 * ROW) / 32 * 4 + e0 % 4;     // and 4 neighbours, the next 4 a quarter row on
  const bool high = is_v ? d.v_high(e0) : d.k_high(e0);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const uint32_t byte = row[is_v ? v_place<V>(slot, e0, j) : k_at + j / 4 * (ROW / 4) + j % 4];
    x[j] = fmaf(sm.x, (float)(high ? byte >> 4 : byte & 15), sm.y);
  }
  RawRow<TYPE, V> y;
  y.put(x);
  y.store(is_v ? v_out : k_out, ((long long)tok * kv.hkv + h) * HD + e0, vec);
}

}  // namespace b200lm
