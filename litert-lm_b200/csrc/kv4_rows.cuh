// Rows of a fused QKV projection: RMSNorm of each query and key head with the rotation in the same pass, keys written out or,
// with the values, put into the cache in 4 bits; and the way back from there.
//
//   y = x / sqrt(mean x^2 + eps) * gain;   (y_i, y_{i + r/2}) -> (y_i c_i - y_{i + r/2} s_i, y_{i + r/2} c_i + y_i s_i)
//   m = fp16(low), s = fp16((high - low) / 15), code = rint((x - m) / s) held to 0 .. 15
//
// Every byte is read and written once: what bounds it is HBM for many tokens, one chain of latencies (row, two warp sums,
// table row) for a few.  A warp takes some heads of one token and keeps the token's rotation in registers; a lane holds hd / 32
// neighbouring elements, so that the other half of a pair lies at the same place of a lane rot / hd * 16 further.
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
  int heads_per_warp;
  int* status;
};

__device__ __forceinline__ void set_status(int* status, int code) {
  if (status) atomicMax(status, code);
}

// V neighbouring elements of a row; one load where the address allows it.
template <int V>
__device__ __forceinline__ void row_load(const void* p, long long i, int type, float (&x)[V]) {
  const char* a = reinterpret_cast<const char*>(p) + i * elem_size(type);
  if (type == kF32) {
    if constexpr (V >= 4) {
      if ((reinterpret_cast<uintptr_t>(a) & 15) == 0) {
#pragma unroll
        for (int j = 0; j < V; j += 4) {
          const float4 v = reinterpret_cast<const float4*>(a)[j / 4];
          x[j] = v.x; x[j + 1] = v.y; x[j + 2] = v.z; x[j + 3] = v.w;
        }
        return;
      }
    }
  } else if ((reinterpret_cast<uintptr_t>(a) & (2 * V - 1)) == 0) {
    uint32_t u[V / 2];
    if constexpr (V == 8) {
      const uint4 v = *reinterpret_cast<const uint4*>(a);
      u[0] = v.x; u[1] = v.y; u[2] = v.z; u[3] = v.w;
    } else if constexpr (V == 4) {
      const uint2 v = *reinterpret_cast<const uint2*>(a);
      u[0] = v.x; u[1] = v.y;
    } else {
      u[0] = *reinterpret_cast<const uint32_t*>(a);
    }
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      const float2 f = gg_pair(u[j], type == kBf16);
      x[2 * j] = f.x;
      x[2 * j + 1] = f.y;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) x[j] = gg_load1(p, i + j, type);
}
template <int V>
__device__ __forceinline__ void row_store(void* p, long long i, int type, const float (&x)[V]) {
  char* a = reinterpret_cast<char*>(p) + i * elem_size(type);
  if (type == kF32) {
    if constexpr (V >= 4) {
      if ((reinterpret_cast<uintptr_t>(a) & 15) == 0) {
#pragma unroll
        for (int j = 0; j < V; j += 4) reinterpret_cast<float4*>(a)[j / 4] = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
        return;
      }
    }
  } else if ((reinterpret_cast<uintptr_t>(a) & (2 * V - 1)) == 0) {
    uint32_t u[V / 2];
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      if (type == kBf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
        u[j] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
        u[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    if constexpr (V == 8) *reinterpret_cast<uint4*>(a) = make_uint4(u[0], u[1], u[2], u[3]);
    else if constexpr (V == 4) *reinterpret_cast<uint2*>(a) = make_uint2(u[0], u[1]);
    else *reinterpret_cast<uint32_t*>(a) = u[0];
    return;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) gg_store1(p, i + j, type, x[j]);
}

// Norm and rotation of the V elements that this lane holds of a head, in T.  `sn` is negative in the lanes of the first half of
// the pairs, so that the same line serves both; `off` is 0 in lanes that do not rotate.
template <typename T, int V>
__device__ __forceinline__ void norm_rotate(const float (&x)[V], bool norm, const float (&gain)[V], float eps, const float (&c)[V], const float (&sn)[V],
                                            int off, int lane, bool rotates, bool any, T (&y)[V]) {
  constexpr int HD = 32 * V;
#pragma unroll
  for (int j = 0; j < V; ++j) y[j] = (T)x[j];
  if (norm) {
    T sum = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) sum += y[j] * y[j];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    T inv;
    if constexpr (sizeof(T) == 8) inv = 1.0 / sqrt(sum / HD + (double)eps);
    else inv = 1.f / sqrtf(sum / HD + eps);
#pragma unroll
    for (int j = 0; j < V; ++j) y[j] = y[j] * inv * (T)gain[j];
  }
  if (any) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const T other = __shfl_sync(0xffffffffu, y[j], lane + off);
      if (rotates) y[j] = y[j] * (T)c[j] + other * (T)sn[j];
    }
  }
}

// Codes of the group that this lane's V elements lie in (GL lanes of it); returns the pair (s, m) as fp16 bits.
template <int V>
__device__ __forceinline__ uint32_t quantise(const float (&x)[V], int gl, uint32_t (&code)[V]) {
  float low = x[0], high = x[0];
  bool odd = !isfinite(x[0]);
#pragma unroll
  for (int j = 1; j < V; ++j) {
    low = fminf(low, x[j]);
    high = fmaxf(high, x[j]);
    odd = odd || !isfinite(x[j]);
  }
  uint32_t bad = odd;
  for (int o = 1; o < gl; o <<= 1) {
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
    bad |= __shfl_xor_sync(0xffffffffu, bad, o);
  }
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
  constexpr int ROW = V >= 4 ? 64 : 32, PLANES = V == 8 ? 2 : 1;     // bytes of a plane's row
  const int plane = e0 / (2 * ROW);
  __syncwarp();                                                      // the row before has been taken away
  if (!d.v_high(e0)) {
#pragma unroll
    for (int j = 0; j < V; ++j) stage[plane * ROW + d.v_byte(slot, e0 + j) - (plane * kKv4Page + slot) * ROW] = (uint8_t)byte[j];
  }
  __syncwarp();
  if (lane * 4 < PLANES * ROW) {
    const int p = lane * 4 / ROW, at = lane * 4 % ROW;
    *reinterpret_cast<uint32_t*>(codes + (p * kKv4Page + slot) * ROW + at) = *reinterpret_cast<const uint32_t*>(stage + lane * 4);
  }
}

// Physical page of (sequence, position), or null (and the status set) where there is none.
__device__ __forceinline__ uint8_t* kv4_page(const Kv4Args& kv, int seq, int pos, int* status) {
  if (seq < 0 || seq >= kv.batch || pos / kKv4Page >= kv.table_stride) { set_status(status, kDevBadPosition); return nullptr; }
  const int page = kv.table[seq * kv.table_stride + pos / kKv4Page];
  if (page < 0 || page >= kv.num_pages) { set_status(status, kDevBadPosition); return nullptr; }
  return kv.pages + (long long)page * kv.hkv * kv.d.head_bytes();
}

template <int HD, bool APPEND>
__global__ void __launch_bounds__(128) qk_norm_rope_kernel(const RowArgs a) {
  constexpr int V = HD / 32;
  __shared__ __align__(16) uint8_t stage[4][APPEND ? HD / 2 : 16];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int heads = a.hq + (APPEND ? 2 : 1) * a.hkv, per = (heads + a.heads_per_warp - 1) / a.heads_per_warp;
  const long long job = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int tok = (int)(job / per), h0 = (int)(job % per) * a.heads_per_warp, h1 = min(h0 + a.heads_per_warp, heads);
  if (tok >= a.tokens) return;
  const int pos = a.pos[tok];
  if (pos < 0) return;
  const int half = a.rot / 2, e0 = lane * V;
  if (a.rot > 0 && pos >= a.rope_rows) { set_status(a.status, kDevBadPosition); return; }
  uint8_t* page = nullptr;
  if constexpr (APPEND) {
    page = kv4_page(a.kv, a.seq ? a.seq[tok] : tok, pos, a.status);
    if (!page) return;
  }
  const bool rotates = e0 < a.rot, first = e0 < half;
  const int off = rotates ? (first ? half / V : -(half / V)) : 0;
  float c[V], sn[V], qg[V], kg[V], ahead[V];
  row_load<V>(a.qkv, tok * a.stride + (long long)h0 * HD + e0, a.type, ahead);
  if (rotates) {
    const long long i = (long long)pos * half + e0 - (first ? 0 : half);
    row_load<V>(a.cos, i, kF32, c);
    row_load<V>(a.sin, i, kF32, sn);
#pragma unroll
    for (int j = 0; j < V; ++j) sn[j] = first ? -sn[j] : sn[j];
  }
  if (a.q_gain) row_load<V>(a.q_gain, e0, kF32, qg);
  if (a.k_gain) row_load<V>(a.k_gain, e0, kF32, kg);
#pragma unroll 1
  for (int h = h0; h < h1; ++h) {
    float x[V];
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = ahead[j];
    if (h + 1 < h1) row_load<V>(a.qkv, tok * a.stride + (long long)(h + 1) * HD + e0, a.type, ahead);
    if (h < a.hq || !APPEND) {
      float y[V];
      if (h < a.hq) norm_rotate<float, V>(x, a.q_gain != nullptr, qg, a.eps, c, sn, off, lane, rotates, a.rot > 0, y);
      else norm_rotate<float, V>(x, a.k_gain != nullptr, kg, a.eps, c, sn, off, lane, rotates, a.rot > 0, y);
      if (h < a.hq) row_store<V>(a.q_out, tok * a.q_stride + (long long)h * HD + e0, a.type, y);
      else row_store<V>(a.k_out, tok * a.k_stride + (long long)(h - a.hq) * HD + e0, a.type, y);
      continue;
    }
    const bool is_v = h >= a.hq + a.hkv;
    if (!is_v) {
      double y[V];
      norm_rotate<double, V>(x, a.k_gain != nullptr, kg, a.eps, c, sn, off, lane, rotates, a.rot > 0, y);
#pragma unroll
      for (int j = 0; j < V; ++j) x[j] = (float)y[j];
    }
    const Kv4Dims d{HD, a.kv.d.group};
    uint8_t* head = page + (long long)(h - a.hq - (is_v ? a.hkv : 0)) * d.head_bytes();
    const int slot = pos % kKv4Page, gl = d.group / V;
    uint32_t code[V];
    const uint32_t pair = quantise<V>(x, gl, code);
    put_codes<V>(head + (is_v ? d.v_codes() : d.k_codes()), d, slot, is_v, lane, code, stage[threadIdx.x >> 5]);
    if (lane % gl == 0)
      reinterpret_cast<uint32_t*>(head + (is_v ? d.v_scales() : d.k_scales()))[slot * d.groups() + lane / gl] = pair;
  }
}

// A warp per (token, kv head, K or V); a lane reads the bytes of V elements and their fellows.
template <int HD>
__global__ void __launch_bounds__(128) kv4_read_kernel(const Kv4Args kv, const int* __restrict__ seq, const int* __restrict__ pos, int tokens, int out_type, void* k_out, void* v_out, int* status) {
  constexpr int V = HD / 32;
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, sides = (k_out != nullptr) + (v_out != nullptr);
  const long long job = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int tok = (int)(job / (sides * kv.hkv)), h = (int)(job % (sides * kv.hkv)) / sides;
  if (tok >= tokens) return;
  const bool is_v = k_out == nullptr || job % sides == 1;
  const int p = pos[tok];
  if (p < 0) return;
  const uint8_t* page = kv4_page(kv, seq ? seq[tok] : tok, p, status);
  if (!page) return;
  const Kv4Dims d{HD, kv.d.group};
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
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int e = e0 + j, plane = e / (2 * ROW);
    const uint32_t byte = row[(is_v ? d.v_byte(slot, e) : d.k_byte(slot, e)) - (plane * kKv4Page + slot) * ROW + plane * ROW];
    const uint32_t c = (is_v ? d.v_high(e) : d.k_high(e)) ? byte >> 4 : byte & 15;
    x[j] = fmaf(sm.x, (float)c, sm.y);
  }
  row_store<V>(is_v ? v_out : k_out, ((long long)tok * kv.hkv + h) * HD + e0, out_type, x);
}

}  // namespace b200lm
