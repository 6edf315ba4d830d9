// Attention of ragged sequences over the cache in 4 bits.
//
// One CTA a query row (token and head): its warps take every eighth key, hold hd / 32 elements a lane, and meet at the end.
#pragma once
#include "kv4_rows.cuh"

namespace b200lm {

struct Kv4AttnArgs {
  Kv4Args kv;
  const void* q;
  int q_type;
  long long q_stride;
  const int *kv_len, *q_start;
  int tokens, max_q, max_kv, hq, window;
  float qscale;                // log2(e) * scale
  void* out;
  long long out_stride;
  int* status;
};

template <int HD>
__global__ void __launch_bounds__(256) kv4_attn_simple_kernel(const Kv4AttnArgs a) {
  constexpr int V = HD / 32;
  __shared__ float so[8][HD], sm[8], sl[8];
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, b = blockIdx.y;
  const int tok0 = a.q_start ? a.q_start[b] : b, n = a.q_start ? a.q_start[b + 1] - tok0 : 1, len = a.kv_len[b];
  const int i = blockIdx.x / a.hq, h = blockIdx.x % a.hq;
  if (tok0 < 0 || n < 0 || n > a.max_q || tok0 + n > a.tokens || len < 0 || len > a.max_kv) {
    if (threadIdx.x == 0) set_status(a.status, kDevBadPosition);
    return;
  }
  if (i >= n) return;
  const int at = len - n + i, lo = a.window > 0 ? max(0, at - a.window + 1) : 0;
  const Kv4Dims d{HD, a.kv.d.group};
  const int kvh = h / (a.hq / a.kv.hkv), e0 = lane * V;
  float q[V], o[V], m = -INFINITY, l = 0.f;
  row_load<V>(a.q, (tok0 + i) * a.q_stride + (long long)h * HD + e0, a.q_type, q);
#pragma unroll
  for (int j = 0; j < V; ++j) o[j] = 0.f;
  for (int p = lo + warp; p <= at; p += 8) {
    const uint8_t* page = kv4_page(a.kv, b, p, a.status);
    if (!page) continue;
    const uint8_t* head = page + (long long)kvh * d.head_bytes();
    const int slot = p % kKv4Page;
    const __half2 ks = reinterpret_cast<const __half2*>(head + d.k_scales())[slot * d.groups() + e0 / d.group];
    const __half2 vs = reinterpret_cast<const __half2*>(head + d.v_scales())[slot * d.groups() + e0 / d.group];
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint32_t byte = head[d.k_codes() + d.k_byte(slot, e0 + j)], c = d.k_high(e0 + j) ? byte >> 4 : byte & 15;
      s = fmaf(q[j], fmaf(__low2float(ks), (float)c, __high2float(ks)), s);
    }
    s = warp_sum(s) * a.qscale;
    const float top = fmaxf(m, s), keep = exp2f(m - top), w = exp2f(s - top);
    m = top;
    l = l * keep + w;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint32_t byte = head[d.v_codes() + d.v_byte(slot, e0 + j)], c = d.v_high(e0 + j) ? byte >> 4 : byte & 15;
      o[j] = fmaf(w, fmaf(__low2float(vs), (float)c, __high2float(vs)), o[j] * keep);
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) so[warp][e0 + j] = o[j];
  if (lane == 0) { sm[warp] = m; sl[warp] = l; }
  __syncthreads();
  if (threadIdx.x >= HD) return;
  float top = -INFINITY, sum = 0.f, v = 0.f;
  for (int w = 0; w < 8; ++w) top = fmaxf(top, sm[w]);
  for (int w = 0; w < 8 && top != -INFINITY; ++w) {
    const float f = exp2f(sm[w] - top);
    sum += f * sl[w];
    v += f * so[w][threadIdx.x];
  }
  gg_store1(a.out, (tok0 + i) * a.out_stride + (long long)h * HD + threadIdx.x, a.q_type, sum == 0.f ? 0.f : v / sum);
}

}  // namespace b200lm
