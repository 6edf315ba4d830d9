// Attention over the cache in 4 bits for many bf16 query rows of a kv head (a prompt's chunk), on the 5th-generation tensor cores.
//
// A CTA owns 128 query rows of a kv head and a range of keys, walked in tiles of 64.
//   S / 2  s (c - 8) / 2 as two fp16 numbers, each exact: s is cut into its upper seven bits and the four below, and c - 8 has four.
//          What the offsets bring, sum over the groups of (m / 2 + 4 s) (sum of q), is one more product of 16: m / 2 and 4 s beside the
//          sums of q over 64 elements, in two terms (2^-22).  (The halves keep 8 s inside fp16's range.)  Queries are bf16 numbers
//          times a power of two of their row, exact in fp16 down to 2^-24 of the row's largest.  So a score is as good as
//          fp32; with K as one fp16 number a score of 50 was off by percents of its key's weight.
//   O      P and V = s c + m as fp16 numbers, one rounding of 2^-11 each, where storing the bf16 row costs 2^-8 (V in two terms and P
//          in two would be three products instead of one, and the rows of V would not fit beside those of K).  P is held times 2^11:
//          a normal number down to 2^-25 of its row's reference, and what lies below is off by 2^-36 of that.
//
//   the others    expand: codes from global memory a tile ahead, K and V rows into swizzled shared memory (two stages each)
//   warp 8        issues the products: S = Q K^T with Q in tensor memory (read from shared memory it would take a third of the
//                 bandwidth that the expanded rows need; the sums of q do come from there), O += P V with P in tensor memory, over
//                 the scores it was made from
//   warps 0 - 7   softmax, two threads a row (half of the keys, half of O each).  A row's reference moves when a score passes it
//                 by 4 powers of two; only then is O read, scaled and written back, behind the products of the tile before.
//
// Order of issue: S(j + 1), then O(j), so that the softmax of a tile runs beside the products of its neighbours.
// Scores of tile j + 1 may overwrite the probabilities of j - 1 when O(j - 1) is complete.
//
// What bounds it: issue slots, 57 % busy, and the tensor pipe, 43 %; most instructions are the expansion's (every CTA of 128 rows
// expands its own keys: 64 of them at head size 256 are 32768 codes), beside it shared memory (96 KB a tile written and read once,
// 1536 cycles, as long as the products take).
// Two chunks of 512 tokens over 4000 and 8192 positions, 8 query heads on 4 of 256: 139 us = 353 TFLOP/s (21 % of the cuBLAS
// rate; 108 us with K in one term), the same of head size 128: 75 us (68); the scores' factor inside the exponent instead of
// beside it took 28 us off, K and V by warps of their own 6.
//
// A NaN in a group of K makes the key's scores NaN, so it spoils the rows that see the key and no others.  One of V is noted for
// those rows, whose dims of the group become NaN at the end; V itself is zero there, as is what no row sees.  All waits are bounded;
// after one that gave up the CTA's threads run to its end without the products, and the status says so.
#pragma once
#include "kv4_attn.cuh"
#include "kv4_chunk_order.h"
#include "prefill_gemm_ts.cuh"
#include "prefill_ops.cuh"
#include "attn_tc.cuh"

namespace b200lm {

constexpr int kKcRows = 128, kKcSoft = 256;
// Powers of two by which a score may pass its row's reference, and by which P is held above that: P <= 2^15 (6 and 9: 135 us instead of 139).
constexpr float kKcLazy = 4.f, kKcRange = 11.f;

template <int HD>
struct KcShape {
  static constexpr int KT = 64;                                      // keys of a tile
  static constexpr int kThreads = kKcSoft + 32 + HD * 2;             // 4 warps for K, 4 for V of every 128 elements
  static constexpr int kTile = KT * HD * 2;                          // V of a tile, or one term of K
  static constexpr int kV = 4 * kTile;                               // two stages of K, then of V
  static constexpr int kLine = 128;                                  // bytes of an operand's row of 64
  static constexpr int kKx = kV + 2 * kTile, kQx = kKx + 2 * KT * kLine;       // offsets of K (two stages) and sums of q: rows of 16 numbers
  static constexpr int kMax = kQx + kKcRows * kLine;                 // [2][128] floats
  static constexpr int kBars = kMax + 2 * 128 * 4;
  static constexpr int kSmem = kBars + 256;
  static constexpr uint32_t kO = 0, kQ = HD, kS = HD + HD / 2;       // tensor memory columns; P of a tile over its scores
  static_assert(kS + 2 * KT <= 512 && kSmem <= 227 * 1024, "budgets");
};
__host__ __device__ constexpr uint32_t kc_idesc(int M, int N) { return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }      // fp16 x fp16 -> fp32

// Two neighbouring codes (nibbles of two bytes, `low` or high) as fp16 numbers (c - 8) / 2, or as V's values.
template <int p>
__device__ __forceinline__ __half2 kc_centred(uint32_t x) {
  const uint32_t y = (x & (p ? 0x00F000F0u : 0x000F000Fu)) | 0x64006400u;       // 1024 + c, or 1024 + 16 c
  const __half2 h = *reinterpret_cast<const __half2*>(&y);
  return p ? __hfma2(h, __float2half2_rn(1.f / 32), __float2half2_rn(-36.f)) : __hfma2(h, __float2half2_rn(0.5f), __float2half2_rn(-516.f));
}
template <int p>
__device__ __forceinline__ uint32_t kc_values(uint32_t x, __half2 s, __half2 m) {
  const uint32_t y = (x & (p ? 0x00F000F0u : 0x000F000Fu)) | 0x64006400u;
  const __half2 h = *reinterpret_cast<const __half2*>(&y);
  const __half2 c = p ? __hfma2(h, __float2half2_rn(1.f / 16), __float2half2_rn(-64.f)) : __hadd2(h, __float2half2_rn(-1024.f));
  const __half2 v = __hfma2(c, s, m);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t kc_product(__half2 a, __half2 b) {
  const __half2 v = __hmul2(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <int HD, int GROUP>
__global__ void __launch_bounds__(KcShape<HD>::kThreads, 1) kv4_chunk_kernel(const Kv4AttnArgs a) {
  using S = KcShape<HD>;
  constexpr int KT = S::KT, P = HD / 128, HK = KT / 2;
  constexpr Kv4Dims d{HD, GROUP};
  extern __shared__ __align__(1024) unsigned char kc_sm[];
  unsigned char *kx = kc_sm + S::kKx, *qx = kc_sm + S::kQx;
  float* row_x = reinterpret_cast<float*>(kc_sm + S::kMax);          // [half][row]
  uint64_t* bars = reinterpret_cast<uint64_t*>(kc_sm + S::kBars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kKcBars);
  int* gave_up = reinterpret_cast<int*>(bars + kKcBars + 1);
  auto wait = [&](KcWait w) { return mbar_wait(bars + w.bar, w.parity(), gave_up); };
  auto wait2 = [&](KcWait w, KcWait x) { return mbar_wait2(bars + w.bar, w.parity(), bars + x.bar, x.parity(), gave_up); };
  __shared__ int last_s, closed_s;                                   // closed: a page that the sequence needs lies outside the pool
  __shared__ unsigned poison[kKcRows];                               // bit i: the row sees a NaN among the elements 64 i .. of V
  const int warp = warp_index(), lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch_dependents();
  // ---- which rows and keys
  const int tile = blockIdx.x % a.row_tiles, split = blockIdx.x / a.row_tiles % a.splits, kvh = blockIdx.x / a.row_tiles / a.splits, b = blockIdx.y;
  const int G = a.hq / a.kv.hkv;
  const int tok0 = a.q_start ? a.q_start[b] : b, nq = a.q_start ? a.q_start[b + 1] - tok0 : 1, len = a.kv_len[b];
  if (tok0 < 0 || nq < 0 || nq > a.max_q || tok0 > a.tokens - nq || len < 0 || len > a.max_kv) {
    if (threadIdx.x == 0) set_status(a.status, kDevBadPosition);
    return;
  }
  const int r0 = tile * kKcRows, rows = min(kKcRows, nq * G - r0);
  if (rows <= 0) return;
  const int first = len - nq + r0 / G, lastp = len - nq + (r0 + rows - 1) / G;
  const int seen0 = a.window > 0 ? max(0, first - a.window + 1) : 0, key0 = seen0 & ~(KT - 1), key1 = lastp + 1;
  const int nsplit = max(1, (key1 - key0 + a.share - 1) / a.share);
  if (split >= nsplit) return;
  const int t0 = (key0 + split * a.share) / KT, n = max(0, (min(key1, key0 + (split + 1) * a.share) + KT - 1) / KT - t0);
  if (threadIdx.x == 0) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars[kKcKFull + s], P * 128);
      mbar_init(&bars[kKcKEmpty + s], 1);
      mbar_init(&bars[kKcVFull + s], P * 128);
      mbar_init(&bars[kKcVEmpty + s], 1);
      mbar_init(&bars[kKcSFull + s], 1);
      mbar_init(&bars[kKcPFull + s], 8);
    }
    mbar_init(&bars[kKcOFull], 1);
    mbar_init(&bars[kKcQReady], 8);
    mbar_init(&bars[kKcODone], 1);
    *gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int i = threadIdx.x; i < (S::kMax - S::kKx) / 16; i += S::kThreads) reinterpret_cast<uint4*>(kx)[i] = make_uint4(0u, 0u, 0u, 0u);      // places of 64 that a head does not have
  if (threadIdx.x < kKcRows) poison[threadIdx.x] = 0u;
  fence_async_smem();
  if (warp == 8) {
    tmem_alloc(tmem_slot, 512);
    const bool closed = __any_sync(0xffffffffu, ka_bad_page(a, a.kv.table + b * a.kv.table_stride, len, nq, lane, 32));
    if (lane == 0) closed_s = closed;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  const int* table = a.kv.table + b * a.kv.table_stride;
  bool ok = true, bad = false;                                       // none of this thread's waits has given up; a page outside the pool
  const int quarter = warp & 3, half = (warp >> 2) & 1, row = quarter * 32 + lane;     // softmax
  const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16);
  float m = -INFINITY, l = 0.f;
  if (n > 0 && warp >= 9) {
    // ---- expansion: the first half of the warps has K rows, the other V rows; thread (key, plane, q): 32 bytes, 64 elements
    const int w = (warp - 9) % (4 * P), key = w / P * 16 + (lane & 15), plane = w % P, q = lane >> 4;
    const bool has_k = warp - 9 < 4 * P;
    const long long page_bytes = (long long)a.kv.hkv * d.head_bytes(), head = (long long)kvh * d.head_bytes();
    uint4 raw[2];
    uint32_t sm[2];                                           // (s, m) of K or V, for each 64 of the plane's elements
    int page_ahead = table[t0 * KT / kKv4Page];               // of the next tile to load: its number is a tile ahead of its rows
    auto load = [&](int j) {
      const int at = (t0 + j) * KT, page = page_ahead, slot = at % kKv4Page + key;
      if (j + 1 < n) page_ahead = table[(at + KT) / kKv4Page];
      if (page < 0 || page >= a.kv.num_pages) {
        bad = true;
        return;
      }
      const uint8_t* h = a.kv.pages + page * page_bytes + head;
      const uint8_t* src = h + (has_k ? d.k_codes() : d.v_codes()) + (plane * kKv4Page + slot) * 64 + q * 32;
      raw[0] = __ldcg(reinterpret_cast<const uint4*>(src));         // not .nc: the kernel before may have written them while this one was set up
      raw[1] = __ldcg(reinterpret_cast<const uint4*>(src) + 1);
      const uint32_t* p = reinterpret_cast<const uint32_t*>(h + (has_k ? d.k_scales() : d.v_scales())) + slot * d.groups() + plane * 128 / GROUP;
      sm[0] = __ldcg(p);
      sm[1] = GROUP == 64 ? __ldcg(p + 1) : sm[0];
    };
    raw[0] = raw[1] = make_uint4(0u, 0u, 0u, 0u);
    sm[0] = sm[1] = 0u;
    load(0);
    auto both = [](uint32_t half) { return __half2half2(__ushort_as_half((unsigned short)half)); };
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      const int st = j & 1;
      const uint32_t word[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
      uint32_t now[2] = {sm[0], sm[1]};
      if (j + 1 < n) load(j + 1);
      const int slot = (t0 + j) * KT % kKv4Page + key, where = (t0 + j) * KT + key;
      if (where < seen0 || where >= key1) now[0] = now[1] = 0u;      // what no row sees: zeros
      if (j >= 2) ok = ok && wait(kc_empty(has_k ? kKcKEmpty : kKcVEmpty, j));
      if (has_k && ok) {
        unsigned char* line = kc_sm + st * 2 * S::kTile + key * S::kLine;
        __half2 hi, lo;
#pragma unroll
        for (int i = 0; i < 4; ++i) {                                // 32 elements: 8 q .. and 16 more, of the words 2 q and 2 q + 1
          if (i == 0 || (GROUP == 64 && i == 2)) {
            hi = both(now[i / 2] & 0xFFF0u);
            lo = __hsub2(both(now[i / 2]), hi);                       // NaN stays NaN
          }
          const uint32_t x[4] = {__byte_perm(word[i], 0, 0x4140), __byte_perm(word[i], 0, 0x4342), __byte_perm(word[4 + i], 0, 0x4140), __byte_perm(word[4 + i], 0, 0x4342)};
          unsigned char* at = line + (plane * 2 + i / 2) * KT * S::kLine;
          const int c = 4 * (i & 1) + q;
          __half2 v[4];
          auto put = [&](int where) {
            unsigned char* to = at + ((where ^ (key & 7)) << 4);
            *reinterpret_cast<uint4*>(to) = make_uint4(kc_product(v[0], hi), kc_product(v[1], hi), kc_product(v[2], hi), kc_product(v[3], hi));
            *reinterpret_cast<uint4*>(to + S::kTile) = make_uint4(kc_product(v[0], lo), kc_product(v[1], lo), kc_product(v[2], lo), kc_product(v[3], lo));
          };
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = kc_centred<0>(x[k]);
          put(c);
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = kc_centred<1>(x[k]);
          put(c + 2);
        }
        // m / 2 of the blocks of 64 elements, then 4 s: beside the first term of the sums (q = 0) and beside the second
        unsigned char* offsets = kx + st * KT * S::kLine + key * S::kLine + ((q ^ (key & 7)) << 4) + plane * 4;
        const uint32_t s2 = __byte_perm(now[0], now[1], 0x5410), m2 = __byte_perm(now[0], now[1], 0x7632);
        *reinterpret_cast<uint32_t*>(offsets) = kc_product(*reinterpret_cast<const __half2*>(&m2), __float2half2_rn(0.5f));
        *reinterpret_cast<uint32_t*>(offsets + 8) = kc_product(*reinterpret_cast<const __half2*>(&s2), __float2half2_rn(4.f));
      }
      // V: this thread has two words of four units; it wants word q of all eight, the partner (lane ^ 16) the other words
      if (!has_k) {
        uint32_t mine[4], got[4], unit[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          mine[i] = q ? word[2 * i + 1] : word[2 * i];
          got[i] = __shfl_xor_sync(0xffffffffu, q ? word[2 * i] : word[2 * i + 1], 16);
        }
        const bool front = q == (slot >> 1 & 1);                         // the units that it has are the first four
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          unit[i] = front ? mine[i] : got[i];
          unit[4 + i] = front ? got[i] : mine[i];
        }
        if (ok) {
          unsigned char* line = kc_sm + S::kV + st * S::kTile + (plane * 2 + q) * KT * S::kLine + key * S::kLine;
          uint32_t pair = q ? now[1] : now[0];
          if ((pair & 0x7C00u) == 0x7C00u) {
            for (int r = 0; r < rows; ++r) {
              const int at = len - nq + (r0 + r) / G;
              if (where <= at && (a.window <= 0 || where > at - a.window)) atomicOr(&poison[r], 1u << (plane * 2 + q));
            }
            pair = 0u;
          }
          const __half2 s = both(pair & 0xFFFFu), low = both(pair >> 16);
#pragma unroll
          for (int i = 0; i < 4; ++i) {                                // byte i of the words: 16 neighbours
            const uint32_t sel = i | (4 + i) << 8;
            const uint32_t x0 = __byte_perm(unit[0], unit[1], sel), x1 = __byte_perm(unit[2], unit[3], sel), x2 = __byte_perm(unit[4], unit[5], sel), x3 = __byte_perm(unit[6], unit[7], sel);
            *reinterpret_cast<uint4*>(line + (((2 * i) ^ (key & 7)) << 4)) = make_uint4(kc_values<0>(x0, s, low), kc_values<0>(x1, s, low), kc_values<0>(x2, s, low), kc_values<0>(x3, s, low));
            *reinterpret_cast<uint4*>(line + (((2 * i + 1) ^ (key & 7)) << 4)) = make_uint4(kc_values<1>(x0, s, low), kc_values<1>(x1, s, low), kc_values<1>(x2, s, low), kc_values<1>(x3, s, low));
          }
        }
      }
      fence_async_smem();
      mbar_arrive(&bars[(has_k ? kKcKFull : kKcVFull) + st]);
      ok = __all_sync(0xffffffffu, ok);
    }
  } else if (n > 0 && warp == 8) {
    // ---- products
    constexpr uint32_t idesc_s = kc_idesc(128, KT), idesc_o = kc_idesc(128, HD) | 1u << 16;      // V: hd contiguous
    const bool leader = elect_one();
    const uint32_t ring = smem_u32(kc_sm);
    auto scores = [&](int j) {
      const uint32_t k = ring + (j & 1) * 2 * S::kTile, to = tmem + S::kS + (j & 1) * KT;
#pragma unroll
      for (int term = 0; term < 2; ++term)
#pragma unroll
        for (int i = 0; i < HD / 16; ++i)
          umma_bf16_ts(to, tmem + S::kQ + i * 8, umma_desc_sw128(k + term * S::kTile + i / 4 * KT * S::kLine) + (uint64_t)(i % 4 * 2), idesc_s, term > 0 || i > 0);
      umma_bf16(to, umma_desc_sw128(smem_u32(qx)), umma_desc_sw128(smem_u32(kx) + (j & 1) * KT * S::kLine), idesc_s, 1);
      umma_commit(&bars[kc_stage(kKcSFull, j)]);
      umma_commit(&bars[kc_stage(kKcKEmpty, j)]);
    };
    ok = __all_sync(0xffffffffu, wait2({kKcQReady, 0}, kc_full(kKcKFull, 0)));
    if (ok) {
      tc_fence_after();
      if (leader) scores(0);
      __syncwarp();
    }
#pragma unroll 1
    for (int j = 0; j < n && ok; ++j) {
      if (j + 1 < n) {
        ok = __all_sync(0xffffffffu, wait(kc_full(kKcKFull, j + 1)) && (j == 0 || wait(kc_o(j - 1))));
        if (!ok) break;
        tc_fence_after();
        if (leader) scores(j + 1);
        __syncwarp();
      }
      ok = __all_sync(0xffffffffu, wait2(kc_full(kKcVFull, j), kc_full(kKcPFull, j)));
      if (!ok) break;
      tc_fence_after();
      if (leader) {
        const uint32_t v = ring + S::kV + (j & 1) * S::kTile;
#pragma unroll
        for (int k = 0; k < KT / 16; ++k)
          umma_bf16_ts(tmem + S::kO, tmem + S::kS + (j & 1) * KT + k * 8, atc_desc_mn(v + k * 2048, KT * S::kLine), idesc_o, j > 0 || k > 0);
        umma_commit(&bars[kKcOFull]);
        umma_commit(&bars[kc_stage(kKcVEmpty, j)]);
        if (j + 1 == n) umma_commit(&bars[kKcODone]);
      }
      __syncwarp();
    }
  } else if (n > 0) {
    // ---- this thread's half of a query row, times a power of two, into tensor memory
    const int at = len - nq + (r0 + row) / G, hi = row < rows ? at : -1, lo = a.window > 0 ? at - a.window + 1 : 0;
    float unit;
    {
      constexpr int V = HD / 2;
      const __nv_bfloat16* src = reinterpret_cast<const __nv_bfloat16*>(a.q) + (long long)(tok0 + (r0 + row) / G) * a.q_stride + (long long)(kvh * G + (r0 + row) % G) * HD + half * V;
      const bool vec = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
      auto get = [&](int i, float (&x)[8]) {
        RawRow<kBf16, 8> raw;
        if (hi >= 0) raw.load(src, i, vec);                          // rows that see nothing are zeros, whatever they hold
        else raw.u[0] = raw.u[1] = raw.u[2] = raw.u[3] = 0u;
        raw.get(x);
      };
      float top = 0.f;
#pragma unroll 4
      for (int i = 0; i < V; i += 8) {
        float x[8];
        get(i, x);
#pragma unroll
        for (int k = 0; k < 8; ++k) top = isfinite(x[k]) ? fmaxf(top, fabsf(x[k])) : INFINITY;
      }
      row_x[half * 128 + row] = top;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      const uint32_t bits = __float_as_uint(fmaxf(row_x[row], row_x[128 + row]));
      const int e = max((int)(bits >> 23), 30);
      const bool spoilt = bits >= 0x7F800000u;
      const float f = spoilt ? 0.f : __uint_as_float((uint32_t)(254 + 7 - e) << 23);             // largest |q| f in [2^7, 2^8)
      // of S / 2; never zero, as masked scores are -inf times this
      unit = spoilt ? __uint_as_float(0x7FC00000u) : fmaxf(__uint_as_float((uint32_t)(e - 6) << 23) * a.qscale, __uint_as_float(1u << 23));
      float sum = 0.f;
#pragma unroll 1
      for (int i = 0; i < V; i += 32) {                              // the second time from the cache
        uint32_t y[16];
#pragma unroll
        for (int k = 0; k < 32; k += 8) {
          float x[8];
          get(i + k, x);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            y[k / 2 + c] = spoilt ? 0u : ka_pack(x[2 * c] * f, x[2 * c + 1] * f);
            sum += spoilt ? 0.f : x[2 * c] * f + x[2 * c + 1] * f;
          }
        }
        tmem_st16(lane_addr + S::kQ + half * (HD / 4) + i / 2, y);
        if (i % 64 == 32) {                                          // below 2^14: a block's sum in two terms, each beside m / 2 and beside 4 s
          const __half t0 = __float2half_rn(sum), t1 = __float2half_rn(sum - __half2float(t0));
          unsigned char* line = qx + row * S::kLine + (half * V + i) / 64 * 2;
          *reinterpret_cast<__half*>(line + ((row & 7) << 4)) = *reinterpret_cast<__half*>(line + ((row & 7) << 4) + 8) = t0;
          *reinterpret_cast<__half*>(line + ((1 ^ (row & 7)) << 4)) = *reinterpret_cast<__half*>(line + ((1 ^ (row & 7)) << 4) + 8) = t1;
          sum = 0.f;
        }
      }
      fence_async_smem();
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[kKcQReady]);
    }
    // keys that every row of the tile sees (rows that it does not have are zeros, and never leave)
    const int open1 = first + 1, open0 = a.window > 0 ? max(0, lastp - a.window + 1) : 0;
    float mz = 0.f;
    bool late = false;
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      const int base = (t0 + j) * KT, mykeys = base + half * HK;
      const bool got = __all_sync(0xffffffffu, wait(kc_full(kKcSFull, j))) && !late;
      float s[HK], mx = -INFINITY;
      if (got) {
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < HK; c += 32) {
          uint32_t x[32];
          tmem_ld32(lane_addr + S::kS + (j & 1) * KT + half * HK + c, x);
#pragma unroll
          for (int i = 0; i < 32; ++i) s[c + i] = __uint_as_float(x[i]);
        }
        if (base < open0 || base + KT > open1) {
#pragma unroll
          for (int i = 0; i < HK; ++i)
            if (mykeys + i > hi || mykeys + i < lo) s[i] = -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < HK; ++i) mx = fmaxf(mx, s[i]);
        mx *= unit;                                                  // positive, or NaN
      }
      if (bar_or<1, 256>(!got || mx > m + kKcLazy)) {
        // the eight warps leave the loop together, or move the references of all rows
        row_x[half * 128 + row] = mx;
        ok = !block_gave_up([&] { return !got; }, bar_or<1, 256>);
        if (!ok) break;
        const float mn = fmaxf(m, fmaxf(row_x[row], row_x[128 + row])), f = mn == m ? 1.f : ka_ex2(m - mn);
        m = mn;
        mz = mn == -INFINITY ? 0.f : mn - kKcRange;
        l *= f;
        if (j > 0) {
          late = !__all_sync(0xffffffffu, wait(kc_o(j - 1)));
          if (!late && __any_sync(0xffffffffu, f != 1.f)) {
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < HD / 2; c += 32) {
              uint32_t x[32];
              tmem_ld32(lane_addr + S::kO + half * (HD / 2) + c, x);
#pragma unroll
              for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * f);
              tmem_st16(lane_addr + S::kO + half * (HD / 2) + c, *reinterpret_cast<const uint32_t(*)[16]>(x));
              tmem_st16(lane_addr + S::kO + half * (HD / 2) + c + 16, *reinterpret_cast<const uint32_t(*)[16]>(x + 16));
            }
          }
        }
      }
#pragma unroll
      for (int c = 0; c < HK; c += 32) {
        uint32_t y[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const float p0 = ka_ex2(fmaf(s[c + i], unit, -mz)), p1 = ka_ex2(fmaf(s[c + i + 1], unit, -mz));
          l += p0 + p1;
          y[i / 2] = ka_pack(p0, p1);
        }
        tmem_st16(lane_addr + S::kS + (j & 1) * KT + half * (HK / 2) + c / 2, y);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[kc_stage(kKcPFull, j)]);
    }
    ok = ok && !late && __all_sync(0xffffffffu, wait(kc_end()));
    tc_fence_after();
  }
  // ---- row sums meet; O out of tensor memory
  const bool spoilt = __syncthreads_or(bad || closed_s) != 0, failed = __syncthreads_or(!ok) != 0;
  const long long u = ((long long)b * a.kv.hkv + kvh) * a.row_tiles + tile;
  constexpr int REC = kKcRows * (HD + 2);
  float* rec = a.parts + (u * a.splits + split) * REC;
  if (warp < 8) row_x[half * 128 + row] = l;
  __syncthreads();
  if (warp < 8 && !failed) {
    const float sum = row_x[row] + row_x[128 + row], inv = sum == 0.f ? 0.f : 1.f / sum;
    const long long out = (long long)(tok0 + (r0 + row) / G) * a.out_stride + (long long)(kvh * G + (r0 + row) % G) * HD + half * (HD / 2);
    const bool vec = (reinterpret_cast<uintptr_t>(reinterpret_cast<__nv_bfloat16*>(a.out) + out) & 15) == 0;
#pragma unroll 1
    for (int c = 0; c < HD / 2; c += 32) {
      uint32_t x[32];
      if (n > 0) tmem_ld32(lane_addr + S::kO + half * (HD / 2) + c, x);
      else {
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] = 0u;
      }
      if (poison[row] >> ((half * (HD / 2) + c) / 64) & 1u) {
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] = 0x7FC00000u;
      }
      if (row < rows && nsplit > 1) {
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          *reinterpret_cast<uint4*>(rec + row * HD + half * (HD / 2) + c + i) = make_uint4(x[i], x[i + 1], x[i + 2], x[i + 3]);
      } else if (row < rows && !spoilt) {
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          RawRow<kBf16, 8> y;
          float v[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = sum == 0.f ? 0.f : __uint_as_float(x[i + k]) * inv;
          y.put(v);
          y.store(a.out, out + c + i, vec);
        }
      }
      __syncwarp();                                                  // the next load is the whole warp's
    }
    if (nsplit > 1 && half == 0) *reinterpret_cast<float2*>(rec + kKcRows * HD + 2 * row) = make_float2(m, spoilt ? -1.f : sum);
  }
  tc_fence_before();
  sync_after_waits(ok);
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (failed) {
    // the other shares of the unit still count this one: its record says that it is lost
    if (nsplit > 1 && threadIdx.x < kKcRows) *reinterpret_cast<float2*>(rec + kKcRows * HD + 2 * threadIdx.x) = make_float2(0.f, -1.f);
    if (threadIdx.x == 0) set_status(a.status, kDevBarrierTimeout);
  } else if (spoilt && threadIdx.x == 0) {
    set_status(a.status, kDevBadPosition);
  }
  if (nsplit == 1) return;
  // ---- the shares' sums: the last CTA of the unit to arrive
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last_s = ticket_last(a.tickets + u, nsplit, [](unsigned* p, unsigned k) { return atomicInc(p, k); });
  __syncthreads();
  if (!last_s) return;
  __threadfence();
  const float* all = a.parts + u * a.splits * REC;
  float* weight = reinterpret_cast<float*>(kc_sm);                   // [nsplit][row], then the rows' sums
  bool lost = false;
  if (threadIdx.x < kKcRows) {
    const float* ml = all + kKcRows * HD + 2 * threadIdx.x;
    float top = -INFINITY, sum = 0.f;
    for (int k = 0; k < nsplit; ++k) top = (int)threadIdx.x < rows ? fmaxf(top, __ldcg(ml + (long long)k * REC)) : 0.f;
    for (int k = 0; k < nsplit; ++k) {
      const float mk = (int)threadIdx.x < rows ? __ldcg(ml + (long long)k * REC) : 0.f, lk = (int)threadIdx.x < rows ? __ldcg(ml + (long long)k * REC + 1) : 1.f, f = mk == top ? 1.f : ka_ex2(mk - top);
      lost = lost || lk < 0.f;
      weight[k * kKcRows + threadIdx.x] = f;
      sum = fmaf(f, lk, sum);
    }
    weight[nsplit * kKcRows + threadIdx.x] = sum;
  }
  if (__syncthreads_or(lost)) return;                                // the CTA that lost it has said so
#pragma unroll 1
  for (int i = threadIdx.x; i < rows * HD / 8; i += S::kThreads) {
    const int r = i / (HD / 8), dim = i % (HD / 8) * 8;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int k = 0; k < nsplit; ++k) {
      const float4* p = reinterpret_cast<const float4*>(all + (long long)k * REC + r * HD + dim);
      const float4 x = __ldcg(p), y = __ldcg(p + 1);
      const float f = weight[k * kKcRows + r];
      v[0] = fmaf(f, x.x, v[0]); v[1] = fmaf(f, x.y, v[1]); v[2] = fmaf(f, x.z, v[2]); v[3] = fmaf(f, x.w, v[3]);
      v[4] = fmaf(f, y.x, v[4]); v[5] = fmaf(f, y.y, v[5]); v[6] = fmaf(f, y.z, v[6]); v[7] = fmaf(f, y.w, v[7]);
    }
    const float sum = weight[nsplit * kKcRows + r], inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = sum == 0.f ? 0.f : v[k] * inv;
    const long long out = (long long)(tok0 + (r0 + r) / G) * a.out_stride + (long long)(kvh * G + (r0 + r) % G) * HD + dim;
    RawRow<kBf16, 8> y;
    y.put(v);
    y.store(a.out, out, (reinterpret_cast<uintptr_t>(reinterpret_cast<__nv_bfloat16*>(a.out) + out) & 15) == 0);
  }
}

}  // namespace b200lm
