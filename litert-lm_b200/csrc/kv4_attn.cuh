// Attention of ragged sequences over the cache in 4 bits, for a few query rows of a kv head (head of its group x token).
//
//   S = scale q K^T,  K = s c + m per group of dims:   S = sum_g s_g (q . c)_g + sum_g m_g (sum of q over g)
//   O = P V,          V = s c + m:                      O = sum_keys (P s_g) (c - 8) + sum_keys P (m_g + 8 s_g)
//
// The codes go from the cache into the A operands of mma.sync as they are, and the precision lies in the other operand:
//   S  int8 products (m16n8k32, unsigned codes): a row of q is cut into four digits of seven bits below its largest power of
//      two (of three bits and three times seven where the codes enter as 16 c: upper nibbles are masked, not shifted), the eight
//      columns are four digits of two rows, the sums are exact integers and enter fp32 once a group.
//   O  fp16 products (m16n8k16) with the codes as numbers c - 8 (exact) and P s in two fp16 terms (2^-22 of each weight).  One
//      term, with P and m + 8 s as fp16 numbers too, took 5.6 us off the 93 of 64 bf16 sequences and put 3 * 2^-11 on each weight:
//      one bf16 result in ten came out a step off.  P s is held in a power of two below fp16's range, one for each group of
//      dims: its reference is the largest scale of the group that the warp has met, so small weights are off by 2^-36 of that.
//      Two nibbles of a half word come out of a mask each (1024 + c and 1024 + 16 c) and a fused product makes them c - 8; as
//      bf16 numbers they would need a shift each, and the logic pipe, half as wide as the others, is what bounds this kernel.
//      Codes centred at zero keep the sums small; the tensor core cuts its sums off, so fp32 rows take them out after every
//      product, 16-bit rows at the end (at most 2^-24 an add).
//
// A warp walks its own tiles of keys (16 at head size 256, else 32) with a ring of its own that it fills by 16-byte asynchronous
// copies: K and V rows lie in the cache in the order in which the fragments want them, so a lane's loads are 8 or 16 bytes
// wide and free of bank conflicts.  Warps meet only at the end.  The softmax keeps a reference per row and warp that moves when a
// score passes it by 4 powers of two, so that an ordinary tile takes one vote and no exchange of maxima.
//
// A CTA serves RB rows over a share of the keys; shares of a sequence are joined by the last CTA to arrive.  How many
// keys a share has is decided on the host from the largest length, how many shares a sequence has on the device from its own.
//
// What bounds it: issue slots (65 % busy with 16 warps an SM) and the logic pipe (52 %), not the bytes.  64 sequences of 300 ..
// 8192 positions, 8 query heads on 4 of 256, bf16: 97.4 us = 3.2 TB/s; three of 40001 .. 65536, 32 on 16 of 128, fp32: 93.7 us =
// 3.7 TB/s; 16 x 5 rows in a window of 1024: 29.4 us; one sequence of 777 positions: 10.1 us, a chain of latencies with the join.
// Tiles of 16 keys at head size 256 because two CTAs an SM leave 14 KB of ring a warp: three stages.
#pragma once
#include "kv4_rows.cuh"
#include "split_ticket.h"

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
  int row_tiles, share, splits;           // row tiles of a kv head, keys of a share, most shares of a sequence
  unsigned* tickets;                      // one per (sequence, kv head, row tile), zero between calls
  float* parts;                           // [unit][split]: O [RB][HD], then maximum and sum (negative: a page outside the pool) of each row
};

constexpr int kKaWarps = 8, kKaThreads = 32 * kKaWarps;
constexpr int kKaTickets = 4096;          // words at the start of a workspace
constexpr int kKaStages = 3;

template <int HD, int GROUP, int RB>
struct KaShape {
  static constexpr int PL = HD < 128 ? HD : 128, P = HD / PL;        // plane, planes
  static constexpr int ROW = PL / 2, NG = HD / GROUP;
  static constexpr int NB = RB / 2;                                  // column blocks of S: two rows of four digits
  static constexpr int CV = RB * 2, NBV = (CV + 7) / 8;              // columns of O (two terms of P s a row), blocks of them
  static constexpr int KT = HD == 256 ? 16 : 32, SUB = KT / 16, MT = HD / 16;
  static constexpr int kCodes = KT * HD / 2, kScales = KT * NG * 4, kStage = 2 * (kCodes + kScales);
  static constexpr int kRing = kKaWarps * kKaStages * kStage;
  static constexpr int kDigits = HD / 64 * NB * 512;
  static constexpr int kUnit = kRing + kDigits;                      // [RB], then the group sums [RB][NG]
  static constexpr int kMergeO = kKaWarps * RB * HD * 4, kMergeOff = kKaWarps * RB * NG * 4;
  static_assert(kMergeO + kMergeOff + kKaWarps * RB * 8 + RB * 8 <= kRing, "the exchange fits over the ring");
  static_assert(RB * KT * 4 <= kCodes, "P of a tile fits over its K codes");
  static_assert(RB * NG <= 32, "a bit for each row and group");
  static constexpr float kLazy = 4.f;                                // powers of two by which a score may pass its row's reference
  static constexpr int kSmem = kUnit + RB * 4 + RB * NG * 4;
};

__device__ __forceinline__ void ka_mma_s(int (&d)[4], const int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
               : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}
__device__ __forceinline__ void ka_mma_o(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ka_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void ka_copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
// The lowest (p = 0) or second nibble of both halves of x as fp16 numbers c - 8.
template <int p>
__device__ __forceinline__ uint32_t ka_codes(uint32_t x) {
  const uint32_t y = (x & (p ? 0x00F000F0u : 0x000F000Fu)) | 0x64006400u;       // 1024 + c, or 1024 + 16 c
  const __half2 h = *reinterpret_cast<const __half2*>(&y);
  const __half2 r = p ? __hfma2(h, __float2half2_rn(1.f / 16), __float2half2_rn(-72.f)) : __hadd2(h, __float2half2_rn(-1032.f));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t ka_pack(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 ka_unpack(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }

// A thread's look at the pages that the rows of a sequence need, from the first that the first row sees to the last: `one` of `all` threads.
// A page outside the pool leaves all rows of the sequence alone, also those of CTAs that would not read it.
__device__ __forceinline__ bool ka_bad_page(const Kv4AttnArgs& a, const int* table, int len, int nq, int one, int all) {
  bool bad = false;
  for (int i = (a.window > 0 ? max(0, len - nq - a.window + 1) : 0) / kKv4Page + one; i < (len + kKv4Page - 1) / kKv4Page; i += all) {
    const int page = table[i];
    bad = bad || page < 0 || page >= a.kv.num_pages;
  }
  return bad;
}

template <int N>
__device__ __forceinline__ void ka_words(const unsigned char* p, uint32_t (&d)[N]) {
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    d[0] = v.x; d[1] = v.y; d[2] = v.z; d[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    d[0] = v.x; d[1] = v.y;
  } else {
    d[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

template <int HD, int GROUP, int RB, bool EXACT>
__global__ void __launch_bounds__(kKaThreads, 2) kv4_attn_kernel(const Kv4AttnArgs a) {
  using S = KaShape<HD, GROUP, RB>;
  constexpr int NG = S::NG, NB = S::NB, NBV = S::NBV, KT = S::KT, SUB = S::SUB, W4 = S::PL / 32;
  extern __shared__ __align__(128) unsigned char ka_sm[];
  __shared__ unsigned poison_s;                                      // bit r NG + g: row r sees a NaN in group g of V
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
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
  const int r0 = tile * RB, rows = min(RB, nq * G - r0);
  if (rows <= 0) return;
  const int first = len - nq + r0 / G, lastp = len - nq + (r0 + rows - 1) / G;              // positions of the first and last row
  const int key0 = (a.window > 0 ? max(0, first - a.window + 1) : 0) & ~(KT - 1), key1 = lastp + 1;     // keys that any of them sees
  const int nsplit = max(1, (key1 - key0 + a.share - 1) / a.share);
  if (split >= nsplit) return;
  const int t0 = (key0 + split * a.share) / KT, t1 = (min(key1, key0 + (split + 1) * a.share) + KT - 1) / KT;

  if (threadIdx.x == 0) poison_s = 0u;
  // ---- this warp's ring
  unsigned char* ring = ka_sm + warp * (kKaStages * S::kStage);
  const Kv4Dims d{HD, GROUP};
  const long long head = (long long)kvh * d.head_bytes(), page_bytes = (long long)a.kv.hkv * d.head_bytes();
  const int* table = a.kv.table + b * a.kv.table_stride;
  bool bad = ka_bad_page(a, table, len, nq, threadIdx.x, kKaThreads);
  int next = t0 + warp, slot_in = 0;
  int page = next < t1 ? table[next * KT / kKv4Page] : 0;
  auto issue = [&]() {
    if (next < t1) {
      if (page < 0 || page >= a.kv.num_pages) bad = true;
      else {
        const unsigned char* src = a.kv.pages + page * page_bytes + head;
        unsigned char* dst = ring + slot_in * S::kStage;
        const int at = next * KT % kKv4Page;
#pragma unroll
        for (int side = 0; side < 2; ++side)
#pragma unroll
          for (int p = 0; p < S::P; ++p)
#pragma unroll
            for (int i = 0; i < KT * S::ROW / 512; ++i)
              ka_copy16(dst + side * S::kCodes + p * KT * S::ROW + i * 512 + lane * 16,
                        src + (side ? d.v_codes() : d.k_codes()) + p * kKv4Page * S::ROW + at * S::ROW + i * 512 + lane * 16);
        constexpr int N = S::kScales / 16;                           // 16-byte pieces of a side's scales: 8 or 16
        if (lane < 2 * N) {
          const int side = lane / N, i = lane % N;
          ka_copy16(dst + 2 * S::kCodes + side * S::kScales + i * 16, src + (side ? d.v_scales() : d.k_scales()) + at * NG * 4 + i * 16);
        }
      }
      next += kKaWarps;
      if (next < t1) page = table[next * KT / kKv4Page];
    }
    if (++slot_in == kKaStages) slot_in = 0;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kKaStages - 1; ++i) issue();

  // ---- query rows as digits; what multiplies their sums, and their sums over the groups
  uint32_t* digits = reinterpret_cast<uint32_t*>(ka_sm + S::kRing);                         // [64 dims][nb][lane][4]
  float* unit_s = reinterpret_cast<float*>(ka_sm + S::kUnit);
  float* qsum_s = unit_s + RB;
  for (int r = warp; r < RB; r += kKaWarps) {
    constexpr int V = HD / 32;
    float x[V];
    const int row = r0 + r;
    if (r < rows) row_load<V>(a.q, (tok0 + row / G) * a.q_stride + (long long)(kvh * G + row % G) * HD + lane * V, a.q_type, x);
    float top = 0.f, sum = 0.f;
    bool odd = false;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (r >= rows) x[j] = 0.f;
      top = fmaxf(top, fabsf(x[j]));
      odd = odd || !isfinite(x[j]);
      sum += x[j];
    }
    const uint32_t bits = __reduce_max_sync(0xffffffffu, odd ? 0x7F800000u : __float_as_uint(top));
    const int e = max((int)(bits >> 23), 30);
    // elements with bit 4 set meet their codes as 16 c: their digits are of a sixteenth, 2^-23 of the row's largest
    const float f = __uint_as_float((uint32_t)(254 + 5 - e - ((lane * V & 16) ? 4 : 0)) << 23);
    const bool spoilt = bits >= 0x7F800000u;
    uint32_t word[4][(V + 3) / 4] = {};
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float y = spoilt ? 0.f : x[j] * f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float q = rintf(y);
        word[i][j / 4] |= ((uint32_t)(int)q & 0xFFu) << (8 * (j % 4));
        y = (y - q) * 128.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // element e0 = 64 T + 32 step + 16 half + 4 t + byte lies in word (T, step, half) of lane (column 4 (r & 1) + i, t)
      const int e0 = lane * V, at = ((e0 / 64 * NB + (r >> 1)) * 32 + (4 * (r & 1) + i) * 4) * 4 + e0 % 64 / 16;
      if constexpr (V == 2) {
        const uint32_t both = word[i][0] | __shfl_down_sync(0xffffffffu, word[i][0], 1) << 16;
        if (!(lane & 1)) digits[at + e0 % 16 / 4 * 4] = both;
      } else {
#pragma unroll
        for (int j = 0; j < V / 4; ++j) digits[at + (e0 + 4 * j) % 16 / 4 * 4] = word[i][j];
      }
    }
#pragma unroll
    for (int o = 1; o < GROUP / V; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane % (GROUP / V) == 0) qsum_s[r * NG + lane / (GROUP / V)] = sum * a.qscale;
    if (lane == 0) unit_s[r] = spoilt ? __uint_as_float(0x7FC00000u) : __uint_as_float((uint32_t)(e - 5) << 23) * a.qscale;
  }
  __syncthreads();
  float unit[NB], qsum[NB][NG], m[NB], mz[NB], l[NB];                  // mz: m, or 0 while there is none
  int hi[NB], lo[NB];                                                // the keys that this lane's rows see
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int r = 2 * nb + (t >> 1);
    unit[nb] = unit_s[r];
#pragma unroll
    for (int i = 0; i < NG; ++i) qsum[nb][i] = qsum_s[r * NG + i];
    const int at = len - nq + (r0 + r) / G;
    hi[nb] = r < rows ? at : -1;
    lo[nb] = a.window > 0 ? at - a.window + 1 : 0;
    m[nb] = -INFINITY;
    mz[nb] = l[nb] = 0.f;
  }
  constexpr int WL = KT * NG / 32;                                   // scales of V of a tile that a lane looks at, of groups (lane WL + i) % NG
  float wk[NG];                                                      // P s is held times this power of two: at first any scale is past it
  uint32_t limit[WL];                                                // and scales (fp16 bits) from this one on are
#pragma unroll
  for (int i = 0; i < NG; ++i) wk[i] = 1099511627776.f;
#pragma unroll
  for (int i = 0; i < WL; ++i) limit[i] = 1u;
  float o[S::MT][NBV][4], off[NBV][NG];                              // off: this lane's sums of P (m + 8 s)
#pragma unroll
  for (int c = 0; c < NBV; ++c) {
#pragma unroll
    for (int i = 0; i < S::MT; ++i) o[i][c][0] = o[i][c][1] = o[i][c][2] = o[i][c][3] = 0.f;
#pragma unroll
    for (int i = 0; i < NG; ++i) off[c][i] = 0.f;
  }
  // keys that every row sees, so that tiles within them need no mask (rows that the tile does not have are zeros, and never leave)
  const int seen0 = a.window > 0 ? max(0, first - a.window + 1) : 0;
  const int open1 = first + 1, open0 = a.window > 0 ? max(0, lastp - a.window + 1) : 0;

  auto add = [](float (&acc)[4], const uint32_t (&x)[4], const uint32_t (&y)[2]) {
    if constexpr (!EXACT) {
      ka_mma_o(acc, x, y[0], y[1]);
    } else {
      float part[4] = {0.f, 0.f, 0.f, 0.f};
      ka_mma_o(part, x, y[0], y[1]);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] += part[i];
    }
  };
  // O += (P s) codes of a tile: lane (g, t) holds column g of P s for the keys t + 4 i, and the codes of unit g of those keys.
  auto products = [&](const unsigned char* st) {
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      float w[NBV][4];
#pragma unroll
      for (int c = 0; c < NBV; ++c) {
        const int r = c * 4 + g / 2;
        const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(st) + (r < RB ? r : 0) * KT + u * 16 + 4 * t);
        w[c][0] = v.x; w[c][1] = v.y; w[c][2] = v.z; w[c][3] = v.w;
      }
      uint32_t vs[4][NG];
#pragma unroll
      for (int i = 0; i < 4; ++i) ka_words<NG>(st + 2 * S::kCodes + S::kScales + (u * 16 + t + 4 * i) * NG * 4, vs[i]);
      uint32_t bt[NBV][2];
#pragma unroll
      for (int pl = 0; pl < S::P; ++pl) {
        constexpr int WU = S::ROW / 32;                              // words of a unit: 2, at head size 64 one
        uint32_t v[4][WU];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int unit_at = S::PL == 128 ? g ^ (4 * (t >> 1)) : g;
          ka_words<WU>(st + S::kCodes + pl * KT * S::ROW + (u * 16 + t + 4 * i) * S::ROW + unit_at * (S::ROW / 8), v[i]);
        }
#pragma unroll
        for (int j = 0; j < WU; ++j) {                               // 64 dims
          const int dim = pl * S::PL + j * 64, grp = dim / GROUP;
          if (dim % GROUP == 0) {
            float sc[4], mn[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&vs[i][grp]));
              sc[i] = f.x * wk[grp];
              mn[i] = fmaf(8.f, f.x, f.y);
            }
#pragma unroll
            for (int c = 0; c < NBV; ++c) {
              float x[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                x[i] = w[c][i] * sc[i];
                off[c][grp] = fmaf(w[c][i], mn[i], off[c][grp]);
              }
              uint32_t b0 = ka_pack(x[0], x[1]), b1 = ka_pack(x[2], x[3]);
              // what the first term left, in the odd columns
              const float2 y0 = ka_unpack(b0), y1 = ka_unpack(b1);
              const uint32_t n0 = ka_pack(x[0] - y0.x, x[1] - y0.y), n1 = ka_pack(x[2] - y1.x, x[3] - y1.y);
              if (g & 1) { b0 = n0; b1 = n1; }
              bt[c][0] = b0;
              bt[c][1] = b1;
            }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {                              // 32 dims: a half of the units' words
            const uint32_t x = __byte_perm(v[0][j], v[1][j], h ? 0x7632 : 0x5410), y = __byte_perm(v[2][j], v[3][j], h ? 0x7632 : 0x5410);
            const uint32_t a0[4] = {ka_codes<0>(x), ka_codes<1>(x), ka_codes<0>(y), ka_codes<1>(y)};
            const uint32_t a1[4] = {ka_codes<0>(x >> 8), ka_codes<1>(x >> 8), ka_codes<0>(y >> 8), ka_codes<1>(y >> 8)};
            const int mt = dim / 16 + 2 * h;
#pragma unroll
            for (int c = 0; c < NBV; ++c) {
              add(o[mt][c], a0, bt[c]);
              add(o[mt + 1][c], a1, bt[c]);
            }
          }
        }
      }
    }
  };
  const int zero[4] = {kGgMagic, kGgMagic, kGgMagic, kGgMagic};
  int slot = 0;
#pragma unroll 1
  for (int tl = t0 + warp; tl < t1; tl += kKaWarps) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kKaStages - 2) : "memory");
    __syncwarp();                                                    // the tile is there, and the tile before is done with
    issue();
    unsigned char* st = ring + slot * S::kStage;
    if (++slot == kKaStages) slot = 0;
    const bool edge = tl * KT < open0 || tl * KT + KT > open1;

    // ---- V's scales: the largest; a NaN spoils its group's sums by itself where every row sees it.  In tiles that not every row sees
    // whole it is taken out and noted for the rows that do; what no row sees may hold anything (zeros do no harm)
    bool over = false;
    uint32_t w[WL];                                                  // every scale of V once in the warp
    {
      uint32_t* scales = reinterpret_cast<uint32_t*>(st + 2 * S::kCodes + S::kScales);
      ka_words<WL>(reinterpret_cast<const unsigned char*>(scales) + lane * WL * 4, w);
#pragma unroll
      for (int i = 0; i < WL; ++i) {
        uint32_t& x = w[i];
        x &= 0xFFFFu;
        if (edge) {
          const int key = tl * KT + (lane * WL + i) / NG;
          const bool seen = key >= seen0 && key < key1;
          if (seen && x >= 0x7C00u) {
            for (int r = 0; r < rows; ++r) {
              const int at = len - nq + (r0 + r) / G;
              if (key <= at && (a.window <= 0 || key > at - a.window)) atomicOr(&poison_s, 1u << (r * NG + (lane * WL + i) % NG));
            }
          }
          if (!seen || x >= 0x7C00u) scales[lane * WL + i] = x = 0u;
        }
        if (x >= 0x7C00u) x = 0u;
        over = over || x >= limit[i];
      }
      if (edge) __syncwarp();
    }

    // ---- S: lane (g, t) gathers the digit pair t & 1 of row 2 nb + (t >> 1) for the keys g and g + 8
    float s[SUB][NB][2], smin[SUB][NB];
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) s[u][nb][0] = s[u][nb][1] = smin[u][nb] = 0.f;
    {
      uint32_t ks[SUB][2][NG];
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) ka_words<NG>(st + 2 * S::kCodes + (u * 16 + g + 8 * h) * NG * 4, ks[u][h]);
      int c[SUB][NB][4];
#pragma unroll
      for (int p = 0; p < S::P; ++p) {
        uint32_t k[SUB][2][W4];
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
          for (int h = 0; h < 2; ++h) ka_words<W4>(st + p * KT * S::ROW + (u * 16 + g + 8 * h) * S::ROW + t * (S::ROW / 4), k[u][h]);
#pragma unroll
        for (int j = 0; j < W4; ++j) {                               // 32 dims
          const int dim = p * S::PL + j * 32, grp = dim / GROUP;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            const uint2 q = *reinterpret_cast<const uint2*>(digits + ((dim / 64 * NB + nb) * 32 + lane) * 4 + (j & 1) * 2);
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
              const uint32_t x = k[u][0][j], y = k[u][1][j];
              constexpr uint32_t n = 0x0F0F0F0Fu;                    // the upper nibbles enter as 16 c, their digits a sixteenth
              if (dim % GROUP == 0) ka_mma_s(c[u][nb], zero, x & n, y & n, x & ~n, y & ~n, q.x, q.y);
              else ka_mma_s(c[u][nb], c[u][nb], x & n, y & n, x & ~n, y & ~n, q.x, q.y);
            }
          }
          if ((dim + 32) % GROUP == 0) {
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
              const float2 s0 = __half22float2(*reinterpret_cast<const __half2*>(&ks[u][0][grp]));
              const float2 s1 = __half22float2(*reinterpret_cast<const __half2*>(&ks[u][1][grp]));
              const float low = t & 1 ? s1.y : s0.y;
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) {
                // both digits' sums carry 1.5 * 2^23; taking that off is exact, the sum of the two is rounded once
                constexpr float big = 12582912.f * (1.f + 1.f / 128);
                const float d0 = fmaf(__int_as_float(c[u][nb][1]), 1.f / 128, __int_as_float(c[u][nb][0]) - big);
                const float d1 = fmaf(__int_as_float(c[u][nb][3]), 1.f / 128, __int_as_float(c[u][nb][2]) - big);
                s[u][nb][0] = fmaf(s0.x, d0, s[u][nb][0]);
                s[u][nb][1] = fmaf(s1.x, d1, s[u][nb][1]);
                smin[u][nb] = fmaf(low, qsum[nb][grp], smin[u][nb]);
              }
            }
          }
        }
      }
    }
    // ---- whole scores: lane keeps key g + 8 (t & 1); softmax against the row's reference
    float p[SUB][NB];
    const float digit = t & 1 ? 1.f / 16384 : 1.f;
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const float mine = (t & 1 ? s[u][nb][1] : s[u][nb][0]) * digit, other = (t & 1 ? s[u][nb][0] : s[u][nb][1]) * digit;
        float x = fmaf(mine + __shfl_xor_sync(0xffffffffu, other, 1), unit[nb], smin[u][nb]);
        if (edge) {
          const int key = tl * KT + u * 16 + g + 8 * (t & 1);
          if (key > hi[nb] || key < lo[nb]) x = -INFINITY;
        }
        p[u][nb] = x;
        over = over || x > m[nb] + S::kLazy;
      }
    if (__any_sync(0xffffffffu, over)) {
      float f[NB], fk[NG];
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        uint32_t largest = 0;
#pragma unroll
        for (int j = 0; j < WL; ++j)
          if ((lane * WL + j) % NG == i) largest = max(largest, w[j]);
        const float top = __half2float(__ushort_as_half((unsigned short)__reduce_max_sync(0xffffffffu, largest)));
        fk[i] = 1.f;
        if (top * wk[i] >= 2048.f) {                                 // largest 2^k in [2^10, 2^11): with P <= 2^4 within fp16's range
          const float power = __uint_as_float(__float_as_uint(top) & 0x7F800000u), k = 1024.f / power;
          fk[i] = k / wk[i];
          wk[i] = k;
#pragma unroll
          for (int j = 0; j < WL; ++j)
            if ((lane * WL + j) % NG == i) limit[j] = power >= 32768.f ? 0x7C00u : (uint32_t)__half_as_ushort(__float2half_rn(2.f * power));
        }
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float top = m[nb];
#pragma unroll
        for (int u = 0; u < SUB; ++u) top = fmaxf(top, p[u][nb]);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
        f[nb] = m[nb] == top ? 1.f : ka_ex2(m[nb] - top);            // equal: both may be -inf
        m[nb] = top;
        mz[nb] = top == -INFINITY ? 0.f : top;
        l[nb] *= f[nb];
      }
      auto of_row = [&](int r) {                                     // factor of row r, from a lane that holds it
        float v = 1.f;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const float x = __shfl_sync(0xffffffffu, f[nb], (r & 1) * 2);
          if (r >> 1 == nb) v = x;
        }
        return v;
      };
#pragma unroll
      for (int c = 0; c < NBV; ++c) {
        const float fr = of_row(c * 4 + t), fo = of_row(c * 4 + g / 2);      // of this lane's columns 2 t and 2 t + 1, and of column g
#pragma unroll
        for (int i = 0; i < S::MT; ++i) {
          const float x = fr * fk[i * 16 / GROUP];
          o[i][c][0] *= x; o[i][c][1] *= x; o[i][c][2] *= x; o[i][c][3] *= x;
        }
#pragma unroll
        for (int i = 0; i < NG; ++i) off[c][i] *= fo;
      }
    }
    // ---- P in the order of the keys in O's products: key t + 4 i of a block of 16 at 4 t + i.  It lies over the K codes.
    __syncwarp();
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const float x = ka_ex2(p[u][nb] - mz[nb]);
        l[nb] += x;
        const int key = g + 8 * (t & 1);
        reinterpret_cast<float*>(st)[(2 * nb + (t >> 1)) * KT + u * 16 + key % 4 * 4 + key / 4] = x;
      }
    __syncwarp();

    products(st);
  }

  // ---- the warps' sums
  float* mo = reinterpret_cast<float*>(ka_sm);                       // [warp][RB][HD]
  float* moff = mo + S::kMergeO / 4;                                 // [warp][RB][NG]
  float* ml = moff + S::kMergeOff / 4;                               // [warp][RB][2]
  const bool spoilt = __syncthreads_or(bad) != 0;                    // every warp is done with its ring, too
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    float x = l[nb];
    x += __shfl_xor_sync(0xffffffffu, x, 1);
#pragma unroll
    for (int w = 4; w < 32; w <<= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
    if (g == 0 && !(t & 1)) {
      ml[(warp * RB + 2 * nb + (t >> 1)) * 2] = m[nb];
      ml[(warp * RB + 2 * nb + (t >> 1)) * 2 + 1] = x;
    }
  }
#pragma unroll
  for (int c = 0; c < NBV; ++c) {
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      float x = off[c][i];
      x += __shfl_xor_sync(0xffffffffu, x, 1);
      x += __shfl_xor_sync(0xffffffffu, x, 2);
      if (t == 0 && !(g & 1) && c * 8 + g < S::CV) moff[(warp * RB + c * 4 + g / 2) * NG + i] = x;
    }
#pragma unroll
    for (int i = 0; i < S::MT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // the two terms of row 4 c + t, out of the group's power of two
        if (c * 4 + t < RB) mo[(warp * RB + c * 4 + t) * HD + i * 16 + h * 8 + g] = (o[i][c][2 * h] + o[i][c][2 * h + 1]) * (1.f / wk[i * 16 / GROUP]);
      }
  }
  __syncthreads();
  // weights of the warps' sums (eight neighbouring lanes a row), the CTA's maximum and sum
  float* total = ml + kKaWarps * RB * 2;                             // [RB][2]
  if (warp * 32 < RB * kKaWarps) {                                   // whole warps: with two rows, lanes 16 .. 31 repeat the second
    const int w = threadIdx.x % kKaWarps, r = min((int)threadIdx.x / kKaWarps, RB - 1);
    const float mw = ml[(w * RB + r) * 2];
    float top = mw, sum = ml[(w * RB + r) * 2 + 1];
#pragma unroll
    for (int k = 1; k < kKaWarps; k <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
    const float f = mw == top ? 1.f : ka_ex2(mw - top);
    sum *= f;
#pragma unroll
    for (int k = 1; k < kKaWarps; k <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
    if (threadIdx.x < RB * kKaWarps) {
      ml[(w * RB + r) * 2] = f;
      if (w == 0) {
        total[2 * r] = top;
        total[2 * r + 1] = sum;
      }
    }
  }
  __syncthreads();
  const long long u = ((long long)b * a.kv.hkv + kvh) * a.row_tiles + tile;
  constexpr int REC = RB * (HD + 2);                                 // a share's record: O, then maximum and sum of its rows
  float* rec = a.parts + (u * a.splits + split) * REC;
  // a thread's elements are four neighbours of a row
  auto store = [&](int r, int dim, const float (&v)[4], float sum) {
    const int row = r0 + r;
    const long long at = (long long)(tok0 + row / G) * a.out_stride + (long long)(kvh * G + row % G) * HD + dim;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int k = 0; k < 4; ++k) gg_store1(a.out, at + k, a.q_type, sum == 0.f ? 0.f : v[k] * inv);
  };
#pragma unroll 1
  for (int i = threadIdx.x; i < RB * HD / 4; i += kKaThreads) {
    const int r = i / (HD / 4), dim = i % (HD / 4) * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kKaWarps; ++w) {
      const float f = ml[(w * RB + r) * 2], add_all = moff[(w * RB + r) * NG + dim / GROUP];
      const float4 x = *reinterpret_cast<const float4*>(mo + (w * RB + r) * HD + dim);
      v[0] = fmaf(f, x.x + add_all, v[0]); v[1] = fmaf(f, x.y + add_all, v[1]); v[2] = fmaf(f, x.z + add_all, v[2]); v[3] = fmaf(f, x.w + add_all, v[3]);
    }
    if (poison_s >> (r * NG + dim / GROUP) & 1u) v[0] = v[1] = v[2] = v[3] = __uint_as_float(0x7FC00000u);
    if (nsplit > 1) *reinterpret_cast<float4*>(rec + r * HD + dim) = make_float4(v[0], v[1], v[2], v[3]);
    else if (r < rows && !spoilt) store(r, dim, v, total[2 * r + 1]);
  }
  if (nsplit == 1) {
    if (spoilt && threadIdx.x == 0) set_status(a.status, kDevBadPosition);
    return;
  }
  if (threadIdx.x < 2 * RB) rec[RB * HD + threadIdx.x] = spoilt && (threadIdx.x & 1) ? -1.f : total[threadIdx.x];
  // ---- the shares' sums: the last CTA of the unit to arrive
  __shared__ int last_s;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last_s = ticket_last(a.tickets + u, nsplit, [](unsigned* p, unsigned n) { return atomicInc(p, n); });
  __syncthreads();
  if (!last_s) return;
  __threadfence();
  const float* all = a.parts + u * a.splits * REC;
  float* weight = reinterpret_cast<float*>(ka_sm);                   // [RB][nsplit] (the host keeps RB * splits below the ring's size)
  bool lost = false;
  for (int i = threadIdx.x; i < RB * nsplit; i += kKaThreads) {
    const float2 x = __ldcg(reinterpret_cast<const float2*>(all + (long long)(i / RB) * REC + RB * HD) + i % RB);
    lost = lost || x.y < 0.f;
    weight[i % RB * nsplit + i / RB] = x.x;
    weight[(RB + i % RB) * nsplit + i / RB] = x.y;
  }
  if (__syncthreads_or(lost)) {
    if (threadIdx.x == 0) set_status(a.status, kDevBadPosition);
    return;
  }
  for (int r = warp; r < RB; r += kKaWarps) {
    float top = -INFINITY, sum = 0.f;
    for (int k = lane; k < nsplit; k += 32) top = fmaxf(top, weight[r * nsplit + k]);
    top = warp_max(top);
    for (int k = lane; k < nsplit; k += 32) {
      const float mk = weight[r * nsplit + k], f = mk == top ? 1.f : ka_ex2(mk - top);
      weight[r * nsplit + k] = f;
      sum = fmaf(f, weight[(RB + r) * nsplit + k], sum);
    }
    sum = warp_sum(sum);
    if (lane == 0) unit_s[r] = sum;
  }
  __syncthreads();
#pragma unroll 1
  for (int i = threadIdx.x; i < rows * HD / 4; i += kKaThreads) {
    const int r = i / (HD / 4), dim = i % (HD / 4) * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int k = 0; k < nsplit; ++k) {
      const float4 x = __ldcg(reinterpret_cast<const float4*>(all + (long long)k * REC + r * HD + dim));
      const float f = weight[r * nsplit + k];
      v[0] = fmaf(f, x.x, v[0]); v[1] = fmaf(f, x.y, v[1]); v[2] = fmaf(f, x.z, v[2]); v[3] = fmaf(f, x.w, v[3]);
    }
    store(r, dim, v, unit_s[r]);
  }
}

// Rows of a CTA for `rows` query rows of a kv head: the fewest that hold them, eight at head size 64 only.  O of eight in two terms
// does not fit the registers at 256, and at 128 takes 300 to 480 bytes of spills: 32 x 8 rows over 2000 .. 4096 keys of four kv
// heads 51.1 us against 47.4 with twice four (fp32 52.6 and 48.4, groups of 128 48.1 and 44.1; five rows 51.0 and 47.2).
constexpr int ka_rows(int hd, long long rows) { return rows <= 2 ? 2 : rows <= 4 || hd >= 128 ? 4 : 8; }

}  // namespace b200lm
