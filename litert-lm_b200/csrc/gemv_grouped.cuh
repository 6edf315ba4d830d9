// int4 matrix-vector products with a scale (and maybe an offset) for each row and group of k, one to eight columns.
//
//   y[c][r] = sum_g s[r][g] sum_{k in g} q[r][k] x[c][k]  +  o[r][g] sum_{k in g} x[c][k]
//
// What has to move is the weights' image, read once (n k / 2 bytes and the scales); the products themselves are small.  So
// the codes go from global memory into the A operand of mma.sync (m16n8k32, int8) with three logic instructions for eight
// of them, and the precision lies in the other operand: x is cut, for each column and block of 128 k, into four digits of
// seven bits, x = 2^e (t0 + t1 / 2^7 + t2 / 2^14 + t3 / 2^21) with |t| <= 64, exact to 2^-28 of the block's largest value.
// The eight columns of a product are four digits of two columns of x; its integer sums are exact.  They enter fp32 once a
// group: an accumulator that starts at the bits of 1.5 * 2^23 is read as a float and 1.5 * 2^23 taken off (|sum| <=
// 128 * 64 * 128 < 2^22, so nothing is rounded).
//
// A CTA has eight warps: RS strips of 16 rows times 8 / RS shares of its blocks of k.  Where the strips are fewer than the
// GPU needs, a cluster of CTAs shares the blocks of the same strips and adds up through distributed shared memory: no
// workspace, and a fixed order of sums.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"
#include "decode_ops.cuh"

namespace b200lm {

enum ElemType : int { kF32 = 0, kBf16 = 1, kF16 = 2 };
__host__ __device__ inline int elem_size(int type) { return type == kF32 ? 4 : 2; }

struct GgArgs {
  const uint8_t* w;
  int n, ncols, strips, blocks;
  long long k;
  const void* x;
  long long ldx;
  void* y;
  long long ldy;
  int x_type, y_type, scale_bf16;
  int rs, cs, chunk;            // strips of a CTA, CTAs of a cluster, blocks of k whose digits are held at once
};

constexpr int kGgThreads = 256;
constexpr int kGgMagic = 0x4B400000;                       // 1.5 * 2^23

template <int GROUP, bool OFF, int NB>
struct GgShape {
  static constexpr int kGroups = 128 / GROUP;              // of a block
  static constexpr int kBlock = 1024 + 32 * kGroups * (OFF ? 2 : 1);
  static constexpr int kAhead = NB == 4 ? 2 : 4;           // blocks of a warp on their way
  static constexpr int kCols = 2 * NB;
  // shared memory of a chunk's block: digits, the columns' powers of two, their group sums
  static constexpr int kPerBlock = NB * 1024 + kCols * 4 + (OFF ? kCols * kGroups * 4 : 0);
  static constexpr int kRed = 8 * kCols * 16 * 4;
  static size_t smem(int chunk) { return (size_t)chunk * kPerBlock + kRed; }
};

__device__ __forceinline__ float gg_load1(const void* p, long long i, int type) {
  if (type == kF32) return reinterpret_cast<const float*>(p)[i];
  if (type == kBf16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(reinterpret_cast<const __half*>(p)[i]);
}
// Elements [i, i + 4) of a row that ends at `end`; zeros behind it.
__device__ __forceinline__ float4 gg_load4(const void* p, long long i, long long end, int type) {
  const char* a = reinterpret_cast<const char*>(p) + i * elem_size(type);
  if (i + 4 <= end && (reinterpret_cast<uintptr_t>(a) & (4 * elem_size(type) - 1)) == 0) {
    if (type == kF32) return *reinterpret_cast<const float4*>(a);
    const uint2 u = *reinterpret_cast<const uint2*>(a);
    if (type == kBf16) return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xFFFF0000u));
    const float2 l = __half22float2(*reinterpret_cast<const __half2*>(&u.x)), h = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
    return make_float4(l.x, l.y, h.x, h.y);
  }
  float4 v;
  v.x = i < end ? gg_load1(p, i, type) : 0.f;
  v.y = i + 1 < end ? gg_load1(p, i + 1, type) : 0.f;
  v.z = i + 2 < end ? gg_load1(p, i + 2, type) : 0.f;
  v.w = i + 3 < end ? gg_load1(p, i + 3, type) : 0.f;
  return v;
}
__device__ __forceinline__ void gg_store1(void* p, long long i, int type, float v) {
  if (type == kF32) reinterpret_cast<float*>(p)[i] = v;
  else if (type == kBf16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16(v);
  else reinterpret_cast<__half*>(p)[i] = __float2half(v);
}

// This lane's part of one block: 16 bytes of each tile, and the scales (and offsets) of its two rows, a word a group.
template <int GROUP, bool OFF>
struct GgBlock {
  static constexpr int G = 128 / GROUP;
  uint4 a, b;
  uint32_t s[G], o[OFF ? G : 1];
  __device__ __forceinline__ static void words(const uint8_t* p, uint32_t (&d)[G]) {
    if constexpr (G == 4) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
      d[0] = v.x; d[1] = v.y; d[2] = v.z; d[3] = v.w;
    } else if constexpr (G == 2) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
      d[0] = v.x; d[1] = v.y;
    } else {
      d[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    }
  }
  __device__ __forceinline__ void load(const uint8_t* p, int lane) {
    a = ldg_nc_v4(reinterpret_cast<const uint4*>(p) + lane);
    b = ldg_nc_v4(reinterpret_cast<const uint4*>(p + 512) + lane);
    words(p + 1024 + (lane >> 2) * 4 * G, s);
    if constexpr (OFF) words(p + 1024 + 32 * G + (lane >> 2) * 4 * G, o);
  }
};

__device__ __forceinline__ float2 gg_pair(uint32_t u, bool bf16) {
  if (bf16) return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}

template <int GROUP, bool OFF, int NB>
__global__ void __launch_bounds__(kGgThreads) gemv_grouped_kernel(const GgArgs a) {
  using S = GgShape<GROUP, OFF, NB>;
  constexpr int G = S::kGroups, AH = S::kAhead;
  extern __shared__ __align__(16) unsigned char gg_sm[];
  uint32_t* digits = reinterpret_cast<uint32_t*>(gg_sm);                                       // [block][tile][nb][lane][4]
  float* unit = reinterpret_cast<float*>(gg_sm + (size_t)a.chunk * NB * 1024);                 // [block][col]
  float* sums = unit + a.chunk * S::kCols;                                                     // [block][col][group]
  float* red = reinterpret_cast<float*>(gg_sm + (size_t)a.chunk * S::kPerBlock);               // [warp][col][16]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = lane & 3;
  const int rank = blockIdx.x % a.cs, tile = blockIdx.x / a.cs;
  const int kw = 8 / a.rs, ks = warp / a.rs;
  const int strip = tile * a.rs + warp % a.rs;
  const int b0 = (int)((long long)a.blocks * rank / a.cs), b1 = (int)((long long)a.blocks * (rank + 1) / a.cs);
  const int last = strip < a.strips ? b1 : b0;                                                 // a warp without a strip has no blocks
  const uint8_t* w = a.w + (long long)strip * a.blocks * S::kBlock;
  pdl_wait();
  pdl_launch_dependents();

  GgBlock<GROUP, OFF> ahead[AH];
#pragma unroll
  for (int i = 0; i < AH; ++i)
    if (b0 + ks + i * kw < last) ahead[i].load(w + (long long)(b0 + ks + i * kw) * S::kBlock, lane);

  float acc[NB][2];
#pragma unroll
  for (int i = 0; i < NB; ++i) acc[i][0] = acc[i][1] = 0.f;

#pragma unroll 1
  for (int c0 = b0; c0 < b1; c0 += a.chunk) {
    const int c1 = min(c0 + a.chunk, b1);
    if (c0 > b0) __syncthreads();                          // the chunk before has been read
#pragma unroll 1
    for (int item = warp; item < (c1 - c0) * a.ncols; item += 8) {
      const int blk = item / a.ncols, c = item % a.ncols;
      const long long k = (long long)(c0 + blk) * 128 + 4 * lane;
      const float4 x = gg_load4(a.x, c * a.ldx + k, c * a.ldx + a.k, a.x_type);
      const float top = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
      const bool odd = !isfinite(x.x) || !isfinite(x.y) || !isfinite(x.z) || !isfinite(x.w);
      const uint32_t bits = __reduce_max_sync(0xffffffffu, odd ? 0x7F800000u : __float_as_uint(top));
      // 2^5 <= largest |x| f < 2^6; the power stays inside fp32 for the smallest and largest x
      const int e = max((int)(bits >> 23), 30);
      const float f = __uint_as_float((uint32_t)(254 + 5 - e) << 23);
      float r[4] = {x.x * f, x.y * f, x.z * f, x.w * f};
      if (bits >= 0x7F800000u) r[0] = r[1] = r[2] = r[3] = 0.f;
      uint32_t* d = digits + ((blk * 2 + (lane >> 4)) * NB + (c >> 1)) * 128 + ((c & 1) * 16 + t) * 4 + ((lane >> 2) & 3);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t word = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float q = rintf(r[j]);
          word |= ((uint32_t)(int)q & 0xFFu) << (8 * j);
          r[j] = (r[j] - q) * 128.f;
        }
        d[i * 16] = word;
      }
      if (lane == 0) unit[blk * S::kCols + c] = bits >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : __uint_as_float((uint32_t)(e - 9) << 23);      // 1/16 of the digits' unit: codes enter as 16 q
      if constexpr (OFF) {
        float sum = (x.x + x.y) + (x.z + x.w);
#pragma unroll
        for (int o = 1; o < GROUP / 4; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane % (GROUP / 4) == 0) sums[(blk * S::kCols + c) * G + lane / (GROUP / 4)] = sum;
      }
    }
    __syncthreads();
    const int end = min(c1, last);
#pragma unroll 1
    for (int base = c0 + ks; base < end; base += AH * kw) {
#pragma unroll
      for (int i = 0; i < AH; ++i) {
        const int b = base + i * kw;
        if (b >= end) break;
        const int at = b - c0;
        const GgBlock<GROUP, OFF>& q = ahead[i];
        constexpr uint32_t m = 0xF0F0F0F0u;
        uint4 x[2][NB];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) x[h][nb] = *reinterpret_cast<const uint4*>(digits + ((at * 2 + h) * NB + nb) * 128 + lane * 4);
        float u[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) u[nb] = unit[at * S::kCols + nb * 2 + (t >> 1)];
        int c[NB][4];
#pragma unroll
        for (int step = 0; step < 4; ++step) {
          const uint4& v = step < 2 ? q.a : q.b;
          const uint32_t lo = step & 1 ? v.z : v.x, hi = step & 1 ? v.w : v.y;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            if (step * 32 % GROUP == 0) c[nb][0] = c[nb][1] = c[nb][2] = c[nb][3] = kGgMagic;
            const uint4& d = x[step >> 1][nb];
            mma_s8s8(c[nb], (lo << 4) & m, lo & m, (hi << 4) & m, hi & m, step & 1 ? d.z : d.x, step & 1 ? d.w : d.y);
          }
          if ((step + 1) * 32 % GROUP == 0) {
            const int grp = step * 32 / GROUP;
            const float2 s = gg_pair(q.s[grp], a.scale_bf16);
            float2 o;
            if constexpr (OFF) o = gg_pair(q.o[grp], a.scale_bf16);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              constexpr float big = 12582912.f;
              const float d0 = __int_as_float(c[nb][0]) - big, d1 = __int_as_float(c[nb][1]) - big;
              const float d2 = __int_as_float(c[nb][2]) - big, d3 = __int_as_float(c[nb][3]) - big;
              acc[nb][0] = fmaf(s.x * u[nb], fmaf(d1, 1.f / 128, d0), acc[nb][0]);
              acc[nb][1] = fmaf(s.y * u[nb], fmaf(d3, 1.f / 128, d2), acc[nb][1]);
              if constexpr (OFF) {
                const float gs = t & 1 ? 0.f : sums[(at * S::kCols + nb * 2 + (t >> 1)) * G + grp];
                acc[nb][0] = fmaf(o.x, gs, acc[nb][0]);
                acc[nb][1] = fmaf(o.y, gs, acc[nb][1]);
              }
            }
          }
        }
        if (b + AH * kw < last) ahead[i].load(w + (long long)(b + AH * kw) * S::kBlock, lane);
      }
    }
  }
  // the two digit pairs of a column sit in neighbouring lanes
  const float f = t & 1 ? 1.f / 16384 : 1.f;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v = acc[nb][h] * f;
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      if (!(t & 1)) red[(warp * S::kCols + nb * 2 + (t >> 1)) * 16 + h * 8 + (lane >> 2)] = v;
    }
  const int rows = a.rs * 16, outs = rows * a.ncols;
  auto share = [&](const float* r, int c, int row) {       // a CTA's sum for column c, row `row` of its strips
    float v = 0.f;
    for (int i = 0; i < kw; ++i) v += r[((i * a.rs + row / 16) * S::kCols + c) * 16 + row % 16];
    return v;
  };
  if (a.cs == 1) {
    __syncthreads();
    for (int i = threadIdx.x; i < outs; i += kGgThreads) {
      const int c = i / rows, row = i % rows;
      if (tile * rows + row < a.n) gg_store1(a.y, c * a.ldy + tile * rows + row, a.y_type, share(red, c, row));
    }
    return;
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  for (int i = rank * kGgThreads + threadIdx.x; i < outs; i += a.cs * kGgThreads) {
    const int c = i / rows, row = i % rows;
    float v = 0.f;
    for (int r = 0; r < a.cs; ++r) {
      uint32_t base;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(base) : "r"((uint32_t)__cvta_generic_to_shared(red)), "r"(r));
      float part = 0.f;
      for (int j = 0; j < kw; ++j) {
        float x;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(base + (uint32_t)(((j * a.rs + row / 16) * S::kCols + c) * 16 + row % 16) * 4) : "memory");
        part += x;
      }
      v += part;
    }
    if (tile * rows + row < a.n) gg_store1(a.y, c * a.ldy + tile * rows + row, a.y_type, v);
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");   // nobody leaves while its sums are read
}

}  // namespace b200lm
