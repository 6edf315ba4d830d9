// int4 matrix-vector products with a scale (and maybe an offset) for each row and group of k, one to eight columns.
//
//   y[c][r] = sum_g s[r][g] sum_{k in g} q[r][k] x[c][k]  +  o[r][g] sum_{k in g} x[c][k]
//
// What has to move is the weights' image, read once (n k / 2 bytes and the scales); the products themselves are small.  So
// the codes go from global memory into the A operand of mma.sync (m16n8k32, int8) with three logic instructions for eight
// of them, and the precision lies in the other operand: x is cut, for each column and block of 128 k, into digits of seven bits,
// x = 2^e (t0 + t1 / 2^7 + t2 / 2^14 [+ t3 / 2^21]) with |t| <= 64, exact to 2^-20 (three) or 2^-27 (four) of the block's
// largest value.  A product of eight columns takes four digits of two columns of x; five to eight columns of a 16-bit type take
// three products, one a digit (their numbers are exact in three unless they are below 2^-9 of the largest).  The integer
// sums are exact.  They enter fp32 once a group: an accumulator that starts at the bits of 1.5 * 2^23 is read as a float and
// 1.5 * 2^23 taken off (|sum| <= 128 * 64 * 128 < 2^22, so nothing is rounded).
//
// The GPU's CTAs (two an SM) are clusters of `cs` that share the blocks of k and take an equal run of strips (16 rows) each.  A
// CTA cuts its part of x into digits once (done for every strip it cost 17 us of 43008 x 5376 with eight columns), then its warps
// stream strips without meeting, with blocks of weights on their way ahead; sums stay in shared memory and meet once, over
// distributed shared memory: no workspace, a fixed order.  Where a run has fewer strips than warps, kw warps share the blocks
// of a strip.
//
// Measured: 262144 x 1152, groups of 128, two fp32 columns 32.2 us = 4.9 TB/s (76 % of the copy rate), bound by HBM (29.0 us where the
// same 158 MB come again at once, part of them from L2); 20480 x 2560, groups of 64 with offsets, three columns 12.3 us = 2.4 TB/s,
// bound by one chain of latencies (digits, first blocks, the cluster's meeting) and the last round of strips; 1536 x 1152, one column
// 3.4 us, a launch; 43008 x 5376, groups of 64, eight bf16 columns 44.8 us = 2.8 TB/s.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

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
  int kw, cs, chunk, run;       // warps of a strip, CTAs of a cluster, blocks of k whose digits are held at once, strips of a cluster
};

constexpr int kGgThreads = 256, kGgWarps = 8;
constexpr int kGgMagic = 0x4B400000;                       // 1.5 * 2^23

// MM products of a step: 1, 2 and 4 are two columns of four digits each, 3 is eight columns of three digits.
template <int GROUP, bool OFF, int MM>
struct GgShape {
  static constexpr int kGroups = 128 / GROUP;              // of a block
  static constexpr int kBlock = 1024 + 32 * kGroups * (OFF ? 2 : 1);
  static constexpr int kAhead = MM >= 3 ? 2 : 4;           // blocks of a warp on their way
  static constexpr int kCols = MM == 3 ? 8 : 2 * MM;
  // shared memory of a chunk's block: digits, the columns' powers of two, their group sums
  static constexpr int kPerBlock = MM * 1024 + kCols * 4 + (OFF ? kCols * kGroups * 4 : 0);
  static constexpr int kChunk = 64 / MM;                   // most blocks held at once
};
inline size_t gg_out_bytes(int run, int ncols, int kw) { return (size_t)run * kw * ncols * 64; }

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

// 16 bytes that are read once.  Not .nc: a kernel before may have written them while this one was set up behind its edge.
__device__ __forceinline__ uint4 gg_stream(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

// This lane's part of one block: 16 bytes of each tile, and the scales (and offsets) of its two rows, a word a group.
template <int GROUP, bool OFF>
struct GgBlock {
  static constexpr int G = 128 / GROUP;
  uint4 a, b;
  uint32_t s[G], o[OFF ? G : 1];
  __device__ __forceinline__ static void words(const uint8_t* p, uint32_t (&d)[G]) {
    if constexpr (G == 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      d[0] = v.x; d[1] = v.y; d[2] = v.z; d[3] = v.w;
    } else if constexpr (G == 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      d[0] = v.x; d[1] = v.y;
    } else {
      d[0] = *reinterpret_cast<const uint32_t*>(p);
    }
  }
  __device__ __forceinline__ void load(const uint8_t* p, int lane) {
    a = gg_stream(reinterpret_cast<const uint4*>(p) + lane);
    b = gg_stream(reinterpret_cast<const uint4*>(p + 512) + lane);
    words(p + 1024 + (lane >> 2) * 4 * G, s);
    if constexpr (OFF) words(p + 1024 + 32 * G + (lane >> 2) * 4 * G, o);
  }
};

__device__ __forceinline__ void gg_mma(int (&d)[4], const int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
               : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}
__device__ __forceinline__ float2 gg_pair(uint32_t u, bool bf16) {
  if (bf16) return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}

template <int GROUP, bool OFF, int MM>
__global__ void __launch_bounds__(kGgThreads, 2) gemv_grouped_kernel(const GgArgs a) {
  using S = GgShape<GROUP, OFF, MM>;
  constexpr int G = S::kGroups, AH = S::kAhead, LC = MM == 3 ? 2 : MM;        // columns of a lane
  extern __shared__ __align__(16) unsigned char gg_sm[];
  uint32_t* digits = reinterpret_cast<uint32_t*>(gg_sm);                                       // [block][tile][product][lane][4]
  float* unit = reinterpret_cast<float*>(gg_sm + (size_t)a.chunk * MM * 1024);                 // [block][col]
  float* sums = unit + a.chunk * S::kCols;                                                     // [block][col][group]
  float* out = reinterpret_cast<float*>(gg_sm + (size_t)a.chunk * S::kPerBlock);               // [share of k][strip][col][16]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = lane & 3;
  const int rank = blockIdx.x % a.cs, first = blockIdx.x / a.cs * a.run, strips = min(a.run, a.strips - first);
  const int rs = kGgWarps / a.kw, ks = warp / rs;                                              // strips at a time, this warp's share
  const int b0 = (int)((long long)a.blocks * rank / a.cs), b1 = (int)((long long)a.blocks * (rank + 1) / a.cs);
  // the first weights into L2 while the kernel before ends (L2 is where it would write them, so nothing stale can come of it)
  if (warp % rs < strips && lane * 128 < min(b1 - b0, AH) * S::kBlock) {
    const uint8_t* p = a.w + ((long long)(first + warp % rs) * a.blocks + b0) * S::kBlock + lane * 128;
    asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
  }
  pdl_wait();
  pdl_launch_dependents();

#pragma unroll 1
  for (int c0 = b0; c0 < b1; c0 += a.chunk) {
    const int c1 = min(c0 + a.chunk, b1);
    // this warp's blocks: of strip warp % rs, warp % rs + rs, ... those from c0 + ks on in steps of kw
    int strip_in = warp % rs, block_in = c0 + ks;
    GgBlock<GROUP, OFF> ahead[AH];
    auto load = [&](GgBlock<GROUP, OFF>& q) {
      if (strip_in < strips && block_in < c1) {
        q.load(a.w + ((long long)(first + strip_in) * a.blocks + block_in) * S::kBlock, lane);
        block_in += a.kw;
        if (block_in >= c1) {
          block_in = c0 + ks;
          strip_in += rs;
        }
      }
    };
#pragma unroll
    for (int i = 0; i < AH; ++i) load(ahead[i]);
    if (c0 > b0) __syncthreads();                          // the chunk before has been read
#pragma unroll 1
    for (int item = warp; item < (c1 - c0) * a.ncols; item += kGgWarps) {
      const int blk = item / a.ncols, c = item % a.ncols;
      const long long k = (long long)(c0 + blk) * 128 + 4 * lane;
      const float4 x = gg_load4(a.x, c * a.ldx + k, c * a.ldx + a.k, a.x_type);
      const float top = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
      const bool odd = !isfinite(x.x) || !isfinite(x.y) || !isfinite(x.z) || !isfinite(x.w);
      const uint32_t bits = __reduce_max_sync(0xffffffffu, odd ? 0x7F800000u : __float_as_uint(top));
      // 2^5 <= largest |x| f < 2^6, for the smallest x (below 2^-117) less; f and the digits' unit below are normal numbers
      const int e = max((int)(bits >> 23), 10);
      const float f = __uint_as_float((uint32_t)(254 + 5 - e) << 23);
      float r[4] = {x.x * f, x.y * f, x.z * f, x.w * f};
      if (bits >= 0x7F800000u) r[0] = r[1] = r[2] = r[3] = 0.f;
      constexpr int ND = MM == 3 ? 3 : 4;
      uint32_t* d = digits + ((blk * 2 + (lane >> 4)) * MM + (MM == 3 ? 0 : c >> 1)) * 128 + ((MM == 3 ? 4 * c : (c & 1) * 16) + t) * 4 + ((lane >> 2) & 3);
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        uint32_t b[4];                                     // rint(r) in the lowest byte of r + 1.5 * 2^23
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float q = r[j] + 12582912.f;
          b[j] = __float_as_uint(q);
          r[j] = (r[j] - (q - 12582912.f)) * 128.f;
        }
        d[i * (MM == 3 ? 128 : 16)] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
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
    const int magic[4] = {kGgMagic, kGgMagic, kGgMagic, kGgMagic};
    // strips and blocks as one sequence, a slot of the ring behind the other
    const int mine = strips > warp % rs ? (strips - warp % rs + rs - 1) / rs : 0, each = c1 - c0 > ks ? (c1 - c0 - ks + a.kw - 1) / a.kw : 0, total = mine * each;
    int s = warp % rs, b = c0 + ks;
    float acc[LC][2];
#pragma unroll
    for (int i = 0; i < LC; ++i) acc[i][0] = acc[i][1] = 0.f;
#pragma unroll 1
    for (int it = 0; it < total; it += AH) {
#pragma unroll
      for (int slot = 0; slot < AH; ++slot) {
        if (it + slot >= total) break;
        const GgBlock<GROUP, OFF>& q = ahead[slot];
        const int at = b - c0;
        constexpr uint32_t m = 0xF0F0F0F0u;
        float part[LC][2];                                 // in units of the column's power of two
#pragma unroll
        for (int i = 0; i < LC; ++i) part[i][0] = part[i][1] = 0.f;
        float off[LC][2];
        if constexpr (OFF) {
#pragma unroll
          for (int i = 0; i < LC; ++i) off[i][0] = off[i][1] = 0.f;
        }
        int c[MM][4];
#pragma unroll
        for (int step = 0; step < 4; ++step) {
          const uint4& v = step < 2 ? q.a : q.b;
          const uint32_t lo = step & 1 ? v.z : v.x, hi = step & 1 ? v.w : v.y;
          const uint32_t a0 = (lo << 4) & m, a1 = lo & m, a2 = (hi << 4) & m, a3 = hi & m;
#pragma unroll
          for (int p = 0; p < MM; ++p) {
            const uint2 d = *reinterpret_cast<const uint2*>(digits + ((at * 2 + (step >> 1)) * MM + p) * 128 + lane * 4 + (step & 1) * 2);
            if (step * 32 % GROUP == 0) gg_mma(c[p], magic, a0, a1, a2, a3, d.x, d.y);
            else gg_mma(c[p], c[p], a0, a1, a2, a3, d.x, d.y);
          }
          if ((step + 1) * 32 % GROUP == 0) {
            const int grp = step * 32 / GROUP;
            const float2 sc = gg_pair(q.s[grp], a.scale_bf16);
            constexpr float big = 12582912.f, two = big + big / 128, three = two + big / 16384;
            if constexpr (MM == 3) {
#pragma unroll
              for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const int x = 2 * h + i;
                  const float v0 = fmaf(__int_as_float(c[1][x]), 1.f / 128, __int_as_float(c[0][x]) - three);
                  part[i][h] = fmaf(h ? sc.y : sc.x, fmaf(__int_as_float(c[2][x]), 1.f / 16384, v0), part[i][h]);
                }
            } else {
#pragma unroll
              for (int p = 0; p < MM; ++p)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                  part[p][h] = fmaf(h ? sc.y : sc.x, fmaf(__int_as_float(c[p][2 * h + 1]), 1.f / 128, __int_as_float(c[p][2 * h]) - two), part[p][h]);
            }
            if constexpr (OFF) {
              const float2 of = gg_pair(q.o[grp], a.scale_bf16);
#pragma unroll
              for (int i = 0; i < LC; ++i) {
                const float gs = sums[(at * S::kCols + (MM == 3 ? 2 * t + i : 2 * i + (t >> 1))) * G + grp];
                off[i][0] = fmaf(of.x, gs, off[i][0]);
                off[i][1] = fmaf(of.y, gs, off[i][1]);
              }
            }
          }
        }
#pragma unroll
        for (int i = 0; i < LC; ++i) {
          const float u = unit[at * S::kCols + (MM == 3 ? 2 * t + i : 2 * i + (t >> 1))];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            acc[i][h] = fmaf(u, part[i][h], acc[i][h]);
            if constexpr (OFF) {
              if (MM == 3 || !(t & 1)) acc[i][h] += off[i][h];       // the other lane of a column has its lower digits only
            }
          }
        }
        load(ahead[slot]);
        b += a.kw;
        if (b < c1) continue;
        // the strip's sums: rows g and g + 8
        float* o = out + (size_t)(ks * a.run + s) * a.ncols * 16 + (lane >> 2);
#pragma unroll
        for (int i = 0; i < LC; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float v = acc[i][h];
            int col = 2 * t + i;
            if constexpr (MM != 3) {                       // the two digit pairs of a column sit in neighbouring lanes
              v = t & 1 ? v * (1.f / 16384) : v;
              v += __shfl_xor_sync(0xffffffffu, v, 1);
              col = t & 1 ? a.ncols : 2 * i + (t >> 1);
            }
            if (col < a.ncols) {
              float* at2 = o + col * 16 + 8 * h;
              *at2 = c0 > b0 ? *at2 + v : v;
            }
            acc[i][h] = 0.f;
          }
        b = c0 + ks;
        s += rs;
      }
    }
  }
  const int outs = strips * a.ncols * 16;
  auto store = [&](int i, float v) {
    const int row = (first + i / (16 * a.ncols)) * 16 + i % 16, c = i / 16 % a.ncols;
    if (row < a.n) gg_store1(a.y, c * a.ldy + row, a.y_type, v);
  };
  if (a.cs == 1) {
    __syncthreads();
    for (int i = threadIdx.x; i < outs; i += kGgThreads) {
      float v = out[i];
      for (int j = 1; j < a.kw; ++j) v += out[j * a.run * a.ncols * 16 + i];
      store(i, v);
    }
    return;
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  for (int i = rank * kGgThreads + threadIdx.x; i < outs; i += a.cs * kGgThreads) {
    float v = 0.f;
    for (int r = 0; r < a.cs; ++r) {
      uint32_t base;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(base) : "r"((uint32_t)__cvta_generic_to_shared(out + i)), "r"(r));
      for (int j = 0; j < a.kw; ++j) {
        float x;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(base + (uint32_t)(j * a.run * a.ncols) * 64) : "memory");
        v += x;
      }
    }
    store(i, v);
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");   // nobody leaves while its sums are read
}

}  // namespace b200lm
