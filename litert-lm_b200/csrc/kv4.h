// Layout of the cache in 4 bits (include/b200lm_ops.h), in one place for host and device.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define B2_KV4_FN __host__ __device__ __forceinline__ constexpr
#else
#define B2_KV4_FN inline constexpr
#endif

namespace b200lm {

constexpr int kKv4Page = 256;                              // positions of a page

// One kv head of one page: K codes, K scales, V codes, V scales.
struct Kv4Dims {
  int hd, group;
  B2_KV4_FN int plane() const { return hd < 128 ? hd : 128; }              // elements of a plane
  B2_KV4_FN int row() const { return plane() / 2; }                        // bytes of a plane's row
  B2_KV4_FN int groups() const { return hd / group; }
  B2_KV4_FN int codes() const { return kKv4Page * hd / 2; }                // bytes
  B2_KV4_FN int scales() const { return kKv4Page * 4 * groups(); }
  B2_KV4_FN int k_codes() const { return 0; }
  B2_KV4_FN int k_scales() const { return codes(); }
  B2_KV4_FN int v_codes() const { return codes() + scales(); }
  B2_KV4_FN int v_scales() const { return 2 * codes() + scales(); }
  B2_KV4_FN int head_bytes() const { return 2 * (codes() + scales()); }
  // Byte of element e of position `slot`, within the codes; the nibble is high for the second of the two that share it.
  B2_KV4_FN int k_byte(int slot, int e) const {
    const int d = e % plane();
    return ((e / plane()) * kKv4Page + slot) * row() + d % 16 / 4 * (row() / 4) + d / 32 * 4 + d % 4;
  }
  B2_KV4_FN bool k_high(int e) const { return e % 32 >= 16; }
  // unit of a V row: 8 units of row / 8 bytes, exchanged with those four further at half of the positions (attention reads
  // positions t, t + 4, ... in the lanes of one t: without the exchange those of t and t + 2 meet in the same banks)
  B2_KV4_FN int v_unit(int slot, int g) const { return plane() == 128 ? g ^ (4 * (slot >> 1 & 1)) : g; }
  B2_KV4_FN int v_byte(int slot, int e) const {
    const int d = e % plane();
    return ((e / plane()) * kKv4Page + slot) * row() + v_unit(slot, d % 8) * (row() / 8) + d / 16;
  }
  B2_KV4_FN bool v_high(int e) const { return e % 16 >= 8; }
};

}  // namespace b200lm
