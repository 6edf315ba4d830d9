// The layout of the 4-bit cache: every element of K and of V has a nibble of its own inside its part of the head's bytes, the
// parts do not overlap, and the byte is where the header's formula has it.
#include "kv4.h"

#include <cstdio>
#include <cstdlib>
#include <vector>

using b200lm::Kv4Dims;

static void require(bool ok, const char* what) {
  if (!ok) { std::fprintf(stderr, "%s\n", what); std::exit(1); }
}

int main() {
  const int dims[][2] = {{64, 64}, {128, 64}, {128, 128}, {256, 64}, {256, 128}};
  for (const auto& x : dims) {
    const Kv4Dims d{x[0], x[1]};
    require(d.k_codes() == 0 && d.k_scales() == d.codes() && d.v_codes() == d.codes() + d.scales() && d.v_scales() == d.v_codes() + d.codes() &&
                d.head_bytes() == d.v_scales() + d.scales() && d.head_bytes() == 512 * (d.hd / 2 + 4 * d.hd / d.group) && d.head_bytes() % 16 == 0, "parts");
    for (int is_v = 0; is_v < 2; ++is_v) {
      std::vector<int> used(2 * d.codes(), 0);
      for (int slot = 0; slot < 256; ++slot)
        for (int e = 0; e < d.hd; ++e) {
          const int byte = is_v ? d.v_byte(slot, e) : d.k_byte(slot, e), high = is_v ? d.v_high(e) : d.k_high(e);
          require(byte >= 0 && byte < d.codes(), "outside");
          require(used[2 * byte + high]++ == 0, "taken twice");
          const int plane = d.hd < 128 ? d.hd : 128, row = plane / 2, in = e % plane;
          int at = (e / plane * 256 + slot) * row;
          if (!is_v) {
            const int j = in / 32, rest = in % 16, t = rest / 4, i = rest % 4;
            at += row / 4 * t + 4 * j + i;
            require(high == (in % 32 >= 16), "K nibble");
          } else {
            int unit = in % 8;
            if (plane == 128 && (slot & 2)) unit = (unit + 4) % 8;
            at += row / 8 * unit + in / 16;
            require(high == (in % 16 >= 8), "V nibble");
          }
          require(byte == at, "formula");
        }
    }
  }
  return 0;
}
