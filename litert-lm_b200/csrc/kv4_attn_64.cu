// Instantiations of the attention over the 4-bit cache at head size 64.
#include "kv4_attn_launch.cuh"

namespace b200lm {
void launch_kv4_attn_64(cudaStream_t st, const Kv4AttnArgs& a, int rb) { launch_kv4_attn<64>(st, a, rb); }
}  // namespace b200lm
