// Launch of the attention over the 4-bit cache for one head size.
#pragma once
#include "kv4_attn.cuh"

namespace b200lm {

template <int HD, int GROUP, int RB, bool EXACT>
void launch_kv4_attn_as(cudaStream_t st, const Kv4AttnArgs& a) {
  using S = KaShape<HD, GROUP, RB>;
  raise_dyn_smem(kv4_attn_kernel<HD, GROUP, RB, EXACT>, S::kSmem);
  launch_pdl(kv4_attn_kernel<HD, GROUP, RB, EXACT>, dim3((unsigned)(a.row_tiles * a.splits * a.kv.hkv), (unsigned)a.kv.batch), dim3(kKaThreads), S::kSmem, st, a);
}

template <int HD, int GROUP, int RB>
void launch_kv4_attn_terms(cudaStream_t st, const Kv4AttnArgs& a) {
  if (a.q_type == kF32) launch_kv4_attn_as<HD, GROUP, RB, true>(st, a);
  else launch_kv4_attn_as<HD, GROUP, RB, false>(st, a);
}

template <int HD, int GROUP>
void launch_kv4_attn_rows(cudaStream_t st, const Kv4AttnArgs& a, int rb) {
  if (rb == 2) launch_kv4_attn_terms<HD, GROUP, 2>(st, a);
  else if (rb == 4) launch_kv4_attn_terms<HD, GROUP, 4>(st, a);
  else if constexpr (HD < 128) launch_kv4_attn_terms<HD, GROUP, 8>(st, a);
}

template <int HD>
void launch_kv4_attn(cudaStream_t st, const Kv4AttnArgs& a, int rb) {
  if constexpr (HD >= 128) {
    if (a.kv.d.group == 128) return launch_kv4_attn_rows<HD, 128>(st, a, rb);
  }
  launch_kv4_attn_rows<HD, 64>(st, a, rb);
}

}  // namespace b200lm
