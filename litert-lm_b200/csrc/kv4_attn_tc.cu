// Instantiations of the attention of chunks over the 4-bit cache.
#include "kv4_attn_tc.cuh"

namespace b200lm {

template <int HD, int GROUP>
static void launch_kv4_chunk_as(cudaStream_t st, const Kv4AttnArgs& a) {
  raise_dyn_smem(kv4_chunk_kernel<HD, GROUP>, KcShape<HD>::kSmem);
  launch_pdl(kv4_chunk_kernel<HD, GROUP>, dim3((unsigned)(a.row_tiles * a.splits * a.kv.hkv), (unsigned)a.kv.batch), dim3(KcShape<HD>::kThreads), KcShape<HD>::kSmem, st, a);
}

void launch_kv4_chunk(cudaStream_t st, const Kv4AttnArgs& a) {
  if (a.kv.d.hd == 256) a.kv.d.group == 64 ? launch_kv4_chunk_as<256, 64>(st, a) : launch_kv4_chunk_as<256, 128>(st, a);
  else a.kv.d.group == 64 ? launch_kv4_chunk_as<128, 64>(st, a) : launch_kv4_chunk_as<128, 128>(st, a);
}

}  // namespace b200lm
