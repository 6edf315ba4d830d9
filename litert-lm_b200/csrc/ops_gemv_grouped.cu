// Entry points of the grouped int4 matrix-vector product (include/b200lm_ops.h).
#include "../../include/b200lm_ops.h"
#include "gemv_grouped.cuh"
#include "op_host.h"

#include <algorithm>

namespace b200lm {

static void check_grouped(int64_t n, int64_t k, int32_t group) {
  B2_CHECK(n > 0 && n <= (1ll << 30) && k > 0 && k <= (1ll << 30) && k % 2 == 0, kInvalidArgument, "n, k: positive, at most 2^30, k even");
  B2_CHECK(group == 32 || group == 64 || group == 128, kUnimplemented, "group must be 32, 64 or 128");
}
static int64_t grouped_block(int group, bool off) { return 1024 + 32 * (128 / group) * (off ? 2 : 1); }
static int64_t grouped_bytes(int64_t n, int64_t k, int group, bool off) { return (n + 15) / 16 * ((k + 127) / 128) * grouped_block(group, off); }

// Runs of strips, clusters and warps a strip: the fewest blocks for the longest warp, where cutting x into digits counts 1/8 of a
// block for each column and block of a CTA, and a cluster's meeting as many blocks as it has CTAs.
template <typename S>
static size_t plan_gg(GgArgs& a, int sms) {
  long long best = -1;
  const int room = 40 << 10;                                // bytes of sums in a CTA
  for (int cs = 1; cs <= 8; cs *= 2)
    for (int kw = 1; kw <= 8; kw *= 2) {
      const int own = (a.blocks + cs - 1) / cs, rs = kGgWarps / kw;
      if (cs > a.blocks || kw > a.blocks / cs) continue;       // every warp has a block
      // clusters that are on the GPU at once: those of four and eight do not fill every GPC (73 of four took two rounds, 68 one)
      const int slots = cs <= 2 ? 2 * sms / cs : cs == 4 ? sms * 46 / 100 : sms * 22 / 100;
      int run = (a.strips + slots - 1) / slots;
      run = std::min(run, room / (64 * a.ncols * kw));
      if (kw > 1 && run > rs) continue;                     // shares of k are for runs shorter than the warps
      const long long waves = ((a.strips + run - 1) / run + slots - 1) / slots;
      const long long cost = waves * (8ll * ((run + rs - 1) / rs) * ((own + kw - 1) / kw) + (long long)own * a.ncols + (cs > 1 ? 8 * cs : 0));
      if (best >= 0 && cost >= best) continue;
      best = cost;
      a.cs = cs;
      a.kw = kw;
      a.run = run;
      a.chunk = std::min(own, S::kChunk);
    }
  return (size_t)a.chunk * S::kPerBlock + gg_out_bytes(a.run, a.ncols, a.kw);
}

template <int GROUP, bool OFF, int MM>
static void launch_gg(cudaStream_t st, GgArgs a, int sms) {
  using S = GgShape<GROUP, OFF, MM>;
  const size_t smem = plan_gg<S>(a, sms);
  raise_dyn_smem(gemv_grouped_kernel<GROUP, OFF, MM>, (size_t)S::kChunk * S::kPerBlock + (40 << 10));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.strips + a.run - 1) / a.run * a.cs));
  cfg.blockDim = dim3(kGgThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)a.cs;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = a.cs > 1 ? 2 : 1;
  B2_CUDA(cudaLaunchKernelEx(&cfg, gemv_grouped_kernel<GROUP, OFF, MM>, (const GgArgs)a));
}

template <int GROUP, bool OFF>
static void launch_gg_cols(cudaStream_t st, const GgArgs& a, int sms) {
  if (a.ncols <= 2) launch_gg<GROUP, OFF, 1>(st, a, sms);
  else if (a.ncols <= 4) launch_gg<GROUP, OFF, 2>(st, a, sms);
  else if (a.x_type == kF32) launch_gg<GROUP, OFF, 4>(st, a, sms);
  else launch_gg<GROUP, OFF, 3>(st, a, sms);
}

}  // namespace b200lm

using namespace b200lm;

extern "C" int B200LmOps_GemvW4GroupedBytes(int64_t n, int64_t k, int32_t group, int32_t has_offset, int64_t* bytes, char** err) {
  OP_TRY
  B2_CHECK(bytes, kInvalidArgument, "null pointer");
  check_grouped(n, k, group);
  *bytes = grouped_bytes(n, k, group, has_offset != 0);
  OP_END
}

extern "C" int B200LmOps_RepackW4Grouped(const uint8_t* packed, const uint16_t* scale, const uint16_t* offset, int64_t n, int64_t k,
                                         int32_t group, uint8_t* out, char** err) {
  OP_TRY
  B2_CHECK(packed && scale && out, kInvalidArgument, "null pointer");
  check_grouped(n, k, group);
  const int64_t blocks = (k + 127) / 128, bytes = grouped_block(group, offset != nullptr), groups = (k + group - 1) / group;
  const int per = 128 / group;
  memset(out, 0, (size_t)grouped_bytes(n, k, group, offset != nullptr));
  for (int64_t r = 0; r < n; ++r) {
    const int g = (int)(r % 8), high = (int)(r % 16 / 8);
    uint8_t* strip = out + r / 16 * blocks * bytes;
    for (int64_t j = 0; j < k; ++j) {
      const int q = (packed[r * (k / 2) + j / 2] >> (4 * (j % 2))) & 15, c = (int)(j % 64);
      uint8_t* tile = strip + j / 128 * bytes + j % 128 / 64 * 512;
      tile[(4 * g + c % 16 / 4) * 16 + (2 * (c / 32) + c % 32 / 16) * 4 + c % 4] |= (uint8_t)(q << (4 * high));
    }
    for (int64_t j = 0; j < groups; ++j) {
      uint8_t* at = strip + j / per * bytes + 1024 + ((g * per + j % per) * 2 + high) * 2;
      memcpy(at, scale + r * groups + j, 2);
      if (offset) memcpy(at + 32 * per, offset + r * groups + j, 2);
    }
  }
  OP_END
}

extern "C" int B200LmOps_GemvW4Grouped(int32_t device, const void* w_dev, int32_t scale_type, int32_t has_offset, int64_t n, int64_t k,
                                       int32_t group, const void* x_dev, int32_t x_type, int64_t ldx, int32_t ncols, void* y_dev,
                                       int32_t y_type, int64_t ldy, void* stream, char** err) {
  OP_TRY
  B2_CHECK(w_dev && x_dev && y_dev, kInvalidArgument, "null pointer");
  check_grouped(n, k, group);
  B2_CHECK(scale_type == kBf16 || scale_type == kF16, kInvalidArgument, "scale_type must be B200LM_BF16 or B200LM_F16");
  B2_CHECK(x_type >= kF32 && x_type <= kF16 && y_type >= kF32 && y_type <= kF16, kInvalidArgument, "unknown element type");
  B2_CHECK(ncols >= 1 && ncols <= 8, kInvalidArgument, "ncols must be 1 .. 8");
  B2_CHECK(ncols == 1 || (ldx >= k && ldy >= n), kInvalidArgument, "a row stride is shorter than its row");
  B2_CHECK((uintptr_t)w_dev % 16 == 0, kInvalidArgument, "w_dev must lie on a 16-byte boundary");
  B2_CHECK((uintptr_t)x_dev % elem_size(x_type) == 0 && (uintptr_t)y_dev % elem_size(y_type) == 0, kInvalidArgument, "x_dev or y_dev is misaligned");
  B2_CHECK((n + 15) / 16 * 8 <= 0x7FFFFFFF, kInvalidArgument, "too many rows");
  require_device(device);
  DeviceScope scope(device);
  GgArgs a{};
  a.w = reinterpret_cast<const uint8_t*>(w_dev);
  a.n = (int)n;
  a.ncols = ncols;
  a.strips = (int)((n + 15) / 16);
  a.blocks = (int)((k + 127) / 128);
  a.k = k;
  a.x = x_dev;
  a.ldx = ldx;
  a.y = y_dev;
  a.ldy = ldy;
  a.x_type = x_type;
  a.y_type = y_type;
  a.scale_bf16 = scale_type == kBf16;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int sms = device_sms(device);
  if (group == 32) has_offset ? launch_gg_cols<32, true>(st, a, sms) : launch_gg_cols<32, false>(st, a, sms);
  else if (group == 64) has_offset ? launch_gg_cols<64, true>(st, a, sms) : launch_gg_cols<64, false>(st, a, sms);
  else has_offset ? launch_gg_cols<128, true>(st, a, sms) : launch_gg_cols<128, false>(st, a, sms);
  OP_END
}
