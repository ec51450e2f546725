// One cache recipe's tcgen05 attention kernels.
#include "kv_attention_tc.cuh"

namespace brc {
namespace kvatt {
int attend_tc_mx_e5m2(const Args& a, int blocks, cudaStream_t st) {
  if (a.c.head_dim == 64) return kvtc::launch_tc<BRC_STE_MXFP8, BRC_FP8_E5M2, 64>(a, blocks, st);
  return kvtc::launch_tc<BRC_STE_MXFP8, BRC_FP8_E5M2, 128>(a, blocks, st);
}
}  // namespace kvatt
}  // namespace brc
