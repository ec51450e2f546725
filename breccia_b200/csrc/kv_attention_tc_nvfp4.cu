// One cache recipe's tcgen05 attention kernels.
#include "kv_attention_tc.cuh"

namespace brc {
namespace kvatt {
int attend_tc_nvfp4(const Args& a, int blocks, cudaStream_t st) {
  return kvtc::launch_tc<BRC_STE_NVFP4, BRC_FP8_E4M3, 128>(a, blocks, st);
}
}  // namespace kvatt
}  // namespace brc
