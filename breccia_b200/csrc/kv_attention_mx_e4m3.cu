// One cache recipe's attention kernels (a file each, so that they compile side by side).
#include "kv_attention.cuh"

namespace brc {
namespace kvatt {
int attend_mx_e4m3(const Args& a, int nt, int blocks, cudaStream_t st) {
  return by_shape<BRC_STE_MXFP8, BRC_FP8_E4M3>(a, nt, blocks, st);
}
}  // namespace kvatt
}  // namespace brc
