// Linear attention on bfloat16 inputs.
#include "linear_attn_kernels.h"

namespace hclsm {

int la_launch_bf16(const LaArgs& a, int da, bool sum, hipStream_t st) {
  return la_launch<HCLSM_BF16>(a, da, sum, st);
}

}  // namespace hclsm
