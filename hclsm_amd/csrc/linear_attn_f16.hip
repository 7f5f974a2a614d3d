// Linear attention on float16 inputs.
#include "linear_attn_kernels.h"

namespace hclsm {

int la_launch_f16(const LaArgs& a, int da, bool sum, hipStream_t st) {
  return la_launch<HCLSM_F16>(a, da, sum, st);
}

}  // namespace hclsm
