// Linear attention on float32 inputs.
#include "linear_attn_kernels.h"

namespace hclsm {

int la_launch_f32(const LaArgs& a, int da, bool sum, hipStream_t st) {
  return la_launch<HCLSM_F32>(a, da, sum, st);
}

}  // namespace hclsm
