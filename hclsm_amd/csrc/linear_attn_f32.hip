// Linear attention on float32 inputs.
#include "linear_attn_kernels.h"

namespace hclsm {

int la_launch_f32(const LaArgs& a, int da, int xt, bool sum, hipStream_t st) {
  return la_launch<HCLSM_F32>(a, da, xt, sum, st);
}

}  // namespace hclsm
