// Cross attention on f32 operands.
#include "cross_attn_kernels.h"

namespace hclsm {

int ca_forward_f32(CaArgs a, int64_t batch, void* ws, int64_t ws_bytes, hipStream_t st) {
  return ca_forward_dt<HCLSM_F32>(a, batch, ws, ws_bytes, st);
}
int ca_backward_f32(CaArgs a, int64_t batch, void* ws, int64_t ws_bytes, hipStream_t st) {
  return ca_backward_dt<HCLSM_F32>(a, batch, ws, ws_bytes, st);
}

}  // namespace hclsm
