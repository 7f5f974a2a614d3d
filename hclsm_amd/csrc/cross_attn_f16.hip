// Cross attention on f16 operands.
#include "cross_attn_kernels.h"

namespace hclsm {

int ca_forward_f16(CaArgs a, int64_t batch, void* ws, int64_t ws_bytes, hipStream_t st) {
  return ca_forward_dt<HCLSM_F16>(a, batch, ws, ws_bytes, st);
}
int ca_backward_f16(CaArgs a, int64_t batch, void* ws, int64_t ws_bytes, hipStream_t st) {
  return ca_backward_dt<HCLSM_F16>(a, batch, ws, ws_bytes, st);
}

}  // namespace hclsm
