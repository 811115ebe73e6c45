// Gradients of attention with one term beside scale q k, in the kernels that many rows and keys take.
#include "attention_backward.h"

namespace hi3d {

int launch_grad_of_one(const TermArgs& a, int dtype, int kind, hipStream_t stream) {
  const bool half = dtype == HI3D_F16;
  switch (kind) {
    case kCap: return half ? launch_grad_type<_Float16, kCap, true>(a, stream) : launch_grad_type<__bf16, kCap, true>(a, stream);
    case kSlopes:
      return half ? launch_grad_type<_Float16, kSlopes, true>(a, stream) : launch_grad_type<__bf16, kSlopes, true>(a, stream);
    default: return half ? launch_grad_type<_Float16, kBias, true>(a, stream) : launch_grad_type<__bf16, kBias, true>(a, stream);
  }
}

}  // namespace hi3d
