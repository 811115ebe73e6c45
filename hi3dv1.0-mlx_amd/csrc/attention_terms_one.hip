// Attention with one term beside scale q k, in the kernels that many rows and keys take.
#include "attention_forward.h"

namespace hi3d {

int launch_rows_of_one(const TermArgs& a, int dtype, int kind, hipStream_t stream) {
  const bool half = dtype == HI3D_F16;
  switch (kind) {
    case kCap: return half ? launch_wide_type<_Float16, kCap>(a, stream) : launch_wide_type<__bf16, kCap>(a, stream);
    case kSlopes: return half ? launch_wide_type<_Float16, kSlopes>(a, stream) : launch_wide_type<__bf16, kSlopes>(a, stream);
    default: return half ? launch_wide_type<_Float16, kBias>(a, stream) : launch_wide_type<__bf16, kBias>(a, stream);
  }
}

}  // namespace hi3d
