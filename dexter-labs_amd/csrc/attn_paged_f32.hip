// Attention over pages for fp32 inputs (attn_paged_kernels.h).
#include "attn_paged_kernels.h"

namespace dx {

hipError_t launch_paged_f32(const PagedArgs& a, const PagedPlan& p, int D, hipStream_t st) {
  switch (D) {
    case 64: return launch_paged<float, 64>(a, p, st);
    case 128: return launch_paged<float, 128>(a, p, st);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace dx
