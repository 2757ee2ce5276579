// Attention over pages for bf16 inputs (attn_paged_kernels.h).
#include "attn_paged_kernels.h"

namespace dx {

hipError_t launch_paged_bf16(const PagedArgs& a, const PagedPlan& p, int D, hipStream_t st) {
  switch (D) {
    case 64: return launch_paged<bf16_t, 64, kPlain>(a, p, st);
    case 128: return launch_paged<bf16_t, 128, kPlain>(a, p, st);
    case 256: return launch_paged<bf16_t, 256, kPlain>(a, p, st);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace dx
