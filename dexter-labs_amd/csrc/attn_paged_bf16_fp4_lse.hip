// Attention over pages in 4 bits for bf16 inputs, with log-sum-exps
// (attn_paged_kernels.h).
#include "attn_paged_kernels.h"

namespace dx {

hipError_t launch_paged_bf16_fp4_lse(const PagedArgs& a, const PagedPlan& p, int D, hipStream_t st) {
  switch (D) {
    case 64: return launch_paged<bf16_t, 64, kFp4Lse>(a, p, st);
    case 128: return launch_paged<bf16_t, 128, kFp4Lse>(a, p, st);
    case 256: return launch_paged<bf16_t, 256, kFp4Lse>(a, p, st);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace dx
