// Serving operators between the projections and behind the lm_head (smelt_kernels_serving.hsaco).
// Built with:  hipcc --offload-arch=gfx950 --genco -O3 -Xclang -target-feature -Xclang -packed-fp32-ops
#include "rope_kernels.hpp"
#include "verify_kernels.hpp"

SMELT_ROPE_KERNELS(f16, smelt::F16)
SMELT_ROPE_KERNELS(bf16, smelt::BF16)
SMELT_VERIFY_KERNELS(f16, smelt::F16)
SMELT_VERIFY_KERNELS(bf16, smelt::BF16)
