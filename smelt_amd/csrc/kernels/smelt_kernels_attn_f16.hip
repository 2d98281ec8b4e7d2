// Attention over the paged cache, f16 (smelt_kernels_attn_f16.hsaco).
// Built with:  hipcc --offload-arch=gfx950 --genco -O3 -Xclang -target-feature -Xclang -packed-fp32-ops
#include "paged_attention.hpp"

SMELT_ATTENTION_KERNELS(f16, smelt::F16, 64, 4, 2, 8, 2, 2)
SMELT_ATTENTION_KERNELS(f16, smelt::F16, 128, 3, 2, 8, 2, 2)
SMELT_ATTENTION_KERNELS(f16, smelt::F16, 256, 2, 1, 4, 1, 1)
