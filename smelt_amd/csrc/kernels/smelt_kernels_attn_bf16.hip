// Attention over the paged cache, bf16 (smelt_kernels_attn_bf16.hsaco).
// Built with:  hipcc --offload-arch=gfx950 --genco -O3 -Xclang -target-feature -Xclang -packed-fp32-ops
#include "paged_attention.hpp"

SMELT_ATTENTION_KERNELS(bf16, smelt::BF16, 64, 4, 2, 8, 2, 2)
SMELT_ATTENTION_KERNELS(bf16, smelt::BF16, 128, 3, 2, 8, 2, 2)
SMELT_ATTENTION_KERNELS(bf16, smelt::BF16, 256, 2, 1, 4, 1, 1)
