// attn_d96.cu — the attention split kernel's instances for head_dim 96.
#include "attn.cuh"

OFB_ATTN_INSTANCES(96)
