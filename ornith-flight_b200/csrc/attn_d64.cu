// attn_d64.cu — the attention split kernel's instances for head_dim 64.
#include "attn.cuh"

OFB_ATTN_INSTANCES(64)
