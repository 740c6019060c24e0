// attn_d256.cu — the attention split kernel's instances for head_dim 256.
#include "attn.cuh"

OFB_ATTN_INSTANCES(256)
