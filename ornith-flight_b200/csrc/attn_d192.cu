// attn_d192.cu — the attention split kernel's instances for head_dim 192.
#include "attn.cuh"

OFB_ATTN_INSTANCES(192)
