// attn_d128.cu — the attention split kernel's instances for head_dim 128.
#include "attn.cuh"

OFB_ATTN_INSTANCES(128)
