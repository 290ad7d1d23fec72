// The attention of many rows over pages of 8 bits: the kernel of paged_attn_prompt.cu, compiled beside it.
#define B200_PAGED_BYTES
#include "paged_attn_prompt.cu"
