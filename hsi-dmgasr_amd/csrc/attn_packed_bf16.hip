// Packed-sequence attention kernels, bf16 (attn_packed.h).
#define HSIDM_ATTN_TYPE bf16
#include "attn_packed_inst.inc"
