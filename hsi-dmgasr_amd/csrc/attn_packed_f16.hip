// Packed-sequence attention kernels, fp16 (attn_packed.h).
#define HSIDM_ATTN_TYPE f16
#include "attn_packed_inst.inc"
