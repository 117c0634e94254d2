// Packed-sequence attention kernels, fp32 (attn_packed.h).
#define HSIDM_ATTN_TYPE float
#include "attn_packed_inst.inc"
