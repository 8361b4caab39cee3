// The attention kernels of csrc/attention.h for one element type.
#include "attention_fwd.h"
#include "attention_bwd.h"

int at_fwd_bf16(const AttnP& p, bool tokens, hipStream_t st) { return at_fwd<__bf16>(p, tokens, st); }
int at_bwd_bf16(const AttnP& dq, const AttnP& dkv, float* stat, hipStream_t st) { return at_bwd<__bf16>(dq, dkv, stat, st); }
