// The attention kernels of csrc/attention.h for one element type.
#include "attention_fwd.h"
#include "attention_bwd.h"

int at_fwd_f32(const AttnP& p, bool tokens, hipStream_t st) { return at_fwd<float>(p, tokens, st); }
int at_bwd_f32(const AttnP& dq, const AttnP& dkv, float* stat, hipStream_t st) { return at_bwd<float>(dq, dkv, stat, st); }
