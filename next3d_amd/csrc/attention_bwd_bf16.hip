// Attention, backward: the kernels of bfloat16 (attention_bwd.h).
#include "attention_bwd.h"

void attn_bwd_bf16(AttnParams& p, hipStream_t stream) { attn_bwd_typed<__bf16>(p, stream); }
