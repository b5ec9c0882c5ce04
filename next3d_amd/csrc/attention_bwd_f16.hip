// Attention, backward: the kernels of float16 (attention_bwd.h).
#include "attention_bwd.h"

void attn_bwd_f16(AttnParams& p, hipStream_t stream) { attn_bwd_typed<_Float16>(p, stream); }
