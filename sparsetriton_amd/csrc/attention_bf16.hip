// Attention kernels for bf16 tensors.
#include "attention.h"

int st::attn_run_bf16(AttnPass pass, const AttnArgs& a, hipStream_t s) { return attn_run<__bf16>(pass, a, s); }
