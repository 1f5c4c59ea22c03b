// Attention kernels for f32 tensors.
#include "attention.h"

int st::attn_run_f32(AttnPass pass, const AttnArgs& a, hipStream_t s) { return attn_run<float>(pass, a, s); }
