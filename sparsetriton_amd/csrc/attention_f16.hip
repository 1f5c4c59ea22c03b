// Attention kernels for f16 tensors.
#include "attention.h"

int st::attn_run_f16(AttnPass pass, const AttnArgs& a, hipStream_t s) { return attn_run<_Float16>(pass, a, s); }
