// Column sums of partial results in a fixed order: the gradients of weights
// that a kernel's workgroups each leave a partial of.
#pragma once

#include "common.h"

namespace st {

constexpr int kPartsThreads = 256;
constexpr int kPartsColumns = 8;  // of a workgroup

// dw, db = the column sums of `groups` partials of 2 C floats: a workgroup for
// eight columns, a thread for a column and each of 32 shares of the partials,
// the shares added in order.
// (32 columns and 8 shares of it took 32 us for 1,024 partials of 64 channels:
// four workgroups, 128 loads one after another.)
template <typename W>
__global__ __launch_bounds__(kPartsThreads) void sum_parts_kernel(const float* __restrict__ parts, int groups, int C,
                                                                  W* __restrict__ dw, W* __restrict__ db) {
  __shared__ float sums[32][9];
  const int in = threadIdx.x & 7, share = threadIdx.x >> 3, col = blockIdx.x * kPartsColumns + in;
  float s = 0.f;
  if (col < 2 * C) {
#pragma unroll 8
    for (int p = share; p < groups; p += 32) s += parts[(int64_t)p * 2 * C + col];
  }
  sums[share][in] = s;
  __syncthreads();
  if (share || col >= 2 * C) return;
#pragma unroll
  for (int o = 1; o < 32; ++o) s += sums[o][in];
  if (col < C) {
    if (dw) dw[col] = (W)s;
  } else if (db) {
    db[col - C] = (W)s;
  }
}

template <typename W>
static int sum_parts(const float* parts, int64_t groups, int C, void* dw, void* db, hipStream_t s) {
  sum_parts_kernel<W><<<st_blocks(2 * (int64_t)C, kPartsColumns), kPartsThreads, 0, s>>>(parts, (int)groups, C, (W*)dw, (W*)db);
  ST_CHECK_LAUNCH();
  return ST_OK;
}

}  // namespace st
