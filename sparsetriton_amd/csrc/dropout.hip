// Dropout with the residual add, its mask from a counter-based generator:
//   Y = keep ? X / (1 - p) : 0   (+ residual),   keep: word(element) >= min(round(p 2^32), 2^32 - 1), none for p = 1
// and, with dY in X's place and no residual, its gradient: the mask is made
// again from the same two numbers and never stored.  An element's word depends
// on its index and the numbers alone, not on the type, the launch or the device.
//
// The words are Philox 4 x 32 with ten rounds (Salmon, Moraes, Dror, Shaw:
// "Parallel random numbers: as easy as 1, 2, 3", 2011): the block of counter
// (index / 4, numbers[1]) under the key numbers[0] holds the words of four
// elements.  A round is two 32 x 32 -> 64 products (a quarter of the vector
// unit's rate) and two three-way exclusive ors.
//
// Bound by memory, and for 16-bit tensors without a residual nearly as much by
// the words: 65,537 x 512 bf16 24.5 us (5.5 TB/s; 29.4 with an exclusive or in two
// instructions), with the residual 38.4 (5.2); 470,532 x 64 fp32 46 us (5.3), its
// gradient the same.  A 1 GiB copy runs at 5.11 TB/s.  (Over tensors that change from call to call: the same ones over and
// over, in part still in the cache behind L2, take 24.4, 32 - 34 and 42.)
#include <math.h>

#include "common.h"

namespace st {

constexpr int kDropThreads = 256;
// Elements of a thread: two blocks of words.  (65,537 x 512 bf16, the same tensors, in us without / with the residual: 24.4 / 34.4; two such
// vectors a thread 24.8 / 36.3, four 30.8 / 41.1: fewer waves, and the words of one do not wait for the other's load anyway.)
constexpr int kDropVec = 8;
constexpr int kDropElements = kDropThreads * kDropVec;  // of a workgroup

// (the compiler takes two instructions for a ^ b ^ c)
__device__ __forceinline__ unsigned xor3(unsigned a, unsigned b, unsigned c) { return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96); }

struct DropWords {
  unsigned w[4];
};

__device__ __forceinline__ DropWords philox(unsigned i_low, unsigned i_high, uint64_t call, uint64_t key) {
  unsigned x0 = i_low, x1 = i_high, x2 = (unsigned)call, x3 = (unsigned)(call >> 32);
  unsigned k0 = (unsigned)key, k1 = (unsigned)(key >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = 0xD2511F53ull * x0, b = 0xCD9E8D57ull * x2;
    x0 = xor3((unsigned)(b >> 32), x1, k0);
    x2 = xor3((unsigned)(a >> 32), x3, k1);
    x1 = (unsigned)b;
    x3 = (unsigned)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{x0, x1, x2, x3}};
}

struct DropArgs {
  const uint64_t* numbers;
  int64_t n, first;    // elements of the launch, and the index of its first one (a multiple of a workgroup's)
  unsigned threshold;
  int none;            // p = 1: no element stays
  float scale;
};

// WIDE: whole vectors of elements at 16-byte addresses, but for the last elements of the tensor.
template <typename T, bool RES, bool WIDE>
__global__ __launch_bounds__(kDropThreads) void dropout_kernel(const T* __restrict__ X, const T* __restrict__ R,
                                                               T* __restrict__ Y, DropArgs g) {
  struct alignas(WIDE ? 16 : sizeof(T)) Vec {
    T e[kDropVec];
  };
  const int64_t block0 = (int64_t)blockIdx.x * kDropElements, at = block0 + (int)threadIdx.x * kDropVec;
  const bool whole = WIDE && at + kDropVec <= g.n;
  Vec x, r;
  if (whole) {
    x = *reinterpret_cast<const Vec*>(X + at);
    if constexpr (RES) r = *reinterpret_cast<const Vec*>(R + at);
  } else {
#pragma unroll
    for (int e = 0; e < kDropVec; ++e) {
      x.e[e] = at + e < g.n ? X[at + e] : (T)0.f;
      if constexpr (RES) r.e[e] = at + e < g.n ? R[at + e] : (T)0.f;
    }
  }
  // The counter's upper half is the same in a workgroup (its first index is a multiple of its elements): a scalar,
  // and with it a product of each of the first two rounds.
  const uint64_t counter0 = (uint64_t)(g.first + block0) >> 2;
  const uint64_t key = g.numbers[0], call = g.numbers[1];
#pragma unroll
  for (int b = 0; b < kDropVec / 4; ++b) {
    const unsigned low = (unsigned)counter0 + threadIdx.x * (kDropVec / 4) + b;
    const DropWords words = philox(low, (unsigned)(counter0 >> 32), call, key);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float y = words.w[e] >= g.threshold && !g.none ? (float)x.e[4 * b + e] * g.scale : 0.f;
      if constexpr (RES) y += (float)r.e[4 * b + e];
      x.e[4 * b + e] = (T)y;
    }
  }
  if (whole) {
    *reinterpret_cast<Vec*>(Y + at) = x;
  } else {
#pragma unroll
    for (int e = 0; e < kDropVec; ++e)
      if (at + e < g.n) Y[at + e] = x.e[e];
  }
}

template <typename T>
static int dropout_run(const void* X, const void* R, void* Y, DropArgs g, hipStream_t s) {
  const bool wide = !(((uintptr_t)X | (uintptr_t)R | (uintptr_t)Y) & 15);
  const int64_t n = g.n, per = kDropElements, most = st_most_blocks(kDropThreads) * per;
  for (int64_t at = 0; at < n; at += most) {
    DropArgs part = g;
    part.n = n - at < most ? n - at : most;
    part.first = at;
    const T *x = (const T*)X + at, *r = R ? (const T*)R + at : nullptr;
    auto kernel = R ? (wide ? dropout_kernel<T, true, true> : dropout_kernel<T, true, false>)
                    : (wide ? dropout_kernel<T, false, true> : dropout_kernel<T, false, false>);
    kernel<<<st_blocks(part.n, (int)per), kDropThreads, 0, s>>>(x, r, (T*)Y + at, part);
    ST_CHECK_LAUNCH();
  }
  return ST_OK;
}

}  // namespace st

extern "C" int st_dropout(const void* X, const void* residual, int64_t n, int dtype, const int64_t* numbers, double p,
                          void* Y, st_stream_t stream) {
  if (n < 0 || !(p >= 0.0 && p <= 1.0)) return ST_ERR_ARG;
  if (n == 0) return ST_OK;
  if (!X || !Y || !numbers) return ST_ERR_ARG;
  const double words = rint(p * 4294967296.0);
  st::DropArgs g{};
  g.numbers = (const uint64_t*)numbers;
  g.n = n;
  g.threshold = words >= 4294967295.0 ? 0xFFFFFFFFu : (unsigned)words;
  g.none = p == 1.0;
  g.scale = p == 1.0 ? 0.f : (float)(1.0 / (1.0 - p));
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case ST_F32:
      return st::dropout_run<float>(X, residual, Y, g, s);
    case ST_F16:
      return st::dropout_run<_Float16>(X, residual, Y, g, s);
    case ST_BF16:
      return st::dropout_run<__bf16>(X, residual, Y, g, s);
    default:
      return ST_ERR_UNSUPPORTED;
  }
}
