// Attention over segments of packed rows: kernels (see attention.hip for the
// host side).  For a segment with queries Q, keys K, values V and the scale c:
//   S = c Q K^T,   P = softmax over the keys that the row may see,   O = P V
// and, from dO and the saved L = log sum exp S,
//   P = exp(S - L),  delta = rowsum(dO o O),  dP = dO V^T,  dS = P o (dP - delta),
//   dQ = c dS K,   dK = c dS^T Q,   dV = P^T dO.
// A row that sees no key has O = 0 and no gradient.
//
// Query heads that share a key head are rows of one matrix: "packed row" r of a
// segment is query r / R, head hk R + r % R for R = heads / kv_heads.  One
// pass over a key head's K and V serves its whole group, dK and dV are summed
// over the group where they are made, and a single query row still fills R
// rows of the matrix product.
//
// Every product is a 32 x 32 MFMA tile, laid out so that no operand goes back
// through memory: the products whose result the next product reduces over are
// computed transposed (S^T = K Q^T: lane = query, registers = keys), so that a
// lane's registers are already its B operand of the next one (O^T += V^T P^T).  The
// reduction index of an MFMA may be permuted if both operands agree: register
// r of half h of the wave is key 8 (r / 4) + 4 h + r % 4, and the other operand
// (V^T, K^T, Q^T, dO^T) is read from LDS in that order -- by transpose reads
// (ds_read_b64_tr_b16) for 16-bit types.  Row sums and maxima of P are sums over a
// lane's own registers and one exchange between the halves.
//
// fp32 tensors use the fp32 MFMA (32 x 32 x 2), eight of them in the place of a
// 32 x 32 x 16, in the same layout: nothing is rounded below 32 bits.  16-bit
// types round P and dS to the type for the second product (their sums, the
// softmax statistics and all accumulators are fp32), and a training pass keeps
// what O's rounding left beside O: delta is a sum of products that cancel dP where
// a row sees few keys, and there the error of one from the rounded O is the
// largest (causal rows of 1 - 8 keys: dQ off by 1.9 times the rounding of dQ
// itself, 1.5 with the rest of O; 1.4 are that rounding and dS's.  No slower).
#pragma once

#include "common.h"
#include "mfma.h"
#include "wave_sum.h"

namespace st {

typedef float v8f __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));

// Rows (or keys) of a workgroup: 32 for each of its waves, four of them or one.
// Four share the tiles in LDS; one alone is for segments that would leave most of
// the four without rows (a workgroup's latency, not its work, is the cost there).
constexpr int kAttnTile = ST_ATTN_TILE;
constexpr int kAttnThreads = 256;  // of the joins

struct AttnItem {  // ST_ATTN_ITEM_WORDS int32, written by the host
  int q0, nq;      // the segment's first query row and their number
  int k0, nk;      // its first key row and their number
  int row0;        // first packed row (first key) of this tile in the segment
  int lo, hi;      // keys (packed rows) to go over
  int part;        // slot of the partial result, -1: the result itself
};
struct AttnJoin {  // ST_ATTN_JOIN_WORDS int32
  int q0, nq, k0, nk, row0;
  int part, parts;  // first slot and number of the partial results
  int unused;
};

struct AttnDivisor {  // d and floor(2^32 / d), 2^32 - 1 for 1
  unsigned d, inv;
};
inline AttnDivisor attn_divisor(int d) { return {(unsigned)d, d > 1 ? (unsigned)((1ull << 32) / d) : ~0u}; }
// x / d for x below 2^31: the product with the inverse is the quotient or one less.
__device__ __forceinline__ int attn_div(int x, AttnDivisor by) {
  const unsigned q = __umulhi((unsigned)x, by.inv);
  return (int)(q + ((unsigned)x - q * by.d >= by.d));
}

struct AttnArgs {
  const void *q, *k, *v, *o, *dout;
  const void* o_rest;  // NULL, or (16-bit) O before its rounding minus O: written by the forward, read for delta
  void *out, *rest, *dq, *dk, *dv;
  float *lse, *delta, *parts;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, do_row, do_head;
  const uint8_t* key_mask;
  const AttnItem* items;
  const AttnJoin* joins;
  int n_items, n_joins;
  AttnDivisor by_items, by_kv_heads, by_group;
  int heads, kv_heads, group, D, causal;
  int tile;        // rows of the items' tiles: ST_ATTN_TILE or ST_ATTN_SMALL_TILE
  int item_major;  // workgroups take an item's key heads in turn, else a key head's items
  float scale, scale_log2;  // c and c / ln 2
};

// ------------------------------------------------------------------ MFMA

template <typename T>
struct AttnFrag;  // eight reduction elements of a lane
template <>
struct AttnFrag<__bf16> {
  using type = v8bf;
};
template <>
struct AttnFrag<_Float16> {
  using type = v8h;
};
template <>
struct AttnFrag<float> {
  using type = v8f;
};

__device__ __forceinline__ v16f mma32(const v8bf& a, const v8bf& b, const v16f& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v16f mma32(const v8h& a, const v8h& b, const v16f& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v16f mma32(const v8f& a, const v8f& b, v16f c) {
#pragma unroll
  for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
  return c;
}
template <typename T>
__device__ __forceinline__ typename AttnFrag<T>::type to_frag(const v8f& x) {
  if constexpr (sizeof(T) == 4)
    return x;
  else
    return __builtin_convertvector(x, typename AttnFrag<T>::type);
}
__device__ __forceinline__ v8f regs8(const v16f& c, int j) {  // registers 8j .. 8j + 7 (j a constant)
  return j == 0 ? __builtin_shufflevector(c, c, 0, 1, 2, 3, 4, 5, 6, 7)
                : __builtin_shufflevector(c, c, 8, 9, 10, 11, 12, 13, 14, 15);
}
// Row (key) of register r in half `half`
__device__ __forceinline__ int reg_row(int r, int half) { return 8 * (r >> 2) + 4 * half + (r & 3); }

// ------------------------------------------------------------------ LDS tiles

// A tile of rows of DP elements, 16-byte chunks permuted within a row by an
// XOR with a few bits of the row, so that both kinds of reads meet 16
// different 16-byte bank groups: 16 consecutive rows at one chunk (row
// fragments), and four consecutive rows at four aligned chunks (transpose
// reads).  Which bits depends on how many rows share 256 bytes.
template <typename T, int DP>
struct AttnTile {
  static constexpr int EPC = 16 / sizeof(T);  // elements of a chunk
  static constexpr int CPR = DP / EPC;        // chunks of a row
  using Frag = typename AttnFrag<T>::type;

  static __device__ __forceinline__ int swz(int row) {
    if constexpr (CPR == 4 || CPR == 12)
      return (row >> 2) & 3;
    else if constexpr (CPR == 8 || CPR == 24)
      return ((row >> 1) & 1) * 4 + ((row >> 2) & 3);
    else
      return (row & 3) * 4 + ((row >> 2) & 3);
  }
  static __device__ __forceinline__ int at(int row, int chunk) { return row * DP + (chunk ^ swz(row)) * EPC; }

  // Elements col .. col + 7 (col a multiple of 8) of a row.
  static __device__ __forceinline__ Frag rows(const T* tile, int row, int col) {
    if constexpr (sizeof(T) == 2) {
      return *reinterpret_cast<const Frag*>(tile + at(row, col / EPC));
    } else {
      const v4f a = *reinterpret_cast<const v4f*>(tile + at(row, col / EPC));
      const v4f b = *reinterpret_cast<const v4f*>(tile + at(row, col / EPC + 1));
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  // Column d0 + lane % 32 of rows row0 + {4 half .. 4 half + 3, 8 + 4 half .. 8 + 4 half + 3}
  // (row0 a multiple of 16, d0 of 32).  16-bit: two transpose reads; in a group of
  // 16 lanes, lane l addresses row l / 4 at columns 4 (l % 4) and receives
  // column l of the four rows.
  static __device__ __forceinline__ Frag cols(const T* tile, int row0, int d0) {
    const int lane = threadIdx.x & 63, half = lane >> 5;
    if constexpr (sizeof(T) == 2) {
      typedef short v4s __attribute__((ext_vector_type(4)));
      typedef short v8s __attribute__((ext_vector_type(8)));
      using lds_v4s = __attribute__((address_space(3))) v4s;
      const int row = row0 + 4 * half + ((lane >> 2) & 3);
      const int chunk = d0 / 8 + ((lane >> 4) & 1) * 2 + ((lane >> 1) & 1), in = (lane & 1) * 4;
      const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(tile + at(row, chunk) + in));
      const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(tile + at(row + 8, chunk) + in));
      const v8s both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      return __builtin_bit_cast(Frag, both);
    } else {
      const int d = d0 + (lane & 31);
      Frag f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int row = row0 + 4 * half + (e & 3) + 8 * (e >> 2);
        f[e] = tile[at(row, d / 4) + d % 4];
      }
      return f;
    }
  }
};

// A product over the rows of a tile that the causal order cuts: the other
// operand is zero where a column must not see a row, but zero times an infinity
// or a NaN is a NaN, so a later row that is not finite would reach earlier ones.
// Such a tile (one check of it, by each wave that the order cuts it for) is
// copied without those elements, the product taken over the copy, and what they
// do to the columns that see them added at the end.
template <typename T, int ROWS, int DP>
__device__ __forceinline__ bool attn_not_finite(const T* tile) {
  using Tile = AttnTile<T, DP>;
  bool bad = false;
#pragma unroll 4
  for (int c = threadIdx.x & 63; c < ROWS * Tile::CPR; c += 64)
#pragma unroll
    for (int e = 0; e < Tile::EPC; ++e) bad |= !(fabsf((float)tile[c * Tile::EPC + e]) < INFINITY);
  return __any(bad);
}
// (Each wave that needs the copy writes all of it, the same values.)
template <typename T, int ROWS, int DP>
__device__ __forceinline__ void attn_copy_finite(const T* tile, T* copy) {
  using Tile = AttnTile<T, DP>;
#pragma unroll 1
  for (int c = (threadIdx.x & 63) * Tile::EPC; c < ROWS * DP; c += 64 * Tile::EPC)
#pragma unroll
    for (int e = 0; e < Tile::EPC; ++e) copy[c + e] = fabsf((float)tile[c + e]) < INFINITY ? tile[c + e] : (T)0.f;
}
// What the left out elements do to a lane's sums (transposed: registers =
// channels), a bit for each: infinities of either sign, both for a NaN.  In
// loops that stay rolled: they take neither time nor registers from the products.
struct AttnNotFinite {
  uint64_t pos = 0, neg = 0;
  template <typename T, int ROWS, int DP>
  __device__ __forceinline__ void add(const T* tile, int first, int last) {  // rows first .. last
    using Tile = AttnTile<T, DP>;
    const int half = (threadIdx.x >> 5) & 1;
#pragma unroll 1
    for (int row = 0; row < ROWS; ++row)
#pragma unroll 1
      for (int r = 0; r < DP / 2; ++r) {
        const int d = (r >> 4) * 32 + reg_row(r & 15, half);
        const float x = (float)tile[Tile::at(row, d / Tile::EPC) + d % Tile::EPC];
        const bool seen = row >= first && row <= last && !(fabsf(x) < INFINITY);
        pos |= (uint64_t)(seen && x != -INFINITY) << r;
        neg |= (uint64_t)(seen && x != INFINITY) << r;
      }
  }
  template <int DB>
  __device__ __forceinline__ void apply(v16f (&acc)[DB]) const {
    if (!__any(pos | neg)) return;
#pragma unroll
    for (int r = 0; r < DB * 16; ++r) {
      if (pos >> r & 1) acc[r / 16][r % 16] += INFINITY;
      if (neg >> r & 1) acc[r / 16][r % 16] -= INFINITY;
    }
  }
};

// Rows of a tile on their way from memory to LDS: each thread carries N chunks.
template <typename T, int DP, int ROWS, int WAVES>
struct AttnStage {
  using Tile = AttnTile<T, DP>;
  static constexpr int THREADS = 64 * WAVES, N = ROWS * Tile::CPR / THREADS;
  static_assert(ROWS * Tile::CPR % THREADS == 0, "whole chunks a thread");
  v4u reg[N];

  static __device__ __forceinline__ int row(int i) { return (threadIdx.x + i * THREADS) / Tile::CPR; }
  static __device__ __forceinline__ int chunk(int i) { return (threadIdx.x + i * THREADS) % Tile::CPR; }
  int off[N];  // byte offsets of this thread's chunks from the tile's first row
  template <typename F>
  __device__ __forceinline__ void place(int D, F offset) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = chunk(i) * Tile::EPC;
      off[i] = c < D ? offset(row(i)) + c * (int)sizeof(T) : kOobOffset;
    }
  }
  // `left` rows from `base` on, zeros after them
  __device__ __forceinline__ void load(const T* base, int left) {
    const __amdgpu_buffer_rsrc_t r = make_rsrc(base, kOobOffset);
#pragma unroll
    for (int i = 0; i < N; ++i) reg[i] = load16<v4u>(r, row(i) < left ? off[i] : kOobOffset);
  }
  __device__ __forceinline__ void store(T* tile) const {
#pragma unroll
    for (int i = 0; i < N; ++i) *reinterpret_cast<v4u*>(tile + Tile::at(row(i), chunk(i))) = reg[i];
  }
};

// Rows from `row` on, to be read at byte offsets of 32 bits.
template <typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t attn_rows(const T* p, int64_t row, int64_t stride) {
  return make_rsrc(p + row * stride, kOobOffset);
}
// Eight elements of a row `off` bytes from a buffer's base (16-byte aligned), zeros past D or for a dead row.
template <typename T>
__device__ __forceinline__ typename AttnFrag<T>::type load_row8(__amdgpu_buffer_rsrc_t base, int off, int col, int D, bool live) {
  using Frag = typename AttnFrag<T>::type;
  const int at = live && col < D ? off + col * (int)sizeof(T) : kOobOffset;
  if constexpr (sizeof(T) == 2) {
    return load16<Frag>(base, at);
  } else {
    const v4f a = load16<v4f>(base, at), b = load16<v4f>(base, at == kOobOffset ? at : at + 16);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}
// The same at an address of its own.
template <typename T>
__device__ __forceinline__ typename AttnFrag<T>::type load_row8(const T* row, int col, int D, bool live) {
  typename AttnFrag<T>::type f;
  if (live && col < D) return *reinterpret_cast<const typename AttnFrag<T>::type*>(row + col);
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = (T)0.f;
  return f;
}

// Stores a lane's row from accumulators that hold it transposed (registers =
// channels): 16-bit halves exchange quads so that each lane stores whole chunks.
template <typename T, int DB>
__device__ __forceinline__ void store_row(T* row, const v16f (&acc)[DB], float scale, int D, bool live) {
  const int half = (threadIdx.x >> 5) & 1;
#pragma unroll
  for (int b = 0; b < DB; ++b) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int d = b * 32 + 8 * j + 4 * half;
        const v4f x = {acc[b][4 * j] * scale, acc[b][4 * j + 1] * scale, acc[b][4 * j + 2] * scale,
                       acc[b][4 * j + 3] * scale};
        if (live && d < D) *reinterpret_cast<v4f*>(row + d) = x;
      }
    } else {
      typedef T v2t __attribute__((ext_vector_type(2)));
      auto pack = [&](int r) {
        const v2f x = {acc[b][r] * scale, acc[b][r + 1] * scale};
        return __builtin_bit_cast(unsigned, __builtin_convertvector(x, v2t));
      };
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const auto x = __builtin_amdgcn_permlane32_swap(pack(4 * j), pack(4 * j + 4), false, false);
        const auto y = __builtin_amdgcn_permlane32_swap(pack(4 * j + 2), pack(4 * j + 6), false, false);
        const int d = b * 32 + 8 * (j + half);
        const v4u w = {x[0], y[0], x[1], y[1]};
        if (live && d < D) *reinterpret_cast<v4u*>(row + d) = w;
      }
    }
  }
}
// What the rounding of acc * scale to T leaves, in acc's place.
template <typename T, int DB>
__device__ __forceinline__ void keep_rest(v16f (&acc)[DB], float scale) {
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float x = acc[b][e] * scale;
      acc[b][e] = x - (float)(T)x;
    }
}
// The same as fp32 partial sums at a row of DP floats.
template <int DB>
__device__ __forceinline__ void store_part(float* row, const v16f (&acc)[DB], bool live) {
  const int half = (threadIdx.x >> 5) & 1;
  if (!live) return;
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<v4f*>(row + b * 32 + 8 * j + 4 * half) =
          (v4f){acc[b][4 * j], acc[b][4 * j + 1], acc[b][4 * j + 2], acc[b][4 * j + 3]};
}

// Work item of a workgroup.  The hardware deals workgroups to the 8 XCDs
// round-robin; runs of 16 consecutive items (tiles of one segment and key
// head, which read the same rows) go to one XCD and its L2.
__device__ __forceinline__ int attn_work(int n) {
  const int id = blockIdx.x, base = id & ~127;
  return base + 128 > n ? id : base + (id & 7) * 16 + ((id & 127) >> 3);
}

// Item and key head of a workgroup.
__device__ __forceinline__ AttnItem attn_item(const AttnArgs& a, int& hk) {
  const int w = attn_work(gridDim.x);
  if (a.item_major) {
    const int i = attn_div(w, a.by_kv_heads);
    hk = w - i * a.kv_heads;
    return a.items[i];
  }
  hk = attn_div(w, a.by_items);
  return a.items[w - hk * a.n_items];
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// For the scheduler: of N fragment reads, each followed by its MFMAs, kAhead
// go out before the first product and one behind each product.  (Left to itself
// it reads, waits ~130 cycles and multiplies, fragment by fragment.)
template <typename T, int N, bool COLS = false>
__device__ __forceinline__ void attn_reads_ahead() {
  constexpr int kAhead = 4, READS = (COLS ? 2 : 1) * (sizeof(T) == 2 ? 1 : COLS ? 4 : 2);
  constexpr int PRODUCTS = sizeof(T) == 2 ? 1 : 8;
  __builtin_amdgcn_sched_group_barrier(0x100, (N < kAhead ? N : kAhead) * READS, 0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, PRODUCTS, 0);
    if (i + kAhead < N) __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
  }
}

// Whether 16 channels of the scores' sum are to be taken: fp32 leaves out those past D, eight slow
// products each (16-bit types take a zero product rather than a branch among theirs).
template <typename T>
__device__ __forceinline__ bool attn_in(int channel, int D) {
  return sizeof(T) == 2 || channel < D;
}

// Waves of a SIMD that the registers leave room for (a limit for the compiler).
template <typename T, int DP>
constexpr int attn_waves() {
  return DP * sizeof(T) <= 256 ? 2 : 1;
}

// ------------------------------------------------------------------ forward

// A tile of packed rows against its keys in steps, K and V of the next step on
// their way to registers while this one is multiplied (two buffers in LDS, one
// barrier a step).  A softmax in one pass: running maximum and sum, the
// accumulators scaled when the maximum rises.  Few tiles: the keys are split
// and the parts joined after it.
//
// (Kernel times here and below are medians by trace.)
// 64 patches of 1,024 rows x 8 heads x 64 bf16: 208 us, 660 TFLOP/s (a large
// product: 1,210).  The vector unit is what it runs on: an exponential, a
// multiply-add, a sum, half a conversion and half a maximum for each score, 64
// instructions a 32 x 32 tile of them, and 32 more by its counter (offsets, bounds, staging); it
// issues 70 % of the time, the matrix unit is busy 37 %, three waves a SIMD.  128 channels do twice the product for the same
// scores: 8,191 rows x 16 heads of 128 (4 key heads), causal, bf16, 330 us, 830
// TFLOP/s of the visible half.  fp32, 24 samples of up to 1,500 rows x 6 x 48: 80
// us, 72 TFLOP/s (a large fp32 product: 153), the matrix unit busy 60 %, a seventh of
// it for the channels 48 .. 63 of the second product.  Single rows over 75,000
// keys of 8 heads x 128: 58 us, 5.3 TB/s.  2,000 windows of up to 96 rows x 4 x
// 32, one wave each: 14.5 us, 3.0 TB/s (8,000 windows 44 us, 4.0), each wave's own chain of loads, products
// and exponentials at 16 waves a unit; bounds of five and six waves a SIMD spill (15, 35 us).

// Keys of a step: 64, or 32 for a wave alone (its lanes carry the whole step on its way to LDS).
template <int WAVES>
constexpr int attn_keys() {
  return WAVES == 1 ? 32 : 64;
}

template <typename T, int DP, int WAVES>
constexpr int attn_fwd_lds(bool causal) {  // two buffers of K and V; causal, a copy of one of them, else two of the keys' terms
  return attn_keys<WAVES>() * (causal ? 5 * DP * (int)sizeof(T) : 4 * DP * (int)sizeof(T) + 2 * (int)sizeof(float));
}

// A running maximum is raised only when a row's maximum passes it by more
// than this (in powers of two): below, exp2(S - m) <= 2^8 loses nothing in
// floating point, and the accumulators need no rescaling.
constexpr float kAttnSlack = 8.f;
// float16 holds P times a power of two, so that small probabilities keep their bits: below 2^-14
// the type has fewer of them.  Forward: P up to 2^8 (kAttnSlack) times 2^7; the keys' pass: P up to 1
// times 2^14 (dP - delta over as much).  The powers are added to the exponents and cost nothing.
// dS has no bound of its own (AttnPower).
template <typename T>
constexpr float kAttnUp = sizeof(T) == 2 && !__is_same(T, __bf16) ? 7.f : 0.f;
template <typename T>
constexpr float kAttnKeysUp = 2.f * kAttnUp<T>;
template <typename T>
constexpr float kAttnKeysDown = kAttnUp<T> == 0.f ? 1.f : 1.f / 16384.f;

// float16 dS: as large as dO V^T (past the type's range under the scale of a loss, where the
// gradients are not) and as small as P makes it (over many keys below 2^-14, where the type
// loses digits).  A lane's column of dS^T (dS) is all that its dQ row (dK row) is a sum of, so each lane
// holds its sums at a power of two of its own, taken from the largest |dS| so far as the
// forward takes its maximum: that one comes to 2^8 .. 2^9 when it sets the power, a later one
// passes 2^15 before the power is set again (and the sums scaled with it), and what
// lies below 2^-14 then is 2^-22 of it or less.  Powers of two: nothing else is rounded.
// (The other types have float's exponents, and none of this.)  Backward without / with it: 64
// patches of 1,024 rows x 8 heads x 64 626 / 685 us, 8,191 causal rows x 16 heads of 128 (4 key
// heads) 1,447 / 1,485, 2,000 windows of up to 96 rows x 4 x 32 85 / 88.
template <typename T>
constexpr bool kAttnHeld = kAttnUp<T> != 0.f;
struct AttnPower {
  float up = 1.f, down = 1.f;  // what dS is held at, and its inverse
  float limit = 0.f;           // of up |dS|: 0 until a first one that is not zero

  // s: up dS of a step (registers and the other half: the lane's column), sums: of dS so far.
  template <int DB>
  __device__ __forceinline__ void hold(v16f& s, v16f (&sums)[DB]) {
    float top = fabsf(s[0]);
#pragma unroll
    for (int e = 1; e < 16; ++e) top = fmaxf(top, fabsf(s[e]));
    top = fmaxf(top, other_half(top));
    const bool raise = top > limit && top < INFINITY;  // (an infinity stays one)
    if (!__any(raise)) return;
    // 2^(9 - e) for a top of 2^(e-1) .. 2^e; below 2^-60 no dS counts in the type's results
    const int e = max((int)(__builtin_bit_cast(unsigned, top) >> 23) - 126, -60);
    const float by = raise ? __builtin_bit_cast(float, (unsigned)(127 + 9 - e) << 23) : 1.f;
    up *= by;
    down *= raise ? __builtin_bit_cast(float, (unsigned)(127 - 9 + e) << 23) : 1.f;
    limit = raise ? 32768.f : limit;
    s *= by;
#pragma unroll
    for (int b = 0; b < DB; ++b) sums[b] *= by;
  }
  template <int DB>
  __device__ __forceinline__ void release(v16f (&sums)[DB]) const {
#pragma unroll
    for (int b = 0; b < DB; ++b) sums[b] *= down;
  }
};

template <typename T, int DP, bool CAUSAL, int WAVES>
__global__ __launch_bounds__(64 * WAVES, (attn_waves<T, DP>())) void attn_forward_kernel(AttnArgs a) {
  using Tile = AttnTile<T, DP>;
  using Frag = typename Tile::Frag;
  constexpr int BK = attn_keys<WAVES>();
  using Stage = AttnStage<T, DP, BK, WAVES>;
  constexpr int KS = DP / 16, DB = DP / 32, NB = BK / 32;
  constexpr int TILE = BK * DP;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  T* tiles = reinterpret_cast<T*>(lds);
  float* bias = reinterpret_cast<float*>(tiles + 4 * TILE);  // two buffers, not CAUSAL: 0 or -inf for each key of a step

  int hk;
  const AttnItem it = attn_item(a, hk);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, half = lane >> 5;
  const int rows = it.nq * a.group, r = it.row0 + wave * 32 + (lane & 31);
  const bool active = it.row0 + wave * 32 < rows, live = r < rows;
  const int qi = attn_div(r, a.by_group), in_group = r - qi * a.group, head = hk * a.group + in_group;
  const int first = attn_div(it.row0, a.by_group);  // query of the tile's first row

  Frag qf[KS];
  {
    const auto base = attn_rows((const T*)a.q + hk * a.group * a.q_head, it.q0 + (int64_t)first, a.q_row);
    const int off = (qi - first) * (int)(a.q_row * sizeof(T)) + in_group * (int)(a.q_head * sizeof(T));
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = load_row8<T>(base, off, 16 * s + 8 * half, a.D, live);
  }
  const int see = CAUSAL ? qi + it.nk - it.nq : 0x7FFFFFFF;  // last key that this lane's row sees

  Stage ks, vs;
  ks.place(a.D, [&](int x) { return x * (int)(a.k_row * sizeof(T)); });
  vs.place(a.D, [&](int x) { return x * (int)(a.v_row * sizeof(T)); });
  uint8_t chunk_kept[Stage::N], key_kept = 1;
  const uint8_t* mask = a.key_mask ? a.key_mask + it.k0 : nullptr;
  auto fetch = [&](int kt) {
    const int left = it.hi - kt;
    const int64_t row = it.k0 + (int64_t)kt;
    if (mask) {
#pragma unroll
      for (int i = 0; i < Stage::N; ++i) chunk_kept[i] = Stage::row(i) < left ? mask[kt + Stage::row(i)] : 0;
      key_kept = lane < left ? mask[kt + lane] : 0;
    }
    ks.load((const T*)a.k + row * a.k_row + hk * a.k_head, left);
    vs.load((const T*)a.v + row * a.v_row + hk * a.v_head, left);
  };

  v16f o[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b) o[b] = (v16f)(0.f);
  float m = -INFINITY, l = 0.f;
  AttnNotFinite left_out;
  if (it.lo < it.hi) fetch(it.lo);
  for (int kt = it.lo, buf = 0; kt < it.hi; kt += BK, buf ^= 1) {
    T* kl = tiles + buf * 2 * TILE;
    T* vl = kl + TILE;
    constexpr uint64_t ALL = ~0ull >> (64 - BK);
    uint64_t seen = ALL;  // keys of this step that exist and are not masked
    if (it.hi - kt < BK) seen >>= BK - (it.hi - kt);
    if (mask) {
      seen &= __ballot(key_kept);
#pragma unroll
      for (int i = 0; i < Stage::N; ++i)  // (whatever a masked row holds, not finite included, stays out of the products)
        if (!chunk_kept[i]) ks.reg[i] = vs.reg[i] = (v4u)(0u);
    }
    if (!CAUSAL && seen != ALL && threadIdx.x < BK) bias[buf * BK + lane] = seen >> lane & 1 ? 0.f : -INFINITY;
    ks.store(kl);
    vs.store(vl);
    __syncthreads();
    if (kt + BK < it.hi) fetch(kt + BK);
    if (!active || (CAUSAL && !__any(live && kt <= see))) continue;

    v16f s[NB];
    auto scores = [&]() {
#pragma unroll
      for (int i = 0; i < KS && attn_in<T>(16 * i, a.D); ++i)
#pragma unroll
        for (int b = 0; b < NB; ++b) s[b] = mma32(Tile::rows(kl, b * 32 + (lane & 31), 16 * i + 8 * half), qf[i], s[b]);
      attn_reads_ahead<T, NB * KS>();
    };
    if (!CAUSAL && seen != ALL) {  // the sums begin at -inf for keys that are left out (their K is zeros)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const v4f x = *reinterpret_cast<const v4f*>(bias + buf * BK + b * 32 + 8 * j + 4 * half);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[b][4 * j + e] = x[e];
        }
      scores();
    } else {
#pragma unroll
      for (int b = 0; b < NB; ++b) s[b] = (v16f)(0.f);
      scores();
    }
    const bool cut = CAUSAL && __any(see - kt < BK - 1);  // by the causal order
    const int last = see - kt;
    const uint64_t keep = last >= 63 ? seen : last < 0 ? 0 : seen & ((2ull << last) - 1);
    if (CAUSAL && (cut || seen != ALL)) {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const unsigned bits = (unsigned)(keep >> (32 * b)) >> (4 * half);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[b][e] = (bits >> reg_row(e, 0)) & 1 ? s[b][e] : -INFINITY;
      }
    }
    float top = s[0][0];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, s[b][e]);
    top = fmaxf(top, other_half(top)) * a.scale_log2;
    const bool raise = top > m + kAttnSlack;
    if (__any(raise)) {  // (each row by its own maximum alone: its bits do not depend on the rows beside it)
      const float shrink = raise ? fast_exp2(m - top) : 1.f;
      m = raise ? top : m;
      l *= shrink;
      if (kt > it.lo) {
#pragma unroll
        for (int b = 0; b < DB; ++b)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[b][e] *= shrink;
      }
    }
    const float base = m == -INFINITY ? 0.f : kAttnUp<T> - m;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[b][e] = fast_exp2(fmaf(s[b][e], a.scale_log2, base));
        sum[e & 3] += s[b][e];
      }
    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    const T* vp = vl;
    if (cut && attn_not_finite<T, BK, DP>(vl)) {
      attn_copy_finite<T, BK, DP>(vl, tiles + 4 * TILE);
      vp = tiles + 4 * TILE;
      left_out.add<T, BK, DP>(vl, 0, last);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const Frag p = to_frag<T>(regs8(s[b], j));
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] = mma32(Tile::cols(vp, b * 32 + 16 * j, d * 32), p, o[d]);
      }
    attn_reads_ahead<T, NB * 2 * DB, true>();
  }

  if (CAUSAL) left_out.apply(o);
  l += other_half(l);
  m -= kAttnUp<T>;
  if (it.part >= 0) {
    // a row of DP sums, then its maximum (in powers of two) and sum
    float* row = a.parts + (((int64_t)it.part * a.kv_heads + hk) * kAttnTile + wave * 32 + (lane & 31)) * (DP + 4);
    store_part<DB>(row, o, live);
    if (live && half == 0) {
      row[DP] = m;
      row[DP + 1] = l;
    }
    return;
  }
  if (!active) return;
  const int64_t q = it.q0 + (int64_t)qi;
  const int64_t at = (q * a.heads + head) * a.D;
  const float inv = l > 0.f ? 1.f / l : l;
  store_row<T, DB>((T*)a.out + at, o, inv, a.D, live);
  if (sizeof(T) == 2 && a.rest) {
    keep_rest<T>(o, inv);
    store_row<T, DB>((T*)a.rest + at, o, 1.f, a.D, live);
  }
  if (a.lse && live && half == 0) a.lse[q * a.heads + head] = l > 0.f ? m + log2f(l) : l == 0.f ? INFINITY : l;
}

// Partial results of split rows into the result, the sums of each weighted
// with 2^(its maximum - the largest): a thread for each four channels.  A row
// has up to some hundred parts (few rows over many keys): more than kAttnFewParts
// are shared between the lanes and joined through LDS in order, fewer are a
// lane's own, and the lanes take rows.  (12 single queries of ~100 parts: 33 us
// unshared, 7 shared; 300 queries x 8 heads of up to 29 parts: 47 and 9 us.)
constexpr int kAttnJoinBlocks = 48;  // workgroups of a tile's join
constexpr int kAttnFewParts = 16;

template <typename T, int DP>
__global__ __launch_bounds__(kAttnThreads) void attn_forward_join_kernel(AttnArgs a) {
  constexpr int QUADS = DP / 4, LANES = kAttnThreads / QUADS;
  __shared__ v4f sums[LANES][QUADS];
  __shared__ float tops[LANES], totals[LANES];
  const int at_join = attn_div(blockIdx.x, a.by_kv_heads), hk = blockIdx.x - at_join * a.kv_heads;
  const AttnJoin jn = a.joins[at_join];
  const int rows = min(a.tile, jn.nq * a.group - jn.row0);
  const int64_t step = (int64_t)a.kv_heads * kAttnTile * (DP + 4);
  const int quad = threadIdx.x % QUADS, lane = threadIdx.x / QUADS;
  const bool share = jn.parts > kAttnFewParts;
  const int stride = share ? 1 : LANES;  // rows of a workgroup at once
  // (m = up, both -inf for parts without keys among them, is weight 1: their sums are zero)
  auto weight = [](float m, float up) { return m == up ? 1.f : fast_exp2(m - up); };
  for (int row0 = blockIdx.y * stride; row0 < rows; row0 += kAttnJoinBlocks * stride) {
    const int row = share ? row0 : row0 + lane;
    const float* p = a.parts + (((int64_t)jn.part * a.kv_heads + hk) * kAttnTile + row) * (DP + 4);
    v4f sum = (v4f)(0.f);
    float m = -INFINITY, l = 0.f;
    if (lane < LANES && row < rows)
      for (int k = share ? lane : 0; k < jn.parts; k += share ? LANES : 1) {
        const float mk = p[k * step + DP], lk = p[k * step + DP + 1];
        const v4f x = *reinterpret_cast<const v4f*>(p + k * step + quad * 4);
        const float up = fmaxf(m, mk), w = weight(m, up), wk = weight(mk, up);
        m = up;
        l = w * l + wk * lk;
        sum = w * sum + wk * x;
      }
    if (share) {
      __syncthreads();
      if (lane < LANES && quad == 0) tops[lane] = m;
      __syncthreads();
      float up = tops[0];
#pragma unroll
      for (int k = 1; k < LANES; ++k) up = fmaxf(up, tops[k]);
      const float w = weight(m, up);
      if (lane < LANES) {
        sums[lane][quad] = w * sum;
        if (quad == 0) totals[lane] = w * l;
      }
      __syncthreads();
      m = up;
      if (lane == 0) {
        l = totals[0];
        sum = sums[0][quad];
#pragma unroll
        for (int k = 1; k < LANES; ++k) {
          l += totals[k];
          sum += sums[k][quad];
        }
      }
    }
    if (lane >= stride || row >= rows) continue;
    const int r = jn.row0 + row, qi = attn_div(r, a.by_group), head = hk * a.group + (r - qi * a.group);
    const int64_t at = (jn.q0 + (int64_t)qi) * a.heads + head;
    if (quad * 4 < a.D) {
      typedef T v4t __attribute__((ext_vector_type(4)));
      const v4f x = sum * (l > 0.f ? 1.f / l : l);
      const v4t y = __builtin_convertvector(x, v4t);
      *reinterpret_cast<v4t*>((T*)a.out + at * a.D + quad * 4) = y;
      if (sizeof(T) == 2 && a.rest)
        *reinterpret_cast<v4t*>((T*)a.rest + at * a.D + quad * 4) =
            __builtin_convertvector(x - __builtin_convertvector(y, v4f), v4t);
    }
    if (a.lse && quad == 0) a.lse[at] = l > 0.f ? m + log2f(l) : l == 0.f ? INFINITY : l;
  }
}

// ------------------------------------------------------------------ backward: queries

// Keys of a step.  At 128 channels of 16 bits the rows of 64 on their way leave no registers for fragments read ahead (the
// products wait for each one): 32 patches of 1,024 x 8 x 128, backward 64 / 32 keys 704 / 692 us.
template <typename T, int DP, int WAVES>
constexpr int attn_dq_keys() {
  return WAVES == 4 && sizeof(T) == 2 && DP == 128 ? 32 : attn_keys<WAVES>();
}
template <typename T, int DP, int WAVES>
constexpr int attn_dq_lds(bool causal) {
  return attn_dq_keys<T, DP, WAVES>() * (causal ? 5 : 4) * DP * (int)sizeof(T);
}

// dQ of a tile of rows, and delta = rowsum(dO o O) for the keys' pass after it:
// the forward's loop with P from the saved L (no running statistics).  dQ in a
// kernel of its own computes S and dP a second time, seven products in all for
// five; one kernel for all three gradients would add dQ with atomics, in an
// order that changes the bits, or write it once for each tile of keys.
//
// As the forward's sizes: 64 channels bf16 272 us (760 TFLOP/s, MFMA busy 44 %, vector
// unit 62: 107 instructions a tile), 128 channels causal 453 us (910, 47 %), fp32 114 us (76, 61 %).
template <typename T, int DP, bool CAUSAL, int WAVES>
__global__ __launch_bounds__(64 * WAVES, (attn_waves<T, DP>())) void attn_dq_kernel(AttnArgs a) {
  using Tile = AttnTile<T, DP>;
  using Frag = typename Tile::Frag;
  constexpr int BK = attn_dq_keys<T, DP, WAVES>();
  using Stage = AttnStage<T, DP, BK, WAVES>;
  constexpr int KS = DP / 16, DB = DP / 32, NB = BK / 32;
  constexpr int TILE = BK * DP;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  T* tiles = reinterpret_cast<T*>(lds);

  int hk;
  const AttnItem it = attn_item(a, hk);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, half = lane >> 5;
  const int rows = it.nq * a.group, r = it.row0 + wave * 32 + (lane & 31);
  const bool active = it.row0 + wave * 32 < rows, live = r < rows;
  const int qi = attn_div(r, a.by_group), in_group = r - qi * a.group, head = hk * a.group + in_group;
  const int first = attn_div(it.row0, a.by_group);  // query of the tile's first row
  const int64_t q = it.q0 + (int64_t)qi, at = q * a.heads + head;

  Frag qf[KS], gf[KS];
  float lse = INFINITY, delta = 0.f;
  {
    const auto qrows = attn_rows((const T*)a.q + hk * a.group * a.q_head, it.q0 + (int64_t)first, a.q_row);
    const auto grows = attn_rows((const T*)a.dout + hk * a.group * a.do_head, it.q0 + (int64_t)first, a.do_row);
    const int qoff = (qi - first) * (int)(a.q_row * sizeof(T)) + in_group * (int)(a.q_head * sizeof(T));
    const int goff = (qi - first) * (int)(a.do_row * sizeof(T)) + in_group * (int)(a.do_head * sizeof(T));
    const T *orow = (const T*)a.o + at * a.D, *rrow = (const T*)a.o_rest + at * a.D;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      qf[s] = load_row8<T>(qrows, qoff, 16 * s + 8 * half, a.D, live);
      gf[s] = load_row8<T>(grows, goff, 16 * s + 8 * half, a.D, live);
      const Frag of = load_row8<T>(orow, 16 * s + 8 * half, a.D, live);
      const Frag rf = load_row8<T>(rrow, 16 * s + 8 * half, a.D, sizeof(T) == 2 && live && a.o_rest);
#pragma unroll
      for (int e = 0; e < 8; ++e) delta = fmaf((float)gf[s][e], (float)of[e] + (float)rf[e], delta);
    }
    delta += other_half(delta);
    if (live) {
      lse = a.lse[at];
      if (half == 0) a.delta[at] = delta;
    }
  }
  const int see = CAUSAL ? qi + it.nk - it.nq : 0x7FFFFFFF;

  Stage ks, vs;
  ks.place(a.D, [&](int x) { return x * (int)(a.k_row * sizeof(T)); });
  vs.place(a.D, [&](int x) { return x * (int)(a.v_row * sizeof(T)); });
  uint8_t chunk_kept[Stage::N], key_kept = 1;
  const uint8_t* mask = a.key_mask ? a.key_mask + it.k0 : nullptr;
  auto fetch = [&](int kt) {
    const int left = it.hi - kt;
    const int64_t row = it.k0 + (int64_t)kt;
    if (mask) {
#pragma unroll
      for (int i = 0; i < Stage::N; ++i) chunk_kept[i] = Stage::row(i) < left ? mask[kt + Stage::row(i)] : 0;
      key_kept = lane < left ? mask[kt + lane] : 0;
    }
    ks.load((const T*)a.k + row * a.k_row + hk * a.k_head, left);
    vs.load((const T*)a.v + row * a.v_row + hk * a.v_head, left);
  };

  v16f dq[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b) dq[b] = (v16f)(0.f);
  AttnPower power;
  if (it.lo < it.hi) fetch(it.lo);
  for (int kt = it.lo, buf = 0; kt < it.hi; kt += BK, buf ^= 1) {
    T* kl = tiles + buf * 2 * TILE;
    T* vl = kl + TILE;
    constexpr uint64_t ALL = ~0ull >> (64 - BK);
    uint64_t seen = ALL;
    if (it.hi - kt < BK) seen >>= BK - (it.hi - kt);
    if (mask) {
      seen &= __ballot(key_kept);
#pragma unroll
      for (int i = 0; i < Stage::N; ++i)
        if (!chunk_kept[i]) ks.reg[i] = vs.reg[i] = (v4u)(0u);
    }
    ks.store(kl);
    vs.store(vl);
    __syncthreads();
    if (kt + BK < it.hi) fetch(kt + BK);
    if (!active || (CAUSAL && !__any(live && kt <= see))) continue;
    const bool cut = CAUSAL && __any(see - kt < BK - 1);
    const int last = see - kt;
    const uint64_t keep = last >= 63 ? seen : last < 0 ? 0 : seen & ((2ull << last) - 1);
    const T* kp = kl;  // (a row that sees a key that is not finite has a dS that is not)
    if (cut && attn_not_finite<T, BK, DP>(kl)) {
      attn_copy_finite<T, BK, DP>(kl, tiles + 4 * TILE);
      kp = tiles + 4 * TILE;
    }
#pragma unroll 1
    for (int b = 0; b < NB; ++b) {
      v16f s = (v16f)(0.f), dp = (v16f)(0.f);
#pragma unroll
      for (int i = 0; i < KS && attn_in<T>(16 * i, a.D); ++i) {
        s = mma32(Tile::rows(kl, b * 32 + (lane & 31), 16 * i + 8 * half), qf[i], s);
        dp = mma32(Tile::rows(vl, b * 32 + (lane & 31), 16 * i + 8 * half), gf[i], dp);
      }
      attn_reads_ahead<T, 2 * KS>();
      const float held = power.up * delta;
#pragma unroll
      for (int e = 0; e < 16; ++e)
        s[e] = fast_exp2(fmaf(s[e], a.scale_log2, -lse)) * (kAttnHeld<T> ? fmaf(dp[e], power.up, -held) : dp[e] - delta);
      if (cut || seen != ALL) {
        const unsigned bits = (unsigned)(keep >> (32 * b)) >> (4 * half);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = (bits >> reg_row(e, 0)) & 1 ? s[e] : 0.f;
      }
      if constexpr (kAttnHeld<T>) power.hold<DB>(s, dq);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const Frag ds = to_frag<T>(regs8(s, j));
#pragma unroll
        for (int d = 0; d < DB; ++d) dq[d] = mma32(Tile::cols(kp, b * 32 + 16 * j, d * 32), ds, dq[d]);
      }
      attn_reads_ahead<T, 2 * DB, true>();
    }
  }

  if constexpr (kAttnHeld<T>) power.release<DB>(dq);
  if (it.part >= 0) {
    store_part<DB>(
        a.parts + (((int64_t)it.part * a.kv_heads + hk) * kAttnTile + wave * 32 + (lane & 31)) * DP, dq, live);
    return;
  }
  if (!active) return;
  store_row<T, DB>((T*)a.dq + at * a.D, dq, a.scale, a.D, live);
}

// ------------------------------------------------------------------ backward: keys

template <typename T, int DP, int WAVES>
constexpr int attn_q_rows() {  // packed rows of a step
  if (WAVES == 1) return 32;
  return DP * (int)sizeof(T) <= 192 ? 64 : 32;
}
template <typename T, int DP, int WAVES>
constexpr int attn_dkv_lds(bool causal) {
  return attn_q_rows<T, DP, WAVES>() * ((causal ? 6 : 4) * DP * (int)sizeof(T) + 4 * 4);
}

// dK and dV of a tile of keys: the waves hold 32 keys each (K, V and both sums in
// registers) while the packed rows' Q, dO, L and delta go by through LDS.
//
// dV and dK of wide 16-bit rows are two launches (WHAT): together K, V and both
// sums of 32 keys take 192 registers of a lane at 128 channels and leave a SIMD
// one wave, whose products and softmax then wait for each other.  Five products
// in the place of four, by two waves a SIMD: 32 patches of 1,024 rows x 8 x 128 bf16,
// the whole backward, 760 -> 680 us (at 96 channels 424 -> 486: one launch there).
//
// As the forward's sizes: 64 channels bf16 345 us (800 TFLOP/s, MFMA busy 45 %, vector
// unit 53: 117 instructions a tile; two waves a SIMD, which wait for each other's products and LDS reads), 128
// channels causal 350 + 470 us (790 and 880, 37 and 42 %), fp32 167
// us (70, 56 %).  (The clock falls to about 1.75 GHz under all of them: fewer cycles buy less time than that.)
constexpr int kAttnDv = 1, kAttnDk = 2;
template <typename T, int DP>
constexpr bool attn_dkv_apart() {
  return sizeof(T) == 2 && DP > 96;
}

template <typename T, int DP, bool CAUSAL, int WAVES, int WHAT>
__global__ __launch_bounds__(64 * WAVES, (WHAT == (kAttnDv | kAttnDk) ? attn_waves<T, DP * 3 / 2>() : attn_waves<T, DP>()))
    void attn_dkv_kernel(AttnArgs a) {
  constexpr bool DV = WHAT & kAttnDv, DK = WHAT & kAttnDk;
  using Tile = AttnTile<T, DP>;
  using Frag = typename Tile::Frag;
  constexpr int BQ = attn_q_rows<T, DP, WAVES>();
  using Stage = AttnStage<T, DP, BQ, WAVES>;
  constexpr int KS = DP / 16, DB = DP / 32, NB = BQ / 32;
  constexpr int TILE = BQ * DP;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  T* tiles = reinterpret_cast<T*>(lds);
  float* stats = reinterpret_cast<float*>(tiles + 4 * TILE);  // two buffers of BQ L, BQ delta
  T* copies = reinterpret_cast<T*>(stats + 4 * BQ);           // CAUSAL: of a Q and a dO tile

  int hk;
  const AttnItem it = attn_item(a, hk);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, half = lane >> 5;
  const int kw = it.row0 + wave * 32, key = kw + (lane & 31);  // in the segment
  const bool active = kw < it.nk, live = key < it.nk;
  const int64_t krow = it.k0 + (int64_t)key;
  const bool kept = live && (!a.key_mask || a.key_mask[krow]);

  Frag kf[KS], vf[DK ? KS : 1];
  const auto krows = attn_rows((const T*)a.k + hk * a.k_head, it.k0 + (int64_t)it.row0, a.k_row);
  const auto vrows = attn_rows((const T*)a.v + hk * a.v_head, it.k0 + (int64_t)it.row0, a.v_row);
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    kf[s] = load_row8<T>(krows, (key - it.row0) * (int)(a.k_row * sizeof(T)), 16 * s + 8 * half, a.D, kept);
    if constexpr (DK) vf[s] = load_row8<T>(vrows, (key - it.row0) * (int)(a.v_row * sizeof(T)), 16 * s + 8 * half, a.D, kept);
  }
  // first packed row that sees this lane's key, and the first that sees any of the wave's
  const int from = CAUSAL ? max(key - (it.nk - it.nq), 0) * a.group : 0;
  const int wave_from = CAUSAL ? max(kw - (it.nk - it.nq), 0) * a.group : 0;

  Stage qs, gs;
  float stat = 0.f;
  auto place = [&](int h0) {  // packed rows from head h0 of a query on
    auto offset = [&](int x, int64_t row, int64_t head) {
      const int dq = attn_div(h0 + x, a.by_group), dh = h0 + x - dq * a.group;
      return dq * (int)(row * sizeof(T)) + dh * (int)(head * sizeof(T));
    };
    qs.place(a.D, [&](int x) { return offset(x, a.q_row, a.q_head); });
    gs.place(a.D, [&](int x) { return offset(x, a.do_row, a.do_head); });
  };
  const bool same_heads = BQ - attn_div(BQ, a.by_group) * a.group == 0;  // every step begins at the same head
  place(it.lo - attn_div(it.lo, a.by_group) * a.group);
  auto fetch = [&](int rt) {
    const int left = it.hi - rt, q0 = attn_div(rt, a.by_group), h0 = rt - q0 * a.group;
    const int64_t q = it.q0 + (int64_t)q0;
    if (!same_heads) place(h0);
    qs.load((const T*)a.q + q * a.q_row + (int64_t)hk * a.group * a.q_head, left);
    gs.load((const T*)a.dout + q * a.do_row + (int64_t)hk * a.group * a.do_head, left);
    if (threadIdx.x < 2 * BQ) {
      const int x = threadIdx.x & (BQ - 1);
      const int dq = attn_div(h0 + x, a.by_group), dh = h0 + x - dq * a.group;
      const int64_t at = (q + dq) * a.heads + hk * a.group + dh;
      // (a row past the end: L = inf makes its P zero)
      stat = threadIdx.x < BQ ? (x < left ? a.lse[at] - kAttnKeysUp<T> : INFINITY)
                              : (x < left ? a.delta[at] * kAttnKeysDown<T> : 0.f);
    }
  };

  v16f dk[DK ? DB : 1], dv[DV ? DB : 1];
#pragma unroll
  for (int b = 0; b < DB; ++b) {
    if constexpr (DK) dk[b] = (v16f)(0.f);
    if constexpr (DV) dv[b] = (v16f)(0.f);
  }
  AttnNotFinite left_out;
  AttnPower power;
  if (it.lo < it.hi) fetch(it.lo);
  for (int rt = it.lo, buf = 0; rt < it.hi; rt += BQ, buf ^= 1) {
    T* ql = tiles + buf * 2 * TILE;
    T* gl = ql + TILE;
    float* st = stats + buf * 2 * BQ;
    qs.store(ql);
    gs.store(gl);
    if (threadIdx.x < 2 * BQ) st[threadIdx.x] = stat;
    __syncthreads();
    if (rt + BQ < it.hi) fetch(rt + BQ);
    if (!active || rt + BQ <= wave_from) continue;
    const bool cut = CAUSAL && __any(from > rt);
    const T *qp = ql, *gp = gl;  // (a row whose Q or dO is not finite has a delta, and so a dS, that is not)
    if (cut && ((DK && attn_not_finite<T, BQ, DP>(ql)) || (DV && attn_not_finite<T, BQ, DP>(gl)))) {
      if constexpr (DK) attn_copy_finite<T, BQ, DP>(ql, copies);
      if constexpr (DV) attn_copy_finite<T, BQ, DP>(gl, copies + TILE);
      qp = copies, gp = copies + TILE;
      if constexpr (DV) left_out.add<T, BQ, DP>(gl, from - rt, BQ);
    }
#pragma unroll 1
    for (int b = 0; b < NB; ++b) {
      v16f s = (v16f)(0.f), dp = (v16f)(0.f);
#pragma unroll
      for (int i = 0; i < KS && attn_in<T>(16 * i, a.D); ++i) {
        s = mma32(Tile::rows(ql, b * 32 + (lane & 31), 16 * i + 8 * half), kf[i], s);
        if constexpr (DK) dp = mma32(Tile::rows(gl, b * 32 + (lane & 31), 16 * i + 8 * half), vf[i], dp);
      }
      attn_reads_ahead<T, (DK ? 2 : 1) * KS>();
      // (L and the rows of the next product are read behind these, out of their count: 8,191 causal rows x 16 x 128 on 4
      // key heads, backward 1,330 -> 1,314 us; 64 patches of 1,024 x 8 x 64 603 -> 595)
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const v4f L = *reinterpret_cast<const v4f*>(st + b * 32 + 8 * j + 4 * half);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[4 * j + e] = fast_exp2(fmaf(s[4 * j + e], a.scale_log2, -L[e]));
      }
      if (cut) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = rt + b * 32 + reg_row(e, half) >= from ? s[e] : 0.f;
      }
      if constexpr (DV) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const Frag p = to_frag<T>(regs8(s, j));
#pragma unroll
        for (int d = 0; d < DB; ++d) dv[d] = mma32(Tile::cols(gp, b * 32 + 16 * j, d * 32), p, dv[d]);
      }
      attn_reads_ahead<T, 2 * DB, true>();
      }
      if constexpr (DK) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const v4f dl = *reinterpret_cast<const v4f*>(st + BQ + b * 32 + 8 * j + 4 * half);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[4 * j + e] *= fmaf(dp[4 * j + e], kAttnKeysDown<T>, -dl[e]);
      }
      if (cut) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = rt + b * 32 + reg_row(e, half) >= from ? s[e] : 0.f;
      }
      if constexpr (kAttnHeld<T>) {
        s *= power.up;
        power.hold<DB>(s, dk);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const Frag ds = to_frag<T>(regs8(s, j));
#pragma unroll
        for (int d = 0; d < DB; ++d) dk[d] = mma32(Tile::cols(qp, b * 32 + 16 * j, d * 32), ds, dk[d]);
      }
      attn_reads_ahead<T, 2 * DB, true>();
      }
    }
  }

  if constexpr (CAUSAL && DV) left_out.apply(dv);
  if constexpr (DK && kAttnHeld<T>) power.release<DB>(dk);
  if (!kept) {  // a masked key gets no gradient
#pragma unroll
    for (int b = 0; b < DB; ++b) {
      if constexpr (DK) dk[b] = (v16f)(0.f);
      if constexpr (DV) dv[b] = (v16f)(0.f);
    }
  }
  if (it.part >= 0) {
    float* row = a.parts + ((((int64_t)it.part * a.kv_heads + hk) * 2) * kAttnTile + wave * 32 + (lane & 31)) * DP;
    if constexpr (DK) store_part<DB>(row, dk, live);
    if constexpr (DV) store_part<DB>(row + kAttnTile * DP, dv, live);
    return;
  }
  if (!active) return;
  const int64_t at = (krow * a.kv_heads + hk) * a.D;
  if constexpr (DK) store_row<T, DB>((T*)a.dk + at, dk, a.scale, a.D, live);
  if constexpr (DV) store_row<T, DB>((T*)a.dv + at, dv, kAttnKeysDown<T>, a.D, live);
}

// Sums of the partial gradients of split tiles, in a fixed order (shares of
// the parts as above): dQ (KEYS = false), or dK and dV.
template <typename T, int DP, bool KEYS>
__global__ __launch_bounds__(kAttnThreads) void attn_sum_parts_kernel(AttnArgs a) {
  typedef T v4t __attribute__((ext_vector_type(4)));
  constexpr int QUADS = DP / 4, LANES = kAttnThreads / QUADS, W = KEYS ? 2 : 1;
  __shared__ v4f sums[LANES][QUADS];
  const int at_join = attn_div(blockIdx.x, a.by_kv_heads), hk = blockIdx.x - at_join * a.kv_heads;
  const AttnJoin jn = a.joins[at_join];
  const int rows = min(a.tile, (KEYS ? jn.nk : jn.nq * a.group) - jn.row0);
  const int64_t step = (int64_t)a.kv_heads * W * kAttnTile * DP;
  const int quad = threadIdx.x % QUADS, lane = threadIdx.x / QUADS;
  const bool share = jn.parts > kAttnFewParts;  // as the forward's join
  for (int i = blockIdx.y * (share ? 1 : LANES); i < W * rows; i += kAttnJoinBlocks * (share ? 1 : LANES)) {
    const int in = share ? i : i + lane;
    const int which = in >= rows, row = in - which * rows;
    const float* p = a.parts + ((((int64_t)jn.part * a.kv_heads + hk) * W + which) * kAttnTile + row) * DP + quad * 4;
    v4f sum = (v4f)(0.f);
    if (lane < LANES && in < W * rows)
      for (int k = share ? lane : 0; k < jn.parts; k += share ? LANES : 1) sum += *reinterpret_cast<const v4f*>(p + k * step);
    if (share) {
      __syncthreads();
      if (lane < LANES) sums[lane][quad] = sum;
      __syncthreads();
      for (int k = 1; k < LANES && lane == 0; ++k) sum += sums[k][quad];
    }
    if (lane >= (share ? 1 : LANES) || in >= W * rows || quad * 4 >= a.D) continue;
    const int r = jn.row0 + row;
    if constexpr (KEYS) {
      const int64_t at = ((jn.k0 + (int64_t)r) * a.kv_heads + hk) * a.D + quad * 4;
      *reinterpret_cast<v4t*>((T*)(which ? a.dv : a.dk) + at) =
          __builtin_convertvector(sum * (which ? kAttnKeysDown<T> : a.scale), v4t);
    } else {
      const int qi = attn_div(r, a.by_group), head = hk * a.group + (r - qi * a.group);
      *reinterpret_cast<v4t*>((T*)a.dq + ((jn.q0 + (int64_t)qi) * a.heads + head) * a.D + quad * 4) =
          __builtin_convertvector(sum * a.scale, v4t);
    }
  }
}

// ------------------------------------------------------------------ launches

enum AttnPass { kAttnForward, kAttnDq, kAttnDkv };

// A workgroup for every item (join) and key head, in as many launches as the grid's limit asks for.
template <typename K>
static int attn_launch(K kernel, int threads, int lds, const AttnArgs& a, hipStream_t s) {
  const int most = (int)(st_most_blocks(threads) / a.kv_heads);
  if (most == 0) return ST_ERR_UNSUPPORTED;
  for (int64_t i = 0; i < a.n_items; i += most) {
    AttnArgs g = a;
    g.items += i;
    g.n_items = (int)(a.n_items - i < most ? a.n_items - i : most);
    g.by_items = attn_divisor(g.n_items);
    kernel<<<(unsigned)(g.n_items * g.kv_heads), threads, lds, s>>>(g);
    ST_CHECK_LAUNCH();
  }
  return ST_OK;
}
template <typename K>
static int attn_join(K kernel, const AttnArgs& a, hipStream_t s) {
  const int most = (int)(st_most_blocks(kAttnThreads) / a.kv_heads);
  if (most == 0) return ST_ERR_UNSUPPORTED;
  for (int64_t i = 0; i < a.n_joins; i += most) {
    AttnArgs g = a;
    g.joins += i;
    g.n_joins = (int)(a.n_joins - i < most ? a.n_joins - i : most);
    kernel<<<dim3((unsigned)(g.n_joins * g.kv_heads), kAttnJoinBlocks), kAttnThreads, 0, s>>>(g);
    ST_CHECK_LAUNCH();
  }
  return ST_OK;
}

template <typename T, int DP, int WAVES>
static int attn_pass(AttnPass pass, const AttnArgs& a, hipStream_t s) {
  auto run = [&](auto kernel, int lds) { return attn_launch(kernel, 64 * WAVES, lds, a, s); };
  if (pass == kAttnForward)
    return run(a.causal ? attn_forward_kernel<T, DP, true, WAVES> : attn_forward_kernel<T, DP, false, WAVES>,
               attn_fwd_lds<T, DP, WAVES>(a.causal));
  if (pass == kAttnDq)
    return run(a.causal ? attn_dq_kernel<T, DP, true, WAVES> : attn_dq_kernel<T, DP, false, WAVES>,
               attn_dq_lds<T, DP, WAVES>(a.causal));
  const int lds = attn_dkv_lds<T, DP, WAVES>(a.causal);
  if constexpr (attn_dkv_apart<T, DP>()) {
    const int rc = run(a.causal ? attn_dkv_kernel<T, DP, true, WAVES, kAttnDv> : attn_dkv_kernel<T, DP, false, WAVES, kAttnDv>, lds);
    if (rc != ST_OK) return rc;
    return run(a.causal ? attn_dkv_kernel<T, DP, true, WAVES, kAttnDk> : attn_dkv_kernel<T, DP, false, WAVES, kAttnDk>, lds);
  } else {
    constexpr int BOTH = kAttnDv | kAttnDk;
    return run(a.causal ? attn_dkv_kernel<T, DP, true, WAVES, BOTH> : attn_dkv_kernel<T, DP, false, WAVES, BOTH>, lds);
  }
}
template <typename T, int DP>
static int attn_dp(AttnPass pass, const AttnArgs& a, hipStream_t s) {
  int rc = ST_ERR_UNSUPPORTED;
  if (a.tile == kAttnTile)
    rc = attn_pass<T, DP, 4>(pass, a, s);
  else if constexpr (DP * sizeof(T) <= ST_ATTN_SMALL_TILE_BYTES)  // (a lane's share of a wider step does not fit its registers)
    rc = attn_pass<T, DP, 1>(pass, a, s);
  if (rc != ST_OK) return rc;
  if (pass == kAttnForward) return attn_join(attn_forward_join_kernel<T, DP>, a, s);
  if (pass == kAttnDq) return attn_join(attn_sum_parts_kernel<T, DP, false>, a, s);
  return attn_join(attn_sum_parts_kernel<T, DP, true>, a, s);
}

template <typename T>
static int attn_run(AttnPass pass, const AttnArgs& a, hipStream_t s) {
  if (a.D <= 32) return attn_dp<T, 32>(pass, a, s);
  if (a.D <= 64) return attn_dp<T, 64>(pass, a, s);
  if (a.D <= 96) return attn_dp<T, 96>(pass, a, s);
  return attn_dp<T, 128>(pass, a, s);
}
int attn_run_bf16(AttnPass pass, const AttnArgs& a, hipStream_t s);
int attn_run_f16(AttnPass pass, const AttnArgs& a, hipStream_t s);
int attn_run_f32(AttnPass pass, const AttnArgs& a, hipStream_t s);

}  // namespace st
