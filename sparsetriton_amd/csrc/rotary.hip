// Rotary positions with several axes: each head's channels are paired, pair p
// belongs to one axis of the row's position and turns by
//   angle = pos[axis(p)] * f(p):   (a, b) -> (a cos - b sin, a sin + b cos),
// channels past the pairs go through unchanged.  The gradient is the turn by
// -angle.  Pairs are (p, p + P) or, interleaved, (2p, 2p + 1).
//
// Bound by memory (each element in and out once), as long as the angles' sines
// are not paid for each head: a workgroup takes `rows` rows, computes their
// rows x P cosines and sines once into LDS, and every head of both tensors
// reads them there.  No table of positions is needed, so any coordinate works.
// The angle is reduced in turns in 64-bit arithmetic (frequency / 2 pi as a
// double, minus the nearest whole turn): an fp32 product pos * f of a few
// hundred radians is already off by 1e-5.
//
// 470,532 rows x 16 heads x 32 bf16: 178 - 185 us (5.3 TB/s; a 1 GiB copy runs at
// 5.1); 60,001 rows x 12 heads x 48 fp32 interleaved: 52 us, its gradient 51 (5.3
// TB/s); 16 rows x 40 heads x 128 bf16: 3.7 us, a launch.
#include "common.h"

namespace st {

constexpr int kRotThreads = 256;
constexpr int kRotTable = 2048;  // cosine / sine pairs in LDS (16 KB)
// Vectors of a workgroup's rows, about, and of a thread's batch.  470,532 rows x 16 x 32 bf16 and 60,001
// rows x 12 x 48 fp32 interleaved: 178 and 45 us; batches of one 184 and 47; 1,024 vectors 189 and 44
// (bf16: an uneven last round of workgroups); one vector at a time, loads behind stores: 181 and 72.
constexpr int kRotItems = 512;
constexpr int kRotBatch = 2;

template <typename T>
struct RotArgs {
  const T* in[2];
  T* out[2];
  int64_t in_row[2], in_head[2];
  int heads[2];
  const void* pos;
  int64_t pos_row;
  const double* turns;
  const int32_t* axis;
  int64_t n;
  int D, P, rows;
  int chunks;                       // vectors of a head: pair vectors, then the unchanged channels'
  int per_row;                      // vectors of a row, both tensors
  uint64_t per_row_inv, chunks_inv; // ceil(2^32 / ...): i / d = i * inv >> 32 for i * d < 2^32
};

template <typename T, int V>
struct RotVec {
  typedef T type __attribute__((ext_vector_type(V)));
};

__device__ __forceinline__ double rot_pos(const int16_t* p, int a) { return p[a]; }
__device__ __forceinline__ double rot_pos(const int32_t* p, int a) { return p[a]; }
__device__ __forceinline__ double rot_pos(const int64_t* p, int a) { return (double)p[a]; }
__device__ __forceinline__ double rot_pos(const float* p, int a) { return p[a]; }

template <typename T, typename PT, int V, bool INTERLEAVED, bool INVERSE>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(RotArgs<T> g) {
  using Vec = typename RotVec<T, V>::type;
  __shared__ float2 table[kRotTable];
  const int64_t row0 = (int64_t)blockIdx.x * g.rows;
  const int rows = g.n - row0 < g.rows ? (int)(g.n - row0) : g.rows;
  const int pair_chunks = INTERLEAVED ? 2 * g.P / V : g.P / V;
  const int items = rows * g.per_row;
  // A thread's next two vectors: their loads all go out before the first store
  // (the compiler keeps a load behind an earlier store), those of the first two
  // before the table is made.
  Vec xa[kRotBatch], xb[kRotBatch];  // a pair's channels, where they are not in one vector
  T* out[kRotBatch];
  int chunk[kRotBatch], at[kRotBatch];
  auto load = [&](int i0) {
#pragma unroll
    for (int u = 0; u < kRotBatch; ++u) {
      const int i = i0 + u * kRotThreads;
      if (i < items) {
        const int r = (int)((uint64_t)i * g.per_row_inv >> 32);
        const int in_row = i - r * g.per_row;
        int h = (int)((uint64_t)in_row * g.chunks_inv >> 32);
        const int ch = in_row - h * g.chunks;
        const int which = h >= g.heads[0];
        h -= which ? g.heads[0] : 0;
        const int d = ch < pair_chunks ? ch * V : 2 * g.P + (ch - pair_chunks) * V;
        const T* in = g.in[which] + (row0 + r) * g.in_row[which] + h * g.in_head[which] + d;
        out[u] = g.out[which] + ((row0 + r) * g.heads[which] + h) * g.D + d;
        chunk[u] = ch;
        at[u] = r * g.P;
        xa[u] = *reinterpret_cast<const Vec*>(in);
        if (!INTERLEAVED && ch < pair_chunks) xb[u] = *reinterpret_cast<const Vec*>(in + g.P);
        if (INTERLEAVED && V == 1 && ch < pair_chunks) xb[u] = *reinterpret_cast<const Vec*>(ch & 1 ? in - 1 : in + 1);
      }
    }
  };
  auto turn = [&](int i0) {
#pragma unroll
    for (int u = 0; u < kRotBatch; ++u) {
      if (i0 + u * kRotThreads < items) {
        const int ch = chunk[u];
        const float2* t = table + at[u];
        if (ch < pair_chunks) {
          if constexpr (INTERLEAVED && V > 1) {
#pragma unroll
            for (int e = 0; e < V; e += 2) {
              const float2 cs = t[ch * (V / 2) + e / 2];
              const float a = (float)xa[u][e], b = (float)xa[u][e + 1];
              xa[u][e] = (T)(a * cs.x - b * cs.y);
              xa[u][e + 1] = (T)(a * cs.y + b * cs.x);
            }
          } else if constexpr (INTERLEAVED) {
            const float2 cs = t[ch >> 1];
            const float a = (float)xa[u][0], b = (float)xb[u][0];
            xa[u][0] = (T)((ch & 1) ? b * cs.y + a * cs.x : a * cs.x - b * cs.y);
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const float2 cs = t[ch * V + e];
              const float a = (float)xa[u][e], b = (float)xb[u][e];
              xa[u][e] = (T)(a * cs.x - b * cs.y);
              xb[u][e] = (T)(a * cs.y + b * cs.x);
            }
            *reinterpret_cast<Vec*>(out[u] + g.P) = xb[u];
          }
        }
        *reinterpret_cast<Vec*>(out[u]) = xa[u];
      }
    }
  };

  load(threadIdx.x);
  for (int i = threadIdx.x; i < rows * g.P; i += kRotThreads) {
    const int r = i / g.P, p = i - r * g.P;
    const PT* pos = (const PT*)g.pos + (row0 + r) * g.pos_row;
    const double t = rot_pos(pos, g.axis[p]) * g.turns[p];
    float s, c;
    sincospif(2.f * (float)(t - rint(t)), &s, &c);
    table[i] = make_float2(c, INVERSE ? -s : s);
  }
  __syncthreads();
  turn(threadIdx.x);
  for (int i0 = threadIdx.x + kRotBatch * kRotThreads; i0 < items; i0 += kRotBatch * kRotThreads) {
    load(i0);
    turn(i0);
  }
}

// Whether vectors of V channels cut every head evenly and lie at their own size's alignment.
template <typename T, int V>
static bool rot_vec_ok(const RotArgs<T>& g, bool interleaved) {
  if (g.D % V || (interleaved ? 2 * g.P : g.P) % V || (2 * g.P) % V) return false;
  for (int w = 0; w < 2; ++w) {
    if (!g.heads[w]) continue;
    if (g.in_row[w] % V || g.in_head[w] % V) return false;
    if (((uintptr_t)g.in[w] | (uintptr_t)g.out[w]) % (V * sizeof(T))) return false;
  }
  return true;
}

template <typename T, typename PT, int V>
static int rot_launch(RotArgs<T> g, bool interleaved, bool inverse, hipStream_t s) {
  const int pairs = interleaved ? 2 * g.P / V : g.P / V;
  g.chunks = pairs + (g.D - 2 * g.P) / V;
  const int64_t per_row = (int64_t)(g.heads[0] + g.heads[1]) * g.chunks;
  if (per_row >= (1 << 15)) return ST_ERR_UNSUPPORTED;
  g.per_row = (int)per_row;
  // rows of a workgroup: what LDS and a few vectors a thread hold, fewer while there are not 1024 workgroups
  int64_t rows = g.P ? kRotTable / g.P : kRotItems;
  if (kRotItems / per_row < rows) rows = kRotItems / per_row;
  if (g.n / 1024 < rows) rows = g.n / 1024;
  g.rows = rows > 0 ? (int)rows : 1;
  g.per_row_inv = ((1ull << 32) + g.per_row - 1) / g.per_row;
  g.chunks_inv = ((1ull << 32) + g.chunks - 1) / g.chunks;
  auto kernel = interleaved ? (inverse ? rotary_kernel<T, PT, V, true, true> : rotary_kernel<T, PT, V, true, false>)
                            : (inverse ? rotary_kernel<T, PT, V, false, true> : rotary_kernel<T, PT, V, false, false>);
  const int64_t n = g.n, most = st_most_blocks(kRotThreads) * g.rows;  // rows of a launch
  for (int64_t row = 0; row < n; row += most) {
    RotArgs<T> part = g;
    part.n = n - row < most ? n - row : most;
    part.pos = (const PT*)g.pos + row * g.pos_row;
    for (int w = 0; w < 2; ++w) {
      part.in[w] = g.in[w] + row * g.in_row[w];
      part.out[w] = g.out[w] + row * g.heads[w] * g.D;
    }
    kernel<<<st_blocks(part.n, g.rows), kRotThreads, 0, s>>>(part);
    ST_CHECK_LAUNCH();
  }
  return ST_OK;
}

template <typename T, typename PT>
static int rot_vectors(const RotArgs<T>& g, bool interleaved, bool inverse, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  if (rot_vec_ok<T, V>(g, interleaved)) return rot_launch<T, PT, V>(g, interleaved, inverse, s);
  if (rot_vec_ok<T, V / 2>(g, interleaved)) return rot_launch<T, PT, V / 2>(g, interleaved, inverse, s);
  return rot_launch<T, PT, 1>(g, interleaved, inverse, s);
}

template <typename T>
static int rot_positions(const st_rotary_args* a, int pos_dtype, hipStream_t s) {
  RotArgs<T> g{};
  g.in[0] = (const T*)a->q, g.in[1] = (const T*)a->k;
  g.out[0] = (T*)a->q_out, g.out[1] = (T*)a->k_out;
  g.in_row[0] = a->q_row, g.in_row[1] = a->k_row;
  g.in_head[0] = a->q_head, g.in_head[1] = a->k_head;
  g.heads[0] = a->q ? a->heads : 0, g.heads[1] = a->k ? a->kv_heads : 0;
  g.pos = a->positions, g.pos_row = a->pos_row;
  g.turns = a->turns, g.axis = a->axis;
  g.n = a->n, g.D = a->dim, g.P = a->pairs;
  const bool il = a->interleaved != 0, inv = a->inverse != 0;
  switch (pos_dtype) {
    case ST_COORD_I16:
      return rot_vectors<T, int16_t>(g, il, inv, s);
    case ST_COORD_I32:
      return rot_vectors<T, int32_t>(g, il, inv, s);
    case ST_COORD_I64:
      return rot_vectors<T, int64_t>(g, il, inv, s);
    case ST_POS_F32:
      return rot_vectors<T, float>(g, il, inv, s);
    default:
      return ST_ERR_UNSUPPORTED;
  }
}

}  // namespace st

extern "C" int st_rotary(const st_rotary_args* a, st_stream_t stream) {
  if (!a || a->n < 0 || a->dim <= 0 || a->pairs < 0 || 2 * a->pairs > a->dim || a->pairs > st::kRotTable) return ST_ERR_ARG;
  if ((!a->q && !a->k) || (a->q && (!a->q_out || a->heads <= 0)) || (a->k && (!a->k_out || a->kv_heads <= 0)))
    return a->n == 0 ? ST_OK : ST_ERR_ARG;
  if (a->n == 0) return ST_OK;
  if (a->pairs && (!a->positions || !a->turns || !a->axis)) return ST_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  switch (a->dtype) {
    case ST_F32:
      return st::rot_positions<float>(a, a->pos_dtype, s);
    case ST_F16:
      return st::rot_positions<_Float16>(a, a->pos_dtype, s);
    case ST_BF16:
      return st::rot_positions<__bf16>(a, a->pos_dtype, s);
    default:
      return ST_ERR_UNSUPPORTED;
  }
}
