// Norm of every head of queries and keys, and their rotary positions, in one
// pass.  For a head x of D channels, the weight w (of the queries' or the keys'
// heads) and the turn R of the row's position (rotary.hip):
//   s = 1 / sqrt(mean_c x^2 + eps),   y = R (x s w)
// and its gradients, with g = R^-1 dy:
//   dx = s (g w - x s^2 mean_c(g w x)),   dw = sum over rows and heads of g x s.
// Nothing but the inputs is kept for the backward: s is a sum over channels
// that it reads anyway.  All sums are fp32, one rounding at the end.
//
// Bound by memory: each element in and out once, as rotary.hip, whose layout
// of a head this is -- a lane holds a vector of V channels and the vector of
// the channels that they turn with -- with the lanes of a head side by side,
// so that both sums over its channels are lane moves.  The row's cosines and
// sines and the weights are in LDS, shared by its heads.  The backward's
// workgroups walk ranges of rows and keep dw of their lanes' channels in
// registers; one partial a workgroup, added in a fixed order by a second kernel.
#include "common.h"
#include "sum_parts.h"
#include "wave_sum.h"

namespace st {

constexpr int kQkThreads = 256;
constexpr int kQkTable = 2048;  // cosine / sine pairs in LDS (16 KB)
constexpr int kQkItems = 512;   // lanes' worth of heads in a forward workgroup, about
constexpr int kQkBatch = 2;     // heads that a forward lane has on their way at once
constexpr int kQkMaxGroups = 1024;  // workgroups of the backward, each leaving one partial

template <typename T>
struct QkArgs {
  const T* in[2];
  const T* dy[2];  // backward
  T* out[2];       // forward: y, backward: dx
  int64_t in_row[2], in_head[2], dy_row[2], dy_head[2];
  const void* w[2];  // NULL: ones
  int w_f32;
  int heads[2], all;
  const void* pos;
  int pos_dtype;
  int64_t pos_row;
  const double* turns;
  const int32_t* axis;
  int64_t n;
  int D, P, rows;
  int chunks, lanes, lane_bits;  // vectors of a head, and the power of two of lanes that hold them
  uint64_t all_inv, heads_inv[2];  // ceil(2^32 / ...): i / d = i * inv >> 32 for i * d < 2^32
  float eps, inv_d;
  float* parts;
};

template <typename T, int V>
struct QkVec {
  typedef T type __attribute__((ext_vector_type(V)));
};

__device__ __forceinline__ double qk_pos(const void* p, int dtype, int64_t i) {
  switch (dtype) {
    case ST_COORD_I16:
      return ((const int16_t*)p)[i];
    case ST_COORD_I32:
      return ((const int32_t*)p)[i];
    case ST_COORD_I64:
      return (double)((const int64_t*)p)[i];
    default:
      return ((const float*)p)[i];
  }
}

// Sums over the lanes of each head.  All lanes of a wave take part.
template <int N>
__device__ __forceinline__ void qk_sum(float (&v)[N], int lanes) {
  auto step = [&](auto other) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += other(v[i]);
  };
  if (lanes >= 2) step([](float x) { return dpp_move<0xB1>(x); });
  if (lanes >= 4) step([](float x) { return dpp_move<0x4E>(x); });
  if (lanes >= 8) step([](float x) { return dpp_move<0x141>(x); });
  if (lanes >= 16) step([](float x) { return dpp_move<0x140>(x); });
  if (lanes >= 32) step([](float x) { return other_row(x); });
  if (lanes >= 64) step([](float x) { return other_half(x); });
}

// How a lane holds its share of a head: NV chunks `lanes` apart.  A chunk is a
// vector of V channels from `at` on and, where its channels turn with others
// (second()), the vector of those, `partner` further on.  Interleaved vectors of
// more than one channel hold both of each pair.
template <typename T, int V, int NV, bool INTERLEAVED>
struct QkLane {
  using Vec = typename QkVec<T, V>::type;
  static constexpr bool kInside = INTERLEAVED && V > 1;
  int ch, pair_chunks, chunks, lanes, P;

  __device__ __forceinline__ QkLane(const QkArgs<T>& g)
      : ch(threadIdx.x & (g.lanes - 1)), pair_chunks(kInside ? 2 * g.P / V : g.P / V), chunks(g.chunks), lanes(g.lanes), P(g.P) {}
  __device__ __forceinline__ int chunk(int k) const { return ch + k * lanes; }
  __device__ __forceinline__ bool live(int k) const { return chunk(k) < chunks; }
  __device__ __forceinline__ bool pair(int k) const { return chunk(k) < pair_chunks; }
  __device__ __forceinline__ bool second(int k) const { return !kInside && pair(k); }
  __device__ __forceinline__ int partner() const { return INTERLEAVED ? 1 : P; }
  __device__ __forceinline__ int at(int k) const {
    const int c = chunk(k);
    return c < pair_chunks ? c * (INTERLEAVED && V == 1 ? 2 : V) : 2 * P + (c - pair_chunks) * V;
  }
  __device__ __forceinline__ void load(const T* head, bool there, Vec (&a)[NV], Vec (&b)[NV]) const {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      a[k] = b[k] = (Vec)(T)0.f;
      if (there && live(k)) {
        a[k] = *reinterpret_cast<const Vec*>(head + at(k));
        if (second(k)) b[k] = *reinterpret_cast<const Vec*>(head + at(k) + partner());
      }
    }
  }
  __device__ __forceinline__ void store(T* head, bool there, const float (&a)[NV][V], const float (&b)[NV][V]) const {
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (there && live(k)) {
        Vec x, y;
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = (T)a[k][e], y[e] = (T)b[k][e];
        *reinterpret_cast<Vec*>(head + at(k)) = x;
        if (second(k)) *reinterpret_cast<Vec*>(head + at(k) + partner()) = y;
      }
  }
  // (a, b) turned by the row's table; forwards or back
  template <bool BACK>
  __device__ __forceinline__ void turn(const float2* table, float (&a)[NV][V], float (&b)[NV][V]) const {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (!pair(k)) continue;
      if constexpr (kInside) {
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          const float2 t = table[chunk(k) * (V / 2) + e / 2];
          const float s = BACK ? -t.y : t.y, x = a[k][e], y = a[k][e + 1];
          a[k][e] = x * t.x - y * s;
          a[k][e + 1] = x * s + y * t.x;
        }
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float2 t = table[chunk(k) * V + e];
          const float s = BACK ? -t.y : t.y, x = a[k][e], y = b[k][e];
          a[k][e] = x * t.x - y * s;
          b[k][e] = x * s + y * t.x;
        }
      }
    }
  }
  // the weights of the lane's channels
  __device__ __forceinline__ void weights(const float* w, float (&a)[NV][V], float (&b)[NV][V]) const {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        a[k][e] = live(k) ? w[at(k) + e] : 0.f;
        b[k][e] = second(k) ? w[at(k) + partner() + e] : 0.f;
      }
  }
};

// Cosines and sines of `rows` rows from row0 on, and the weights, in LDS.
template <typename T>
__device__ __forceinline__ void qk_table(const QkArgs<T>& g, int64_t row0, int rows, float2* table) {
  for (int i = threadIdx.x; i < rows * g.P; i += kQkThreads) {
    const int r = i / g.P, p = i - r * g.P;
    const double t = qk_pos(g.pos, g.pos_dtype, (row0 + r) * g.pos_row + g.axis[p]) * g.turns[p];
    float s, c;
    sincospif(2.f * (float)(t - rint(t)), &s, &c);
    table[i] = make_float2(c, s);
  }
}
template <typename T>
__device__ __forceinline__ void qk_weights(const QkArgs<T>& g, float* weights) {
  for (int i = threadIdx.x; i < 2 * ST_QK_MAX_DIM; i += kQkThreads) {
    const int which = i / ST_QK_MAX_DIM, d = i % ST_QK_MAX_DIM;
    const void* w = g.w[which];
    if (d < g.D) weights[i] = !w ? 1.f : g.w_f32 ? ((const float*)w)[d] : (float)((const T*)w)[d];
  }
}

template <typename T, int V, int NV, bool INTERLEAVED>
__global__ __launch_bounds__(kQkThreads) void qk_forward_kernel(QkArgs<T> g) {
  using Lane = QkLane<T, V, NV, INTERLEAVED>;
  using Vec = typename Lane::Vec;
  __shared__ float2 table[kQkTable];
  __shared__ __attribute__((aligned(16))) float weights[2 * ST_QK_MAX_DIM];
  const int64_t row0 = (int64_t)blockIdx.x * g.rows;
  const int rows = g.n - row0 < g.rows ? (int)(g.n - row0) : g.rows;
  const int items = rows * g.all, side = kQkThreads >> g.lane_bits, group = threadIdx.x >> g.lane_bits;
  const Lane lane(g);
  // (the loads of the first heads go out before the table is made, those of a batch before its first store)
  Vec xa[kQkBatch][NV], xb[kQkBatch][NV];
  T* out[kQkBatch];
  int row[kQkBatch], which[kQkBatch];
  bool there[kQkBatch];
  auto load = [&](int i0) {
#pragma unroll
    for (int u = 0; u < kQkBatch; ++u) {
      const int i = i0 + u * side + group;
      there[u] = i < items;
      const int r = there[u] ? (int)((uint64_t)i * g.all_inv >> 32) : 0;
      int h = there[u] ? i - r * g.all : 0;
      row[u] = r;
      which[u] = h >= g.heads[0];
      h -= which[u] ? g.heads[0] : 0;
      const T* in = which[u] ? g.in[1] + (row0 + r) * g.in_row[1] + h * g.in_head[1] : g.in[0] + (row0 + r) * g.in_row[0] + h * g.in_head[0];
      out[u] = (which[u] ? g.out[1] : g.out[0]) + ((row0 + r) * (which[u] ? g.heads[1] : g.heads[0]) + h) * g.D;
      lane.load(in, there[u], xa[u], xb[u]);
    }
  };
  load(0);
  qk_table(g, row0, rows, table);
  qk_weights(g, weights);
  __syncthreads();
  for (int i0 = 0; i0 < items; i0 += kQkBatch * side) {
    if (i0) load(i0);
    float sum[kQkBatch];
#pragma unroll
    for (int u = 0; u < kQkBatch; ++u) {
      sum[u] = 0.f;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) sum[u] += (float)xa[u][k][e] * (float)xa[u][k][e] + (float)xb[u][k][e] * (float)xb[u][k][e];
    }
    qk_sum(sum, g.lanes);
#pragma unroll
    for (int u = 0; u < kQkBatch; ++u) {
      const float s = 1.f / sqrtf(sum[u] * g.inv_d + g.eps);
      float a[NV][V], b[NV][V];
      lane.weights(weights + which[u] * ST_QK_MAX_DIM, a, b);
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) a[k][e] *= (float)xa[u][k][e] * s, b[k][e] *= (float)xb[u][k][e] * s;
      lane.template turn<false>(table + row[u] * g.P, a, b);
      lane.store(out[u], there[u], a, b);
    }
  }
}

template <typename T, int V, int NV, bool INTERLEAVED>
__global__ __launch_bounds__(kQkThreads) void qk_backward_kernel(QkArgs<T> g) {
  using Lane = QkLane<T, V, NV, INTERLEAVED>;
  using Vec = typename Lane::Vec;
  __shared__ float2 table[kQkTable];
  __shared__ __attribute__((aligned(16))) float weights[2 * ST_QK_MAX_DIM];
  const int side = kQkThreads >> g.lane_bits, group = threadIdx.x >> g.lane_bits;
  const Lane lane(g);
  const int64_t per = (g.n + gridDim.x - 1) / gridDim.x, end = per * (blockIdx.x + 1) < g.n ? per * (blockIdx.x + 1) : g.n;
  float da[2][NV][V], db[2][NV][V];
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) da[w][k][e] = db[w][k][e] = 0.f;
  qk_weights(g, weights);
  for (int64_t row0 = per * blockIdx.x; row0 < end; row0 += g.rows) {
    const int rows = end - row0 < g.rows ? (int)(end - row0) : g.rows;
    qk_table(g, row0, rows, table);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const int items = rows * g.heads[w];
      for (int i0 = 0; i0 < items; i0 += side) {
        const int i = i0 + group;
        const bool there = i < items;
        const int r = there ? (int)((uint64_t)i * g.heads_inv[w] >> 32) : 0, h = there ? i - r * g.heads[w] : 0;
        Vec xa[NV], xb[NV], ga[NV], gb[NV];
        lane.load(g.in[w] + (row0 + r) * g.in_row[w] + h * g.in_head[w], there, xa, xb);
        lane.load(g.dy[w] + (row0 + r) * g.dy_row[w] + h * g.dy_head[w], there, ga, gb);
        float a[NV][V], b[NV][V], wa[NV][V], wb[NV][V];
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
          for (int e = 0; e < V; ++e) a[k][e] = (float)ga[k][e], b[k][e] = (float)gb[k][e];
        lane.template turn<true>(table + r * g.P, a, b);
        lane.weights(weights + w * ST_QK_MAX_DIM, wa, wb);
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float x = (float)xa[k][e], y = (float)xb[k][e];
            wa[k][e] *= a[k][e], wb[k][e] *= b[k][e];
            sum[0] += x * x + y * y;
            sum[1] += wa[k][e] * x + wb[k][e] * y;
          }
        qk_sum(sum, g.lanes);
        const float s = there ? 1.f / sqrtf(sum[0] * g.inv_d + g.eps) : 0.f, c = sum[1] * g.inv_d * s * s;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float x = (float)xa[k][e], y = (float)xb[k][e];
            da[w][k][e] += a[k][e] * x * s, db[w][k][e] += b[k][e] * y * s;
            a[k][e] = s * (wa[k][e] - x * c), b[k][e] = s * (wb[k][e] - y * c);
          }
        lane.store(g.out[w] + ((row0 + r) * g.heads[w] + h) * g.D, there, a, b);
      }
    }
    __syncthreads();
  }
  if (!g.parts) return;
  // the heads side by side in a wave, then the four waves, in a fixed order; the table's room holds three waves' sums
  static_assert(3 * 2 * ST_QK_MAX_DIM * sizeof(float) <= sizeof(table), "three waves' sums");
  float* sums = reinterpret_cast<float*>(table);
  const int wave = threadIdx.x >> 6;
  const bool mine = (threadIdx.x & 63) < g.lanes;
  float* out = g.parts + (int64_t)blockIdx.x * 2 * g.D;
  auto each = [&](auto f) {
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if (lane.live(k)) f(w * g.D + lane.at(k) + e, da[w][k][e]);
          if (lane.second(k)) f(w * g.D + lane.at(k) + lane.partner() + e, db[w][k][e]);
        }
  };
  for (int o = g.lanes; o < 64; o *= 2)
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          da[w][k][e] += __shfl_xor(da[w][k][e], o, 64);
          db[w][k][e] += __shfl_xor(db[w][k][e], o, 64);
        }
  if (wave > 0 && mine) each([&](int at, float v) { sums[(wave - 1) * 2 * ST_QK_MAX_DIM + at] = v; });
  __syncthreads();
  if (wave == 0 && mine)
    each([&](int at, float v) {
#pragma unroll
      for (int o = 0; o < 3; ++o) v += sums[o * 2 * ST_QK_MAX_DIM + at];
      out[at] = v;
    });
}

// ------------------------------------------------------------------ host

// Whether vectors of V channels cut every head evenly and lie at their own size's alignment.
template <typename T, int V>
static bool qk_vec_ok(const QkArgs<T>& g, bool interleaved) {
  if (g.D % V || (interleaved ? 2 * g.P : g.P) % V) return false;
  for (int w = 0; w < 2; ++w) {
    if (!g.heads[w]) continue;
    if (g.in_row[w] % V || g.in_head[w] % V) return false;
    if (g.dy[w] && (g.dy_row[w] % V || g.dy_head[w] % V)) return false;
    if (((uintptr_t)g.in[w] | (uintptr_t)g.dy[w] | (uintptr_t)g.out[w]) % (V * sizeof(T))) return false;
  }
  return true;
}

// Rows whose table is in LDS at once.
static int64_t qk_table_rows(int P) { return P ? kQkTable / P : kQkTable; }

// Workgroups of the backward: a row each while there are fewer than its limit.
static int64_t qk_groups(int64_t n) { return n < kQkMaxGroups ? (n > 0 ? n : 1) : kQkMaxGroups; }

template <typename T, int V, int NV, bool INTERLEAVED>
static int qk_launch(QkArgs<T> g, bool backward, hipStream_t s) {
  auto inv = [](int64_t d) { return d ? ((1ull << 32) + d - 1) / d : 0; };
  g.all_inv = inv(g.all);
  for (int w = 0; w < 2; ++w) g.heads_inv[w] = inv(g.heads[w]);
  if (backward) {
    // rows of a table: what LDS holds, and i * heads within the inverse's reach
    int64_t rows = qk_table_rows(g.P);
    const int64_t most = g.heads[0] > g.heads[1] ? g.heads[0] : g.heads[1];
    while (rows > 1 && rows * most * most >= (1ll << 32)) rows /= 2;
    g.rows = (int)rows;
    qk_backward_kernel<T, V, NV, INTERLEAVED><<<(unsigned)qk_groups(g.n), kQkThreads, 0, s>>>(g);
    ST_CHECK_LAUNCH();
    return ST_OK;
  }
  // rows of a workgroup: what LDS and a few heads a lane hold, fewer while there are not 1024 workgroups
  int64_t rows = qk_table_rows(g.P);
  const int64_t per_row = (int64_t)g.all * g.lanes;
  if (kQkItems / per_row < rows) rows = kQkItems / per_row;
  if (g.n / 1024 < rows) rows = g.n / 1024;
  g.rows = rows > 0 ? (int)rows : 1;
  const int64_t n = g.n, most = st_most_blocks(kQkThreads) * g.rows;  // rows of a launch
  for (int64_t row = 0; row < n; row += most) {
    QkArgs<T> part = g;
    part.n = n - row < most ? n - row : most;
    const int64_t esz = g.pos_dtype == ST_COORD_I16 ? 2 : g.pos_dtype == ST_COORD_I64 ? 8 : 4;
    part.pos = (const char*)g.pos + row * g.pos_row * esz;
    for (int w = 0; w < 2; ++w) {
      part.in[w] = g.in[w] + row * g.in_row[w];
      part.out[w] = g.out[w] + row * g.heads[w] * g.D;
    }
    qk_forward_kernel<T, V, NV, INTERLEAVED><<<st_blocks(part.n, g.rows), kQkThreads, 0, s>>>(part);
    ST_CHECK_LAUNCH();
  }
  return ST_OK;
}

template <typename T, int V>
static int qk_vectors(QkArgs<T> g, bool interleaved, bool backward, hipStream_t s) {
  g.chunks = (interleaved && V > 1 ? 2 * g.P / V : g.P / V) + (g.D - 2 * g.P) / V;
  g.lanes = 1, g.lane_bits = 0;
  while (g.lanes < g.chunks && g.lanes < 64) g.lanes *= 2, ++g.lane_bits;
  if (g.chunks <= 64)
    return interleaved ? qk_launch<T, V, 1, true>(g, backward, s) : qk_launch<T, V, 1, false>(g, backward, s);
  if constexpr (ST_QK_MAX_DIM / V > 64)  // (heads longer than 64 vectors)
    return interleaved ? qk_launch<T, V, ST_QK_MAX_DIM / V / 64, true>(g, backward, s)
                       : qk_launch<T, V, ST_QK_MAX_DIM / V / 64, false>(g, backward, s);
  return ST_ERR_UNSUPPORTED;
}

template <typename T>
static int qk_run(const st_qk_norm_args* a, bool backward, hipStream_t s) {
  QkArgs<T> g{};
  const void *in[2] = {a->q, a->k}, *dy[2] = {a->dq_out, a->dk_out}, *w[2] = {a->q_weight, a->k_weight};
  void* out[2] = {backward ? a->dq : a->q_out, backward ? a->dk : a->k_out};
  const int64_t rows[2] = {a->q_row, a->k_row}, heads[2] = {a->q_head, a->k_head};
  const int64_t dy_rows[2] = {a->dq_row, a->dk_row}, dy_heads[2] = {a->dq_head, a->dk_head};
  for (int t = 0; t < 2; ++t) {
    g.heads[t] = in[t] ? (t ? a->kv_heads : a->heads) : 0;
    g.in[t] = (const T*)in[t], g.out[t] = (T*)out[t], g.w[t] = w[t];
    g.in_row[t] = rows[t], g.in_head[t] = heads[t];
    if (backward) g.dy[t] = (const T*)dy[t], g.dy_row[t] = dy_rows[t], g.dy_head[t] = dy_heads[t];
  }
  g.w_f32 = a->weight_dtype == ST_F32;
  g.all = g.heads[0] + g.heads[1];
  g.pos = a->positions, g.pos_dtype = a->pos_dtype, g.pos_row = a->pos_row;
  g.turns = a->turns, g.axis = a->axis;
  g.n = a->n, g.D = a->dim, g.P = a->pairs;
  g.eps = a->eps, g.inv_d = 1.f / (float)a->dim;
  g.parts = backward && (a->dq_weight || a->dk_weight) ? a->workspace : nullptr;
  const bool il = a->interleaved != 0;
  constexpr int V = 16 / sizeof(T);
  int rc = ST_OK;
  if (g.n == 0)
    ;  // (no rows: the weights' gradients are sums of nothing)
  else if (qk_vec_ok<T, V>(g, il))
    rc = qk_vectors<T, V>(g, il, backward, s);
  else if (qk_vec_ok<T, V / 2>(g, il))
    rc = qk_vectors<T, V / 2>(g, il, backward, s);
  else
    rc = qk_vectors<T, 1>(g, il, backward, s);
  if (rc != ST_OK || !g.parts) return rc;
  const int64_t groups = g.n ? qk_groups(g.n) : 0;
  return g.w_f32 ? sum_parts<float>(g.parts, groups, g.D, a->dq_weight, a->dk_weight, s)
                 : sum_parts<T>(g.parts, groups, g.D, a->dq_weight, a->dk_weight, s);
}

static int qk_check(const st_qk_norm_args* a, bool backward) {
  if (!a || a->n < 0 || a->dim <= 0 || a->pairs < 0 || 2 * a->pairs > a->dim || !(a->eps >= 0.f)) return ST_ERR_ARG;
  if (a->dim > ST_QK_MAX_DIM) return ST_ERR_UNSUPPORTED;
  if (a->dtype != ST_F32 && a->dtype != ST_F16 && a->dtype != ST_BF16) return ST_ERR_UNSUPPORTED;
  if (a->weight_dtype != a->dtype && a->weight_dtype != ST_F32) return ST_ERR_UNSUPPORTED;
  if (a->pos_dtype != ST_COORD_I16 && a->pos_dtype != ST_COORD_I32 && a->pos_dtype != ST_COORD_I64 &&
      a->pos_dtype != ST_POS_F32)
    return ST_ERR_UNSUPPORTED;
  const int64_t heads = a->q ? a->heads : 0, kv_heads = a->k ? a->kv_heads : 0;
  if (heads < 0 || kv_heads < 0 || heads + kv_heads >= (1 << 15)) return ST_ERR_UNSUPPORTED;
  if (a->n == 0) return ST_OK;
  if (heads + kv_heads == 0 || (a->q && (heads == 0 || !(backward ? a->dq : a->q_out))) ||
      (a->k && (kv_heads == 0 || !(backward ? a->dk : a->k_out))))
    return ST_ERR_ARG;
  if (backward && ((a->q && !a->dq_out) || (a->k && !a->dk_out))) return ST_ERR_ARG;
  if (a->pairs && (!a->positions || !a->turns || !a->axis)) return ST_ERR_ARG;
  return ST_OK;
}

static int qk_dispatch(const st_qk_norm_args* a, bool backward, hipStream_t s) {
  if (a->dtype == ST_F32) return qk_run<float>(a, backward, s);
  if (a->dtype == ST_F16) return qk_run<_Float16>(a, backward, s);
  return qk_run<__bf16>(a, backward, s);
}

}  // namespace st

extern "C" int st_qk_norm_rotary(const st_qk_norm_args* a, st_stream_t stream) {
  const int rc = st::qk_check(a, false);
  if (rc != ST_OK || a->n == 0) return rc;
  return st::qk_dispatch(a, false, (hipStream_t)stream);
}

extern "C" int st_qk_norm_rotary_workspace(int64_t n, int dim, int64_t* floats) {
  if (n < 0 || dim <= 0 || dim > ST_QK_MAX_DIM || !floats) return ST_ERR_ARG;
  *floats = st::qk_groups(n) * 2 * dim;
  return ST_OK;
}

extern "C" int st_qk_norm_rotary_backward(const st_qk_norm_args* a, st_stream_t stream) {
  const int rc = st::qk_check(a, true);
  if (rc != ST_OK) return rc;
  const bool weights = a->dq_weight || a->dk_weight;
  if (a->n == 0 && !weights) return ST_OK;
  int64_t need = 0;
  st_qk_norm_rotary_workspace(a->n, a->dim, &need);
  if (weights && (!a->workspace || a->workspace_floats < need)) return ST_ERR_ARG;
  return st::qk_dispatch(a, true, (hipStream_t)stream);
}
