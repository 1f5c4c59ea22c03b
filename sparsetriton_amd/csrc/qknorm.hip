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
//
// Kernel times (a 1 GiB copy runs at 5.11 TB/s), forward / backward: 470,532 rows x
// (8 + 8) heads x 32 bf16 181 / 317 us (5.3 and 4.6 TB/s), 65,537 x (16 + 4) x 128
// bf16 116 / 223 (5.8, 4.5), 60,001 x (6 + 6) x 48 fp32 interleaved 52 / 89 (5.3,
// 4.7); the rotation alone, rotary.hip, takes 182, 118 and 44.  Offsets that grow
// by steps for ones computed anew at each head, and each head's loads ahead of
// the one before it: forward 212, 145, 78 us before.
#include "common.h"
#include "mfma.h"
#include "sum_parts.h"
#include "wave_sum.h"

namespace st {

constexpr int kQkThreads = 256;
constexpr int kQkTable = 2048;  // cosine / sine pairs in LDS (16 KB)
// Lanes' worth of heads in a forward workgroup, about (512 / 1,024: 65,537 x (16 + 4) x 128 bf16 142 / 125 us,
// 470,532 x (8 + 8) x 32 184 / 185).
constexpr int kQkItems = 1024;
constexpr int64_t kQkReach = ST_QK_REACH;  // bytes from a workgroup's first head to its last one's end
static_assert(kQkReach <= kOobOffset - 4 * ST_QK_MAX_DIM, "a head's last channel is below the offset that reads zeros");
// Workgroups of the backward, each leaving one partial: three a compute unit, what the 159 - 162 registers of whole 16-bit vectors,
// apart or inside, leave room for (1,024 of them, a last quarter alone: 364 us at 470,532 x 16 x 32 bf16 for 316).  The other
// forms (63 - 123 registers; a channel a lane up to 154) have room for up to seven and are given as many, which is not tuned for them.
constexpr int kQkMaxGroups = 768;

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
  int chunks, lanes, lane_bits;  // of a head, and the power of two of lanes that hold them
  int table_row;                 // entries of a row's table: the pairs, and one for each of the other chunks' turns
  float heads_inv[2];              // 1 / heads: (i + 1/2) / heads tells i's row, for the i < 256 of a first step
  int step_row[2], step_h[2];      // a step of `side` heads, in rows and heads
  float eps, inv_d;
  int64_t per;  // backward: rows of a workgroup
  float* parts;
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

typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));

// N bytes at an offset from a buffer's base: zeros past its end (kOobOffset on), where nothing is stored either.
template <typename T, int V>
struct QkVec {
  typedef T type __attribute__((ext_vector_type(V)));
  static constexpr int kBytes = V * (int)sizeof(T);
  using Rsrc = __amdgpu_buffer_rsrc_t;
  template <typename F>
  static __device__ __forceinline__ void load(Rsrc r, unsigned at, F (&x)[V]) {
    type v;
    if constexpr (kBytes == 16)
      v = __builtin_bit_cast(type, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0));
    else if constexpr (kBytes == 8)
      v = __builtin_bit_cast(type, __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, 0));
    else if constexpr (kBytes == 4)
      v = __builtin_bit_cast(type, __builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0));
    else
      v = __builtin_bit_cast(type, __builtin_amdgcn_raw_buffer_load_b16(r, at, 0, 0));
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = (F)v[e];
  }
  static __device__ __forceinline__ void store(Rsrc r, unsigned at, const float (&x)[V]) {
    type v;
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (T)x[e];
    if constexpr (kBytes == 16)
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, v), r, at, 0, 0);
    else if constexpr (kBytes == 8)
      __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(v2u, v), r, at, 0, 0);
    else if constexpr (kBytes == 4)
      __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, v), r, at, 0, 0);
    else
      __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, v), r, at, 0, 0);
  }
};

// How a lane holds its share of a head: NV chunks `lanes` apart.  A chunk is
//   kQkApart       a vector of V channels and the vector of those that they turn with,
//   kQkPairs       the same of single channels, interleaved pairs,
//   kQkInside      a vector that holds both of each (interleaved) pair, or
//   kQkExchanged   a vector whose channels' partners are with other lanes, at any distance:
// the lanes write their values to a row of LDS for each place in the vector and read their
// partners'; for pairs whose number V does not divide.  200,000 rows x (8 + 8) x 64 bf16, forward /
// backward in us: 32 pairs apart 156 / 275, 15 pairs exchanged 207 / 352 (a channel a lane, apart, 720 / 1,112),
// 20 pairs exchanged 203 / 352 (apart in half vectors 237 / 424), 15 interleaved pairs inside 152 / 263.
// Channels past the pairs turn by nothing: the table has (1, 0) for them (kQkExchanged; the
// other forms leave them as they are, whatever lies beside them), and a
// second vector that is not there, like all of a chunk that the head does not have, is
// read as zeros and not stored, by an offset past the buffers.
enum QkMode { kQkApart, kQkPairs, kQkInside, kQkExchanged };
constexpr int kQkExchange = kQkThreads / 64 * (8 * 64 + 1);  // floats: for each wave eight rows and a zero
template <typename T, int V, int NV, int MODE>
struct QkLane {
  using Vec = QkVec<T, V>;
  static constexpr bool kInside = MODE == kQkInside, kOne = kInside || MODE == kQkExchanged;
  static constexpr int H = kOne ? 1 : 2, M = NV * H;  // vectors of a chunk, of the lane
  unsigned off[M];  // bytes from the head's first channel
  int w[M];         // channel (any where there is none: its x is zero)
  int turns[NV];    // of the table's row
  int pairs;        // of the head
  int partner[MODE == kQkExchanged ? V : 1];  // where the partners are in LDS
  float* exchange;                            // the wave's

  __device__ __forceinline__ QkLane(const QkArgs<T>& g, float* lds) : pairs(g.P) {
    const int pair_chunks = g.P / V;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (threadIdx.x & (g.lanes - 1)) + k * g.lanes;
      const bool live = c < g.chunks, pair = !kOne && c < pair_chunks;
      const int at = kOne ? c * V : pair ? c * (MODE == kQkPairs ? 2 : V) : 2 * g.P + (c - pair_chunks) * V;
      off[k * H] = live ? at * (unsigned)sizeof(T) : (unsigned)kOobOffset;
      w[k * H] = live ? at : 0;
      if constexpr (!kOne) {
        const int second = at + (MODE == kQkPairs ? 1 : g.P);
        off[k * H + 1] = pair ? second * (unsigned)sizeof(T) : (unsigned)kOobOffset;
        w[k * H + 1] = pair ? second : 0;
      }
      turns[k] = live ? c * (kInside ? V / 2 : V) : 0;
    }
    if constexpr (MODE == kQkExchanged) {
      static_assert(NV == 1, "a head's lanes are neighbours");
      exchange = lds + (threadIdx.x >> 6) * (8 * 64 + 1);
      const int lane = threadIdx.x & 63, head = lane & ~(g.lanes - 1);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int c = (lane - head) * V + e, to = c < g.P ? c + g.P : c - g.P;
        partner[e] = c < 2 * g.P ? to % V * 64 + head + to / V : 8 * 64;
      }
      if (lane == 0) exchange[8 * 64] = 0.f;
    }
  }
  // the weights of vector m, `all` the tensor's
  __device__ __forceinline__ void weights(const float* all, int m, float (&x)[V]) const {
    typedef float F __attribute__((ext_vector_type(V)));
    const F v = *reinterpret_cast<const F*>(all + w[m]);
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = v[e];
  }
  __device__ __forceinline__ bool has(int m) const { return off[m] != (unsigned)kOobOffset; }
  // `head`: the head's offset, kOobOffset for none (the sum of two such does not wrap)
  template <typename F>
  __device__ __forceinline__ void load(typename Vec::Rsrc r, unsigned head, F (&x)[M][V]) const {
#pragma unroll
    for (int m = 0; m < M; ++m) Vec::load(r, head + off[m], x[m]);
  }
  __device__ __forceinline__ void store(typename Vec::Rsrc r, unsigned head, const float (&x)[M][V]) const {
#pragma unroll
    for (int m = 0; m < M; ++m) Vec::store(r, head + off[m], x[m]);
  }
  // x turned by the row's table, forwards or back
  template <bool BACK>
  __device__ __forceinline__ void turn(const float2* table, float (&x)[M][V]) const {
    if constexpr (MODE == kQkExchanged) {  // (within a wave, whose LDS accesses keep their order)
#pragma unroll
      for (int e = 0; e < V; ++e) exchange[e * 64 + (threadIdx.x & 63)] = x[0][e];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 t = table[turns[0] + e];
        const float y = exchange[partner[e]] * t.y;
        x[0][e] = x[0][e] * t.x + (BACK ? -y : y);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      return;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < (kInside ? V / 2 : V); ++i) {
        const float2 t = table[turns[k] + i];
        float& a = kInside ? x[k][2 * i] : x[k * H][i];
        float& b = kInside ? x[k][2 * i + 1] : x[k * H + H - 1][i];
        const float s = BACK ? -t.y : t.y, u = a * t.x - b * s, v = a * s + b * t.x;
        // Past the pairs: as they are (zero times an infinity is a NaN).  A second vector that is not there is zeros when it
        // turns back, and what a weight makes of them when it turns.
        const bool turned = kInside ? turns[k] + i < pairs : has(k * H + H - 1);
        a = turned || (BACK && !kInside) ? u : a;
        b = turned ? v : kInside ? b : 0.f;
      }
  }
};

// Cosines and sines of `rows` rows from row0 on, and the weights, in LDS.  kQkExchanged: an entry for each channel, with the
// sign that its partner's sine has there.
template <int MODE, typename T>
__device__ __forceinline__ void qk_table(const QkArgs<T>& g, int64_t row0, int rows, float2* table) {
#pragma unroll 1
  for (int i = threadIdx.x; i < rows * g.table_row; i += kQkThreads) {
    const int r = i / g.table_row, d = i - r * g.table_row;
    const bool second = MODE == kQkExchanged && d >= g.P && d < 2 * g.P;
    const int p = second ? d - g.P : d;
    float s = 0.f, c = 1.f;
    if (p < g.P) {
      const double t = qk_pos(g.pos, g.pos_dtype, (row0 + r) * g.pos_row + g.axis[p]) * g.turns[p];
      sincospif(2.f * (float)(t - rint(t)), &s, &c);
      if (MODE == kQkExchanged && !second) s = -s;
    }
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

// The heads of one tensor over the rows of a workgroup, a group of lanes' heads
// one after another, `side` apart: 32-bit byte offsets from the workgroup's first
// row that grow by the same amounts at each step (products and divisions are
// quarter-rate, in 64 bits several of them).
template <int STREAMS>
struct QkWalk {
  int row, h, table;
  unsigned off[STREAMS];

  template <typename T>
  __device__ __forceinline__ void first(const QkArgs<T>& g, int w, int group, const int64_t (&strides)[STREAMS][2]) {
    row = (int)(((float)group + 0.5f) * g.heads_inv[w]);
    h = group - row * g.heads[w];
    table = row * g.table_row;
#pragma unroll
    for (int i = 0; i < STREAMS; ++i) off[i] = ((unsigned)row * (unsigned)strides[i][0] + (unsigned)h * (unsigned)strides[i][1]) * (unsigned)sizeof(T);
  }
  template <typename T>
  __device__ __forceinline__ void next(const QkArgs<T>& g, int w, const int64_t (&strides)[STREAMS][2]) {
    h += g.step_h[w];
    const bool wrap = h >= g.heads[w];
    h -= wrap ? g.heads[w] : 0;
    row += g.step_row[w] + wrap;
    table += (wrap ? g.step_row[w] + 1 : g.step_row[w]) * g.table_row;
#pragma unroll
    for (int i = 0; i < STREAMS; ++i) {
      const unsigned in_row = (unsigned)strides[i][0] * (unsigned)sizeof(T), in_head = (unsigned)strides[i][1] * (unsigned)sizeof(T);
      const unsigned by = g.step_row[w] * in_row + g.step_h[w] * in_head, more = in_row - g.heads[w] * in_head;
      off[i] += wrap ? by + more : by;
    }
  }
};

template <typename T, int V, int NV, int MODE>
__global__ __launch_bounds__(kQkThreads) void qk_forward_kernel(QkArgs<T> g) {
  using Lane = QkLane<T, V, NV, MODE>;
  constexpr int M = Lane::M;
  __shared__ float2 table[kQkTable];
  __shared__ __attribute__((aligned(32))) float weights[2 * ST_QK_MAX_DIM];
  const int64_t row0 = (int64_t)blockIdx.x * g.rows;
  const int rows = g.n - row0 < g.rows ? (int)(g.n - row0) : g.rows;
  const int side = kQkThreads >> g.lane_bits, group = threadIdx.x >> g.lane_bits;
  __shared__ float exchange[MODE == kQkExchanged ? kQkExchange : 1];
  const Lane lane(g, exchange);
  // q's heads, then k's, each in steps of a head a group of lanes; a head's loads go out while the one before it is at
  // work, the first one's before the table is made
  const int q_steps = (rows * g.heads[0] + side - 1) / side, steps = q_steps + (rows * g.heads[1] + side - 1) / side;
  T next[M][V];
  QkWalk<2> walk;
  auto load = [&](int step) {
    const int w = step >= q_steps;
    const int64_t strides[2][2] = {{g.in_row[w], g.in_head[w]}, {(int64_t)g.heads[w] * g.D, g.D}};
    if (step == 0 || step == q_steps)
      walk.first(g, w, group, strides);
    else
      walk.next(g, w, strides);
    lane.load(make_rsrc(g.in[w] + row0 * g.in_row[w], kOobOffset), walk.row < rows ? walk.off[0] : kOobOffset, next);
  };
  load(0);
  qk_table<MODE>(g, row0, rows, table);
  qk_weights(g, weights);
  __syncthreads();
#pragma unroll 1
  for (int step = 0; step < steps; ++step) {
    float x[M][V], sum[1] = {0.f};
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int e = 0; e < V; ++e) x[m][e] = (float)next[m][e];
    const int w = step >= q_steps;
    const bool live = walk.row < rows;
    const unsigned to = live ? walk.off[1] : kOobOffset;
    const float2* turns = table + (live ? walk.table : 0);
    if (step + 1 < steps) load(step + 1);
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int e = 0; e < V; ++e) sum[0] += x[m][e] * x[m][e];
    qk_sum(sum, g.lanes);
    const float s = rsqrtf(sum[0] * g.inv_d + g.eps);
#pragma unroll
    for (int m = 0; m < M; ++m) {
      float wm[V];
      lane.weights(weights + w * ST_QK_MAX_DIM, m, wm);
#pragma unroll
      for (int e = 0; e < V; ++e) x[m][e] *= wm[e] * s;
    }
    lane.template turn<false>(turns, x);
    lane.store(make_rsrc(g.out[w] + row0 * g.heads[w] * g.D, kOobOffset), to, x);
  }
}

// q's heads of all of a workgroup's rows, then k's: the sums of one weight's
// gradient in registers at a time, for a second table.
template <typename T, int V, int NV, int MODE>
__global__ __launch_bounds__(kQkThreads) void qk_backward_kernel(QkArgs<T> g) {
  using Lane = QkLane<T, V, NV, MODE>;
  constexpr int M = Lane::M;
  __shared__ float2 table[kQkTable];
  __shared__ __attribute__((aligned(32))) float weights[2 * ST_QK_MAX_DIM];
  __shared__ float sums[3][ST_QK_MAX_DIM];
  const int side = kQkThreads >> g.lane_bits, group = threadIdx.x >> g.lane_bits;
  __shared__ float exchange[MODE == kQkExchanged ? kQkExchange : 1];
  const Lane lane(g, exchange);
  const int64_t first = g.per * blockIdx.x, end = first + g.per < g.n ? first + g.per : g.n;
  qk_weights(g, weights);
#pragma unroll 1
  for (int w = 0; w < 2; ++w) {
    const int64_t strides[3][2] = {{g.in_row[w], g.in_head[w]}, {g.dy_row[w], g.dy_head[w]}, {(int64_t)g.heads[w] * g.D, g.D}};
    float dw[M][V];
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int e = 0; e < V; ++e) dw[m][e] = 0.f;
    for (int64_t row0 = first; row0 < end && g.heads[w]; row0 += g.rows) {
      const int rows = end - row0 < g.rows ? (int)(end - row0) : g.rows;
      const int steps = (rows * g.heads[w] + side - 1) / side;
      const auto in = make_rsrc(g.in[w] + row0 * g.in_row[w], kOobOffset);
      const auto dy = make_rsrc(g.dy[w] + row0 * g.dy_row[w], kOobOffset);
      const auto out = make_rsrc(g.out[w] + row0 * g.heads[w] * g.D, kOobOffset);
      QkWalk<3> walk;
      T next_x[M][V], next_g[M][V];
      auto load = [&]() {
        const bool live = walk.row < rows;
        lane.load(in, live ? walk.off[0] : kOobOffset, next_x);
        lane.load(dy, live ? walk.off[1] : kOobOffset, next_g);
      };
      walk.first(g, w, group, strides);
      load();
      qk_table<MODE>(g, row0, rows, table);
      __syncthreads();
#pragma unroll 1
      for (int step = 0; step < steps; ++step) {
        float x[M][V], d[M][V], gw[M][V];
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int e = 0; e < V; ++e) x[m][e] = (float)next_x[m][e], d[m][e] = (float)next_g[m][e];
        const bool live = walk.row < rows;
        const unsigned to = live ? walk.off[2] : kOobOffset;
        const float2* turns = table + (live ? walk.table : 0);
        walk.next(g, w, strides);
        if (step + 1 < steps) load();
        lane.template turn<true>(turns, d);
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int m = 0; m < M; ++m) {
          lane.weights(weights + w * ST_QK_MAX_DIM, m, gw[m]);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            gw[m][e] *= d[m][e];
            sum[0] += x[m][e] * x[m][e];
            sum[1] += gw[m][e] * x[m][e];
          }
        }
        qk_sum(sum, g.lanes);
        const float s = live ? rsqrtf(sum[0] * g.inv_d + g.eps) : 0.f, c = sum[1] * g.inv_d * s * s;
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            dw[m][e] += d[m][e] * (x[m][e] * s);
            d[m][e] = s * (gw[m][e] - x[m][e] * c);
          }
        lane.store(out, to, d);
      }
      __syncthreads();
    }
    if (!g.parts) continue;
    // the heads side by side in a wave, then the four waves, in a fixed order
    for (int o = g.lanes; o < 64; o *= 2)
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int e = 0; e < V; ++e) dw[m][e] += __shfl_xor(dw[m][e], o, 64);
    const int wave = threadIdx.x >> 6;
    const bool mine = (threadIdx.x & 63) < g.lanes;
    float* part = g.parts + (int64_t)blockIdx.x * 2 * g.D + w * g.D;
#pragma unroll
    for (int m = 0; m < M; ++m)
      if (wave > 0 && mine && lane.has(m))
#pragma unroll
        for (int e = 0; e < V; ++e) sums[wave - 1][lane.w[m] + e] = dw[m][e];
    __syncthreads();
#pragma unroll
    for (int m = 0; m < M; ++m)
      if (wave == 0 && mine && lane.has(m))
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int at = lane.w[m] + e;
          part[at] = dw[m][e] + sums[0][at] + sums[1][at] + sums[2][at];
        }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ host

// Whether vectors of V channels cut every head evenly and lie at their own size's alignment.
template <typename T, int V>
static bool qk_vec_ok(const QkArgs<T>& g) {
  if (g.D % V) return false;
  for (int w = 0; w < 2; ++w) {
    if (!g.heads[w]) continue;
    if (g.in_row[w] % V || g.in_head[w] % V) return false;
    if (g.dy[w] && (g.dy_row[w] % V || g.dy_head[w] % V)) return false;
    if (((uintptr_t)g.in[w] | (uintptr_t)g.dy[w] | (uintptr_t)g.out[w]) % (V * sizeof(T))) return false;
  }
  return true;
}

// Rows whose table is in LDS at once.
static int64_t qk_table_rows(int table_row) { return kQkTable / table_row; }

// Workgroups of the backward: a row each while there are fewer than its limit.
static int64_t qk_groups(int64_t n) { return n < kQkMaxGroups ? (n > 0 ? n : 1) : kQkMaxGroups; }

template <typename T, int V, int NV, int MODE>
static int qk_launch(QkArgs<T> g, bool backward, hipStream_t s) {
  for (int w = 0; w < 2; ++w) {
    const int d = g.heads[w], side = kQkThreads / g.lanes;
    g.heads_inv[w] = d ? 1.f / (float)d : 0.f;
    g.step_row[w] = d ? side / d : 0, g.step_h[w] = d ? side % d : 0;
  }
  // rows whose heads are within a 32-bit offset of the first
  int64_t reach = 1ll << 31;
  for (int w = 0; w < 2; ++w) {
    if (!g.heads[w]) continue;
    const int64_t row[3] = {g.in_row[w], backward ? g.dy_row[w] : 0, (int64_t)g.heads[w] * g.D};
    const int64_t head[3] = {g.in_head[w], backward ? g.dy_head[w] : 0, g.D};
    for (int i = 0; i < 3; ++i) {
      const int64_t left = kQkReach / (int64_t)sizeof(T) - g.heads[w] * head[i];
      if (left < row[i]) return ST_ERR_UNSUPPORTED;
      if (row[i] && left / row[i] < reach) reach = left / row[i];
    }
  }
  if (backward) {
    const int64_t rows = qk_table_rows(g.table_row);  // of a table
    g.rows = (int)(reach < rows ? reach : rows);
    g.per = (g.n + qk_groups(g.n) - 1) / qk_groups(g.n);
    qk_backward_kernel<T, V, NV, MODE><<<(unsigned)qk_groups(g.n), kQkThreads, 0, s>>>(g);
    ST_CHECK_LAUNCH();
    return ST_OK;
  }
  // rows of a workgroup: what LDS and a few heads a lane hold, fewer while there are not 1024 workgroups
  int64_t rows = qk_table_rows(g.table_row);
  const int64_t per_row = (int64_t)g.all * g.lanes;
  if (kQkItems / per_row < rows) rows = kQkItems / per_row;
  if (g.n / 1024 < rows) rows = g.n / 1024;
  if (reach < rows) rows = reach;
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
    qk_forward_kernel<T, V, NV, MODE><<<st_blocks(part.n, g.rows), kQkThreads, 0, s>>>(part);
    ST_CHECK_LAUNCH();
  }
  return ST_OK;
}

template <typename T, int V>
static int qk_vectors(QkArgs<T> g, bool interleaved, bool backward, hipStream_t s) {
  auto lanes = [&](int nv) {
    g.lanes = 1, g.lane_bits = 0;
    while (g.lanes * nv < g.chunks) g.lanes *= 2, ++g.lane_bits;
    return g.lanes <= 64;
  };
  if constexpr (V > 1) {
    g.chunks = g.D / V;
    if (interleaved) {  // (two vectors a lane: as many bytes as with the two of a chunk in the other modes)
      g.table_row = g.D / 2;
      return lanes(2) ? qk_launch<T, V, 2, kQkInside>(g, backward, s) : ST_ERR_UNSUPPORTED;
    }
    if (g.P % V) {
      g.table_row = g.D;
      return lanes(1) ? qk_launch<T, V, 1, kQkExchanged>(g, backward, s) : ST_ERR_UNSUPPORTED;
    }
  }
  g.table_row = g.D - g.P;
  g.chunks = (g.D - g.P) / V;
  constexpr int NV = ST_QK_MAX_DIM / V > 64 ? ST_QK_MAX_DIM / V / 64 : 1;
  const bool one = lanes(1);
  if (!one) lanes(NV);  // (heads longer than 64 vectors)
  if constexpr (V == 1) {
    if (interleaved) return one ? qk_launch<T, V, 1, kQkPairs>(g, backward, s) : qk_launch<T, V, NV, kQkPairs>(g, backward, s);
  }
  return one ? qk_launch<T, V, 1, kQkApart>(g, backward, s) : qk_launch<T, V, NV, kQkApart>(g, backward, s);
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
  else if (qk_vec_ok<T, V>(g))
    rc = qk_vectors<T, V>(g, il, backward, s);
  else if (qk_vec_ok<T, V / 2>(g) && (il || g.P % (V / 2) == 0 || g.D / (V / 2) <= 64))
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
  for (int64_t stride : {a->q_row, a->q_head, a->k_row, a->k_head, a->dq_row, a->dq_head, a->dk_row, a->dk_head})
    if (stride < 0 || stride >= (1ll << 31)) return ST_ERR_UNSUPPORTED;
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
