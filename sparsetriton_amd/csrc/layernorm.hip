// Layer norm over the channels of each row, with the residual add of a
// pre-norm block in the same pass:
//   h = x + r          (rounded to the stream's type: the block's stream goes on as h)
//   y = (h - mu) s w + b,   mu = mean_c h,   s = 1 / sqrt(mean_c (h - mu)^2 + eps)
// and its gradients, with g = dy w and xh = (h - mu) s:
//   dh = s (g - mean_c g - xh mean_c(g xh)) + (the gradient that arrives at h)
//   dw = sum_n dy xh,   db = sum_n dy.
//
// Both passes are bound by memory: a row's channels sit in the registers of
// LANES lanes, NV vectors of V channels each, from the load to the store, so
// every tensor moves once; the variance is a second sum over the registers (no
// cancellation of a one-pass E[h^2] - mu^2).  All sums are fp32.  The
// backward's workgroups walk the rows with a stride and keep dw and db of
// their lanes' channels in registers; one partial per workgroup goes to the
// workspace and a second kernel adds the partials in a fixed order, so the
// gradients are the same bits on every run.
//
// Forward / backward / sum of the partials, 470,532 x 64 fp32: 45 / 68 / 4 us
// (5.3 and 5.3 TB/s of what each moves); 65,537 x 512 bf16 with the residual and
// its gradient: 47 / 55 / 4 us (5.7 and 4.9 TB/s); a 1 GiB copy runs at 5.1 TB/s.
// 16 x 512 bf16: 2.8 us, a launch.
#include "common.h"
#include "wave_sum.h"

#define ST_LN_DISPATCH(dt, T, ...) \
  switch (dt) {                    \
    case ST_F32: {                 \
      using T = float;             \
      return __VA_ARGS__;          \
    }                              \
    case ST_F16: {                 \
      using T = _Float16;          \
      return __VA_ARGS__;          \
    }                              \
    case ST_BF16: {                \
      using T = __bf16;            \
      return __VA_ARGS__;          \
    }                              \
    default:                       \
      return ST_ERR_UNSUPPORTED;   \
  }

namespace st {

constexpr int kLnThreads = 256;
constexpr int kLnMaxGroups = 1024;  // workgroups of the backward, each leaving one partial

// How a row of C channels lies over lanes: vectors of V channels, lane l of
// LANES holding vectors l, l + LANES, ...  (V = 1 where a row is not whole
// 16-byte vectors at 16-byte addresses.)  lanes = 0: rows longer than the
// registers hold, read again for each sum.
struct LnGeom {
  int V, lanes, nv;
};
static LnGeom ln_geom(int C, int esz, bool aligned) {
  const int V = 16 / esz;
  if (aligned && C % V == 0) {
    const int vecs = C / V;
    if (vecs <= 64) {
      int lanes = 2;
      while (lanes < vecs) lanes *= 2;
      return {V, lanes, 1};
    }
    if (vecs <= 128) return {V, 64, 2};
    for (int nv = 1; nv <= 4; nv *= 2)
      if (vecs <= 256 * nv) return {V, 256, nv};
    return {V, 0, 0};
  }
  if (C <= 64) return {1, 64, 1};
  if (C <= 256) return {1, 64, 4};
  if (C <= 1024) return {1, 256, 4};
  if (C <= 4096) return {1, 256, 16};
  return {1, 0, 0};
}

// Workgroups of the backward: one for each CU while there are rows, then as
// many as keep eight steps of rows each for the partial that they leave (2 C
// floats against 3 C elements a row), at most 1024.
static int64_t ln_groups(int64_t n, const LnGeom& g) {
  const int side = g.lanes ? kLnThreads / g.lanes : 1;
  const int64_t steps = (n + side - 1) / side;
  int64_t w = steps < 256 ? steps : 256;
  if (steps / 8 > w) w = steps / 8;
  if (w > kLnMaxGroups) w = kLnMaxGroups;
  return w > 0 ? w : 1;
}

template <typename T, int V>
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) LnVec {
  T e[V];
};
template <typename T, int V>
__device__ __forceinline__ void ln_load(const T* __restrict__ p, float (&v)[V]) {
  const LnVec<T, V> u = *reinterpret_cast<const LnVec<T, V>*>(p);
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = (float)u.e[e];
}
template <typename T, int V>
__device__ __forceinline__ void ln_store(T* __restrict__ p, const float (&v)[V]) {
  LnVec<T, V> u;
#pragma unroll
  for (int e = 0; e < V; ++e) u.e[e] = (T)v[e];
  *reinterpret_cast<LnVec<T, V>*>(p) = u;
}

// Sum over the lanes of a row; LANES = 256 goes through LDS (`scratch`, four
// floats; two calls in a row take different ones).
template <int LANES>
__device__ __forceinline__ float ln_sum(float v, float* scratch) {
  if constexpr (LANES <= 64) return group_sum<LANES>(v);
  v = group_sum<64>(v);
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  return (scratch[0] + scratch[1]) + (scratch[2] + scratch[3]);
}

template <typename T, typename W, int V, int LANES, int NV, bool RES>
__global__ __launch_bounds__(kLnThreads) void ln_forward_kernel(const T* __restrict__ X, const T* __restrict__ R,
                                                                int64_t n, int C, const W* __restrict__ w,
                                                                const W* __restrict__ b, float eps,
                                                                T* __restrict__ H, T* __restrict__ Y,
                                                                float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float scratch[8];
  const int lane = threadIdx.x % LANES;
  const int64_t row = (int64_t)blockIdx.x * (kLnThreads / LANES) + threadIdx.x / LANES;
  if (LANES <= 64 && row >= n) return;  // (LANES = 256: the grid is exact)
  const float inv = 1.f / (float)C;
  float h[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * LANES + lane) * V;
    if (c < C) {
      ln_load<T, V>(X + row * C + c, h[i]);
      if constexpr (RES) {
        float r[V];
        ln_load<T, V>(R + row * C + c, r);
#pragma unroll
        for (int e = 0; e < V; ++e) h[i][e] = (float)(T)(h[i][e] + r[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) h[i][e] = 0.f;
    }
  }
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) s += h[i][e];
  const float mu = ln_sum<LANES>(s, scratch) * inv;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if ((i * LANES + lane) * V < C) {
#pragma unroll
      for (int e = 0; e < V; ++e) s += (h[i][e] - mu) * (h[i][e] - mu);
    }
  }
  const float rs = 1.f / sqrtf(ln_sum<LANES>(s, scratch + 4) * inv + eps);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * LANES + lane) * V;
    if (c < C) {
      float wv[V], bv[V], y[V];
      if (w) ln_load<W, V>(w + c, wv);
      if (b) ln_load<W, V>(b + c, bv);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        y[e] = (h[i][e] - mu) * rs;
        if (w) y[e] *= wv[e];
        if (b) y[e] += bv[e];
      }
      if constexpr (RES) ln_store<T, V>(H + row * C + c, h[i]);
      ln_store<T, V>(Y + row * C + c, y);
    }
  }
  if (mean && lane == 0) {
    mean[row] = mu;
    rstd[row] = rs;
  }
}

template <typename T, typename W, int V, int LANES, int NV>
__global__ __launch_bounds__(kLnThreads) void ln_backward_kernel(
    const T* __restrict__ H, const T* __restrict__ dY, const T* __restrict__ dH, int64_t n, int C,
    const W* __restrict__ w, const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dX,
    float* __restrict__ parts) {
  __shared__ float scratch[16];
  constexpr int SIDE = kLnThreads / LANES;
  const int lane = threadIdx.x % LANES;
  const float inv = 1.f / (float)C;
  float wv[NV][V], aw[NV][V], ab[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * LANES + lane) * V;
    if (w && c < C) {
      ln_load<W, V>(w + c, wv[i]);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) wv[i][e] = 1.f;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) aw[i][e] = ab[i][e] = 0.f;
  }
  // one step: the rows side by side in this workgroup (LANES = 256: one row, two sets of LDS slots in turn)
  int turn = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * SIDE; r0 < n; r0 += (int64_t)gridDim.x * SIDE, turn ^= 8) {
    const int64_t row = r0 + threadIdx.x / LANES;
    const bool live = LANES == 256 || row < n;
    float xh[NV][V], g[NV][V], sg = 0.f, sx = 0.f, rs = 0.f;
    if (live) {
      const float mu = mean[row];
      rs = rstd[row];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * LANES + lane) * V;
        if (c < C) {
          ln_load<T, V>(H + row * C + c, xh[i]);
          ln_load<T, V>(dY + row * C + c, g[i]);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            xh[i][e] = (xh[i][e] - mu) * rs;
            aw[i][e] += g[i][e] * xh[i][e];
            ab[i][e] += g[i][e];
            g[i][e] *= wv[i][e];
            sg += g[i][e];
            sx += g[i][e] * xh[i][e];
          }
        }
      }
    }
    sg = ln_sum<LANES>(sg, scratch + turn) * inv;
    sx = ln_sum<LANES>(sx, scratch + turn + 4) * inv;
    if (live && dX) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * LANES + lane) * V;
        if (c < C) {
          float d[V];
#pragma unroll
          for (int e = 0; e < V; ++e) d[e] = rs * (g[i][e] - sg - xh[i][e] * sx);
          if (dH) {
            float in[V];
            ln_load<T, V>(dH + row * C + c, in);
#pragma unroll
            for (int e = 0; e < V; ++e) d[e] += in[e];
          }
          ln_store<T, V>(dX + row * C + c, d);
        }
      }
    }
  }
  if (!parts) return;
  // the rows side by side in one wave, then the four waves, in a fixed order
  float* out = parts + (int64_t)blockIdx.x * 2 * C;
  if constexpr (LANES < 64) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e)
#pragma unroll
        for (int o = LANES; o < 64; o *= 2) {
          aw[i][e] += __shfl_xor(aw[i][e], o, 64);
          ab[i][e] += __shfl_xor(ab[i][e], o, 64);
        }
  }
  if constexpr (LANES < 256) {
    constexpr int ROW = LANES * NV * V;  // channels that the lanes hold, padding included
    __shared__ float sums[3][2][ROW];
    const int wave = threadIdx.x >> 6;
    const bool mine = (threadIdx.x & 63) < LANES;
    if (wave > 0 && mine) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          sums[wave - 1][0][(i * LANES + lane) * V + e] = aw[i][e];
          sums[wave - 1][1][(i * LANES + lane) * V + e] = ab[i][e];
        }
    }
    __syncthreads();
    if (wave > 0 || !mine) return;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e)
#pragma unroll
        for (int o = 0; o < 3; ++o) {
          aw[i][e] += sums[o][0][(i * LANES + lane) * V + e];
          ab[i][e] += sums[o][1][(i * LANES + lane) * V + e];
        }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * LANES + lane) * V;
    if (c < C) {
      ln_store<float, V>(out + c, aw[i]);
      ln_store<float, V>(out + C + c, ab[i]);
    }
  }
}

// ------------------------------------------------- rows longer than the registers hold

__device__ __forceinline__ float ln_block_sum(float v, float* scratch) {
  __syncthreads();
  return ln_sum<256>(v, scratch);
}

template <typename T, typename W>
__global__ __launch_bounds__(kLnThreads) void ln_forward_long_kernel(const T* __restrict__ X, const T* __restrict__ R,
                                                                     int C, const W* __restrict__ w,
                                                                     const W* __restrict__ b, float eps,
                                                                     T* __restrict__ H, T* __restrict__ Y,
                                                                     float* __restrict__ mean,
                                                                     float* __restrict__ rstd) {
  __shared__ float scratch[4];
  const int64_t row = blockIdx.x;
  const T* x = X + row * C;
  const T* r = R ? R + row * C : nullptr;
  const float inv = 1.f / (float)C;
  auto value = [&](int c) { return r ? (float)(T)((float)x[c] + (float)r[c]) : (float)x[c]; };
  float s = 0.f;
  for (int c = threadIdx.x; c < C; c += kLnThreads) s += value(c);
  const float mu = ln_block_sum(s, scratch) * inv;
  s = 0.f;
  for (int c = threadIdx.x; c < C; c += kLnThreads) {
    const float d = value(c) - mu;
    s += d * d;
  }
  const float rs = 1.f / sqrtf(ln_block_sum(s, scratch) * inv + eps);
  for (int c = threadIdx.x; c < C; c += kLnThreads) {
    const float h = value(c);
    if (r) H[row * C + c] = (T)h;
    Y[row * C + c] = (T)((h - mu) * rs * (w ? (float)w[c] : 1.f) + (b ? (float)b[c] : 0.f));
  }
  if (mean && threadIdx.x == 0) {
    mean[row] = mu;
    rstd[row] = rs;
  }
}

// dX only: the weight and bias gradients of long rows go column by column (ln_columns_kernel)
template <typename T, typename W>
__global__ __launch_bounds__(kLnThreads) void ln_backward_long_kernel(
    const T* __restrict__ H, const T* __restrict__ dY, const T* __restrict__ dH, int C, const W* __restrict__ w,
    const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dX) {
  __shared__ float scratch[4];
  const int64_t row = blockIdx.x;
  const float mu = mean[row], rs = rstd[row], inv = 1.f / (float)C;
  float sg = 0.f, sx = 0.f;
  for (int c = threadIdx.x; c < C; c += kLnThreads) {
    const float g = (float)dY[row * C + c] * (w ? (float)w[c] : 1.f);
    sg += g;
    sx += g * ((float)H[row * C + c] - mu) * rs;
  }
  sg = ln_block_sum(sg, scratch) * inv;
  sx = ln_block_sum(sx, scratch) * inv;
  for (int c = threadIdx.x; c < C; c += kLnThreads) {
    const float g = (float)dY[row * C + c] * (w ? (float)w[c] : 1.f);
    const float xh = ((float)H[row * C + c] - mu) * rs;
    const float d = rs * (g - sg - xh * sx);
    dX[row * C + c] = (T)(dH ? d + (float)dH[row * C + c] : d);
  }
}

// Column sums over a share of the rows (blockIdx.y of gridDim.y) for one column a thread.
template <typename T>
__global__ __launch_bounds__(kLnThreads) void ln_columns_kernel(const T* __restrict__ H, const T* __restrict__ dY,
                                                                int64_t n, int C, const float* __restrict__ mean,
                                                                const float* __restrict__ rstd,
                                                                float* __restrict__ parts) {
  const int c = blockIdx.x * kLnThreads + threadIdx.x;
  if (c >= C) return;
  float aw = 0.f, ab = 0.f;
  for (int64_t row = blockIdx.y; row < n; row += gridDim.y) {
    const float g = (float)dY[row * C + c];
    aw += g * ((float)H[row * C + c] - mean[row]) * rstd[row];
    ab += g;
  }
  parts[(int64_t)blockIdx.y * 2 * C + c] = aw;
  parts[(int64_t)blockIdx.y * 2 * C + C + c] = ab;
}

// dw, db = the partials' column sums: a workgroup for eight columns, a thread
// for a column and each of 32 shares of the partials, the shares added in order.
// (32 columns and 8 shares of it took 32 us for 1,024 partials of 64 channels:
// four workgroups, 128 loads one after another.)
template <typename W>
__global__ __launch_bounds__(kLnThreads) void ln_reduce_kernel(const float* __restrict__ parts, int groups, int C,
                                                               W* __restrict__ dw, W* __restrict__ db) {
  __shared__ float sums[32][9];
  const int in = threadIdx.x & 7, share = threadIdx.x >> 3, col = blockIdx.x * 8 + in;
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

// ------------------------------------------------------------------ host

// F<V, LANES, NV>() for the geometry.  (VV: the type's whole vector.)
template <int VV, typename F>
static int ln_select(const LnGeom& g, F f) {
  auto is = [&](int v, int lanes, int nv) { return g.V == v && g.lanes == lanes && g.nv == nv; };
#define ST_LN_CASE(v, l, k) \
  if (is(v, l, k)) return f(std::integral_constant<int, v>(), std::integral_constant<int, l>(), std::integral_constant<int, k>())
  ST_LN_CASE(VV, 2, 1);
  ST_LN_CASE(VV, 4, 1);
  ST_LN_CASE(VV, 8, 1);
  ST_LN_CASE(VV, 16, 1);
  ST_LN_CASE(VV, 32, 1);
  ST_LN_CASE(VV, 64, 1);
  ST_LN_CASE(VV, 64, 2);
  ST_LN_CASE(VV, 256, 1);
  ST_LN_CASE(VV, 256, 2);
  ST_LN_CASE(VV, 256, 4);
  ST_LN_CASE(1, 64, 1);
  ST_LN_CASE(1, 64, 4);
  ST_LN_CASE(1, 256, 4);
  ST_LN_CASE(1, 256, 16);
#undef ST_LN_CASE
  return ST_ERR_UNSUPPORTED;
}

// Rows of a launch, `side` of them to a workgroup.
static int64_t ln_most_rows(int side) { return st_most_blocks(kLnThreads) * side; }

static bool ln_aligned(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if ((uintptr_t)p & 15) return false;
  return true;
}

template <typename T, typename W>
static int ln_forward(const void* X, const void* R, int64_t n, int C, const void* w, const void* b, float eps, void* H,
                      void* Y, float* mean, float* rstd, hipStream_t s) {
  const T *x = (const T*)X, *r = (const T*)R;
  T *h = (T*)H, *y = (T*)Y;
  const W *wp = (const W*)w, *bp = (const W*)b;
  const LnGeom g = ln_geom(C, sizeof(T), ln_aligned({X, R, H, Y, w, b}));
  const int64_t most = ln_most_rows(g.lanes ? kLnThreads / g.lanes : 1);
  for (int64_t row = 0; row < n; row += most) {
    const int64_t m = n - row < most ? n - row : most, at = row * C;
    const T *xr = x + at, *rr = r ? r + at : nullptr;
    T *hr = h ? h + at : nullptr, *yr = y + at;
    float *mr = mean ? mean + row : nullptr, *sr = rstd ? rstd + row : nullptr;
    int rc = ST_OK;
    if (!g.lanes)
      ln_forward_long_kernel<T, W><<<(unsigned)m, kLnThreads, 0, s>>>(xr, rr, C, wp, bp, eps, hr, yr, mr, sr);
    else
      rc = ln_select<16 / sizeof(T)>(g, [&](auto v, auto lanes, auto nv) -> int {
        constexpr int V = decltype(v)::value, L = decltype(lanes)::value, N = decltype(nv)::value;
        const unsigned blocks = st_blocks(m, kLnThreads / L);
        if (r)
          ln_forward_kernel<T, W, V, L, N, true><<<blocks, kLnThreads, 0, s>>>(xr, rr, m, C, wp, bp, eps, hr, yr, mr, sr);
        else
          ln_forward_kernel<T, W, V, L, N, false><<<blocks, kLnThreads, 0, s>>>(xr, rr, m, C, wp, bp, eps, hr, yr, mr, sr);
        return ST_OK;
      });
    if (rc != ST_OK) return rc;
    ST_CHECK_LAUNCH();
  }
  return ST_OK;
}

template <typename T, typename W>
static int ln_backward(const void* H, const void* dY, const void* dH, int64_t n, int C, const void* w,
                       const float* mean, const float* rstd, float* ws, void* dX, void* dw, void* db, hipStream_t s) {
  const T *h = (const T*)H, *dy = (const T*)dY, *dh = (const T*)dH;
  const W* wp = (const W*)w;
  const LnGeom g = ln_geom(C, sizeof(T), ln_aligned({H, dY, dH, dX, w}));
  const int64_t groups = ln_groups(n, g);
  const bool columns = dw || db;
  int rc = ST_OK;
  if (!g.lanes) {
    const int64_t most = ln_most_rows(1);
    for (int64_t row = 0; dX && row < n; row += most) {
      const int64_t m = n - row < most ? n - row : most, at = row * C;
      ln_backward_long_kernel<T, W><<<(unsigned)m, kLnThreads, 0, s>>>(h + at, dy + at, dh ? dh + at : nullptr, C, wp,
                                                                      mean + row, rstd + row, (T*)dX + at);
      ST_CHECK_LAUNCH();
    }
    if (columns)
      ln_columns_kernel<T>
          <<<dim3(st_blocks(C, kLnThreads), (unsigned)groups), kLnThreads, 0, s>>>(h, dy, n, C, mean, rstd, ws);
    ST_CHECK_LAUNCH();
  } else {
    rc = ln_select<16 / sizeof(T)>(g, [&](auto v, auto lanes, auto nv) -> int {
      constexpr int V = decltype(v)::value, L = decltype(lanes)::value, N = decltype(nv)::value;
      ln_backward_kernel<T, W, V, L, N><<<(unsigned)groups, kLnThreads, 0, s>>>(h, dy, dh, n, C, wp, mean, rstd,
                                                                               (T*)dX, columns ? ws : nullptr);
      ST_CHECK_LAUNCH();
      return ST_OK;
    });
  }
  if (rc != ST_OK || !columns) return rc;
  ln_reduce_kernel<W><<<st_blocks(2 * (int64_t)C, 8), kLnThreads, 0, s>>>(ws, (int)groups, C, (W*)dw, (W*)db);
  ST_CHECK_LAUNCH();
  return ST_OK;
}

}  // namespace st

// n rows of C channels that the kernels take
static bool ln_sizes_ok(int64_t n, int C) { return n >= 0 && n < (1ll << 31) && C > 0; }

extern "C" int st_ln_forward(const void* X, const void* residual, int64_t n, int C, int dtype, const void* weight,
                             const void* bias, int weight_dtype, float eps, void* H, void* Y, float* mean, float* rstd,
                             st_stream_t stream) {
  if (!ln_sizes_ok(n, C) || (!mean != !rstd)) return ST_ERR_ARG;
  if (n == 0) return ST_OK;
  if (!X || !Y || (!residual != !H)) return ST_ERR_ARG;
  if (weight_dtype != dtype && weight_dtype != ST_F32) return ST_ERR_UNSUPPORTED;
  hipStream_t s = (hipStream_t)stream;
  if (weight_dtype == ST_F32) {
    ST_LN_DISPATCH(dtype, T, (st::ln_forward<T, float>(X, residual, n, C, weight, bias, eps, H, Y, mean, rstd, s)));
  }
  ST_LN_DISPATCH(dtype, T, (st::ln_forward<T, T>(X, residual, n, C, weight, bias, eps, H, Y, mean, rstd, s)));
}

extern "C" int st_ln_backward_workspace(int64_t n, int C, int dtype, int64_t* floats) {
  if (!ln_sizes_ok(n, C) || !floats) return ST_ERR_ARG;
  if (dtype != ST_F32 && dtype != ST_F16 && dtype != ST_BF16) return ST_ERR_UNSUPPORTED;
  // (whichever of the two layouts the call's pointers lead to)
  const int esz = dtype == ST_F32 ? 4 : 2;
  const int64_t a = st::ln_groups(n, st::ln_geom(C, esz, true)), b = st::ln_groups(n, st::ln_geom(C, esz, false));
  *floats = (a > b ? a : b) * 2 * C;
  return ST_OK;
}

extern "C" int st_ln_backward(const void* H, const void* dY, const void* dH, int64_t n, int C, int dtype,
                              const void* weight, int weight_dtype, const float* mean, const float* rstd,
                              float* workspace, int64_t workspace_floats, void* dX, void* dweight, void* dbias,
                              st_stream_t stream) {
  int64_t need = 0;
  const int rc = st_ln_backward_workspace(n, C, dtype, &need);
  if (rc != ST_OK) return rc;
  // (the sum of the partials is one launch, eight of 2 C columns to a workgroup)
  if ((dweight || dbias) && (2 * (int64_t)C + 7) / 8 > st_most_blocks(st::kLnThreads)) return ST_ERR_UNSUPPORTED;
  if (weight_dtype != dtype && weight_dtype != ST_F32) return ST_ERR_UNSUPPORTED;
  if (n > 0 && (!H || !dY || !mean || !rstd)) return ST_ERR_ARG;
  if ((dweight || dbias) && (!workspace || workspace_floats < need || ((uintptr_t)workspace & 15))) return ST_ERR_ARG;
  if (n == 0 && !dweight && !dbias) return ST_OK;
  hipStream_t s = (hipStream_t)stream;
  if (weight_dtype == ST_F32) {
    ST_LN_DISPATCH(dtype, T,
                   (st::ln_backward<T, float>(H, dY, dH, n, C, weight, mean, rstd, workspace, dX, dweight, dbias, s)));
  }
  ST_LN_DISPATCH(dtype, T,
                 (st::ln_backward<T, T>(H, dY, dH, n, C, weight, mean, rstd, workspace, dX, dweight, dbias, s)));
}
