// Layer norm over the columns of a row, forward and backward (the norm of
// src/model/KGAT/multi_head_attention.py:30, trainable):
//   mean = sum x / d,  var = sum (x - mean)^2 / d,  rstd = 1 / sqrt(var + eps),  xhat = (x - mean) rstd
//   y  = xhat w + b
//   g  = dy w,  dx = rstd (g - mean(g) - xhat mean(g xhat))
//   dw = sum over rows of dy xhat,  db = sum over rows of dy
#include "dense.hpp"

namespace kgat {

namespace {

// A weight vector of the rows' type or of float, element by element (read once a block).
struct NormVec {
  const void* p;
  int32_t dtype;
  __device__ __forceinline__ float at(int64_t j) const {
    if (dtype == KGAT_F32) return static_cast<const float*>(p)[j];
    if (dtype == KGAT_BF16) return static_cast<float>(static_cast<const __bf16*>(p)[j]);
    return static_cast<float>(static_cast<const _Float16*>(p)[j]);
  }
  __device__ __forceinline__ void put(int64_t j, float v) const {
    void* q = const_cast<void*>(p);
    if (dtype == KGAT_F32) static_cast<float*>(q)[j] = v;
    else if (dtype == KGAT_BF16) static_cast<__bf16*>(q)[j] = static_cast<__bf16>(v);
    else static_cast<_Float16*>(q)[j] = static_cast<_Float16>(v);
  }
};

// Sums of K values over the G threads of a row (G a power of two; G > 64: the whole block, through LDS).
template <int G, int K>
__device__ __forceinline__ void group_sum(float (&v)[K], float* lds) {
#pragma unroll
  for (int o = (G < 64 ? G : 64) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < K; ++i) v[i] += __shfl_xor(v[i], o);
  if constexpr (G > 64) {
    constexpr int kWaves = G / 64;
    const int wave = threadIdx.x >> 6;
    __syncthreads();  // the last sum's readers are done with lds
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < K; ++i) lds[i * kWaves + wave] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < K; ++i) {
      float s = 0.f;
      for (int w = 0; w < kWaves; ++w) s += lds[i * kWaves + w];
      v[i] = s;
    }
  }
}

struct NormFwd {
  const void* x;
  int64_t ldx;
  void* y;
  int64_t ldy;
  NormVec w, b;
  float* mean;
  float* rstd;
  int64_t n;
  int32_t d;
  float eps;
};

// G threads hold a row as NV vectors each.
template <typename T, int G, int NV, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_fwd_kernel(NormFwd a) {
  constexpr int V = Vec<T>::N;
  __shared__ float lds[2 * (THREADS / 64)];
  const int lane = threadIdx.x % G;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (THREADS / G);
  const float d = static_cast<float>(a.d);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * (THREADS / G) + threadIdx.x / G; row - threadIdx.x / G < a.n;
       row += step) {
    const bool live = row < a.n;
    const T* x = static_cast<const T*>(a.x) + (live ? row : 0) * a.ldx;
    float v[NV][V];
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + lane) * V;
      const Vec<T> t = load_vec(x + c, live ? a.d - c : 0);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[i][j] = static_cast<float>(t.e[j]);
        s[0] += v[i][j];
      }
    }
    group_sum<G>(s, lds);
    const float mean = s[0] / d;
    float q[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[i][j] -= mean;
        if ((i * G + lane) * V + j < a.d) q[0] += v[i][j] * v[i][j];
      }
    group_sum<G>(q, lds);
    const float rstd = 1.f / sqrtf(q[0] / d + a.eps);
    if (!live) continue;
    T* y = static_cast<T*>(a.y) + row * a.ldy;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + lane) * V;
      Vec<T> t;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float r = v[i][j] * rstd;
        if (c + j < a.d) {
          if (a.w.p != nullptr) r *= a.w.at(c + j);
          if (a.b.p != nullptr) r += a.b.at(c + j);
        }
        t.e[j] = static_cast<T>(r);
      }
      store_vec(y + c, t, a.d - c);
    }
    if (lane == 0 && a.mean != nullptr) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

// Rows wider than a block's registers: the row is read three times (from the cache the second and third time).
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_fwd_wide_kernel(NormFwd a) {
  constexpr int V = Vec<T>::N;
  __shared__ float lds[2 * (THREADS / 64)];
  const float d = static_cast<float>(a.d);
  for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    T* y = static_cast<T*>(a.y) + row * a.ldy;
    float s[1] = {0.f}, q[1] = {0.f};
    for (int64_t c = threadIdx.x * V; c < a.d; c += THREADS * V) {
      const Vec<T> t = load_vec(x + c, a.d - c);
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] += static_cast<float>(t.e[j]);
    }
    group_sum<THREADS>(s, lds);
    const float mean = s[0] / d;
    for (int64_t c = threadIdx.x * V; c < a.d; c += THREADS * V) {
      const Vec<T> t = load_vec(x + c, a.d - c);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float e = static_cast<float>(t.e[j]) - mean;
        if (c + j < a.d) q[0] += e * e;
      }
    }
    group_sum<THREADS>(q, lds);
    const float rstd = 1.f / sqrtf(q[0] / d + a.eps);
    for (int64_t c = threadIdx.x * V; c < a.d; c += THREADS * V) {
      Vec<T> t = load_vec(x + c, a.d - c);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (c + j < a.d) {
          float r = (static_cast<float>(t.e[j]) - mean) * rstd;
          if (a.w.p != nullptr) r *= a.w.at(c + j);
          if (a.b.p != nullptr) r += a.b.at(c + j);
          t.e[j] = static_cast<T>(r);
        }
      store_vec(y + c, t, a.d - c);
    }
    if (threadIdx.x == 0 && a.mean != nullptr) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

struct NormBwd {
  const void* dy;
  int64_t lddy;
  const void* x;
  int64_t ldx;
  const float* mean;
  const float* rstd;
  NormVec w, dw, db;
  void* dx;
  int64_t lddx;
  int64_t n;
  int32_t d;
  float* part;  // [parts][2][d]: the row blocks' sums of dy xhat and of dy
  int32_t parts;
};

// dx, a block per row (rows of any width).
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_dx_kernel(NormBwd a) {
  constexpr int V = Vec<T>::N;
  __shared__ float lds[2 * (THREADS / 64)];
  const float d = static_cast<float>(a.d);
  for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* dy = static_cast<const T*>(a.dy) + row * a.lddy;
    T* dx = static_cast<T*>(a.dx) + row * a.lddx;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s[2] = {0.f, 0.f};
    for (int64_t c = threadIdx.x * V; c < a.d; c += THREADS * V) {
      const Vec<T> tx = load_vec(x + c, a.d - c), tg = load_vec(dy + c, a.d - c);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (c + j < a.d) {
          float g = static_cast<float>(tg.e[j]);
          if (a.w.p != nullptr) g *= a.w.at(c + j);
          s[0] += g;
          s[1] += g * ((static_cast<float>(tx.e[j]) - mean) * rstd);
        }
    }
    group_sum<THREADS>(s, lds);
    const float mg = s[0] / d, mgx = s[1] / d;
    for (int64_t c = threadIdx.x * V; c < a.d; c += THREADS * V) {
      const Vec<T> tx = load_vec(x + c, a.d - c), tg = load_vec(dy + c, a.d - c);
      Vec<T> t;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float g = static_cast<float>(tg.e[j]);
        if (a.w.p != nullptr && c + j < a.d) g *= a.w.at(c + j);
        t.e[j] = static_cast<T>(rstd * (g - mg - (static_cast<float>(tx.e[j]) - mean) * rstd * mgx));
      }
      store_vec(dx + c, t, a.d - c);
    }
  }
}

// The rows' sums by column: a block takes 64 columns and a share of the rows, its 4 waves every fourth row.
template <typename T>
__global__ __launch_bounds__(256) void norm_cols_kernel(NormBwd a) {
  __shared__ float lds[2][4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + lane;
  const int64_t per = (a.n + a.parts - 1) / a.parts, r0 = blockIdx.y * per, r1 = r0 + per < a.n ? r0 + per : a.n;
  float sw = 0.f, sb = 0.f;
  if (c < a.d)
    for (int64_t row = r0 + wave; row < r1; row += 4) {
      const float g = static_cast<float>(static_cast<const T*>(a.dy)[row * a.lddy + c]);
      const float x = static_cast<float>(static_cast<const T*>(a.x)[row * a.ldx + c]);
      sw += g * ((x - a.mean[row]) * a.rstd[row]);
      sb += g;
    }
  lds[0][wave][lane] = sw;
  lds[1][wave][lane] = sb;
  __syncthreads();
  if (wave < 2 && c < a.d) {
    const float s = (lds[wave][0][lane] + lds[wave][1][lane]) + (lds[wave][2][lane] + lds[wave][3][lane]);
    a.part[(static_cast<int64_t>(blockIdx.y) * 2 + wave) * a.d + c] = s;
  }
}

// dw and db from the parts, in their order: 64 columns of the [2 d] sums a block, 16 waves over the parts.
__global__ __launch_bounds__(1024) void norm_cols_join_kernel(NormBwd a) {
  __shared__ float lds[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + lane, width = 2 * static_cast<int64_t>(a.d);
  float s = 0.f;
  if (c < width)
    for (int p = wave; p < a.parts; p += 16) s += a.part[p * width + c];
  lds[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || c >= width) return;
  s = 0.f;
#pragma unroll
  for (int w = 0; w < 16; ++w) s += lds[w][lane];
  const NormVec& to = c < a.d ? a.dw : a.db;
  if (to.p != nullptr) to.put(c < a.d ? c : c - a.d, s);
}

template <typename T, int G, int NV, int THREADS>
int launch_fwd(const NormFwd& a, hipStream_t st) {
  const int rows = THREADS / G;
  const int grid = blocks_for(a.n, rows, 1 << 20);
  hipLaunchKernelGGL((norm_fwd_kernel<T, G, NV, THREADS>), dim3(grid), dim3(THREADS), 0, st, a);
  KGAT_LAUNCH_CHECK();
  return KGAT_OK;
}

template <typename T>
int norm_fwd(const NormFwd& a, hipStream_t st) {
  const int nvec = (a.d + Vec<T>::N - 1) / Vec<T>::N;
  if (nvec <= 16) return launch_fwd<T, 16, 1, 256>(a, st);
  if (nvec <= 64) return launch_fwd<T, 64, 1, 256>(a, st);
  if (nvec <= 256) return launch_fwd<T, 64, 4, 256>(a, st);
  if (nvec <= 1024) return launch_fwd<T, 256, 4, 256>(a, st);
  hipLaunchKernelGGL((norm_fwd_wide_kernel<T, 1024>), dim3(blocks_for(a.n, 1, 1 << 20)), dim3(1024), 0, st, a);
  KGAT_LAUNCH_CHECK();
  return KGAT_OK;
}

int norm_parts(int64_t n, int32_t d) {
  const int64_t cols = (static_cast<int64_t>(d) + 63) / 64;
  int64_t p = (1024 + cols - 1) / cols;  // about 1024 blocks in all, 16 rows at least in each
  if (p > (n + 15) / 16) p = (n + 15) / 16;
  return p < 1 ? 1 : static_cast<int>(p);
}

template <typename T>
int norm_bwd(const NormBwd& a, hipStream_t st) {
  if (a.dx != nullptr && a.n > 0) {
    hipLaunchKernelGGL((norm_dx_kernel<T, 256>), dim3(blocks_for(a.n, 1, 1 << 20)), dim3(256), 0, st, a);
    KGAT_LAUNCH_CHECK();
  }
  if (a.dw.p == nullptr && a.db.p == nullptr) return KGAT_OK;
  hipLaunchKernelGGL(norm_cols_kernel<T>, dim3((a.d + 63) / 64, a.parts), dim3(256), 0, st, a);
  KGAT_LAUNCH_CHECK();
  hipLaunchKernelGGL(norm_cols_join_kernel, dim3((2 * a.d + 63) / 64), dim3(1024), 0, st, a);
  KGAT_LAUNCH_CHECK();
  return KGAT_OK;
}

bool norm_vec_ok(int32_t w_dtype, int32_t dtype) { return w_dtype == KGAT_F32 || w_dtype == dtype; }

}  // namespace

}  // namespace kgat

extern "C" int kgat_layer_norm_fwd(int32_t dtype, const void* x, int64_t ldx, int32_t w_dtype, const void* weight,
                                   const void* bias, void* y, int64_t ldy, float* mean, float* rstd, int64_t n,
                                   int32_t d, float eps, void* stream) {
  using namespace kgat;
  if (!x || !y || n < 0 || d < 1 || d > KGAT_NORM_MAX_D || ldx < 0 || ldy < d || !(eps >= 0.f) ||
      (mean == nullptr) != (rstd == nullptr) || !norm_vec_ok(w_dtype, dtype))
    return KGAT_ERR_INVALID;
  NormFwd a{x, ldx, y, ldy, {weight, w_dtype}, {bias, w_dtype}, mean, rstd, n, d, eps};
  return with_dtype(dtype, [&](auto t) {
    return n == 0 ? static_cast<int>(KGAT_OK) : norm_fwd<decltype(t)>(a, reinterpret_cast<hipStream_t>(stream));
  });
}

extern "C" int64_t kgat_layer_norm_bwd_workspace(int64_t n, int32_t d) {
  if (n < 0 || d < 1 || d > KGAT_NORM_MAX_D) return -1;
  return static_cast<int64_t>(kgat::norm_parts(n, d)) * 2 * d;
}

extern "C" int kgat_layer_norm_bwd(int32_t dtype, const void* dy, int64_t lddy, const void* x, int64_t ldx,
                                   const float* mean, const float* rstd, int32_t w_dtype, const void* weight, void* dx,
                                   int64_t lddx, void* dweight, void* dbias, int64_t n, int32_t d, float* workspace,
                                   int64_t workspace_floats, void* stream) {
  using namespace kgat;
  if (!dy || !x || !mean || !rstd || n < 0 || d < 1 || d > KGAT_NORM_MAX_D || lddy < 0 || ldx < 0 ||
      (dx != nullptr && lddx < d) || !norm_vec_ok(w_dtype, dtype))
    return KGAT_ERR_INVALID;
  const bool cols = dweight != nullptr || dbias != nullptr;
  if (cols && (!workspace || workspace_floats < kgat_layer_norm_bwd_workspace(n, d))) return KGAT_ERR_WORKSPACE;
  NormBwd a{dy, lddy, x, ldx, mean, rstd, {weight, w_dtype}, {dweight, w_dtype}, {dbias, w_dtype}, dx, lddx, n, d,
            workspace, norm_parts(n, d)};
  return with_dtype(dtype, [&](auto t) { return norm_bwd<decltype(t)>(a, reinterpret_cast<hipStream_t>(stream)); });
}
