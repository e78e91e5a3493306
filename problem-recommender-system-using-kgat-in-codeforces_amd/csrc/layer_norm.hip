// Layer norm over the columns of a row, forward and backward (the norm of
// src/model/KGAT/multi_head_attention.py:30, trainable):
//   mean = sum x / d,  var = sum (x - mean)^2 / d,  rstd = 1 / sqrt(var + eps),  xhat = (x - mean) rstd
//   y  = xhat w + b
//   g  = dy w,  dx = rstd (g - mean(g) - xhat mean(g xhat))
//   dw = sum over rows of dy xhat,  db = sum over rows of dy
#include <type_traits>

#include "dense.hpp"

namespace kgat {

namespace {

// A weight vector, of float or of the rows' type T.
struct NormVec {
  void* p;
  int32_t dtype;
  __device__ __forceinline__ void put(int64_t j, float v) const {
    if (dtype == KGAT_F32) static_cast<float*>(p)[j] = v;
    else if (dtype == KGAT_BF16) static_cast<__bf16*>(p)[j] = static_cast<__bf16>(v);
    else static_cast<_Float16*>(p)[j] = static_cast<_Float16>(v);
  }
};

// A thread's columns of a weight vector; `none` where there is no vector.  The choices are uniform: with a choice of
// type for every element under the lane's own bound, hipcc 7.2 lost a live address register on the fp16 path.
template <typename W, int V, int NV>
__device__ __forceinline__ void load_columns_of(const W* p, int lane, int G, int32_t d, float (&out)[NV][V]) {
  constexpr int N = Vec<W>::N < V ? Vec<W>::N : V;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; j += N) {
      const Vec<W> v = load_row(p, (i * G + lane) * V + j, d);
#pragma unroll
      for (int k = 0; k < N; ++k) out[i][j + k] = static_cast<float>(v.e[k]);
    }
}

template <typename T, int V, int NV>
__device__ __forceinline__ void load_columns(const NormVec& w, int lane, int G, int32_t d, float none,
                                             float (&out)[NV][V]) {
  if (w.p == nullptr) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) out[i][j] = none;
  } else if (sizeof(T) == 4 || w.dtype == KGAT_F32) {
    load_columns_of(static_cast<const float*>(w.p), lane, G, d, out);
  } else {
    load_columns_of(static_cast<const T*>(w.p), lane, G, d, out);
  }
}

// Sums of K values over the G threads of a row (a power of two up to 64, or whole waves, through LDS).  Every thread of
// the block calls it.  `turn` alternates between two LDS halves, so one barrier a sum is enough: who writes a half
// again has passed the barrier of the sum between, and with it every reader of the half.
template <int G, int THREADS, int K>
__device__ __forceinline__ void group_sum(float (&v)[K], float* lds, int& turn) {
#pragma unroll
  for (int i = 0; i < K; ++i) v[i] = lanes_sum<(G < 64 ? G : 64)>(v[i]);
  if constexpr (G > 64) {
    constexpr int kWaves = THREADS / 64;
    const int wave = threadIdx.x >> 6;
    float* at = lds + turn * K * kWaves;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < K; ++i) at[i * kWaves + wave] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < K; ++i) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < G / 64; ++w) s += at[i * kWaves + wave / (G / 64) * (G / 64) + w];
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

// The statistics from the sums of D = x - mean and of D^2 (inv = 1 / d), mean being a rounded 32-bit sum over d: D is
// exact near the mean, so what the mean is off by stands in D's own sum, to a rounding of D's size.  `shift` is to be
// taken from every D; var = sum D^2 / d - shift^2, which is 0 for a constant row, not a rounding below it, and infinite
// where the squares are.
struct RowStat {
  float shift, mean, rstd;
  __device__ __forceinline__ RowStat(float mean_, float sum, float sum2, float inv, float eps) : shift(sum * inv), mean(mean_ + shift) {
    const float q = sum2 * inv, s = shift * shift;
    const float var = s < q ? q - s : q < INFINITY ? 0.f : q;
    rstd = 1.f / sqrtf(var + eps);
  }
};

// G threads hold a row as NV vectors each, and the weights of their columns over all the rows they take (a row's
// weights are 8 bytes a column: read again for every row they would be up to four times its own bytes, from the
// cache).  The next row is on its way while one is normalised.  Two passes over the registers, not sums of x and x^2:
// a row far from 0 keeps its digits (see RowStat).
// Bound by memory: 1M x 64 float 86 us (512 MB, 6.0 TB/s), 8192 x 4096 bf16 24 us (134 MB, 5.5 TB/s).  At odd widths
// the 16-byte accesses straddle cache lines: 16484 x 1021 bf16 16.1 us (4.2 TB/s), x 1024 13.6.  The correction by D's own sum
// costs 16-bit rows of 1024 columns and more 2 to 4 % (8192 x 4096 23.8 us without it), narrower and float ones nothing.
template <typename T, int G, int NV, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_fwd_kernel(NormFwd a) {
  constexpr int V = Vec<T>::N;
  static_assert(THREADS % G == 0, "whole rows");
  __shared__ float lds[4 * (THREADS / 64)];
  int turn = 0;
  const int lane = threadIdx.x % G;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (THREADS / G);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (THREADS / G);
  const float d = static_cast<float>(a.d), inv = 1.f / d;
  float w[NV][V], b[NV][V];
  load_columns<T>(a.w, lane, G, a.d, 1.f, w);
  load_columns<T>(a.b, lane, G, a.d, 0.f, b);
  Vec<T> next[NV];
  auto fetch = [&](int64_t row) {
    const T* x = static_cast<const T*>(a.x) + (row < a.n ? row : a.n - 1) * a.ldx;
#pragma unroll
    for (int i = 0; i < NV; ++i) next[i] = load_row(x, (i * G + lane) * V, a.d);
  };
  fetch(first + threadIdx.x / G);
  for (int64_t base = first; base < a.n; base += step) {
    const int64_t row = base + threadIdx.x / G;
    float v[NV][V];
    float s[1] = {0.f}, q[2] = {0.f, 0.f};  // q: sums of D and of D^2, D = x - mean
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[i][j] = static_cast<float>(next[i].e[j]);
        s[0] += v[i][j];
      }
    if (base + step < a.n) fetch(row + step);
    group_sum<G, THREADS>(s, lds, turn);
    const float mean = s[0] / d;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[i][j] = (i * G + lane) * V + j < a.d ? v[i][j] - mean : 0.f;
        q[0] += v[i][j];
        q[1] += v[i][j] * v[i][j];
      }
    group_sum<G, THREADS>(q, lds, turn);
    const RowStat r(mean, q[0], q[1], inv, a.eps);
    const float shift = r.shift * r.rstd;
    if (row < a.n) {
      T* y = static_cast<T*>(a.y) + row * a.ldy;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * G + lane) * V;
        Vec<T> t;
#pragma unroll
        for (int j = 0; j < V; ++j) t.e[j] = static_cast<T>((v[i][j] * r.rstd - shift) * w[i][j] + b[i][j]);
        store_row(y, c, a.d, t);
      }
      if (lane == 0 && a.mean != nullptr) {
        a.mean[row] = r.mean;
        a.rstd[row] = r.rstd;
      }
    }
  }
}

// A vector's weights; `none` where there is no vector of them.
template <typename T>
__device__ __forceinline__ void load_weights(const NormVec& w, int64_t c, int32_t d, float none,
                                             float (&out)[Vec<T>::N]) {
  constexpr int V = Vec<T>::N;
  if (w.p == nullptr) {
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = none;
  } else if (sizeof(T) == 4 || w.dtype == KGAT_F32) {
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      const Vec<float> v = load_row(static_cast<const float*>(w.p), c + j, d);
#pragma unroll
      for (int k = 0; k < 4; ++k) out[j + k] = v.e[k];
    }
  } else {
    const Vec<T> v = load_row(static_cast<const T*>(w.p), c, d);
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = static_cast<float>(v.e[j]);
  }
}

// Rows wider than a block's registers: the row is read three times (from the cache the second and third time).
// 2048 x 32768 bf16 83 us (268 MB, 3.2 TB/s); a weight at a time instead of a vector 279.
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_fwd_wide_kernel(NormFwd a) {
  constexpr int V = Vec<T>::N;
  __shared__ float lds[4 * (THREADS / 64)];
  int turn = 0;
  const float d = static_cast<float>(a.d), inv = 1.f / d;
  for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    T* y = static_cast<T*>(a.y) + row * a.ldy;
    float s[1] = {0.f}, q[2] = {0.f, 0.f};
#pragma unroll 4
    for (int64_t c = threadIdx.x * V; c < a.d; c += THREADS * V) {
      const Vec<T> t = load_row(x, c, a.d);
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] += static_cast<float>(t.e[j]);
    }
    group_sum<THREADS, THREADS>(s, lds, turn);
    const float mean = s[0] / d;
#pragma unroll 4
    for (int64_t c = threadIdx.x * V; c < a.d; c += THREADS * V) {
      const Vec<T> t = load_row(x, c, a.d);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float e = c + j < a.d ? static_cast<float>(t.e[j]) - mean : 0.f;
        q[0] += e;
        q[1] += e * e;
      }
    }
    group_sum<THREADS, THREADS>(q, lds, turn);
    const RowStat r(mean, q[0], q[1], inv, a.eps);
    const float shift = r.shift * r.rstd;
#pragma unroll 4
    for (int64_t c = threadIdx.x * V; c < a.d; c += THREADS * V) {
      Vec<T> t = load_row(x, c, a.d);
      float w[V], b[V];
      load_weights<T>(a.w, c, a.d, 1.f, w);
      load_weights<T>(a.b, c, a.d, 0.f, b);
#pragma unroll
      for (int j = 0; j < V; ++j) t.e[j] = static_cast<T>(((static_cast<float>(t.e[j]) - mean) * r.rstd - shift) * w[j] + b[j]);
      store_row(y, c, a.d, t);
    }
    if (threadIdx.x == 0 && a.mean != nullptr) {
      a.mean[row] = r.mean;
      a.rstd[row] = r.rstd;
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

// The backward in one pass over x and dy: G threads hold a row as NV vectors, keep the weights of their columns and
// the columns' sums of dy xhat and dy over all the rows they take, and write dx.  At the end the block joins its row
// groups' sums in their order (by lane exchange within a wave, then through LDS) into its part.  With LDS_SUMS (16
// columns a thread, one row group) the columns' sums lie in LDS instead, four of a thread together; 128 of its 160 KB.
// One pass because the sums are free beside it: dx alone takes 8192 x 4096 bf16 34 us, with the sums 41 and their join 4.5
// (201 MB, 4.9 TB/s), where a second pass would read 134 MB again.  1M x 64 float 155 us (768 MB, 5.0 TB/s: memory);
// 4096 x 16384 bf16 101 us with the join, by norm_dx_kernel and norm_cols_kernel 446.  Between rows of whole waves the
// instructions count too (16 waves a CU are all that its registers hold): a second row in flight gained nothing.
template <typename T, int G, int NV, int THREADS, bool LDS_SUMS>
__global__ __launch_bounds__(THREADS) void norm_bwd_kernel(NormBwd a) {
  constexpr int V = Vec<T>::N, kGroups = THREADS / (G < 64 ? 64 : G), kSums = LDS_SUMS ? NV * V / 4 : 0;
  static_assert(THREADS % G == 0, "whole rows");
  static_assert(!LDS_SUMS || kGroups == 1, "one row group");
  __shared__ float lds[4 * (THREADS / 64)];
  __shared__ float4 sums[LDS_SUMS ? 2 * kSums * THREADS : 1];
  __shared__ float cols[kGroups > 1 ? G * NV * V : 1];
  int turn = 0;
  const int lane = threadIdx.x % G;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (THREADS / G);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (THREADS / G);
  const float d = static_cast<float>(a.d);
  float w[NV][V], dw[NV][V], db[NV][V];
  load_columns<T>(a.w, lane, G, a.d, 1.f, w);
  if constexpr (LDS_SUMS) {
#pragma unroll
    for (int k = 0; k < 2 * kSums; ++k) sums[k * THREADS + threadIdx.x] = float4{0.f, 0.f, 0.f, 0.f};
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) dw[i][j] = db[i][j] = 0.f;
  }
  Vec<T> nx[NV], ng[NV];
  float nmean = 0.f, nrstd = 0.f;
  auto fetch = [&](int64_t row) {
    const bool live = row < a.n;  // behind the last row: no column is read, dy is 0
    const int64_t at = live ? row : a.n - 1;
    const T* x = static_cast<const T*>(a.x) + at * a.ldx;
    const T* dy = static_cast<const T*>(a.dy) + at * a.lddy;
    nmean = live ? a.mean[at] : 0.f;
    nrstd = live ? a.rstd[at] : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = live ? (i * G + lane) * V : a.d;
      nx[i] = load_row(x, c, a.d);
      ng[i] = load_row(dy, c, a.d);
    }
  };
  fetch(first + threadIdx.x / G);
  for (int64_t base = first; base < a.n; base += step) {
    const int64_t row = base + threadIdx.x / G;
    const float mean = nmean, rstd = nrstd;
    float xh[NV][V], g[NV][V];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        xh[i][j] = (static_cast<float>(nx[i].e[j]) - mean) * rstd;
        g[i][j] = static_cast<float>(ng[i].e[j]);
        if constexpr (!LDS_SUMS) {
          db[i][j] += g[i][j];
          dw[i][j] += g[i][j] * xh[i][j];
        }
      }
    // Behind the row's end dy is 0 and xhat -mean rstd, which must not be infinite: 0 times it is NaN.  Rows of whole waves
    // ask first (8192 x 4096 bf16 41.0 us, 43.7 without asking), narrow ones do not (798403 x 17 fp16 38.6 and 40.7).
    if (G < 64 || __any(!(fabsf(mean * rstd) < INFINITY)))
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j)
          if ((i * G + lane) * V + j >= a.d) xh[i][j] = 0.f;
    if constexpr (LDS_SUMS) {
      if (a.part != nullptr)
#pragma unroll
        for (int k = 0; k < kSums; ++k) {
          const float *gk = &g[k * 4 / V][k * 4 % V], *xk = &xh[k * 4 / V][k * 4 % V];
          float4* at = sums + k * THREADS + threadIdx.x;
          float4 t = at[0];
          t.x += gk[0] * xk[0];
          t.y += gk[1] * xk[1];
          t.z += gk[2] * xk[2];
          t.w += gk[3] * xk[3];
          at[0] = t;
          t = at[kSums * THREADS];
          t.x += gk[0];
          t.y += gk[1];
          t.z += gk[2];
          t.w += gk[3];
          at[kSums * THREADS] = t;
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        g[i][j] *= w[i][j];
        s[0] += g[i][j];
        s[1] += g[i][j] * xh[i][j];
      }
    if (base + step < a.n) fetch(row + step);
    if (a.dx == nullptr) continue;
    group_sum<G, THREADS>(s, lds, turn);
    const float mg = s[0] / d, mgx = s[1] / d;
    if (row < a.n) {
      T* dx = static_cast<T*>(a.dx) + row * a.lddx;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * G + lane) * V;
        Vec<T> t;
#pragma unroll
        for (int j = 0; j < V; ++j) t.e[j] = static_cast<T>(rstd * (g[i][j] - mg - xh[i][j] * mgx));
        store_row(dx, c, a.d, t);
      }
    }
  }
  if (a.part == nullptr) return;
  if constexpr (LDS_SUMS) {
#pragma unroll
    for (int k = 0; k < kSums; ++k) {
      const float4 p = sums[k * THREADS + threadIdx.x], q = sums[(kSums + k) * THREADS + threadIdx.x];
      float *pk = &dw[k * 4 / V][k * 4 % V], *qk = &db[k * 4 / V][k * 4 % V];
      pk[0] = p.x; pk[1] = p.y; pk[2] = p.z; pk[3] = p.w;
      qk[0] = q.x; qk[1] = q.y; qk[2] = q.z; qk[3] = q.w;
    }
  }
  auto join = [&](float (&v)[NV][V], int which) {
    if constexpr (G < 64)
#pragma unroll
      for (int o = G; o < 64; o <<= 1)
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) v[i][j] += __shfl_xor(v[i][j], o);
    const int group = threadIdx.x / (G < 64 ? 64 : G);
    if constexpr (kGroups > 1) {
      __syncthreads();
      for (int k = 1; k < kGroups; ++k) {  // one group after the other: the sums' order is fixed
        if (group == k && (threadIdx.x & 63) < G)
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
              float* at = cols + (i * V + j) * G + lane;
              *at = k == 1 ? v[i][j] : *at + v[i][j];
            }
        __syncthreads();
      }
    }
    if (group == 0 && (threadIdx.x & 63) < G) {
      float* to = a.part + (static_cast<int64_t>(blockIdx.x) * 2 + which) * a.d;
      const NormVec& only = which == 0 ? a.dw : a.db;  // a single part is the result: one launch for the smallest calls
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int c = (i * G + lane) * V + j;
          const float sum = kGroups > 1 ? v[i][j] + cols[(i * V + j) * G + lane] : v[i][j];
          if (c >= a.d) continue;
          if (a.parts > 1) to[c] = sum;
          else if (only.p != nullptr) only.put(c, sum);
        }
    }
  };
  join(dw, 0);
  join(db, 1);
}

// dx of rows wider than a block's registers: a block per row, which it reads twice (the second time from the cache):
// 2048 x 32768 bf16 112 us (403 MB, 3.6 TB/s).
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_dx_kernel(NormBwd a) {
  constexpr int V = Vec<T>::N;
  __shared__ float lds[4 * (THREADS / 64)];
  int turn = 0;
  const float d = static_cast<float>(a.d);
  for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* dy = static_cast<const T*>(a.dy) + row * a.lddy;
    T* dx = static_cast<T*>(a.dx) + row * a.lddx;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s[2] = {0.f, 0.f}, w[V];
#pragma unroll 4
    for (int64_t c = threadIdx.x * V; c < a.d; c += THREADS * V) {
      const Vec<T> tx = load_row(x, c, a.d), tg = load_row(dy, c, a.d);
      load_weights<T>(a.w, c, a.d, 1.f, w);
#pragma unroll
      for (int j = 0; j < V; ++j) {  // behind the row's end dy is 0, and xhat must not be infinite: see norm_bwd_kernel
        const float g = static_cast<float>(tg.e[j]) * w[j];
        s[0] += g;
        s[1] += g * (c + j < a.d ? (static_cast<float>(tx.e[j]) - mean) * rstd : 0.f);
      }
    }
    group_sum<THREADS, THREADS>(s, lds, turn);
    const float mg = s[0] / d, mgx = s[1] / d;
#pragma unroll 4
    for (int64_t c = threadIdx.x * V; c < a.d; c += THREADS * V) {
      const Vec<T> tx = load_row(x, c, a.d), tg = load_row(dy, c, a.d);
      load_weights<T>(a.w, c, a.d, 1.f, w);
      Vec<T> t;
#pragma unroll
      for (int j = 0; j < V; ++j)
        t.e[j] = static_cast<T>(rstd * (static_cast<float>(tg.e[j]) * w[j] - mg - (static_cast<float>(tx.e[j]) - mean) * rstd * mgx));
      store_row(dx, c, a.d, t);
    }
  }
}

// The rows' sums by column, of rows wider than a block's registers: a block takes 64 vectors of columns and a share of
// the rows, its 4 waves every fourth row.  2048 x 32768 bf16 50 us with the join (268 MB, 5.4 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void norm_cols_kernel(NormBwd a) {
  constexpr int V = Vec<T>::N;
  __shared__ float lds[2][4][64 * V];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c0 = static_cast<int64_t>(blockIdx.x) * 64 * V, c = c0 + lane * V;
  const int64_t per = (a.n + a.parts - 1) / a.parts, r0 = blockIdx.y * per, r1 = r0 + per < a.n ? r0 + per : a.n;
  float sw[V], sb[V];
#pragma unroll
  for (int j = 0; j < V; ++j) sw[j] = sb[j] = 0.f;
  for (int64_t row = r0 + wave; row < r1; row += 4) {
    const Vec<T> x = load_row(static_cast<const T*>(a.x) + row * a.ldx, c, a.d);
    const Vec<T> g = load_row(static_cast<const T*>(a.dy) + row * a.lddy, c, a.d);
    const float mean = a.mean[row], rstd = a.rstd[row];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      sw[j] += static_cast<float>(g.e[j]) * ((static_cast<float>(x.e[j]) - mean) * rstd);
      sb[j] += static_cast<float>(g.e[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    lds[0][wave][j * 64 + lane] = sw[j];
    lds[1][wave][j * 64 + lane] = sb[j];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * 64 * V; i += 256) {
    const int which = i / (64 * V), at = i % (64 * V);  // column c0 + (at % 64) V + at / 64
    const int64_t to = c0 + at % 64 * V + at / 64;
    const float s = (lds[which][0][at] + lds[which][1][at]) + (lds[which][2][at] + lds[which][3][at]);
    if (to < a.d) a.part[(static_cast<int64_t>(blockIdx.y) * 2 + which) * a.d + to] = s;
  }
}

// dw and db from the parts, in their order: 64 columns of the [2 d] sums a block, 16 waves over the parts.  Bound by
// its loads' latency: 256 parts of 2 x 4096 in 4.5 us (8 MB) with 8 loads of a wave on their way, 8 us with one.
__global__ __launch_bounds__(1024) void norm_cols_join_kernel(NormBwd a) {
  __shared__ float lds[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + lane, width = 2 * static_cast<int64_t>(a.d);
  float s = 0.f;
  if (c < width)
#pragma unroll 8
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

// The rows' shape: G threads a row, NV vectors a thread, E elements of a thread at most; a narrow row shares its wave
// with others (1M x 4 float forward 11 us with 2 threads a row, 31 with 8), a wide one takes 1, 2, 3, 4, 6, 8, 12 or 16
// waves (a wave without a column costs as much as any: 16384 x 1032 bf16 backward 39 us with 4 waves a row, 35 with 3).
// f(G, NV) as integral constants; false: wider than 1024 E columns.
template <typename T, int E, typename F>
bool with_shape(int32_t d, F&& f) {
  constexpr int NV = E / Vec<T>::N;
  const int nvec = (d + Vec<T>::N - 1) / Vec<T>::N;
  bool done = false;
  const auto offer = [&](auto g, auto nv) {
    if (done || nvec > decltype(g)::value * decltype(nv)::value) return;
    f(g, nv);
    done = true;
  };
  const auto one = [&](auto g) { offer(g, std::integral_constant<int, 1>{}); };
  const auto all = [&](auto g) { offer(g, std::integral_constant<int, NV>{}); };
  one(std::integral_constant<int, 2>{});
  one(std::integral_constant<int, 4>{});
  one(std::integral_constant<int, 8>{});
  one(std::integral_constant<int, 16>{});
  one(std::integral_constant<int, 32>{});
  one(std::integral_constant<int, 64>{});
  if constexpr (NV > 1) all(std::integral_constant<int, 64>{});
  all(std::integral_constant<int, 128>{});
  all(std::integral_constant<int, 192>{});
  all(std::integral_constant<int, 256>{});
  all(std::integral_constant<int, 384>{});
  all(std::integral_constant<int, 512>{});
  all(std::integral_constant<int, 768>{});
  all(std::integral_constant<int, 1024>{});
  return done;
}

// Elements of a thread: the forward keeps two weights beside each, the backward also two sums, which leaves 8 in the
// 128 registers of a 1024-thread block (16 spilled 34 to 63 of them); with the sums in LDS it is 16.
constexpr int kFwdElems = 16, kBwdElems = 8, kBwdLdsElems = 16;
constexpr int kBwdThreads = 1024;
constexpr int bwd_threads(int G) { return kBwdThreads / G * G; }  // whole rows

template <typename T>
int norm_fwd(const NormFwd& a, hipStream_t st) {
  const bool done = with_shape<T, kFwdElems>(a.d, [&](auto g, auto nv) {
    constexpr int G = decltype(g)::value, NV = decltype(nv)::value, kThreads = G > 256 ? G : 256 / G * G;
    const int grid = blocks_for(a.n, kThreads / G, kCUs * (kThreads > 512 ? 1 : 1024 / kThreads));  // 16 waves a CU
    hipLaunchKernelGGL((norm_fwd_kernel<T, G, NV, kThreads>), dim3(grid), dim3(kThreads), 0, st, a);
  });
  if (!done)
    hipLaunchKernelGGL((norm_fwd_wide_kernel<T, 1024>), dim3(blocks_for(a.n, 1, 1 << 20)), dim3(1024), 0, st, a);
  KGAT_LAUNCH_CHECK();
  return KGAT_OK;
}

// Blocks for n rows, `rows` of them at a time in each.  Up to five steps as few as take no more steps than all CUs would,
// for every block's column sums are written and read (300 x 8192 bf16 19.8 us with 150 blocks, 22.6 with 256); for more
// rows all CUs (4169 x 3757 36.0 us, 36.8 with 232).
int bwd_blocks(int64_t n, int rows) {
  const int64_t all = static_cast<int64_t>(rows) * kCUs, steps = (n + all - 1) / all;
  if (steps > 5) return kCUs;
  return steps < 1 ? 1 : static_cast<int>((n + rows * steps - 1) / (rows * steps));
}

// The row shares whose column sums are kept apart.
template <typename T>
int norm_parts(int64_t n, int32_t d) {
  int parts = 0;
  if (with_shape<T, kBwdElems>(d, [&](auto g, auto) { parts = bwd_blocks(n, kBwdThreads / decltype(g)::value); })) return parts;
  if (d <= kBwdThreads * kBwdLdsElems) return bwd_blocks(n, 1);
  const int64_t cols = (static_cast<int64_t>(d) + 64 * Vec<T>::N - 1) / (64 * Vec<T>::N);
  int64_t p = (1024 + cols - 1) / cols;  // wide rows: about 1024 blocks in all, 16 rows at least in each
  if (p > (n + 15) / 16) p = (n + 15) / 16;
  return p < 1 ? 1 : static_cast<int>(p);
}

template <typename T>
int norm_bwd(NormBwd a, hipStream_t st) {
  const bool cols = a.dw.p != nullptr || a.db.p != nullptr;
  a.parts = norm_parts<T>(a.n, a.d);
  if (!cols) a.part = nullptr;
  bool done = with_shape<T, kBwdElems>(a.d, [&](auto g, auto nv) {
    constexpr int G = decltype(g)::value, NV = decltype(nv)::value;
    hipLaunchKernelGGL((norm_bwd_kernel<T, G, NV, bwd_threads(G), false>), dim3(a.parts), dim3(bwd_threads(G)), 0, st, a);
  });
  if (!done && a.d <= kBwdThreads * kBwdLdsElems) {
    constexpr int NV = kBwdLdsElems / Vec<T>::N;
    hipLaunchKernelGGL((norm_bwd_kernel<T, kBwdThreads, NV, kBwdThreads, true>), dim3(a.parts), dim3(kBwdThreads), 0, st, a);
    done = true;
  }
  KGAT_LAUNCH_CHECK();
  if (!done && a.dx != nullptr && a.n > 0) {
    hipLaunchKernelGGL((norm_dx_kernel<T, 1024>), dim3(blocks_for(a.n, 1, 1 << 20)), dim3(1024), 0, st, a);
    KGAT_LAUNCH_CHECK();
  }
  if (!cols || (done && a.parts == 1)) return KGAT_OK;
  if (!done) {
    const int width = 64 * Vec<T>::N;
    hipLaunchKernelGGL(norm_cols_kernel<T>, dim3((a.d + width - 1) / width, a.parts), dim3(256), 0, st, a);
    KGAT_LAUNCH_CHECK();
  }
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
  NormFwd a{x, ldx, y, ldy, {const_cast<void*>(weight), w_dtype}, {const_cast<void*>(bias), w_dtype}, mean, rstd, n, d, eps};
  return with_dtype(dtype, [&](auto t) {
    return n == 0 ? static_cast<int>(KGAT_OK) : norm_fwd<decltype(t)>(a, reinterpret_cast<hipStream_t>(stream));
  });
}

extern "C" int64_t kgat_layer_norm_bwd_workspace(int32_t dtype, int64_t n, int32_t d) {
  using namespace kgat;
  if (n < 0 || d < 1 || d > KGAT_NORM_MAX_D) return -1;
  if (dtype != KGAT_F32 && dtype != KGAT_BF16 && dtype != KGAT_F16) return -1;
  return static_cast<int64_t>(dtype == KGAT_F32 ? norm_parts<float>(n, d) : norm_parts<__bf16>(n, d)) * 2 * d;
}

extern "C" int kgat_layer_norm_bwd(int32_t dtype, const void* dy, int64_t lddy, const void* x, int64_t ldx,
                                   const float* mean, const float* rstd, int32_t w_dtype, const void* weight, void* dx,
                                   int64_t lddx, void* dweight, void* dbias, int64_t n, int32_t d, float* workspace,
                                   int64_t workspace_floats, void* stream) {
  using namespace kgat;
  if (!dy || !x || !mean || !rstd || n < 0 || d < 1 || d > KGAT_NORM_MAX_D || lddy < 0 || ldx < 0 ||
      (dx != nullptr && lddx < d) || !norm_vec_ok(w_dtype, dtype) || dtype < KGAT_F32 || dtype > KGAT_F16)
    return KGAT_ERR_INVALID;
  const bool cols = dweight != nullptr || dbias != nullptr;
  if (cols && (!workspace || workspace_floats < kgat_layer_norm_bwd_workspace(dtype, n, d))) return KGAT_ERR_WORKSPACE;
  NormBwd a{dy, lddy, x, ldx, mean, rstd, {const_cast<void*>(weight), w_dtype}, {dweight, w_dtype}, {dbias, w_dtype}, dx, lddx, n, d,
            workspace, 0};
  return with_dtype(dtype, [&](auto t) { return norm_bwd<decltype(t)>(a, reinterpret_cast<hipStream_t>(stream)); });
}
