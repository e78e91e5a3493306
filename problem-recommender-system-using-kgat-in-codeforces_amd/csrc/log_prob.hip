// Log probabilities of given items under a row of scores, the row's entropy and its best items, and the gradient
// into the scores (the distribution over the catalogue that src/model/KGAT/main.py:70-130 only ranks).
// For a row s of C scores, z = scale s, m = max s:
//   S = sum e^(z - scale m),  W = sum (z - scale m) e^(z - scale m)
//   lse = scale m + log S,  logp_j = z_j - lse,  H = -sum p log p = log S - W / S   (both terms >= 0: no cancellation)
//   ds_j = scale (sum_t g_t [item_t = j] - p_j (sum_t g_t + g_H (logp_j + H)))
// m, S and W come from one pass: a thread that meets a larger score rescales what it has,
//   S <- S f,  W <- f (W + delta S),  delta = (old m - new m) scale,  f = e^delta.
// Everything is kept in base 2 (t = (s - m) scale log2 e, one v_exp_f32 an element).  The difference is taken before
// the product, so that rows of one single value, were it the type's lowest, come out uniform.
//
// Masked scores (-inf) have p = 0 and count nowhere.  A row of nothing else has no distribution: logp and lse -inf,
// H 0, gradient 0.  A row with a NaN or a +inf: everything NaN, best items -1, gradient NaN.
// A negative item is padding (logp 0, no gradient); one beyond the catalogue makes its logp and the row's gradient NaN.
#include "dense.hpp"

namespace kgat {

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLow = -1e30f;  // a base-2 exponent whose power is 0, and whose products with 0 are 0

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// A part of a row: its maximum, and S and W relative to it.
struct Stat {
  float m, s, w;
};

// The factor that brings sums relative to `from` to `to` >= from (-inf: nothing was summed).
__device__ __forceinline__ Stat rebase(Stat a, float to, float c) {
  const float delta = fmaxf((a.m - to) * c, kLow);  // from -inf (or NaN from two of them): kLow
  const float f = exp2_fast(delta);
  return {to, a.s * f, f * (a.w + delta * a.s)};
}

__device__ __forceinline__ Stat combine(Stat a, Stat b, float c) {
  const float m = fmaxf(a.m, b.m);
  a = rebase(a, m, c);
  b = rebase(b, m, c);
  return {m, a.s + b.s, a.w + b.w};
}

// ------------------------------------------------------------------------------------------------- best items
// A key orders by score, then by lower item: the upper half is the score's ordered bits (never 0), the lower half the
// item's complement.  0: no item.
__device__ __forceinline__ uint64_t item_key(float s, uint32_t item) {
  const uint32_t b = __float_as_uint(s + 0.f);  // -0 and +0 are one score
  const uint32_t o = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (static_cast<uint64_t>(o) << 32) | (0xFFFFFFFFu - item);
}
__device__ __forceinline__ float key_score(uint64_t k) {
  const uint32_t o = static_cast<uint32_t>(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
__device__ __forceinline__ int32_t key_item(uint64_t k) {
  return static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(k));
}

// A wave's list of its 64 E largest keys, descending: element 64 i + lane in k[i].
template <int E>
struct Best {
  uint64_t k[E];
};

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int o) {
  const uint32_t lo = static_cast<uint32_t>(__shfl_xor(static_cast<int>(static_cast<uint32_t>(v)), o));
  const uint32_t hi = static_cast<uint32_t>(__shfl_xor(static_cast<int>(static_cast<uint32_t>(v >> 32)), o));
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

// Orders a wave's LDS writes before its later LDS reads by other lanes (LDS works in order within a wave: this holds
// the compiler, and costs no instruction).
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Sorts a bitonic list of 64 E descending.
template <int E>
__device__ __forceinline__ void merge_down(Best<E>& b, int lane) {
#pragma unroll
  for (int i = E / 2; i > 0; i >>= 1)
#pragma unroll
    for (int j = 0; j < E; ++j)
      if ((j & i) == 0) {
        const uint64_t x = b.k[j], y = b.k[j + i];
        b.k[j] = x > y ? x : y;
        b.k[j + i] = x > y ? y : x;
      }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const uint64_t x = b.k[j], y = shfl_xor64(x, o);
      b.k[j] = ((lane & o) == 0) == (x > y) ? x : y;
    }
}

// 64 keys, one a lane, sorted descending.
__device__ __forceinline__ uint64_t sort64(uint64_t v, int lane) {
#pragma unroll
  for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o > 0; o >>= 1) {
      const uint64_t y = shfl_xor64(v, o);
      const bool down = (lane & size) == 0, low = (lane & o) == 0;
      v = (down == low) == (v > y) ? v : y;
    }
  return v;
}

// The 64 E largest of the list and of another sorted one: the larger of element i of one and of the last but i of
// the other are those, and bitonic.
template <int E>
__device__ __forceinline__ void merge(Best<E>& a, const Best<E>& b, int lane) {
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const uint64_t y = shfl_xor64(b.k[E - 1 - i], 63);
    a.k[i] = a.k[i] > y ? a.k[i] : y;
  }
  merge_down(a, lane);
}

template <int E>
__device__ __forceinline__ uint64_t key_at(const Best<E>& b, int i) {  // i uniform
  uint64_t v = b.k[0];
  if (E > 1 && i >= 64) v = b.k[E - 1];
  const uint32_t lo = static_cast<uint32_t>(__shfl(static_cast<int>(static_cast<uint32_t>(v)), i & 63));
  const uint32_t hi = static_cast<uint32_t>(__shfl(static_cast<int>(static_cast<uint32_t>(v >> 32)), i & 63));
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

struct LogProb {
  const void* s;
  int64_t ld;
  int32_t rows, cols;
  float scale;
  const int64_t* items;  // [rows][t]
  int32_t t, k;
  float* logp;           // [rows][t]
  float* stats;          // [4][rows]: m, log2 S, H, lse
  int64_t* top_item;     // [rows][k]
  float* top_logp;       // [rows][k]
  int32_t splits;        // blocks of a row
  int32_t per;           // columns of a split
  float* part;           // [rows][splits][4]: m, S, W
  uint64_t* lists;       // [rows][splits][k]
};

// What a whole row's sums say: written by one block.
template <typename T>
__device__ __forceinline__ void finish_row(const LogProb& a, int row, Stat r) {
  const T* s = static_cast<const T*>(a.s) + static_cast<int64_t>(row) * a.ld;
  const bool none = r.s == 0.f;  // nothing but -inf
  const float l2 = none ? 0.f : log2f(r.s);
  const float ls = l2 * kLn2;
  if (threadIdx.x == 0) {
    a.stats[row] = none ? -INFINITY : r.s != r.s ? r.s : r.m;
    a.stats[a.rows + row] = l2;
    a.stats[2 * static_cast<int64_t>(a.rows) + row] = none ? 0.f : ls - r.w / r.s * kLn2;
    a.stats[3 * static_cast<int64_t>(a.rows) + row] = none ? -INFINITY : r.m * a.scale + ls;
  }
  for (int i = threadIdx.x; i < a.t; i += blockDim.x) {
    const int64_t at = static_cast<int64_t>(row) * a.t + i, j = a.items[at];
    float v = 0.f;
    if (j >= a.cols) v = NAN;
    else if (j >= 0) v = none ? -INFINITY : (static_cast<float>(s[j]) - r.m) * a.scale - ls;
    a.logp[at] = v;
  }
}

template <int E>
__device__ __forceinline__ void write_best(const LogProb& a, int row, Stat r, const Best<E>& b, int lane) {
  const bool none = r.s == 0.f, bad = r.s != r.s;
  const float ls = none ? 0.f : log2f(r.s) * kLn2;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int at = i * 64 + lane;
    if (at < a.k) {
      const int64_t o = static_cast<int64_t>(row) * a.k + at;
      a.top_item[o] = bad ? -1 : key_item(b.k[i]);
      a.top_logp[o] = bad ? NAN : none ? -INFINITY : (key_score(b.k[i]) - r.m) * a.scale - ls;
    }
  }
}

// One block per row (splits = 1) or per share of a row.  E: 64-key registers of the lists (0: no best items).
template <typename T, int E, int THREADS>
__global__ __launch_bounds__(THREADS) void log_prob_kernel(LogProb a) {
  constexpr int V = Vec<T>::N, kWaves = THREADS / 64, kList = E > 0 ? 64 * E : 1;
  __shared__ Stat part[kWaves];
  __shared__ uint64_t queue[E > 0 ? kWaves * 128 : 1];
  __shared__ uint64_t lists[E > 0 ? kWaves * kList : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = blockIdx.x, split = blockIdx.y;
  const T* s = static_cast<const T*>(a.s) + static_cast<int64_t>(row) * a.ld;
  const int64_t c0 = static_cast<int64_t>(split) * a.per;
  const int64_t c1 = c0 + a.per < a.cols ? c0 + a.per : a.cols;
  const float c = a.scale * kLog2e;

  Stat r{-INFINITY, 0.f, 0.f};
  Best<E < 1 ? 1 : E> best;
  uint64_t* mine = queue + (E > 0 ? wave * 128 : 0);
  int queued = 0, held = 0;    // keys in the queue; keys that reached the list
  float floor = -INFINITY;     // the list's k-th score once it holds k,
  uint64_t floor_key = 0;      // and its key
  bool full = false;
  if constexpr (E > 0) {
#pragma unroll
    for (int i = 0; i < E; ++i) best.k[i] = 0;
  }
  // Takes the queue's first 64 keys (fewer at the end) into the list.
  auto drain = [&]() {
    if constexpr (E > 0) {
      const int take = queued < 64 ? queued : 64;
      Best<E> b;
#pragma unroll
      for (int i = 1; i < E; ++i) b.k[i] = 0;
      b.k[0] = sort64(lane < take ? mine[lane] : 0, lane);
      const uint64_t rest = 64 + lane < queued ? mine[64 + lane] : 0;
      wave_fence();
      mine[lane] = rest;
      wave_fence();
      merge<E>(best, b, lane);
      queued -= take;
      held += take;
      if (held >= a.k) {
        full = true;
        floor_key = key_at<E>(best, a.k - 1);
        floor = key_score(floor_key);
      }
    }
  };
  for (int64_t base = c0 + static_cast<int64_t>(wave) * 64 * V; base < c1; base += static_cast<int64_t>(THREADS) * V) {
    const int64_t col = base + lane * V;
    const Vec<T> t = load_vec(s + col, c1 - col, -INFINITY);
    float f[V], top = -INFINITY;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      f[j] = static_cast<float>(t.e[j]);
      top = fmaxf(top, f[j]);
    }
    const float m = fmaxf(r.m, top);
    r = rebase(r, m, c);
    const float ms = fmaxf(m, -3.402823466e38f);  // no score yet: -inf - ms stays -inf
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float x = (f[j] - ms) * c, e = exp2_fast(x);
      r.s += e;
      r.w += e * fmaxf(x, kLow);
    }
    if constexpr (E > 0) {
      // Columns rise from vector to vector of a wave, so a score equal to the list's k-th ranks behind it: once the
      // list holds k, only a larger one opens the vector (within it, the keys decide).
      if (__any(top > floor || !full)) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const uint64_t key = item_key(f[j], static_cast<uint32_t>(col + j));
          const bool in = (key > floor_key || !full) && col + j < c1;
          const uint64_t who = __ballot(in);
          if (who != 0) {
            if (in) mine[queued + __popcll(who & ((1ull << lane) - 1))] = key;
            queued += __popcll(who);
            wave_fence();
            if (queued >= 64) drain();
          }
        }
      }
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const Stat b{__shfl_xor(r.m, o), __shfl_xor(r.s, o), __shfl_xor(r.w, o)};
    r = combine(r, b, c);
  }
  if (lane == 0) part[wave] = r;
  if constexpr (E > 0) {
    if (queued > 0) drain();
#pragma unroll
    for (int i = 0; i < E; ++i) lists[wave * kList + i * 64 + lane] = best.k[i];
  }
  __syncthreads();
  r = part[0];
  for (int w = 1; w < kWaves; ++w) r = combine(r, part[w], c);
  if constexpr (E > 0) {
    if (wave == 0) {
      for (int w = 1; w < kWaves; ++w) {
        Best<E> b;
#pragma unroll
        for (int i = 0; i < E; ++i) b.k[i] = lists[w * kList + i * 64 + lane];
        merge<E>(best, b, lane);
      }
      if (a.splits == 1) {
        write_best<E>(a, row, r, best, lane);
      } else {
        uint64_t* to = a.lists + (static_cast<int64_t>(row) * a.splits + split) * a.k;
#pragma unroll
        for (int i = 0; i < E; ++i)
          if (i * 64 + lane < a.k) to[i * 64 + lane] = best.k[i];
      }
    }
  }
  if (a.splits == 1) {
    finish_row<T>(a, row, r);
  } else if (threadIdx.x == 0) {
    float* to = a.part + (static_cast<int64_t>(row) * a.splits + split) * 4;
    to[0] = r.m;
    to[1] = r.s;
    to[2] = r.w;
  }
}

// Joins a row's shares in their order.
template <typename T, int E>
__global__ __launch_bounds__(256) void log_prob_join_kernel(LogProb a) {
  constexpr int kList = E > 0 ? 64 * E : 1;
  __shared__ uint64_t lists[E > 0 ? 4 * kList : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = blockIdx.x;
  const float c = a.scale * kLog2e;
  const float* part = a.part + static_cast<int64_t>(row) * a.splits * 4;
  Stat r{-INFINITY, 0.f, 0.f};
  for (int p = lane; p < a.splits; p += 64) r = combine(r, {part[4 * p], part[4 * p + 1], part[4 * p + 2]}, c);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const Stat b{__shfl_xor(r.m, o), __shfl_xor(r.s, o), __shfl_xor(r.w, o)};
    r = combine(r, b, c);
  }
  if constexpr (E > 0) {
    Best<E> best;
#pragma unroll
    for (int i = 0; i < E; ++i) best.k[i] = 0;
    for (int p = wave; p < a.splits; p += 4) {
      const uint64_t* from = a.lists + (static_cast<int64_t>(row) * a.splits + p) * a.k;
      Best<E> b;
#pragma unroll
      for (int i = 0; i < E; ++i) b.k[i] = i * 64 + lane < a.k ? from[i * 64 + lane] : 0;
      merge<E>(best, b, lane);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) lists[wave * kList + i * 64 + lane] = best.k[i];
    __syncthreads();
    if (wave == 0) {
      for (int w = 1; w < 4; ++w) {
        Best<E> b;
#pragma unroll
        for (int i = 0; i < E; ++i) b.k[i] = lists[w * kList + i * 64 + lane];
        merge<E>(best, b, lane);
      }
      write_best<E>(a, row, r, best, lane);
    }
  }
  finish_row<T>(a, row, r);
}

struct LogProbBwd {
  const void* s;
  int64_t ld;
  int32_t rows, cols;
  float scale;
  const int64_t* items;
  int32_t t;
  const float* stats;
  const float* dlogp;     // [rows][t]
  const float* dentropy;  // [rows] (nullable)
  void* ds;
  int64_t ldds;
  int32_t per;  // columns of a block
};

// A block per row and share of its columns.  The given items' columns are computed first, from the scores and the
// whole list (the first of equal items sums their gradients in list order), and written last: ds may be s itself.
template <typename T>
__global__ __launch_bounds__(256) void log_prob_bwd_kernel(LogProbBwd a) {
  constexpr int V = Vec<T>::N, kMine = KGAT_LOGPROB_MAX_ITEMS / 256;
  __shared__ int64_t item[KGAT_LOGPROB_MAX_ITEMS];
  __shared__ float grad[KGAT_LOGPROB_MAX_ITEMS];
  __shared__ float sums[4];
  const int row = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c0 = static_cast<int64_t>(blockIdx.y) * a.per;
  const int64_t c1 = c0 + a.per < a.cols ? c0 + a.per : a.cols;
  const T* s = static_cast<const T*>(a.s) + static_cast<int64_t>(row) * a.ld;
  T* ds = static_cast<T*>(a.ds) + static_cast<int64_t>(row) * a.ldds;
  const float m = a.stats[row], l2 = a.stats[a.rows + row], h = a.stats[2 * static_cast<int64_t>(a.rows) + row];
  const float gh = a.dentropy != nullptr ? a.dentropy[row] : 0.f;
  const float c = a.scale * kLog2e;
  const bool none = m == -INFINITY;
  float g = 0.f;
  for (int i = threadIdx.x; i < a.t; i += 256) {
    const int64_t at = static_cast<int64_t>(row) * a.t + i, j = a.items[at];
    const float v = j < 0 ? 0.f : j >= a.cols ? NAN : a.dlogp[at];
    item[i] = j;
    grad[i] = v;
    g += v;
  }
  g = wave_sum(g);
  if (lane == 0) sums[wave] = g;
  __syncthreads();
  g = (sums[0] + sums[1]) + (sums[2] + sums[3]);

  auto slope = [&](float x, float own) {
    const float b = (x - m) * c - l2, p = exp2_fast(b);
    return none ? 0.f : a.scale * (own - p * (g + gh * (fmaxf(b, kLow) * kLn2 + h)));
  };
  float mine[kMine];
  int32_t column[kMine];  // -1: not this thread's to write
#pragma unroll
  for (int q = 0; q < kMine; ++q) {
    const int i = q * 256 + threadIdx.x;
    mine[q] = 0.f;
    column[q] = -1;
    if (i < a.t && item[i] >= c0 && item[i] < c1) {
      float own = 0.f;
      bool first = true;
      for (int o = 0; o < a.t; ++o)
        if (item[o] == item[i]) {
          first = first && o >= i;
          own += grad[o];
        }
      if (first) {
        column[q] = static_cast<int32_t>(item[i]);
        mine[q] = slope(static_cast<float>(s[item[i]]), own);
      }
    }
  }
  __syncthreads();
  for (int64_t col = c0 + threadIdx.x * V; col < c1; col += 256 * V) {
    Vec<T> t = load_vec(s + col, c1 - col);
#pragma unroll
    for (int j = 0; j < V; ++j) t.e[j] = static_cast<T>(slope(static_cast<float>(t.e[j]), 0.f));
    store_vec(ds + col, t, c1 - col);
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kMine; ++q)
    if (column[q] >= 0) ds[column[q]] = static_cast<T>(mine[q]);
}

struct Plan {
  int32_t splits, per;
};

// Shares of a row: enough blocks for the chip where there are few rows, and no share under 8192 columns.
Plan plan_rows(int32_t rows, int32_t cols) {
  if (rows < 1) return {1, cols};
  int64_t splits = (4 * kCUs + rows - 1) / rows;
  const int64_t most = (static_cast<int64_t>(cols) + 8191) / 8192;
  if (splits > most) splits = most;
  if (cols <= 16384) splits = 1;
  const int64_t per = ((cols + splits - 1) / splits + 2047) / 2048 * 2048;
  if (splits == 1 || per >= cols) return {1, cols};
  return {static_cast<int32_t>((cols + per - 1) / per), static_cast<int32_t>(per)};
}

int64_t work_floats(int32_t rows, int32_t cols, int32_t k) {
  const Plan p = plan_rows(rows, cols);
  return p.splits == 1 ? 0 : static_cast<int64_t>(rows) * p.splits * (4 + 2 * static_cast<int64_t>(k));
}

template <typename T, int E>
int log_prob(const LogProb& a, hipStream_t st) {
  const dim3 grid(a.rows, a.splits);
  if (a.splits == 1 && a.cols > 4096 && a.rows <= 2 * kCUs)
    hipLaunchKernelGGL((log_prob_kernel<T, E, 1024>), grid, dim3(1024), 0, st, a);
  else
    hipLaunchKernelGGL((log_prob_kernel<T, E, 256>), grid, dim3(256), 0, st, a);
  KGAT_LAUNCH_CHECK();
  if (a.splits > 1) {
    hipLaunchKernelGGL((log_prob_join_kernel<T, E>), dim3(a.rows), dim3(256), 0, st, a);
    KGAT_LAUNCH_CHECK();
  }
  return KGAT_OK;
}

bool scores_ok(const void* s, int64_t ld, int32_t rows, int32_t cols, const int64_t* items, int32_t t, float scale) {
  return s != nullptr && rows >= 0 && cols >= 1 && ld >= 0 && t >= 0 && t <= KGAT_LOGPROB_MAX_ITEMS &&
         (t == 0 || items != nullptr) && scale >= 0x1p-64f && scale <= 0x1p64f;
}

}  // namespace

}  // namespace kgat

extern "C" int64_t kgat_log_prob_workspace(int32_t rows, int32_t cols, int32_t k) {
  if (rows < 0 || cols < 1 || k < 0 || k > KGAT_LOGPROB_MAX_K) return -1;
  return kgat::work_floats(rows, cols, k);
}

extern "C" int kgat_log_prob_fwd(int32_t dtype, const void* scores, int64_t ld, int32_t rows, int32_t cols, float scale,
                                 const int64_t* items, int32_t t, int32_t k, float* logp, float* stats,
                                 int64_t* top_item, float* top_logp, float* workspace, int64_t workspace_floats,
                                 void* stream) {
  using namespace kgat;
  if (!scores_ok(scores, ld, rows, cols, items, t, scale) || !stats || (t > 0 && !logp) || k < 0 || k > cols ||
      k > KGAT_LOGPROB_MAX_K || (k > 0 && (!top_item || !top_logp)))
    return KGAT_ERR_INVALID;
  const int64_t need = work_floats(rows, cols, k);
  if (need > 0 && (!workspace || workspace_floats < need || (reinterpret_cast<uintptr_t>(workspace) & 7)))
    return KGAT_ERR_WORKSPACE;
  const Plan p = plan_rows(rows, cols);
  LogProb a{scores, ld, rows, cols, scale, items, t, k, logp, stats, top_item, top_logp, p.splits, p.per, workspace,
            reinterpret_cast<uint64_t*>(workspace + (p.splits == 1 ? 0 : static_cast<int64_t>(rows) * p.splits * 4))};
  return with_dtype(dtype, [&](auto e) -> int {
    using T = decltype(e);
    if (rows == 0) return KGAT_OK;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    return k == 0 ? log_prob<T, 0>(a, st) : k <= 64 ? log_prob<T, 1>(a, st) : log_prob<T, 2>(a, st);
  });
}

extern "C" int kgat_log_prob_bwd(int32_t dtype, const void* scores, int64_t ld, int32_t rows, int32_t cols, float scale,
                                 const int64_t* items, int32_t t, const float* stats, const float* dlogp,
                                 const float* dentropy, void* dscores, int64_t ld_dscores, void* stream) {
  using namespace kgat;
  if (!scores_ok(scores, ld, rows, cols, items, t, scale) || !stats || (t > 0 && !dlogp) || !dscores ||
      ld_dscores < cols)
    return KGAT_ERR_INVALID;
  constexpr int32_t per = 16384;
  LogProbBwd a{scores, ld, rows, cols, scale, items, t, stats, dlogp, dentropy, dscores, ld_dscores, per};
  const int64_t shares = (static_cast<int64_t>(cols) + per - 1) / per;
  if (shares > 65535) return KGAT_ERR_INVALID;
  return with_dtype(dtype, [&](auto e) -> int {
    using T = decltype(e);
    if (rows == 0) return KGAT_OK;
    hipLaunchKernelGGL(log_prob_bwd_kernel<T>, dim3(rows, static_cast<uint32_t>(shares)), dim3(256), 0,
                       reinterpret_cast<hipStream_t>(stream), a);
    KGAT_LAUNCH_CHECK();
    return KGAT_OK;
  });
}
