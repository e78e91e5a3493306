// Log probabilities of given items under a row of scores, the row's entropy and its best items, and the gradient
// into the scores (the distribution over the catalogue that src/model/KGAT/main.py:70-130 only ranks).
// For a row s of C scores, z = scale s, m = max s:
//   S = sum e^(z - scale m),  W = sum (z - scale m) e^(z - scale m)
//   lse = scale m + log S,  logp_j = z_j - lse,  H = -sum p log p = log S - W / S   (both terms >= 0: no cancellation)
//   ds_j = scale (sum_t g_t [item_t = j] - p_j (sum_t g_t + g_H (logp_j + H)))
// m, S and W come from one pass: who meets a larger score rescales what it has,
//   S <- S f,  W <- f (W + delta S),  delta = (old m - new m) scale,  f = e^delta.
// Exponents are kept in base 2, x = s c - rho with c = scale log2 e and rho = m c rounded: one fma and one v_exp_f32 an
// element, and rho's rounding is the same in every x and in lse.  x at the maximum is that rounding, m c - rho: 2^-5 at
// most while |m c| < 2^20.  Farther from zero (a row of nothing but a mask's -1e10) its power would leave the floats' range, so
// there x = (s - m) c, which is 0 at the maximum.
//
// Masked scores (-inf) have p = 0 and count nowhere.  A row of nothing else has no distribution: logp and lse -inf,
// H 0, gradient 0.  A row with a NaN or a +inf: everything NaN, best items -1, gradient NaN.
// A negative item is padding (logp 0, no gradient); one beyond the catalogue makes its logp and the row's gradient NaN.
#include <type_traits>

#include "dense.hpp"

namespace kgat {

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLow = -1e30f;  // a base-2 exponent whose power is 0, and whose products with 0 are 0
constexpr float kNone = -200.f;  // the same, and whose products with any gradient are finite

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }  // NaN wins

// A maximum m and the reference rho that stands for it in base 2.
struct Ref {
  float m, rho;
  bool far;  // rho's rounding is not small, or no number
  __device__ __forceinline__ Ref(float m_, float c) : m(m_), rho(m_ * c), far(!(fabsf(m_ * c) < 0x1p20f)) {}
  __device__ __forceinline__ float operator()(float s, float c) const {
    return far ? (s - m) * c : __builtin_fmaf(s, c, -rho);
  }
  __device__ __forceinline__ float at_max(float c) const { return far ? 0.f : __builtin_fmaf(m, c, -rho); }  // x of m
};

// A part of a row: its maximum, and S and W relative to it.
struct Stat {
  float m, s, w;
};

// Brings sums relative to a.m to `to` >= a.m (-inf: nothing was summed).
__device__ __forceinline__ Stat rebase(Stat a, float to, float c) {
#pragma clang fp contract(off)
  const Ref from(a.m, c), ref(to, c);
  // The new x of a score less its old one.
  float delta = from.far || ref.far ? (a.m - to) * c + (ref.at_max(c) - from.at_max(c)) : from.rho - ref.rho;
  delta = fmaxf(delta, kLow);  // from -inf, or NaN from two of them
  const float f = exp2_fast(delta);
  return {to, a.s * f, f * (a.w + delta * a.s)};
}

// Joins the parts of N lanes (a power of two): the largest maximum first, one rescaling each, then plain sums.
template <int N>
__device__ __forceinline__ Stat join_lanes(Stat a, float c) {
  const float m = lanes_all<N>(a.m, max_nan);
  a = rebase(a, m, c);
  a.s = lanes_sum<N>(a.s);
  a.w = lanes_sum<N>(a.w);
  return a;
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
  uint64_t* lists;       // [rows][splits][k], best first, 0 behind the last
  int32_t row0;          // of this launch
};

// What a whole row's sums say.
struct Row {
  bool none, bad;
  Ref ref;
  float l2;
  __device__ __forceinline__ Row(Stat r, float c)
      : none(r.m == -INFINITY), bad(!(r.m < INFINITY)), ref(r.m, c), l2(none ? 0.f : log2f(r.s)) {}
  __device__ __forceinline__ float logp(float s, float c, float scale) const {
    const float x = ref(s, c);
    if (bad || none) return bad ? NAN : -INFINITY;
    return x > -1e37f ? (x - l2) * kLn2 : (s - ref.m) * scale;  // a mask of the lowest value: s c may pass the floats' range
  }
};

// A given item of the row and its score, loaded long before they are needed.
struct Given {
  int64_t item;
  float score;
};

template <typename T>
__device__ __forceinline__ Given load_given(const LogProb& a, int row, int i) {
  Given g{-1, 0.f};
  if (i < a.t) {
    g.item = a.items[static_cast<int64_t>(row) * a.t + i];
    if (g.item >= 0 && g.item < a.cols) g.score = static_cast<float>((static_cast<const T*>(a.s) + static_cast<int64_t>(row) * a.ld)[g.item]);
  }
  return g;
}

// `g`: load_given of the thread's first item.
template <typename T>
__device__ __forceinline__ void finish_row(const LogProb& a, int row, Stat r, const Row& w, float c, Given g) {
  const int64_t rows = a.rows;
  if (threadIdx.x == 0) {
    a.stats[row] = w.bad ? NAN : r.m;
    a.stats[rows + row] = w.l2;
    a.stats[2 * rows + row] = w.bad ? NAN : w.none ? 0.f : (w.l2 - r.w / r.s) * kLn2;
    a.stats[3 * rows + row] = w.bad ? NAN : w.none ? -INFINITY : w.ref.far ? r.m * a.scale + w.l2 * kLn2 : (w.ref.rho + w.l2) * kLn2;
  }
  for (int i = threadIdx.x; i < a.t; i += blockDim.x) {
    if (i != static_cast<int>(threadIdx.x)) g = load_given<T>(a, row, i);
    a.logp[static_cast<int64_t>(row) * a.t + i] = g.item < 0 ? 0.f : g.item >= a.cols ? NAN : w.logp(g.score, c, a.scale);
  }
}

// ------------------------------------------------------------------------------------------------- best items
// A key orders by score, then by lower item: the upper half is the score's ordered bits (never 0), the lower half the
// item's complement.  0: no item.
__device__ __forceinline__ uint32_t ordered(float s) {
  const uint32_t b = __float_as_uint(s + 0.f);  // -0 and +0 are one score
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
__device__ __forceinline__ uint32_t lanes_max_bits(uint32_t v) {
  return __float_as_uint(lanes_all<64>(__uint_as_float(v), [](float x, float y) {
    const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
    return __uint_as_float(a > b ? a : b);
  }));
}
__device__ __forceinline__ uint64_t item_key(float s, uint32_t item) {
  return (static_cast<uint64_t>(ordered(s)) << 32) | (0xFFFFFFFFu - item);
}
__device__ __forceinline__ float key_score(uint64_t k) { return unordered(static_cast<uint32_t>(k >> 32)); }
__device__ __forceinline__ int32_t key_item(uint64_t k) {
  return static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(k));
}

// A block's candidates.  Scores at or above a floor enter; when the pool fills up, the k best stay and the k-th
// becomes the floor.  Every key is one of a kind, so an element's place is the number of larger keys: ranks are counted,
// not sorted, and do not depend on the order in which the candidates came.
template <int NT>
struct Pool {
  static constexpr int kSize = NT + 256;  // what is kept (at most 128) and one key of every thread always fit
  alignas(16) uint64_t key[2][kSize];
  alignas(16) uint32_t group[256];  // ordered bits of the groups' maxima, 0: empty
  int count, first_lost, now;
  uint64_t floor_key;  // the k-th key, once k were kept (0: none)
  float floor;         // no smaller score enters: behind the columns of the keys kept, an equal one ranks after them
};

template <int NT>
__device__ __forceinline__ void pool_start(Pool<NT>& p) {
  if (threadIdx.x == 0) {
    p.count = p.now = 0;
    p.first_lost = 0x7FFFFFFF;
    p.floor_key = 0;
    p.floor = -INFINITY;
  }
}

// Ranks the first n keys: f(rank, key) for those among the k best.
template <int NT, typename F>
__device__ __forceinline__ void pool_rank(const Pool<NT>& p, int n, int k, F&& f) {
  const uint64_t* key = p.key[p.now];
  for (int i = threadIdx.x; i < n; i += NT) {
    const uint64_t mine = key[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n / 2; ++j) {  // two keys a read, the same ones in all lanes
      const ulonglong2 two = reinterpret_cast<const ulonglong2*>(key)[j];
      rank += (two.x > mine ? 1 : 0) + (two.y > mine ? 1 : 0);
    }
    if ((n & 1) != 0) rank += key[n - 1] > mine ? 1 : 0;
    if (rank < k) f(rank, mine);
  }
}

// Keeps the k best of the first n keys.  The whole block calls it, between barriers of its own.
template <int NT>
__device__ __forceinline__ void pool_keep(Pool<NT>& p, int n, int k) {
  uint64_t* to = p.key[1 - p.now];
  pool_rank(p, n, k, [&](int rank, uint64_t key) { to[rank] = key; });
  __syncthreads();
  if (threadIdx.x == 0) {
    p.now = 1 - p.now;
    p.count = n < k ? n : k;
    p.first_lost = 0x7FFFFFFF;
    if (n >= k) {
      p.floor_key = to[k - 1];
      p.floor = nextafterf(key_score(to[k - 1]), INFINITY);
    }
  }
  __syncthreads();
}

// One key of every thread that has one, with room for all made before.  The whole block calls it.
template <int NT>
__device__ __forceinline__ void pool_step(Pool<NT>& p, bool in, uint64_t key, int k) {
  __syncthreads();
  const int n = p.count;
  __syncthreads();  // everyone has read the count
  if (n > Pool<NT>::kSize - NT) pool_keep(p, n, k);
  in = in && key > p.floor_key;
  const uint64_t who = __ballot(in);
  if (who != 0) {
    int base = 0;
    if ((threadIdx.x & 63) == 0) base = atomicAdd(&p.count, __popcll(who));
    base = __shfl(base, 0);
    if (in) p.key[p.now][base + __popcll(who & ((1ull << (threadIdx.x & 63)) - 1))] = key;
  }
}

// The floor from the maxima of G = 64 or 256 > k groups of the columns: with the k-th largest of them as the floor, k
// scores at least reach it, and of unordered scores hardly more: -G log(1 - k / G) on average.  `add(i, x)` puts a score
// into the group i mod G; k groups at least must have one, or all scores are candidates (4013 rows of 271, k = 20:
// 42 us so, 16 us with a floor).  One wave finds it: 64 groups by counting each one's rank; 256 bit by bit, from the
// first in which the maxima differ, until k to 9/8 k of them are left (6155 rows of 3781, k = 100: 61 us, 77 by ranks;
// 8192 rows of 1000, k = 20: 31 us by ranks, 33 by bits).
__device__ __forceinline__ uint32_t pool_groups(int k) { return k <= 48 ? 64 : 256; }

template <typename T, int NT, typename F>
__device__ __forceinline__ void pool_floor(Pool<NT>& p, int k, F&& fill) {
  if (threadIdx.x < 256) p.group[threadIdx.x] = 0;
  __syncthreads();
  const uint32_t last = pool_groups(k) - 1;
  fill([&](uint32_t i, float x) { atomicMax(&p.group[i & last], ordered(x)); });
  __syncthreads();
  if (threadIdx.x < 64) {
    uint32_t floor;
    if (last < 64) {
      const uint32_t mine = p.group[threadIdx.x];
      int reach = 0;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const uint4 g = reinterpret_cast<const uint4*>(p.group)[j];
        reach += (g.x >= mine ? 1 : 0) + (g.y >= mine ? 1 : 0) + (g.z >= mine ? 1 : 0) + (g.w >= mine ? 1 : 0);
      }
      floor = lanes_max_bits(reach >= k ? mine : 0);
    } else {
      const uint4 g = reinterpret_cast<const uint4*>(p.group)[threadIdx.x];
      const uint32_t one = __builtin_amdgcn_readfirstlane(g.x);
      uint32_t differ = (g.x ^ one) | (g.y ^ one) | (g.z ^ one) | (g.w ^ one);
      differ = __builtin_amdgcn_readfirstlane(lanes_max_bits(differ));  // its first bit is that of all together
      constexpr int kLow = std::is_same_v<T, float> ? 0 : std::is_same_v<T, __bf16> ? 16 : 13;  // the type's last bit
      const int most = k + k / 8;
      int bit = 31 - __builtin_clz(differ | 1);
      floor = one >> bit >> 1 << bit << 1;  // the bits that all share
      for (int count = 256; bit >= kLow && count > most; --bit) {
        const uint32_t v = floor | 1u << bit;
        const int more = __popcll(__ballot(g.x >= v)) + __popcll(__ballot(g.y >= v)) + __popcll(__ballot(g.z >= v)) +
                         __popcll(__ballot(g.w >= v));
        if (more >= k) {
          floor = v;
          count = more;
        }
      }
    }
    if (threadIdx.x == 0) p.floor = floor > ordered(-INFINITY) ? unordered(floor) : -INFINITY;
  }
  __syncthreads();
}

// A block takes a row (splits = 1) or a share of one, NT M columns at a time, all in registers: maximum, sums, and with
// TOP the scores that reach the pool's floor.
// Without TOP bound by memory, and nearly so by its instructions (one v_exp_f32 and seven more an element): 4096 x 65537
// float 184 us (1.07 GB, 5.8 TB/s), bf16 117 (537 MB, 4.6 TB/s; 128 with every load's and element's end of the row
// looked at).  With it the candidates' comparisons and ranks come on top: bf16 with k = 20 192 us, k = 100 282;
// 6155 x 3781 fp16, k = 100 52 us (24 without best items; candidates 17, ranks 12).  Small calls
// are a block's latency: 1 x 9500 float, k = 20 7.0 us (load, maximum, sums, floor, ranks, one after the other), 256 rows
// with k = 100 10.8.  3 x 1000003 float, k = 20: 11 us and 5.7 for the join.
// 5 waves a SIMD where 16-bit scores leave the registers for them (600 x 200003 bf16, k = 100 142 us; with 4 173).
template <typename T, bool TOP, int NT, int M>
__global__ __launch_bounds__(NT, sizeof(T) == 2 && NT == 256 ? 5 : 4) void log_prob_kernel(LogProb a) {
  constexpr int V = Vec<T>::N, U = M / V, kWaves = NT / 64;
  __shared__ Stat part[kWaves];
  __shared__ Pool<TOP ? NT : 0> pool;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = a.row0 + static_cast<int>(blockIdx.x), split = blockIdx.y;
  const T* s = static_cast<const T*>(a.s) + static_cast<int64_t>(row) * a.ld;
  const int64_t c0 = static_cast<int64_t>(split) * a.per;
  const int64_t c1 = c0 + a.per < a.cols ? c0 + a.per : a.cols;
  const float c = a.scale * kLog2e;
  if constexpr (TOP) pool_start(pool);
  Given given{-1, 0.f};
  if (a.splits == 1) given = load_given<T>(a, row, threadIdx.x);

  Stat r{-INFINITY, 0.f, 0.f};
  Vec<T> t[U];
  auto fetch = [&](int64_t base) __attribute__((always_inline)) {
    if (base + NT * M <= c1) {  // uniform; a scalar address and the thread's offset
      const T* at = s + base;
#pragma unroll
      for (int u = 0; u < U; ++u) t[u].raw = *reinterpret_cast<const u32x4_any*>(at + u * NT * V + threadIdx.x * V);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) t[u] = load_row(s, base + (u * NT + threadIdx.x) * V, c1);
    }
  };
  if constexpr (!TOP) fetch(c0);
  for (int64_t base = c0; base < c1; base += NT * M) {
    if constexpr (TOP) fetch(base);
    float f[M];
    const bool whole = base + NT * M <= c1;  // uniform
    float top = -INFINITY, tops[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      tops[u] = -INFINITY;
      if (whole || base + u * NT * V < c1) {  // uniform, as the next one: a row's last columns seldom fill a step
#pragma unroll
        for (int j = 0; j < V; ++j) f[u * V + j] = static_cast<float>(t[u].e[j]);
        if (!whole && base + (u + 1) * NT * V > c1) {
          const int64_t left = c1 - base - (u * NT + threadIdx.x) * V;
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (j >= left) f[u * V + j] = -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) tops[u] = max_nan(tops[u], f[u * V + j]);
        top = max_nan(top, tops[u]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) f[u * V + j] = -INFINITY;
      }
    }
    if constexpr (!TOP) {  // the next columns are on their way meanwhile (with the candidates' registers: other blocks)
      if (base + NT * M < c1) fetch(base + NT * M);
    }
    r = rebase(r, max_nan(r.m, top), c);
    const Ref ref(r.m, c);
    const bool far = __any(ref.far && r.m != -INFINITY);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (base + u * NT * V >= c1) break;  // uniform
      if (!far) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float x = fmaxf(__builtin_fmaf(f[u * V + j], c, -ref.rho), kLow);  // -inf (and NaN, which r.m holds): kLow
          const float e = exp2_fast(x);
          r.s += e;
          r.w += e * x;
        }
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float x = fmaxf(ref(f[u * V + j], c), kLow);
          const float e = exp2_fast(x);
          r.s += e;
          r.w += e * x;
        }
      }
    }
    if constexpr (TOP) {
      if (base == c0)
        pool_floor<T>(pool, a.k, [&](auto add) {
          const int have = static_cast<int>(c1 - c0 < NT * V ? c1 - c0 : NT * V);  // scores of first vectors
          if (have >= static_cast<int>(pool_groups(a.k)) * V) {  // the threads' maxima
            if (threadIdx.x * V < have) add(threadIdx.x, top);
          } else {  // all columns lie there: one by one, numbered so that lanes meet in no group
            const int stride = (have + V - 1) / V;
#pragma unroll
            for (int j = 0; j < V; ++j)
              if (threadIdx.x * V + j < have) add(j * stride + threadIdx.x, f[j]);
          }
        });
      // Candidates: a wave reserves room for all of its own at once.  Few vectors hold one, and few of their elements
      // reach it, so the loops are a comparison and a scalar branch an element.
      const float floor = pool.floor;
      const bool bounded = whole || floor > -INFINITY;  // uniform; else the filled-up columns would enter
      auto item = [&](int i) { return static_cast<uint32_t>(base) + (i / V * NT + threadIdx.x) * V + i % V; };
      auto enters = [&](int i) { return f[i] >= floor && (bounded || item(i) < static_cast<uint32_t>(c1)); };
      bool lost = false;
      if (__any(top >= floor)) {
        int mine = 0;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (__any(tops[u] >= floor))
#pragma unroll
            for (int j = 0; j < V; ++j) mine += __popcll(__ballot(enters(u * V + j)));
        int at = 0;
        if (lane == 0 && mine > 0) at = atomicAdd(&pool.count, mine);
        at = __shfl(at, 0);
        lost = mine > 0 && at + mine > Pool<NT>::kSize;
        if (lost) {
          if (lane == 0) atomicMin(&pool.first_lost, at);
        } else {
          uint64_t* key = pool.key[pool.now];
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (__any(tops[u] >= floor))
#pragma unroll
              for (int j = 0; j < V; ++j) {
                const int i = u * V + j;
                const bool in = enters(i);
                const uint64_t who = __ballot(in);
                if (who != 0) {
                  if (in) key[at + __popcll(who & ((1ull << lane) - 1))] = item_key(f[i], item(i));
                  at += __popcll(who);
                }
              }
        }
      }
      __syncthreads();
      const int n = pool.count, held = pool.first_lost < n ? pool.first_lost : n;
      __syncthreads();
      if (n > Pool<NT>::kSize) {
        // More candidates than room (many equal scores, or rising ones): what is held is cut to the k best, and the waves
        // that found no room go on one element at a time.
        pool_keep(pool, held, a.k);
#pragma unroll
        for (int i = 0; i < M; ++i) {
          const bool in = lost && item(i) < static_cast<uint32_t>(c1) && f[i] == f[i];
          pool_step(pool, in, item_key(f[i], item(i)), a.k);
        }
        __syncthreads();
      } else if (n > a.k + a.k / 2 + 24 && base + NT * M < c1) {
        pool_keep(pool, n, a.k);  // raises the floor for the columns to come
      }
    }
  }
  r = join_lanes<64>(r, c);
  if (lane == 0) part[wave] = r;
  __syncthreads();
  r = join_lanes<kWaves>(part[lane % kWaves], c);
  if (a.splits == 1) {
    const Row w(r, c);
    finish_row<T>(a, row, r, w, c, given);
    if constexpr (TOP) {
      const int64_t o = static_cast<int64_t>(row) * a.k;
      if (w.bad) {
        for (int i = threadIdx.x; i < a.k; i += NT) {
          a.top_item[o + i] = -1;
          a.top_logp[o + i] = NAN;
        }
      } else {
        pool_rank(pool, pool.count, a.k, [&](int rank, uint64_t key) {
          a.top_item[o + rank] = key_item(key);
          a.top_logp[o + rank] = w.logp(key_score(key), c, a.scale);
        });
      }
    }
  } else {
    const int64_t at = static_cast<int64_t>(row) * a.splits + split;
    if (threadIdx.x == 0) {
      a.part[at * 4] = r.m;
      a.part[at * 4 + 1] = r.s;
      a.part[at * 4 + 2] = r.w;
    }
    if constexpr (TOP) {
      uint64_t* to = a.lists + at * a.k;
      const int n = pool.count;
      for (int i = n + threadIdx.x; i < a.k; i += NT) to[i] = 0;
      pool_rank(pool, n, a.k, [&](int rank, uint64_t key) { to[rank] = key; });
    }
  }
}

// Joins a row's shares in their order.
template <typename T, bool TOP>
__global__ __launch_bounds__(1024) void log_prob_join_kernel(LogProb a) {
  constexpr int NT = 1024;
  __shared__ Pool<TOP ? NT : 0> pool;
  const int lane = threadIdx.x & 63, row = blockIdx.x;
  const float c = a.scale * kLog2e;
  const float* part = a.part + static_cast<int64_t>(row) * a.splits * 4;
  const Given given = load_given<T>(a, row, threadIdx.x);
  Stat r{-INFINITY, 0.f, 0.f};
  for (int p = lane; p < a.splits; p += 64) {
    const Stat b{part[4 * p], part[4 * p + 1], part[4 * p + 2]};
    const float m = max_nan(r.m, b.m);
    const Stat x = rebase(r, m, c), y = rebase(b, m, c);
    r = {m, x.s + y.s, x.w + y.w};
  }
  r = join_lanes<64>(r, c);
  const Row w(r, c);
  finish_row<T>(a, row, r, w, c, given);
  if constexpr (TOP) {
    const int64_t o = static_cast<int64_t>(row) * a.k;
    if (w.bad) {  // uniform
      for (int i = threadIdx.x; i < a.k; i += NT) {
        a.top_item[o + i] = -1;
        a.top_logp[o + i] = NAN;
      }
      return;
    }
    pool_start(pool);
    __syncthreads();
    const uint64_t* lists = a.lists + static_cast<int64_t>(row) * a.splits * a.k;
    auto score_at = [&](int64_t i) { return lists[i] != 0 ? key_score(lists[i]) : -INFINITY; };
    const int64_t n = static_cast<int64_t>(a.splits) * a.k;
    const int stride = a.splits >= a.k ? a.k : 1;  // enough lists: their best scores give the floor, else all do
    pool_floor<T>(pool, a.k, [&](auto add) {
      for (int64_t i = threadIdx.x * static_cast<int64_t>(stride), p = threadIdx.x; i < n; i += NT * static_cast<int64_t>(stride), p += NT)
        add(static_cast<uint32_t>(p), score_at(i));
    });
    const float floor = pool.floor;
    for (int64_t base = 0; base < n; base += NT) {
      const uint64_t key = base + threadIdx.x < n ? lists[base + threadIdx.x] : 0;
      const bool in = key != 0 && key_score(key) >= floor;
      const uint64_t who = __ballot(in);
      if (who != 0) {
        int at = 0;
        if (lane == 0) at = atomicAdd(&pool.count, __popcll(who));
        at = __shfl(at, 0) + __popcll(who & ((1ull << lane) - 1));
        if (in && at < Pool<NT>::kSize) pool.key[0][at] = key;
      }
    }
    __syncthreads();
    if (pool.count > Pool<NT>::kSize) {  // many equal scores: again, cut to the k best whenever the pool fills up
      __syncthreads();
      if (threadIdx.x == 0) pool.count = 0;
      for (int64_t base = 0; base < n; base += NT) {
        const uint64_t key = base + threadIdx.x < n ? lists[base + threadIdx.x] : 0;
        pool_step(pool, key != 0 && key_score(key) >= floor, key, a.k);
      }
    }
    __syncthreads();
    pool_rank(pool, pool.count, a.k, [&](int rank, uint64_t key) {
      a.top_item[o + rank] = key_item(key);
      a.top_logp[o + rank] = w.logp(key_score(key), c, a.scale);
    });
  }
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
  int32_t per;   // columns of a block
  int32_t row0;  // of this launch
};

// A block per row and share of its columns.  The given items' columns are computed first, from the scores and the
// whole list (the first of equal items sums their gradients in list order), and written last: ds may be s itself.
// Bound by memory: 4096 x 65537 bf16 212 us (1.07 GB, 5.1 TB/s).  Every block compares the items of its columns with the
// whole list: with 128 items a row the call takes 267 us, with 1024 2150 (256 x 9500 float 16 and 231).
template <typename T>
__global__ __launch_bounds__(256) void log_prob_bwd_kernel(LogProbBwd a) {
  constexpr int V = Vec<T>::N, kMine = KGAT_LOGPROB_MAX_ITEMS / 256;
  __shared__ int64_t item[KGAT_LOGPROB_MAX_ITEMS];
  __shared__ float grad[KGAT_LOGPROB_MAX_ITEMS];
  __shared__ float sums[4];
  const int row = a.row0 + static_cast<int>(blockIdx.x), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c0 = static_cast<int64_t>(blockIdx.y) * a.per;
  const int64_t c1 = c0 + a.per < a.cols ? c0 + a.per : a.cols;
  const T* s = static_cast<const T*>(a.s) + static_cast<int64_t>(row) * a.ld;
  T* ds = static_cast<T*>(a.ds) + static_cast<int64_t>(row) * a.ldds;
  const int64_t rows = a.rows;
  const float m = a.stats[row], l2 = a.stats[rows + row], h = a.stats[2 * rows + row];
  const float gh = a.dentropy != nullptr ? a.dentropy[row] : 0.f;
  const float c = a.scale * kLog2e;
  const bool none = m == -INFINITY;
  const Ref ref(m, c);
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
    const float b = ref(x, c) - l2, p = exp2_fast(b);
    return none ? 0.f : a.scale * (own - p * (g + gh * (fmaxf(b, kNone) * kLn2 + h)));
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
    Vec<T> t = load_row(s, col, c1);
#pragma unroll
    for (int j = 0; j < V; ++j) t.e[j] = static_cast<T>(slope(static_cast<float>(t.e[j]), 0.f));
    store_row(ds, col, c1, t);
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kMine; ++q)
    if (column[q] >= 0) ds[column[q]] = static_cast<T>(mine[q]);
}

struct Plan {
  int32_t splits, per;
};

// Rows of a launch, a block of 256 threads each: a grid holds fewer than 2^32 threads along x.
constexpr int32_t kLaunchRows = 1 << 23;

constexpr int32_t kTileCols = 8192;   // a 256-thread block's, 32 a thread
constexpr int32_t kWideCols = 16384;  // a 1024-thread block's, 16 a thread

// One block a row where a row fits a block's registers, or there are rows enough; else shares of whole tiles, about 4
// blocks a CU in all: 16 rows of 627037 float, k = 64 take 33 us in 77 shares and 36 in 39; 103 rows of 457241, k = 100
// 78 us in 10 shares and 89 in 19, whose lists are joined too.
Plan plan_rows(int32_t rows, int32_t cols) {
  if (rows < 1 || cols <= kWideCols || rows >= 4 * kCUs) return {1, cols};
  const int64_t tiles = (static_cast<int64_t>(cols) + kTileCols - 1) / kTileCols;
  const int64_t want = (4 * kCUs + rows - 1) / rows;
  const int64_t each = (2 * tiles + want) / (2 * want);  // tiles of a share, to the nearest
  const int64_t per = (each < 1 ? 1 : each) * kTileCols;
  if (per >= cols) return {1, cols};
  return {static_cast<int32_t>((cols + per - 1) / per), static_cast<int32_t>(per)};
}

int64_t work_floats(int32_t rows, int32_t cols, int32_t k) {
  const Plan p = plan_rows(rows, cols);
  return p.splits == 1 ? 0 : static_cast<int64_t>(rows) * p.splits * (4 + 2 * static_cast<int64_t>(k));
}

template <typename T, bool TOP>
int log_prob(LogProb a, hipStream_t st) {
  for (int64_t row0 = 0; row0 < a.rows; row0 += kLaunchRows) {
    a.row0 = static_cast<int32_t>(row0);
    const dim3 grid(a.rows - a.row0 < kLaunchRows ? a.rows - a.row0 : kLaunchRows, a.splits);
    // The smallest block that holds a row in one step: 8192 rows of 1000, k = 20 29 us with 256 x 8 columns and 51 with
    // 256 x 32.  Few longer rows: a whole CU's threads for each, 256 rows of 9500, k = 100 10.4 us, 256 x 32 15.7; from
    // 512 rows on the small block is as fast (13.9 and 13.2), at 2048 rows faster (50 and 32).  Candidates of float scores
    // want the registers that more waves need: 611 rows of 113711, k = 64 91 us with 16 columns a thread, 109 with 32;
    // with more of them the steps count (8192 rows of 9500, k = 100 174 and 148), as in 16 bits (219 rows of 436892 109
    // and 99); a row of 3781 fp16, which is one step of either, 52 and 59 for 6155.
    if (a.cols <= 2048)
      hipLaunchKernelGGL((log_prob_kernel<T, TOP, 256, 8>), grid, dim3(256), 0, st, a);
    else if (a.cols <= kWideCols && a.rows <= 2 * kCUs)
      hipLaunchKernelGGL((log_prob_kernel<T, TOP, 1024, 16>), grid, dim3(1024), 0, st, a);
    else if (a.cols <= 4096 || (TOP && sizeof(T) == 4 && a.k <= 64))
      hipLaunchKernelGGL((log_prob_kernel<T, TOP, 256, 16>), grid, dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((log_prob_kernel<T, TOP, 256, 32>), grid, dim3(256), 0, st, a);
    KGAT_LAUNCH_CHECK();
  }
  if (a.splits > 1) {
    hipLaunchKernelGGL((log_prob_join_kernel<T, TOP>), dim3(a.rows), dim3(1024), 0, st, a);
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
            reinterpret_cast<uint64_t*>(workspace + (p.splits == 1 ? 0 : static_cast<int64_t>(rows) * p.splits * 4)), 0};
  return with_dtype(dtype, [&](auto e) -> int {
    using T = decltype(e);
    if (rows == 0) return KGAT_OK;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    return k == 0 ? log_prob<T, false>(a, st) : log_prob<T, true>(a, st);
  });
}

extern "C" int kgat_log_prob_bwd(int32_t dtype, const void* scores, int64_t ld, int32_t rows, int32_t cols, float scale,
                                 const int64_t* items, int32_t t, const float* stats, const float* dlogp,
                                 const float* dentropy, void* dscores, int64_t ld_dscores, void* stream) {
  using namespace kgat;
  if (!scores_ok(scores, ld, rows, cols, items, t, scale) || !stats || (t > 0 && !dlogp) || !dscores ||
      ld_dscores < cols)
    return KGAT_ERR_INVALID;
  int32_t per = 16384;
  while ((static_cast<int64_t>(cols) + per - 1) / per > 65535) per *= 2;  // a grid's limit along y
  const uint32_t shares = static_cast<uint32_t>((static_cast<int64_t>(cols) + per - 1) / per);
  LogProbBwd a{scores, ld, rows, cols, scale, items, t, stats, dlogp, dentropy, dscores, ld_dscores, per, 0};
  return with_dtype(dtype, [&](auto e) -> int {
    using T = decltype(e);
    for (int64_t row0 = 0; row0 < rows; row0 += kLaunchRows) {
      a.row0 = static_cast<int32_t>(row0);
      const dim3 grid(rows - a.row0 < kLaunchRows ? rows - a.row0 : kLaunchRows, shares);
      hipLaunchKernelGGL(log_prob_bwd_kernel<T>, grid, dim3(256), 0, reinterpret_cast<hipStream_t>(stream), a);
      KGAT_LAUNCH_CHECK();
    }
    return KGAT_OK;
  });
}
