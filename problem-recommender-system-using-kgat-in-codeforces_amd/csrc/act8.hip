// Activations kept in 8 bits between the forward and the backward.
//
// A row's columns are cut into blocks of 32.  With A the largest |x| of a block,
//   e = floor(log2 A) - 6  (at least -126),   q = clamp(round_half_even(x 2^-e), -127, 127),   value = q 2^e,
// so |x - value| <= 2^-7 A: A lies in [64, 128) steps of 2^e, rounding costs half a step of 64 or more, and clipping a
// steps to 127 costs (a - 127) / a < 1 / 128 (at the least e, 2^-127 in place of it).  A block that holds an infinity or
// a NaN has the exponent code 255 and stands for NaN in all its columns: a diverged step stays visible.
// Stored: q as int8 [n, 32 ceil(d/32)] (zeros behind column d), the code e + 127 as one byte a block.
//
// The power-of-two scale costs up to one bit against max / 127, and buys exactness: q 2^e has 7 bits of mantissa,
// so it IS a bf16 number, and the weight gradient dW = dy^T x runs on the bf16 matrix instructions without any
// further rounding of x.  dy goes in as it is (bf16) or as the exact sum of two (fp16) or three (float) bf16 terms: of a
// float its digits down to bf16's last, 2^-133, which is all of them from 2^-110 up.
// Where x was fp16 its value is an fp16 number too, and fp16 dy goes in as it is: q has 7 bits, |q 2^e| <= 127 * 2^9, and
// where 2^e lies below fp16's last bit, 2^-24, x 2^-e is an even integer below 128, so that q 2^e is x itself.
#include <type_traits>

#include "dense.hpp"

namespace kgat {

namespace {

constexpr int kBlock = KGAT_ACT8_BLOCK;

__device__ __forceinline__ float scale_of(uint32_t code) { return __uint_as_float(code << 23); }  // 255: inf

struct Pack {
  const void* x;
  int64_t ldx;
  int8_t* q;
  uint8_t* e;
  int64_t n;
  int32_t d;
};

// A thread packs one 16-byte vector of a row, the 8 (float) or 4 (16-bit) threads of a block share its maximum.
// Bound by memory: 1M x 128 float 138 us (644 MB, 4.7 TB/s), 16384 x 4096 bf16 40 us (203 MB, 5.1 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void act8_pack_kernel(Pack a) {
  constexpr int V = Vec<T>::N, kLanes = kBlock / V;
  const int32_t nb = (a.d + kBlock - 1) / kBlock;
  const uint32_t per_row = static_cast<uint32_t>(nb) * kLanes;  // vectors of a padded row
  const int64_t first = static_cast<int64_t>(blockIdx.x) * 256;
  const int64_t row0 = first / per_row;  // uniform
  const uint32_t at = static_cast<uint32_t>(first - row0 * per_row) + threadIdx.x;
  const int64_t row = row0 + at / per_row;
  const int32_t vec = static_cast<int32_t>(at % per_row), c = vec * V;
  const bool live = row < a.n;
  const Vec<T> t = load_row(static_cast<const T*>(a.x) + (live ? row : a.n - 1) * a.ldx, c, a.d);
  uint32_t top = 0;
  float f[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    f[j] = static_cast<float>(t.e[j]);
    const uint32_t b = __float_as_uint(f[j]) & 0x7FFFFFFFu;  // |f| orders as its bits; inf and NaN are the largest
    top = top > b ? top : b;
  }
  // Bits of values >= 0 order as integers: the maximum over the block's lanes.
  top = __float_as_uint(lanes_all<kLanes>(__uint_as_float(top), [](float x, float y) {
    const uint32_t p = __float_as_uint(x), q = __float_as_uint(y);
    return __uint_as_float(p > q ? p : q);
  }));
  if (!live) return;
  const uint32_t ex = top >> 23;  // biased exponent of the maximum
  const uint32_t code = ex == 255 ? 255u : ex < 7 ? 1u : ex - 6;
  const float inv = __uint_as_float((254u - code) << 23);  // 2^-e (code 255: unused)
  uint32_t w[V / 4] = {};
  if (code != 255) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int v = static_cast<int>(fminf(fmaxf(rintf(f[j] * inv), -127.f), 127.f));
      w[j / 4] |= (static_cast<uint32_t>(v) & 255u) << (8 * (j % 4));
    }
  }
  uint32_t* q = reinterpret_cast<uint32_t*>(a.q + row * (static_cast<int64_t>(nb) * kBlock) + c);
#pragma unroll
  for (int j = 0; j < V / 4; ++j) q[j] = w[j];
  if (vec % kLanes == 0) a.e[row * nb + vec / kLanes] = static_cast<uint8_t>(code);
}

struct Unpack {
  const int8_t* q;
  const uint8_t* e;
  void* x;
  int64_t ldx;
  int64_t n;
  int32_t d;
};

// A thread a 16-byte vector.  1M x 128 float 127 us (644 MB, 5.1 TB/s): memory.
template <typename T>
__global__ __launch_bounds__(256) void act8_unpack_kernel(Unpack a) {
  constexpr int V = Vec<T>::N;
  const int32_t nb = (a.d + kBlock - 1) / kBlock;
  const uint32_t per_row = (static_cast<uint32_t>(a.d) + V - 1) / V;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * 256;
  const int64_t row0 = first / per_row;
  const uint32_t at = static_cast<uint32_t>(first - row0 * per_row) + threadIdx.x;
  const int64_t row = row0 + at / per_row;
  const int32_t c = static_cast<int32_t>(at % per_row) * V;
  if (row >= a.n) return;
  const uint32_t* q = reinterpret_cast<const uint32_t*>(a.q + row * (static_cast<int64_t>(nb) * kBlock) + c);
  const float s = scale_of(a.e[row * nb + c / kBlock]);
  Vec<T> t;
#pragma unroll
  for (int j = 0; j < V; ++j)
    t.e[j] = static_cast<T>(static_cast<float>(static_cast<int8_t>(q[j / 4] >> (8 * (j % 4)))) * s);
  store_row(static_cast<T*>(a.x) + row * a.ldx, c, a.d, t);
}

// ---------------------------------------------------------------------------------------------- weight gradient
// dW[o, i] = sum_n dy[n, o] x[n, i]: a block of 2 B threads takes a B x B tile of dW and a share of the rows (split
// over the grid, the shares' tiles summed in order by act8_join_kernel), 64 rows a step.  The reduction runs over the
// rows, which both operands store apart: a thread takes 8 rows x 4 columns and turns them in its registers (v_perm
// pairs the halves of two rows; x is decoded on the way: v_cvt_f32_ubyte, one fma with the scale, the upper halves), so
// that LDS holds [column][row] with the 8 rows of a lane's operand together, one ds_read_b128 for a
// v_mfma_f32_32x32x16_bf16.  Column 4 c + j of the tile lies at LDS row (B / 4) j + c: the threads of a row write
// neighbouring LDS rows at a pitch of 36 dwords, which spreads 16 of them over all 64 banks.
//
// bf16 dy, n = 16384, o = d = 4096: 517 us called again and again on the same operands (1.06 PFLOP/s; a library's
// product of 16-bit operands 565), 580 to 716, mean 631, in a trace of the first 20 calls with their packs.  The matrix
// instructions are busy half of the time at 2.0 GHz; without the decoding the kernel takes 402 us, so what is left of it is
// LDS reads and their waits beside the products.  fp16 dy and x 531; fp16 dy as two terms 950, float as three 1374.
// Narrow outputs are bound by the decoding, which every tile repeats for its own columns: n = 100003, o = 131, d = 257 in
// fp16 36 us and 4 for the join (15 tiles of 64; two terms 59).
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __fp16 half2v __attribute__((ext_vector_type(2)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

constexpr int kDepth = 64;                  // rows a step
constexpr int kLdsPitch = kDepth * 2 + 16;  // bytes
constexpr int32_t kNarrow = 4;              // fewer columns of dy are no quad: the NARROW kernel

struct Wgrad {
  const void* dy;
  int64_t lddy;
  const int8_t* q;
  const uint8_t* e;
  float* out;      // [splits][o][d]
  float* bias;     // [splits][o] (nullable): the column sums of dy
  int64_t n, per;  // rows, rows of a split (a multiple of kDepth; every split has one at least)
  int32_t o, d, nb;
  int32_t tiles_o, tiles_d, splits;
};

// How dy goes in: its type, and whether the matrix instructions take fp16 (x was fp16, as dy is).
template <typename T, bool HALF>
struct Dy {
  typedef T type;
  static constexpr bool kHalf = HALF;
  static constexpr int kPlanes = sizeof(T) == 4 ? 3 : std::is_same_v<T, __bf16> || HALF ? 1 : 2;  // terms
  // LDS buffers: two (the next step is written while one is multiplied) where the operands fit twice beside a second
  // block, one and two barriers a step for dy's two and three terms.
  static constexpr int kStages = kPlanes == 1 ? 2 : 1;
};

__device__ __forceinline__ uint32_t high_halves(uint32_t lo, uint32_t hi) {  // [hi's upper 16 : lo's upper 16]
  return __builtin_amdgcn_perm(hi, lo, 0x07060302);
}

// f's next bf16 term: its upper 16 bits; what is left of f is exact.
__device__ __forceinline__ uint32_t take_term(float& f) {
  const uint32_t h = __float_as_uint(f) & 0xFFFF0000u;
  f -= __uint_as_float(h);
  return h;
}

template <typename T>
struct Quad {  // 4 columns of one row, as they lie in memory
  uint32_t w[sizeof(T)];
  __device__ __forceinline__ float at(int j) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[j]);
    else return static_cast<float>(__builtin_bit_cast(T, static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)))));
  }
};

typedef u32x2 u32x2_any __attribute__((aligned(2)));
#define KGAT_GLOBAL __attribute__((address_space(1)))  // of pointers that came through integers
template <typename P>
__device__ __forceinline__ const KGAT_GLOBAL P* global_at(uint64_t base, uint64_t offset) {
  return reinterpret_cast<const KGAT_GLOBAL P*>(reinterpret_cast<const KGAT_GLOBAL char*>(base) + offset);
}

// NARROW: a row of `width` < 4 columns.
template <typename T, bool NARROW>
__device__ __forceinline__ Quad<T> load_quad(uint64_t base, uint64_t offset, int32_t width) {
  Quad<T> v;
  if constexpr (NARROW) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = j < width ? j : width - 1;
      if constexpr (sizeof(T) == 4) {
        v.w[j] = global_at<uint32_t>(base, offset)[c];
      } else {
        const uint32_t e = global_at<uint16_t>(base, offset)[c];
        v.w[j >> 1] = (j & 1) != 0 ? v.w[j >> 1] | e << 16 : e;
      }
    }
  } else if constexpr (sizeof(T) == 4) {
    const u32x4 q = *global_at<u32x4_any>(base, offset);
#pragma unroll
    for (int j = 0; j < 4; ++j) v.w[j] = q[j];
  } else {
    const u32x2 q = *global_at<u32x2_any>(base, offset);
    v.w[0] = q[0];
    v.w[1] = q[1];
  }
  return v;
}

// NARROW: dy has fewer than 4 columns.
template <typename D, int B, bool NARROW>
__global__ __launch_bounds__(2 * B) void act8_wgrad_kernel(Wgrad a) {
  typedef typename D::type T;
  constexpr int P = D::kPlanes, kPlane = B * kLdsPitch, kBuffer = (P + 1) * kPlane;
  // Waves along d; 32 x 32 tiles of a wave along o and d.
  constexpr int kWavesN = B == 64 ? 2 : B / 64, FM = B == 64 ? 2 : B / 64, FN = B == 64 ? 1 : 2;
  static_assert(kWavesN * FN * 32 == B && (2 * B / 64) / kWavesN * FM * 32 == B, "the waves cover the tile");
  __shared__ __align__(16) char lds[D::kStages * kBuffer];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int cg = tid % (B / 4), kg = tid / (B / 4);
  // Blocks b, b + 8, ... run on one XCD: give it neighbouring tiles (4 along o at a time), whose operands its L2 shares
  // (15 tiles of 100003 rows 41 us, with the blocks in their own order 69).
  const int total = a.tiles_o * a.tiles_d * a.splits;
  int id = blockIdx.x;
  const int xcd = id % 8, more = total % 8;
  id = xcd * (total / 8) + (xcd < more ? xcd : more) + id / 8;
  const int split = id / (a.tiles_o * a.tiles_d);
  id -= split * (a.tiles_o * a.tiles_d);
  const int strip = id / (4 * a.tiles_d), rows_here = a.tiles_o - strip * 4 < 4 ? a.tiles_o - strip * 4 : 4;
  id -= strip * 4 * a.tiles_d;
  const int32_t o0 = (strip * 4 + id % rows_here) * B, i0 = id / rows_here * B;

  const int64_t r0 = split * a.per, r1 = r0 + a.per < a.n ? r0 + a.per : a.n;
  const int32_t ldq = a.nb * kBlock;
  // A quad that would pass the last column starts earlier: its columns are computed twice, and written twice with the
  // same value.
  auto first_of = [](int32_t c, int32_t width) { return c < width - 4 ? c : width > 4 ? width - 4 : 0; };
  // A wave's rows start at a uniform address (scalar registers, a scalar addition a row); a thread adds its 32-bit
  // column offset, and where a wave holds several row groups their rows.
  const int kg0 = __builtin_amdgcn_readfirstlane(kg);
  const int64_t pitch_y = a.lddy * static_cast<int64_t>(sizeof(T)), pitch_q = ldq;
  const int32_t oc = first_of(o0 + cg * 4, a.o) * static_cast<int32_t>(sizeof(T)), ic = first_of(i0 + cg * 4, ldq);
  uint64_t dy = reinterpret_cast<uint64_t>(a.dy) + (r0 + kg0 * 8) * pitch_y;
  uint64_t qp = reinterpret_cast<uint64_t>(a.q) + (r0 + kg0 * 8) * pitch_q;
  typedef std::conditional_t<B == 256, uint32_t, int64_t> offset_t;
  const offset_t off_y = B == 256 ? oc : oc + (kg - kg0) * 8 * pitch_y, off_q = B == 256 ? ic : ic + (kg - kg0) * 8 * pitch_q;
  // The scales of 8 rows and the tile's blocks are one byte for each of the B / 4 threads of a row group: a thread loads
  // one, and takes its 8 rows' by lane exchange (a load for each was a sixth of the kernel's time).
  constexpr int kTileBlocks = B / kBlock;
  const int32_t eb = i0 / kBlock + cg % kTileBlocks < a.nb ? i0 / kBlock + cg % kTileBlocks : a.nb - 1;
  const uint8_t* ep = a.e + (r0 + kg * 8 + cg / kTileBlocks) * a.nb + eb;
  const int code_lane = (lane - cg % 64 + cg / (kBlock / 4)) * 4;  // of the group's first row, for ds_bpermute

  floatx16 acc[FM][FN];
#pragma unroll
  for (int m = 0; m < FM; ++m)
#pragma unroll
    for (int n = 0; n < FN; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[m][n][i] = 0.f;
  const int wm = (wave / kWavesN) * FM * 32, wn = (wave % kWavesN) * FN * 32;

  Quad<T> y[8];
  uint32_t x[8], codes;
  // The column sums of dy: every block forms them, one instruction for two terms, and the first of its strip writes them.
  float bias[4] = {0.f, 0.f, 0.f, 0.f};
  // The next kDepth rows' operands.
  auto fetch_all = [&]() __attribute__((always_inline)) {
    // The bases are scalars, and new ones every step: left to itself the compiler steps 16 vector addresses instead.
    uint64_t y0 = dy, q0 = qp;
    asm("" : "+s"(y0), "+s"(q0));
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      y[k] = load_quad<T, NARROW>(y0 + k * pitch_y, off_y, a.o);
      x[k] = *global_at<uint32_t>(q0 + k * pitch_q, off_q);
    }
    codes = *ep;
    dy += kDepth * pitch_y;
    qp += kDepth * pitch_q;
    ep += kDepth * static_cast<int64_t>(a.nb);
  };
  // The same where the share ends after `left` < kDepth of them: behind its last row x repeats it and dy is 0.
  auto fetch_last = [&](int64_t left) __attribute__((always_inline)) {
    const int32_t last = static_cast<int32_t>(left) - 1 - kg * 8;  // from this thread's first row
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int64_t at = k < last ? k : last;
      y[k] = load_quad<T, NARROW>(dy, off_y + at * pitch_y, a.o);
      x[k] = *global_at<uint32_t>(qp, off_q + at * pitch_q);
      if (k > last)
#pragma unroll
        for (int j = 0; j < static_cast<int>(sizeof(T)); ++j) y[k].w[j] = 0;
    }
    const int64_t beyond = kg * 8 + cg / kTileBlocks - (left - 1);  // rows from the share's last to the one whose byte this is
    codes = *(beyond > 0 ? ep - beyond * a.nb : ep);
  };
  auto fetch = [&](int64_t left) __attribute__((always_inline)) {
    if (left >= kDepth) fetch_all();
    else fetch_last(left);
  };
  auto scales = [&](float (&s)[8]) __attribute__((always_inline)) {
    const int mine = static_cast<int>(codes);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      s[k] = scale_of(static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(code_lane + k * kTileBlocks * 4, mine)));
  };
  // Column j of the thread's quads into a buffer.
  auto store = [&](char* buffer, int j, const float (&scale)[8]) __attribute__((always_inline)) {
    char* at = buffer + ((B / 4) * j + cg) * kLdsPitch + kg * 16;
    if constexpr (P == 1) {
      u32x4 w;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t lo = y[2 * k].w[j >> 1], hi = y[2 * k + 1].w[j >> 1];
        const uint32_t pair = __builtin_amdgcn_perm(hi, lo, (j & 1) != 0 ? 0x07060302 : 0x05040100);
        if constexpr (D::kHalf)
          bias[j] = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2v, pair), half2v{1, 1}, bias[j], false);
        else
          bias[j] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), bf16x2{1, 1}, bias[j], false);
        w[k] = pair;
      }
      *reinterpret_cast<u32x4*>(at) = w;
    } else {
      float f[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = y[k].at(j);
      bias[j] += ((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7]));
#pragma unroll
      for (int p = 0; p < P; ++p) {
        u32x4 w;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t lo = take_term(f[2 * k]), hi = take_term(f[2 * k + 1]);
          w[k] = high_halves(lo, hi);
        }
        *reinterpret_cast<u32x4*>(at + p * kPlane) = w;
      }
    }
    u32x4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float f[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)  // exact; NaN where the scale is inf
        f[h] = static_cast<float>(static_cast<int8_t>(x[2 * k + h] >> (8 * j))) * scale[2 * k + h];
      if constexpr (D::kHalf) w[k] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(f[0], f[1]));
      else w[k] = high_halves(__float_as_uint(f[0]), __float_as_uint(f[1]));
    }
    *reinterpret_cast<u32x4*>(at + P * kPlane) = w;
  };
  // The operands of 16 rows: a wave's columns of x and of each of dy's terms.
  struct Operands {
    u32x4 b[FN], a[P][FM];
  };
  auto read = [&](Operands& v, const char* buffer, int s) __attribute__((always_inline)) {
    const int off = (lane & 31) * kLdsPitch + s * 32 + (lane >> 5) * 16;
#pragma unroll
    for (int n = 0; n < FN; ++n)
      v.b[n] = *reinterpret_cast<const u32x4*>(buffer + P * kPlane + (wn + n * 32) * kLdsPitch + off);
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int m = 0; m < FM; ++m)
        v.a[p][m] = *reinterpret_cast<const u32x4*>(buffer + p * kPlane + (wm + m * 32) * kLdsPitch + off);
  };
  auto multiply = [&](const Operands& v) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int m = 0; m < FM; ++m)
#pragma unroll
        for (int n = 0; n < FN; ++n)
          if constexpr (D::kHalf)
            acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, v.a[p][m]),
                                                               __builtin_bit_cast(half8, v.b[n]), acc[m][n], 0, 0, 0);
          else
            acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v.a[p][m]),
                                                                __builtin_bit_cast(bf16x8, v.b[n]), acc[m][n], 0, 0, 0);
  };

  float scale[8];
  int64_t left = r1 - r0;  // rows not multiplied yet
  fetch(left);
  if constexpr (D::kStages == 2) {
    scales(scale);
#pragma unroll
    for (int j = 0; j < 4; ++j) store(lds, j, scale);
    if (left > kDepth) fetch(left - kDepth);
    __syncthreads();
    char* now = lds;
    char* then = lds + kBuffer;
    auto turn = [&]() {
      char* t = now;
      now = then;
      then = t;
    };
    Operands v[2];
    // While two whole steps follow: no branch between the products of a step, the next one's operands on their way into
    // the other buffer and the loads of the one behind it.  Each phase reads the next 16 rows' operands, decodes a
    // column and multiplies (groups laid down with sched_group_barrier were 3 % slower than the compiler's own mix).
    for (; left >= 3 * kDepth; left -= kDepth) {
      read(v[0], now, 0);
      scales(scale);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        if (s < 3) read(v[(s + 1) & 1], now, s + 1);
        store(then, s, scale);
        if (s == 3) fetch_all();
        multiply(v[s & 1]);
      }
      __syncthreads();
      turn();
    }
    for (; left > 0; left -= kDepth) {  // the last two
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        read(v[0], now, s);
        multiply(v[0]);
      }
      if (left > kDepth) {
        scales(scale);
#pragma unroll
        for (int j = 0; j < 4; ++j) store(then, j, scale);
      }
      if (left > 2 * kDepth) fetch(left - 2 * kDepth);
      __syncthreads();
      turn();
    }
  } else {
    Operands v;
    do {
      scales(scale);
      __syncthreads();  // the last step's operands are read
#pragma unroll
      for (int j = 0; j < 4; ++j) store(lds, j, scale);
      if (left > kDepth) fetch(left - kDepth);
      __syncthreads();
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        read(v, lds, s);
        multiply(v);
      }
      left -= kDepth;
    } while (left > 0);
  }
  if (a.bias != nullptr && i0 == 0) {  // the 8 row groups' sums, in their order
    float* sums = reinterpret_cast<float*>(lds);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[kg * B + (B / 4) * j + cg] = bias[j];
    __syncthreads();
    if (tid < B) {
      const int32_t row = first_of(o0 + tid % (B / 4) * 4, a.o) + tid / (B / 4);
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) v += sums[k * B + tid];
      if (!NARROW || row < a.o) a.bias[static_cast<int64_t>(split) * a.o + row] = v;
    }
  }
  float* out = a.out + static_cast<int64_t>(split) * a.o * a.d;
#pragma unroll
  for (int n = 0; n < FN; ++n) {
    const int ln = wn + n * 32 + (lane & 31);
    const int32_t col = first_of(i0 + ln % (B / 4) * 4, ldq) + ln / (B / 4);
    if (col >= a.d) continue;
#pragma unroll
    for (int m = 0; m < FM; ++m)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int lm = wm + m * 32 + (i >> 2) * 8 + (lane >> 5) * 4 + (i & 3);
        const int32_t row = first_of(o0 + lm % (B / 4) * 4, a.o) + lm / (B / 4);
        if (!NARROW || row < a.o) out[static_cast<int64_t>(row) * a.d + col] = acc[m][n][i];
      }
  }
}

// Sums of parts, in their order: the first blocks take dW's elements, the others db's.  64 elements a block at a time,
// its 4 waves every fourth part.  68 parts of 131 x 257 in 4.6 us (9 MB): launch and latency.
struct Join {
  const float* part[2];
  float* out[2];
  int64_t size[2];
  int32_t parts[2];
  uint32_t blocks;  // of the first
};

__global__ __launch_bounds__(256) void act8_join_kernel(Join a) {
  __shared__ float lds[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int which = blockIdx.x < a.blocks ? 0 : 1;
  const uint32_t first = which != 0 ? a.blocks : 0, count = which != 0 ? gridDim.x - a.blocks : a.blocks;
  const int64_t size = a.size[which];
  const float* part = a.part[which];
  const int parts = a.parts[which];
  for (int64_t base = static_cast<int64_t>(blockIdx.x - first) * 64; base < size; base += static_cast<int64_t>(count) * 64) {
    const int64_t i = base + lane;
    float s = 0.f;
    if (i < size)
#pragma unroll 8
      for (int p = wave; p < parts; p += 4) s += part[p * size + i];
    lds[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && i < size) a.out[which][i] = (lds[0][lane] + lds[1][lane]) + (lds[2][lane] + lds[3][lane]);
    __syncthreads();
  }
}

struct Splits {
  int32_t tile;  // B
  int32_t tiles_o, tiles_d;
  int32_t w;     // row shares
  int64_t per;   // rows of a share
  // Workspace: the shares' tiles, and their column sums; one share writes its results.
  int64_t floats(int32_t o, int32_t d) const {
    return w == 1 ? 0 : static_cast<int64_t>(w) * o * (static_cast<int64_t>(d) + 1);
  }
};

// Microseconds of a step of 64 rows with `occ` blocks on a CU, measured (n = 16384, o = d = 1024 and 4096): a
// step of bf16 dy takes 0.73 / 1.4 us with 1 / 4 blocks of 64, 1.25 / 1.7 with 1 / 2 of 128, 2.25 with one of 256; of
// fp16 dy 2.3 with 4 (64), 1.9 / 2.4 (128) and 4.1 (256); of float dy 1.6 / 2.4 (64), 2.45 / 2.95 (128) and 5.8 (256).
double step_us(int planes, int32_t tile, int64_t occ) {
  const double n = static_cast<double>(occ);
  if (tile == 256) return planes == 1 ? 2.25 : planes == 2 ? 4.1 : 5.8;
  if (tile == 128) return planes == 1 ? 0.8 + 0.45 * n : planes == 2 ? 1.3 + 0.55 * n : 1.7 + 0.62 * n;
  return planes == 1 ? 0.6 + 0.2 * n : planes == 2 ? 0.9 + 0.35 * n : 1.35 + 0.26 * n;
}

// The tile and the number of row shares with the least estimated time: the blocks' steps (4, 2 or 1 of them on a CU at
// once), and the shares' tiles written and read again at 5 TB/s.  One rule for every size: at o = d = 4096 tiles of 256
// take 504 us and of 128 822 us (fp16 950 and 1140, float 1375 and 1575); at 2048 x 512 (n = 8192) 63 and 50; at
// o = d = 64 (n = 2048) one share takes 53 us, 16 of them 18.  Outputs of fewer than 4 columns have a kernel of 64 alone.
Splits wgrad_splits(int planes, int64_t n, int32_t o, int32_t d) {
  Splits best{};
  double least = 1e300;
  for (int32_t tile = 64; tile <= (o < kNarrow ? 64 : 256); tile *= 2) {
    const int32_t tiles_o = (o + tile - 1) / tile, tiles_d = (d + tile - 1) / tile;
    const int64_t tiles = static_cast<int64_t>(tiles_o) * tiles_d, occ = tile == 256 ? 1 : tile == 128 ? 2 : 4;
    // Shares: 1, 2, 3, 4, 6, 8, 12, ... and as many as fill the chip once.
    const int64_t once = kCUs * occ / tiles;
    for (int step = 0; step < 24; ++step) {
      int64_t w = step == 23 ? once : step < 2 ? step + 1 : (int64_t{2} + (step & 1)) << (step / 2 - 1);
      if (w < 1 || (w > 1 && w * 128 > n)) continue;
      const int64_t per = n < 1 ? kDepth : ((n + w - 1) / w + kDepth - 1) / kDepth * kDepth;
      const int64_t shares = n < 1 ? 1 : (n + per - 1) / per, blocks = tiles * shares;
      const int64_t full = blocks / (kCUs * occ), rest = blocks % (kCUs * occ);
      const double steps = static_cast<double>(per / kDepth) + 3;  // 3: a block's start and end
      double us = full * steps * step_us(planes, tile, occ);
      if (rest > 0) us += steps * step_us(planes, tile, (rest + kCUs - 1) / kCUs);
      if (shares > 1) us += 3 + 8e-6 / 5 * static_cast<double>(shares) * o * d;
      if (us < least) {
        least = us;
        best = {tile, tiles_o, tiles_d, static_cast<int32_t>(shares), per};
      }
    }
  }
  return best;
}

bool act8_shape_ok(int64_t n, int32_t d) { return n >= 0 && d >= 1 && d <= KGAT_ACT8_MAX_D; }

// A grid holds fewer than 2^32 threads along x.
constexpr int64_t kLaunchThreads = int64_t{1} << 31;

// f(first row, rows, blocks of 256 threads) for n rows of per_row vectors, a thread each, in as many launches as it takes.
template <typename F>
int launch_rows(int64_t n, int64_t per_row, F&& f) {
  if (n > (int64_t{1} << 52) / per_row) return KGAT_ERR_INVALID;  // more than any memory holds
  const int64_t most = kLaunchThreads / per_row;
  for (int64_t row = 0; row < n; row += most) {
    const int64_t rows = n - row < most ? n - row : most;
    f(row, rows, dim3(static_cast<uint32_t>((rows * per_row + 255) / 256)));
    KGAT_LAUNCH_CHECK();
  }
  return KGAT_OK;
}

}  // namespace

}  // namespace kgat

extern "C" int kgat_act8_pack(int32_t dtype, const void* x, int64_t ldx, int64_t n, int32_t d, int8_t* q, uint8_t* e,
                              void* stream) {
  using namespace kgat;
  if (!x || !q || !e || !act8_shape_ok(n, d) || ldx < 0 || (reinterpret_cast<uintptr_t>(q) & 15))
    return KGAT_ERR_INVALID;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const int64_t nb = (d + kBlock - 1) / kBlock;
    return launch_rows(n, nb * (kBlock / Vec<T>::N), [&](int64_t row, int64_t rows, dim3 grid) {
      const Pack a{static_cast<const T*>(x) + row * ldx, ldx, q + row * nb * kBlock, e + row * nb, rows, d};
      hipLaunchKernelGGL(act8_pack_kernel<T>, grid, dim3(256), 0, reinterpret_cast<hipStream_t>(stream), a);
    });
  });
}

extern "C" int kgat_act8_unpack(int32_t dtype, const int8_t* q, const uint8_t* e, int64_t n, int32_t d, void* x,
                                int64_t ldx, void* stream) {
  using namespace kgat;
  if (!x || !q || !e || !act8_shape_ok(n, d) || ldx < d || (reinterpret_cast<uintptr_t>(q) & 15))
    return KGAT_ERR_INVALID;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const int64_t nb = (d + kBlock - 1) / kBlock;
    return launch_rows(n, (d + Vec<T>::N - 1) / Vec<T>::N, [&](int64_t row, int64_t rows, dim3 grid) {
      const Unpack a{q + row * nb * kBlock, e + row * nb, static_cast<T*>(x) + row * ldx, ldx, rows, d};
      hipLaunchKernelGGL(act8_unpack_kernel<T>, grid, dim3(256), 0, reinterpret_cast<hipStream_t>(stream), a);
    });
  });
}

namespace kgat {
namespace {

// f(Dy<...>{}) for dy's type and the type that x was packed from; an unknown one is KGAT_ERR_INVALID.
template <typename F>
int with_dy(int32_t dtype, int32_t x_dtype, F&& f) {
  if (x_dtype < KGAT_F32 || x_dtype > KGAT_F16) return KGAT_ERR_INVALID;
  if (dtype == KGAT_F16 && x_dtype == KGAT_F16) return f(Dy<_Float16, true>{});
  return with_dtype(dtype, [&](auto t) { return f(Dy<decltype(t), false>{}); });
}

}  // namespace
}  // namespace kgat

extern "C" int64_t kgat_act8_wgrad_workspace(int32_t dtype, int32_t x_dtype, int64_t n, int32_t o, int32_t d) {
  using namespace kgat;
  if (!act8_shape_ok(n, d) || o < 1 || o > KGAT_ACT8_MAX_D) return -1;
  int64_t floats = -1;
  with_dy(dtype, x_dtype, [&](auto t) {
    floats = wgrad_splits(decltype(t)::kPlanes, n, o, d).floats(o, d);
    return static_cast<int>(KGAT_OK);
  });
  return floats;
}

extern "C" int kgat_act8_wgrad(int32_t dtype, const void* dy, int64_t lddy, int32_t x_dtype, const int8_t* q,
                               const uint8_t* e, int64_t n, int32_t o, int32_t d, float* dW, float* db,
                               float* workspace, int64_t workspace_floats, void* stream) {
  using namespace kgat;
  if (!dy || !q || !e || !dW || !act8_shape_ok(n, d) || o < 1 || o > KGAT_ACT8_MAX_D || lddy < 0 ||
      (reinterpret_cast<uintptr_t>(q) & 15))
    return KGAT_ERR_INVALID;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return with_dy(dtype, x_dtype, [&](auto t) -> int {
    using D = decltype(t);
    const Splits s = wgrad_splits(D::kPlanes, n, o, d);
    const int64_t need = s.floats(o, d), size = static_cast<int64_t>(o) * d;
    if (need > 0 && (!workspace || workspace_floats < need)) return KGAT_ERR_WORKSPACE;
    float* part_b = need > 0 ? workspace + s.w * size : nullptr;
    Join j{{workspace, part_b}, {dW, db}, {size, o}, {s.w, s.w}, 0};
    if (n == 0) {  // sums of nothing
      j.parts[0] = j.parts[1] = 0;
    } else {
      const Wgrad a{dy, lddy, q, e, s.w == 1 ? dW : workspace, db == nullptr ? nullptr : j.parts[1] == 1 ? db : part_b,
                    n, s.per, o, d, (d + kBlock - 1) / kBlock, s.tiles_o, s.tiles_d, s.w};
      const int64_t blocks = static_cast<int64_t>(s.tiles_o) * s.tiles_d * s.w;
      if (blocks > kLaunchThreads / 512) return KGAT_ERR_INVALID;  // a dW of 2^38 bytes
      const dim3 grid(static_cast<uint32_t>(blocks));
      if (o < kNarrow) hipLaunchKernelGGL((act8_wgrad_kernel<D, 64, true>), grid, dim3(128), 0, st, a);
      else if (s.tile == 64) hipLaunchKernelGGL((act8_wgrad_kernel<D, 64, false>), grid, dim3(128), 0, st, a);
      else if (s.tile == 128) hipLaunchKernelGGL((act8_wgrad_kernel<D, 128, false>), grid, dim3(256), 0, st, a);
      else hipLaunchKernelGGL((act8_wgrad_kernel<D, 256, false>), grid, dim3(512), 0, st, a);
      KGAT_LAUNCH_CHECK();
    }
    const int64_t blocks_w = j.parts[0] == 1 ? 0 : blocks_for(size, 64, 1 << 22);
    const int64_t blocks_b = db == nullptr || j.parts[1] == 1 ? 0 : (o + 63) / 64;
    if (blocks_w + blocks_b > 0) {
      j.blocks = static_cast<uint32_t>(blocks_w);
      hipLaunchKernelGGL(act8_join_kernel, dim3(static_cast<uint32_t>(blocks_w + blocks_b)), dim3(256), 0, st, j);
      KGAT_LAUNCH_CHECK();
    }
    return KGAT_OK;
  });
}
