// Layer norm of matrix rows with the activation behind it, forward and backward (enable_LN branch of the DNN tower).
//
//   xhat = (x - mean) rstd,  u = gamma xhat + beta,  y = act(u)
//   du = dy act'(u),  t = du gamma,  dx = rstd (t - mean(t) - xhat mean(t xhat)),
//   dgamma = sum_rows du xhat,  dbeta = sum_rows du
//
// Bound by memory: forward 2 passes over the data (read x, write y), backward 3 (read x and dy, write dx), ~10 and ~25
// operations an element.  So a row is loaded once, stays in registers until it is stored, and the next one is under way
// meanwhile; y is not kept for the backward pass (u is formed again from x); blocks are as many as the chip holds at
// once and walk the rows, so that gamma, beta and the weights' gradients stay with a thread's columns.
//   1024 x 65536 fp32 relu, forward     91 us, 5.9 TB/s of 6.2 that a plain streaming addition reaches
//    512 x 65536 fp32 relu, backward    73 us, 5.5 TB/s, 5 of them in the second launch that joins 256 partial sums
//   2496 x 16384 bf16, backward         49 us, 5.0 TB/s, 4.7 of them in the second launch
// Rows that the registers of a block do not hold (16384 elements backward; 18432, of 16 bits 20480, forward) take a slower
// way: 20483 x 533 fp32 29 us forward and 63 backward, 3.0 and 2.1 TB/s; few rows leave CUs idle (400001 x 21 fp32 136 and
// 215 us).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "xdfm_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxWaves = 16;  // of a block that shares a row

// ------------------------------------------------------------------ rows in registers
// 16 bytes of a row: 4 or 8 elements at any address of the type
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

// How rows are read and written.  kStream: past the caches, for a pass over more than half of the Infinity Cache
// (256 MB), of which its neighbours would find little there: by 3 to 14 % faster from 150 MB on (forward 1024 x 65536 fp32
// 98 -> 91 us, backward 512 x 65536 80 -> 73), even at 100 MB, up to 20 % slower at 60 MB.
enum { kPlain, kStream };

// The pieces of a row that a thread holds.  Element j of piece k is column c[k] + j and counts where j >= skip[k]:
// a piece that would pass the row's end is moved back to end there and leaves out what its neighbour holds, so that
// loads need no condition (one inside the loop would wait for the loads under way); one that lies behind the end
// counts nowhere.  Rows shorter than a piece (c < 0) are the exception.
template <typename T, int NV>
struct Pieces {
  int c[NV], skip[NV];
  __device__ __forceinline__ Pieces(int c0, int step, int cols) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int at = c0 + k * step;
      c[k] = min(at, cols - kVec<T>);
      skip[k] = at - c[k];
    }
  }
  // whether every piece of the wave counts as a whole: one branch then saves the forward pass four operations an
  // element (1024 x 65536 bf16 54.7 -> 51.5 us; in the backward pass it gained and lost 1 %)
  __device__ __forceinline__ bool whole() const {
    bool all = true;
#pragma unroll
    for (int k = 0; k < NV; ++k) all &= skip[k] == 0;
    return __all(all);
  }
};

template <typename T>
__device__ __forceinline__ void unpack(u32x4 w, float (&v)[kVec<T>]) {
  T e[kVec<T>];
  __builtin_memcpy(e, &w, 16);
#pragma unroll
  for (int j = 0; j < kVec<T>; ++j) v[j] = (float)e[j];
}

// the elements that do not count: 0
template <int V>
__device__ __forceinline__ void mask(float (&v)[V], int skip) {
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = j >= skip ? v[j] : 0.f;
}

template <int MODE>
__device__ __forceinline__ u32x4 load_16(const void* from) {
  return MODE == kStream ? __builtin_nontemporal_load((const u32x4_any*)from) : *(const u32x4_any*)from;
}

template <int MODE, typename T, int NV>
__device__ __forceinline__ void load_row(const T* row, const Pieces<T, NV>& at, bool tiny, u32x4 (&w)[NV]) {
  if (!tiny) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const u32x4_any* from = reinterpret_cast<const u32x4_any*>(row + at.c[k]);
      w[k] = MODE == kStream ? __builtin_nontemporal_load(from) : *from;
    }
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      T e[kVec<T>];
#pragma unroll
      for (int j = 0; j < kVec<T>; ++j) e[j] = j >= at.skip[k] ? row[at.c[k] + j] : (T)0.f;
      __builtin_memcpy(&w[k], e, 16);
    }
  }
}

template <typename T, int NV>
__device__ __forceinline__ void load_weights(const float* __restrict__ w, const Pieces<T, NV>& at, bool tiny,
                                             float (&v)[NV][kVec<T>]) {
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int j = 0; j < kVec<T>; j += 4)
      if (!tiny) {
        const u32x4 raw = *reinterpret_cast<const u32x4_any*>(w + at.c[k] + j);
        __builtin_memcpy(&v[k][j], &raw, 16);
      } else {
#pragma unroll
        for (int i = j; i < j + 4; ++i) v[k][i] = i >= at.skip[k] ? w[at.c[k] + i] : 0.f;
      }
}

// what counts of V elements to `to` (column c)
template <int MODE, typename T, int V>
__device__ __forceinline__ void store_piece(T* to, int skip, const float (&v)[V]) {
  T e[V];
#pragma unroll
  for (int j = 0; j < V; ++j) e[j] = (T)v[j];
  if (skip == 0) {
#pragma unroll
    for (int i = 0; i < V * (int)sizeof(T) / 16; ++i) {
      u32x4 w;
      __builtin_memcpy(&w, (const char*)e + 16 * i, 16);
      if (MODE == kStream)
        __builtin_nontemporal_store(w, reinterpret_cast<u32x4_any*>(to) + i);
      else
        reinterpret_cast<u32x4_any*>(to)[i] = w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j >= skip) to[j] = e[j];
  }
}

// ------------------------------------------------------------------ sums
// a value moved within the lanes of a row of 16, without a trip through LDS
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xF, 0xF, true));
}

// sum over groups of G neighbouring lanes, the same in each of them
template <int G>
__device__ __forceinline__ float group_sum(float v) {
  v += dpp<0xB1>(v);                     // lane ^ 1
  v += dpp<0x4E>(v);                     // lane ^ 2
  if (G > 4) v += dpp<0x141>(v);         // 7 - lane of 8
  if (G > 8) v += dpp<0x140>(v);         // 15 - lane of 16
  if (G > 16) {
    const auto h = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(h[0]) + __uint_as_float(h[1]);
  }
  if (G > 32) {
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(h[0]) + __uint_as_float(h[1]);
  }
  return v;
}

// sum over the lanes of a wave that are equal modulo G, the same in each of them
template <int G>
__device__ __forceinline__ float groups_sum(float v) {
  if (G <= 8) v += dpp<0x128>(v);  // turned by 8 within 16
  if (G <= 16) {
    const auto h = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(h[0]) + __uint_as_float(h[1]);
  }
  const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(h[0]) + __uint_as_float(h[1]);
}

// N sums over `waves` neighbouring waves at once, the same in each of their threads, in an order that does not depend
// on timing.  One barrier: `sh` is one of two buffers that consecutive calls take in turn, so a wave that comes to
// write it again has passed the barrier of the call between, behind every reader of this one.
template <int N>
__device__ __forceinline__ void waves_sum(float (&v)[N], int waves, float (*sh)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = group_sum<64>(v[k]);
  const int wave = (int)threadIdx.x >> 6, first = wave - wave % waves;
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int k = 0; k < N; ++k) sh[wave][k] = v[k];
  __syncthreads();
  const int mine = (int)threadIdx.x & 15;  // (16 waves at most: each 16 lanes add them up for themselves)
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = group_sum<16>(mine < waves ? sh[first + mine][k] : 0.f);
}

// over a row: G of its lanes (G <= 64), or (G = 0) `waves` waves
template <int G, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], int waves, float (*sh)[N]) {
  if constexpr (G == 0) {
    waves_sum(v, waves, sh);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = group_sum<G>(v[k]);
  }
}

// ------------------------------------------------------------------ activations
// e^u to about 1.5 units of the last place: 2^(u log2 e) with what the product's rounding cut off put back, one
// hardware exponential in all.  (Beyond 2^126 the correction would meet infinities: left out.)
__device__ __forceinline__ float exp_of(float u) {
  const float hi = u * 1.44269504f;
  const float lo = fmaf(u, 1.44269504f, -hi) + u * 1.92596303e-8f;  // log2 e in two parts
  const float e = __builtin_amdgcn_exp2f(hi);
  return fabsf(hi) < 126.f ? fmaf(e * lo, 0.693147181f, e) : e;
}

__device__ __forceinline__ float sigmoid_of(float u) { return __builtin_amdgcn_rcpf(1.f + exp_of(-u)); }

// 1 - 2 / (e^2|u| + 1); below 0.6, where that cancels, u (1 + u^2 P(u^2)) with P interpolated (error 3e-9).  (Here the
// exponent's rounding needs no correction: it moves the result by less than one unit of the last place.  Slopes over |u| < 6
// are off by 0.509 x 2^-24 in the mean, 2.26 at most; corrected by 0.502 and 2.21, and 1001 x 4099 fp32 takes 9.7 us
// instead of 8.7.)
__device__ __forceinline__ float tanh_of(float u) {
  const float w = u * u;
  float p = fmaf(w, -0.00584964391f, 0.0207513491f);
  p = fmaf(w, p, -0.0537679835f);
  p = fmaf(w, p, 0.133316796f);
  p = fmaf(w, p, -0.333332828f);
  const float small = fmaf(u * w, p, u);
  const float large = copysignf(fmaf(-2.f, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(2.88539008f * fabsf(u)) + 1.f), 1.f), u);
  return fabsf(u) < 0.6f ? small : large;
}

// e^u - 1 for u <= 0; above -0.5 u (1 + u Q(u)) with Q interpolated (error 2e-9), below without the exponent's correction
// for tanh's reason (|u| e^u < 0.4: the result moves by less than one unit of the last place)
__device__ __forceinline__ float expm1_of(float u) {
  float q = fmaf(u, 0.00112340425f, 0.00818961363f);
  q = fmaf(u, q, 0.0416300728f);
  q = fmaf(u, q, 0.166662419f);
  q = fmaf(u, q, 0.499999819f);
  return u > -0.5f ? fmaf(u * u, q, u) : __builtin_amdgcn_exp2f(1.44269504f * u) - 1.f;
}

// Where a result is stored in 16 bits, and for slopes there, the exponent's own rounding may stay: |u| 2^-24 of the value,
// 2^-17 at most before the value itself is out of range, a hundredth of the storage's half step and less; a slope is off
// by less than 2^-24 so (|u| e^-|u| < 0.4).  Half the operations of a sigmoid: 632 x 12980 bf16 11.9 against 14.4 us.
// Slopes over |u| < 6, off in the mean and at most, in 2^-24: sigmoid 0.228, 1.65 (corrected 0.222, 1.66), tanh 0.516, 2.26
// (0.502, 2.21), elu 0.046, 0.80 (0.035, 0.80); corrected, 2496 x 16384 bf16 backward takes 55 us instead of 53 with
// sigmoid, 53.4 and 50.8 with elu, 63 and 53 with tanh, and 409 x 54188 with tanh 50 and 38.5.
__device__ __forceinline__ float exp_quick(float u) { return __builtin_amdgcn_exp2f(u * 1.44269504f); }
__device__ __forceinline__ float sigmoid_quick(float u) { return __builtin_amdgcn_rcpf(1.f + exp_quick(-u)); }
// (up to 0.1 the series, to 2^-23 and 2^-20; from there on 2^-22 of 1 is 2^-18 of the value, a sixtieth of fp16's half
// step.  Tanh 409 x 54188 bf16 29.2 against 32.0 us.)
__device__ __forceinline__ float tanh_16(float u) {
  const float w = u * u;
  const float small = fmaf(u * w, fmaf(w, 0.133333333f, -0.333333333f), u);
  const float large = copysignf(fmaf(-2.f, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(2.88539008f * fabsf(u)) + 1.f), 1.f), u);
  return fabsf(u) < 0.1f ? small : large;
}
__device__ __forceinline__ float expm1_16(float u) {
  const float small = fmaf(u * u, fmaf(u, fmaf(u, 0.0416666667f, 0.166666667f), 0.5f), u);
  return u > -0.1f ? small : exp_quick(u) - 1.f;
}
// tanh |u|, off by 2^-22 at most: near 0 only a slope can bear that
__device__ __forceinline__ float tanh_quick(float u) {
  return fmaf(-2.f, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(2.88539008f * fabsf(u)) + 1.f), 1.f);
}

// v <- act(v).  (One switch for all of a thread's elements: the cases are straight code.)
template <typename T, int NV, int V>
__device__ __forceinline__ void activate_all(float (&v)[NV][V], int act) {
  constexpr bool kQuick = sizeof(T) == 2;
#define XDFM_EACH(EXPR)              \
  _Pragma("unroll") for (int k = 0; k < NV; ++k) _Pragma("unroll") for (int j = 0; j < V; ++j) { \
    const float u = v[k][j];         \
    v[k][j] = EXPR;                  \
  }                                  \
  break;
  switch (act) {
    case XDFM_ACT_RELU: XDFM_EACH(u <= 0.f ? 0.f : u)  // (NaN stays: a row without statistics is no row of zeros)
    case XDFM_ACT_SIGMOID: XDFM_EACH(kQuick ? sigmoid_quick(u) : sigmoid_of(u))
    case XDFM_ACT_TANH: XDFM_EACH(kQuick ? tanh_16(u) : tanh_of(u))
    case XDFM_ACT_ELU: XDFM_EACH(u > 0.f ? u : kQuick ? expm1_16(u) : expm1_of(u))
    default: break;
  }
#undef XDFM_EACH
}

// The slope of relu, from 64 bits: 32 bits lose the sign of u where gamma xhat and beta nearly cancel
// (three roundings of 2^-24 of |beta|: near_zero)
__device__ __forceinline__ bool near_zero(float u, float b) { return fabsf(u) <= 6e-7f * fabsf(b); }
__device__ __forceinline__ float on_exactly(float x, float mean, float rstd, float g, float b) {
  return ((double)x - (double)mean) * (double)rstd * (double)g + (double)b > 0.0 ? 1.f : 0.f;
}
__device__ __forceinline__ float relu_slope(float u, float x, float mean, float rstd, float g, float b) {
  return near_zero(u, b) ? on_exactly(x, mean, rstd, g, b) : u > 0.f ? 1.f : 0.f;
}

// d <- d act'(gamma xhat + beta) for all of a thread's elements; x: the raw pieces of the row
template <typename T, int NV, int V>
__device__ __forceinline__ void through_act(float (&d)[NV][V], const float (&xh)[NV][V], const u32x4 (&x)[NV],
                                            const float (&g)[NV][V], const float (&b)[NV][V], float mean, float rstd,
                                            int act) {
  constexpr bool kQuick = sizeof(T) == 2;
#define XDFM_EACH(EXPR)                              \
  _Pragma("unroll") for (int k = 0; k < NV; ++k) _Pragma("unroll") for (int j = 0; j < V; ++j) { \
    const float u = xh[k][j] * g[k][j] + b[k][j];    \
    EXPR;                                            \
  }
  switch (act) {
    case XDFM_ACT_RELU: {
      bool near = false;
      XDFM_EACH(near |= near_zero(u, b[k][j]))
      if (near) {  // hardly ever
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          float xv[V];
          unpack<T>(x[k], xv);
#pragma unroll
          for (int j = 0; j < V; ++j)
            d[k][j] *= relu_slope(xh[k][j] * g[k][j] + b[k][j], xv[j], mean, rstd, g[k][j], b[k][j]);
        }
      } else {
        XDFM_EACH(d[k][j] *= u > 0.f ? 1.f : 0.f)
      }
      break;
    }
    case XDFM_ACT_SIGMOID: XDFM_EACH(const float s = kQuick ? sigmoid_quick(u) : sigmoid_of(u); d[k][j] *= s * (1.f - s)) break;
    case XDFM_ACT_TANH: XDFM_EACH(const float t = kQuick ? tanh_quick(u) : tanh_of(u); d[k][j] *= 1.f - t * t) break;
    case XDFM_ACT_ELU: XDFM_EACH(d[k][j] *= u > 0.f ? 1.f : kQuick ? exp_quick(u) : exp_of(u)) break;
    default: break;
  }
#undef XDFM_EACH
}

// ------------------------------------------------------------------ forward
// waves of a CU that hold `each` elements a lane (by their registers)
constexpr int places(int each) { return each <= 16 ? 16 : each <= 24 ? 12 : 8; }

// One pass over the data: a row lies in the registers of its G lanes (or of the block's threads) from the load to the
// store, so the variance is taken around the mean and not from the sum of squares.  A thread keeps its columns from
// row to row, and with them gamma and beta.  (Re-reading the row for each of the three sums instead, one block a row:
// 226 against 91 us at 1024 x 65536 fp32.  gamma and beta by single elements instead of 16 bytes: 21 against 6 us at
// 1001 x 4099 fp16, where most waves see one row.)
// (Two pieces of 16 bits take 97 registers where five waves a SIMD leave 96 to each: asked for, 1001 x 4099 fp16 tanh 7.35
// against 7.75 us, 1001 x 5000 7.8 and 9.3.)
template <typename T, int G, int NV, int MODE>
__global__ __launch_bounds__(G ? kThreads : 64 * places(NV * kVec<T>),
                             G == 64 && NV == 2 && sizeof(T) == 2 ? 5 : 1) void layer_norm_fwd_kernel(
    const T* x, int64_t xs, int64_t rows, int cols, const float* __restrict__ gamma, const float* __restrict__ beta,
    float eps, int act, T* y, int64_t ys, float* __restrict__ stats) {
  constexpr int V = kVec<T>;
  __shared__ float sh[2][kMaxWaves][1];
  const int per_row = G ? G : (int)blockDim.x, waves = (int)blockDim.x >> 6;
  const int lane = G ? (int)threadIdx.x & (G - 1) : (int)threadIdx.x;
  const int64_t at_once = G ? kThreads / (G ? G : 1) : 1;
  const Pieces<T, NV> at(lane * V, per_row * V, cols);
  const bool tiny = G == 8 && cols < V, whole = at.whole();
  const float n = (float)cols;
  float g[NV][V], b[NV][V];
  load_weights<T, NV>(gamma, at, tiny, g);
  load_weights<T, NV>(beta, at, tiny, b);
  const int64_t stride = gridDim.x * at_once;
  // (every lane of a wave takes part in the sums: a group past the last row works on that one and stores nothing)
  const int64_t first = blockIdx.x * at_once + (G ? (int64_t)threadIdx.x / (G ? G : 1) : 0);
  u32x4 raw[NV];
  load_row<MODE, T, NV>(x + (first < rows ? first : rows - 1) * xs, at, tiny, raw);
  int64_t r = first;
  for (int64_t r0 = blockIdx.x * at_once; r0 < rows; r0 += stride, r += stride) {
    float v[NV][V], s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) unpack<T>(raw[k], v[k]);
    if (!whole) {
#pragma unroll
      for (int k = 0; k < NV; ++k) mask(v[k], at.skip[k]);
    }
    if (r0 + stride < rows)  // the next row is under way while this one is worked on
      load_row<MODE, T, NV>(x + (r + stride < rows ? r + stride : rows - 1) * xs, at, tiny, raw);
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] += v[k][j];
    row_sum<G>(s, waves, sh[0]);
    const float mean = s[0] / n;
    float q[1] = {0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) v[k][j] -= mean;
    if (!whole) {
#pragma unroll
      for (int k = 0; k < NV; ++k) mask(v[k], at.skip[k]);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) q[0] = fmaf(v[k][j], v[k][j], q[0]);
    row_sum<G>(q, waves, sh[1]);
    const float rstd = 1.f / sqrtf(q[0] / n + eps);
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) v[k][j] = v[k][j] * rstd * g[k][j] + b[k][j];
    activate_all<T>(v, act);
    if (r < rows) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (at.skip[k] < V) store_piece<MODE, T, V>(y + r * ys + at.c[k], at.skip[k], v[k]);
      if (stats && lane == 0) {
        stats[r] = mean;
        stats[rows + r] = rstd;
      }
    }
  }
}

// Rows that the registers of a block do not hold: three passes over the row, which the caches serve.  The pieces' sums
// are added up in 64 bits: a thread has up to 2^18 of them, and equal terms would round the same way every time.
template <typename T>
__global__ __launch_bounds__(64 * kMaxWaves) void layer_norm_fwd_long_kernel(
    const T* x, int64_t xs, int64_t rows, int cols, const float* __restrict__ gamma, const float* __restrict__ beta,
    float eps, int act, T* y, int64_t ys, float* __restrict__ stats) {
  constexpr int V = kVec<T>;
  __shared__ float sh[2][kMaxWaves][1];
  const int waves = (int)blockDim.x >> 6, c0 = (int)threadIdx.x * V, step = (int)blockDim.x * V;
  const float n = (float)cols;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const auto piece = [&](int c, float (&v)[1][V]) {
      const Pieces<T, 1> at(c, 0, cols);
      u32x4 w[1];
      load_row<kPlain, T, 1>(x + r * xs, at, false, w);
      unpack<T>(w[0], v[0]);
      return at;
    };
    float v[1][V];
    double sum = 0.;
    for (int c = c0; c < cols; c += step) {
      const Pieces<T, 1> at = piece(c, v);
      mask(v[0], at.skip[0]);
      float p = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) p += v[0][j];
      sum += p;
    }
    float s[1] = {(float)sum};
    waves_sum(s, waves, sh[0]);
    const float mean = s[0] / n;
    sum = 0.;
    for (int c = c0; c < cols; c += step) {
      const Pieces<T, 1> at = piece(c, v);
#pragma unroll
      for (int j = 0; j < V; ++j) v[0][j] -= mean;
      mask(v[0], at.skip[0]);
      float p = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) p = fmaf(v[0][j], v[0][j], p);
      sum += p;
    }
    float q[1] = {(float)sum};
    waves_sum(q, waves, sh[1]);
    const float rstd = 1.f / sqrtf(q[0] / n + eps);
    for (int c = c0; c < cols; c += step) {
      const Pieces<T, 1> at = piece(c, v);
      float g[1][V], b[1][V];
      load_weights<T, 1>(gamma, at, false, g);
      load_weights<T, 1>(beta, at, false, b);
#pragma unroll
      for (int j = 0; j < V; ++j) v[0][j] = (v[0][j] - mean) * rstd * g[0][j] + b[0][j];
      activate_all<T>(v, act);
      store_piece<kPlain, T, V>(y + r * ys + at.c[0], at.skip[0], v[0]);
    }
    if (stats && threadIdx.x == 0) {
      stats[r] = mean;
      stats[rows + r] = rstd;
    }
  }
}

// ------------------------------------------------------------------ backward
// x and dy are read once and dx is written: a thread keeps its columns from row to row, so it carries their dgamma and
// dbeta along in registers.  A block works on blockDim / (lanes of a row) rows at once; at the end it adds up what its
// row groups hold (pairwise, through LDS) and leaves one partial sum per column in part_g, part_b [block][column].
// `waves`: of a row, for G = 0.  Dynamic LDS: blockDim / 2 * NV * V * 2 floats.
template <typename T, int G, int NV, int MODE>
__global__ __launch_bounds__(64 * kMaxWaves) void layer_norm_bwd_kernel(
    const T* x, int64_t xs, const T* dy, int64_t dys, int64_t rows, int cols, const float* __restrict__ gamma,
    const float* __restrict__ beta, const float* __restrict__ stats, int act, T* dx, int64_t dxs,
    float* __restrict__ part_g, float* __restrict__ part_b, int waves) {
  constexpr int V = kVec<T>;
  __shared__ float sh[2][kMaxWaves][2];
  extern __shared__ float acc[];
  const int per_row = G ? G : waves * 64;
  const int group = (int)threadIdx.x / per_row, lane = (int)threadIdx.x - group * per_row;
  const int64_t at_once = (int)blockDim.x / per_row;
  const Pieces<T, NV> at(lane * V, per_row * V, cols);
  const bool tiny = G == 8 && cols < V;
  const float n = (float)cols;
  float g[NV][V], b[NV][V], sg[NV][V], sb[NV][V];
  load_weights<T, NV>(gamma, at, tiny, g);
  load_weights<T, NV>(beta, at, tiny, b);
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) sg[k][j] = sb[k][j] = 0.f;
  const int64_t stride = gridDim.x * at_once, first = blockIdx.x * at_once + group;
  u32x4 xn[NV], dn[NV];
  float mean_n, rstd_n;
  const auto fetch = [&](int64_t row) {
    row = row < rows ? row : rows - 1;
    load_row<MODE, T, NV>(x + row * xs, at, tiny, xn);
    load_row<MODE, T, NV>(dy + row * dys, at, tiny, dn);
    mean_n = stats[row];
    rstd_n = stats[rows + row];
  };
  fetch(first);
  int64_t r = first;
  int turn = 0;
  for (int64_t r0 = blockIdx.x * at_once; r0 < rows; r0 += stride, r += stride, turn ^= 1) {
    const float mean = mean_n, rstd = rstd_n;
    const bool live = r < rows;
    u32x4 xw[NV];
    float xh[NV][V], t[NV][V], s[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      // (a group past the last row adds nothing to any sum: dy = 0, and x = 0 because dx may lie on x, so that what
      // it read there can be the last row's dx already, and infinite)
      const u32x4 none = {0u, 0u, 0u, 0u};
      xw[k] = live ? xn[k] : none;
      unpack<T>(dn[k], t[k]);
      mask(t[k], live ? at.skip[k] : V);
    }
    if (r0 + stride < rows) fetch(r + stride);  // the next row is under way while this one is worked on
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      unpack<T>(xw[k], xh[k]);
#pragma unroll
      for (int j = 0; j < V; ++j) xh[k][j] = (xh[k][j] - mean) * rstd;
    }
    through_act<T>(t, xh, xw, g, b, mean, rstd, act);
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        sg[k][j] = fmaf(t[k][j], xh[k][j], sg[k][j]);
        sb[k][j] += t[k][j];
        t[k][j] *= g[k][j];
        s[0] += t[k][j];
        s[1] = fmaf(t[k][j], xh[k][j], s[1]);
      }
    row_sum<G>(s, waves, sh[turn]);
    const float ma = s[0] / n, mq = s[1] / n;
    if (live) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int j = 0; j < V; ++j) t[k][j] = rstd * fmaf(-mq, xh[k][j], t[k][j] - ma);
        if (at.skip[k] < V) store_piece<MODE, T, V>(dx + r * dxs + at.c[k], at.skip[k], t[k]);
      }
    }
  }
  // the groups of a wave first; then the upper half of the waves (G = 0: of the groups) hands its sums to the lower
  // one, until one is left
  if constexpr (G != 0 && G < 64) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        sg[k][j] = groups_sum<G>(sg[k][j]);
        sb[k][j] = groups_sum<G>(sb[k][j]);
      }
  }
  const bool holder = G == 0 || (int)(threadIdx.x & 63) < G;
  const int number = G ? (int)threadIdx.x >> 6 : group;
  for (int groups = G ? (int)blockDim.x >> 6 : (int)at_once; groups > 1;) {
    const int half = (groups + 1) / 2;
    const bool give = holder && number >= half && number < groups, take = holder && number < groups - half;
    float* slot = acc + (give ? number - half : number) * (NV * V * 2) * per_row + lane;
    if (give)
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          slot[(k * V + j) * 2 * per_row] = sg[k][j];
          slot[((k * V + j) * 2 + 1) * per_row] = sb[k][j];
        }
    __syncthreads();
    if (take)
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          sg[k][j] += slot[(k * V + j) * 2 * per_row];
          sb[k][j] += slot[((k * V + j) * 2 + 1) * per_row];
        }
    __syncthreads();
    groups = half;
  }
  if (holder && number == 0) {
    float* pg = part_g + (int64_t)blockIdx.x * cols;
    float* pb = part_b + (int64_t)blockIdx.x * cols;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (at.skip[k] < V) {
        store_piece<kPlain, float, V>(pg + at.c[k], at.skip[k], sg[k]);
        store_piece<kPlain, float, V>(pb + at.c[k], at.skip[k], sb[k]);
      }
  }
}

// Rows in 1, 2, 4 or 8 waves (W) with up to 40 elements of 16 bits or 32 of fp32 a lane.  A block is eight waves of up to
// 256 registers: they have more bytes under way (80 KB of a CU's reads at 5 pieces) than the sixteen of 8 elements a thread
// (30 KB), and the sums of a row alone in its wave need no barrier.  What is not needed all the time makes room for that:
// gamma and beta lie in LDS, xhat is formed again for dx.  us, against the kernel above (beyond 8192 columns: below):
//   bf16   640 x 16384  16.7, 21.3    2496 x 16384  49, 54 (with tanh 53, 74)    4346 x 8192  48, 65    8192 x 8192  77, 78
//          12288 x 8192  109, 269     16384 x 64  14.6, 16.7
//   fp32   640 x 16384  23.2, 25.3    1280 x 4096  15.4, 18.1    1280 x 65536  182, 170    12288 x 8192  212, 460
constexpr int kRowWaves = 8;
template <typename T, int W, int NV, int MODE, bool ACT>
__global__ __launch_bounds__(64 * kRowWaves) void layer_norm_bwd_wave_kernel(
    const T* x, int64_t xs, const T* dy, int64_t dys, int64_t rows, int cols, const float* __restrict__ gamma,
    const float* __restrict__ beta, const float* __restrict__ stats, int act, T* dx, int64_t dxs,
    float* __restrict__ part_g, float* __restrict__ part_b) {
  constexpr int V = kVec<T>;
  constexpr int kGroups = kRowWaves / W;  // rows at once
  __shared__ u32x4 weights[2][NV][V / 4][64 * W];
  // (read V apart: the padding spreads them over the banks)
  __shared__ float acc[kGroups > 1 ? 2 : 1][kGroups > 1 ? kRowWaves : 1][2 * V][64 + 64 / V];
  __shared__ float sh[2][kMaxWaves][2];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), group = wave / W;
  const int lane = (int)threadIdx.x - 64 * W * group;
  const Pieces<T, NV> at(lane * V, 64 * W * V, cols);
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (group == k % kGroups) {
#pragma unroll
      for (int i = 0; i < V / 4; ++i) {
        weights[0][k][i][lane] = *reinterpret_cast<const u32x4_any*>(gamma + at.c[k] + 4 * i);
        weights[1][k][i][lane] = *reinterpret_cast<const u32x4_any*>(beta + at.c[k] + 4 * i);
      }
    }
  __syncthreads();
  const auto weight = [&](int which, int k, int l, float (&v)[1][V]) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      const u32x4 w = weights[which][k][i][l];
      __builtin_memcpy(&v[0][4 * i], &w, 16);
    }
  };
  uint32_t byte[NV];  // of the pieces in their row (32 bits, so that the row's address stays in scalar registers)
#pragma unroll
  for (int k = 0; k < NV; ++k) byte[k] = (uint32_t)at.c[k] * (uint32_t)sizeof(T);
  const float n = (float)cols;
  float sg[NV][V], sb[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) sg[k][j] = sb[k][j] = 0.f;
  const int64_t stride = (int64_t)gridDim.x * kGroups;
  int64_t r = (int64_t)blockIdx.x * kGroups + group;
  u32x4 xn[NV], dn[NV];
  float mean_n = 0.f, rstd_n = 0.f;
  const auto fetch = [&](int64_t row) {
    const char *xr = (const char*)(x + row * xs), *dr = (const char*)(dy + row * dys);
#pragma unroll
    for (int k = 0; k < NV; ++k) xn[k] = load_16<MODE>(xr + byte[k]);
#pragma unroll
    for (int k = 0; k < NV; ++k) dn[k] = load_16<MODE>(dr + byte[k]);
    mean_n = stats[row];
    rstd_n = stats[rows + row];
  };
  if (r < rows) fetch(r);
  int turn = 0;
  // (waves that share rows meet at barriers: all of a block's take every turn, with or without a row)
  for (; (W == 1 ? r : r - group) < rows; r += stride, turn ^= 1) {
    const bool live = W == 1 || kGroups == 1 || r < rows;
    const float mean = mean_n, rstd = rstd_n;
    u32x4 xw[NV], dw[NV];
    float t[NV][V], s[2] = {0.f, 0.f};
    int l = lane;
    asm volatile("" : "+v"(l));  // (this and the others below: or the compiler keeps the weights and xhat in registers
                                 // all the same, and leaves the sums to the loop's end with all that goes into them)
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      xw[k] = xn[k];
      dw[k] = dn[k];
    }
    if (r + stride < rows) fetch(r + stride);  // the next row is under way while this one is worked on
    if (live) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        __builtin_amdgcn_sched_barrier(0);
        float xh[1][V], g[1][V], d[1][V];
        unpack<T>(xw[k], xh[0]);
        weight(0, k, l, g);
#pragma unroll
        for (int j = 0; j < V; ++j) xh[0][j] = (xh[0][j] - mean) * rstd;
        asm volatile("" : "+v"(dw[k]));
        unpack<T>(dw[k], d[0]);
        if (k == NV - 1) mask(d[0], at.skip[k]);
        if constexpr (ACT) {
          float b[1][V];
          const u32x4 xk[1] = {xw[k]};
          weight(1, k, l, b);
          through_act<T>(d, xh, xk, g, b, mean, rstd, act);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
          sg[k][j] = fmaf(d[0][j], xh[0][j], sg[k][j]);
          sb[k][j] += d[0][j];
          asm volatile("" : "+v"(sg[k][j]), "+v"(sb[k][j]));
          t[k][j] = d[0][j] * g[0][j];
          s[0] += t[k][j];
          s[1] = fmaf(t[k][j], xh[0][j], s[1]);
        }
        asm volatile("" : "+v"(s[0]), "+v"(s[1]));
      }
    }
    row_sum<W == 1 ? 64 : 0>(s, W, sh[turn]);
    if (!live) continue;
    const float a = -(s[0] / n) * rstd, b = -(s[1] / n) * rstd * rstd;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float x0[V];
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("" : "+v"(xw[k]));
      unpack<T>(xw[k], x0);
#pragma unroll
      for (int j = 0; j < V; ++j) t[k][j] = fmaf(t[k][j], rstd, fmaf(x0[j] - mean, b, a));
      T* to = (T*)((char*)(dx + r * dxs) + byte[k]);
      if (k < NV - 1)
        store_piece<MODE, T, V>(to, 0, t[k]);
      else if (at.skip[k] < V)
        store_piece<MODE, T, V>(to, at.skip[k], t[k]);
    }
  }
  if constexpr (kGroups == 1) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (at.skip[k] < V) {
        store_piece<kPlain, float, V>(part_g + (int64_t)blockIdx.x * cols + at.c[k], at.skip[k], sg[k]);
        store_piece<kPlain, float, V>(part_b + (int64_t)blockIdx.x * cols + at.c[k], at.skip[k], sb[k]);
      }
    return;
  }
  // the groups' sums, a piece at a time through one of two buffers: [wave][sum][lane] -> one sum per column
#pragma unroll
  for (int k = 0; k < NV; ++k) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      acc[k & 1][wave][j][lane & 63] = sg[k][j];
      acc[k & 1][wave][V + j][lane & 63] = sb[k][j];
    }
    __syncthreads();
    constexpr int kSums = V * 64 * W;  // of one kind; whole turns of the block
    static_assert(2 * kSums % (64 * kRowWaves) == 0, "");
#pragma unroll
    for (int i = 0; i < 2 * kSums; i += 64 * kRowWaves) {
      const int e = i + (int)threadIdx.x;
      // neighbours in a block take neighbouring columns of one of the two sums
      const int which = e / kSums, l = e % kSums / V, j = e % V;
      const int at0 = (k * 64 * W + l) * V, c = min(at0, cols - V), skip = at0 - c;
      float sum = 0.f;
#pragma unroll
      for (int q = 0; q < kGroups; ++q) sum += acc[k & 1][q * W + (l >> 6)][which * V + j][l & 63];
      if (j >= skip) (which ? part_b : part_g)[(int64_t)blockIdx.x * cols + c + j] = sum;
    }
  }
}

// A piece of a long row: du in t, xhat in xh, and what counts of it.
template <typename T>
struct LongPiece {
  float g[1][kVec<T>], xh[1][kVec<T>], t[1][kVec<T>];
  Pieces<T, 1> at;
  __device__ __forceinline__ LongPiece(const T* x, const T* dy, const float* __restrict__ gamma,
                                       const float* __restrict__ beta, float mean, float rstd, int act, int c, int cols)
      : at(c, 0, cols) {
    u32x4 xw[1], dw[1];
    float b[1][kVec<T>];
    load_row<kPlain, T, 1>(x, at, false, xw);
    load_row<kPlain, T, 1>(dy, at, false, dw);
    load_weights<T, 1>(gamma, at, false, g);
    load_weights<T, 1>(beta, at, false, b);
    unpack<T>(xw[0], xh[0]);
    unpack<T>(dw[0], t[0]);
    mask(t[0], at.skip[0]);
#pragma unroll
    for (int j = 0; j < kVec<T>; ++j) xh[0][j] = (xh[0][j] - mean) * rstd;
    through_act<T>(t, xh, xw, g, b, mean, rstd, act);
  }
};

// Rows that the registers of a block do not hold: x and dy are read three times, twice here (the second time out of the
// caches) and once for the weights' gradients.
template <typename T>
__global__ __launch_bounds__(64 * kMaxWaves) void layer_norm_bwd_long_kernel(
    const T* x, int64_t xs, const T* dy, int64_t dys, int64_t rows, int cols, const float* __restrict__ gamma,
    const float* __restrict__ beta, const float* __restrict__ stats, int act, T* dx, int64_t dxs) {
  constexpr int V = kVec<T>;
  __shared__ float sh[2][kMaxWaves][2];
  const int waves = (int)blockDim.x >> 6, c0 = (int)threadIdx.x * V, step = (int)blockDim.x * V;
  const float n = (float)cols;
  int turn = 0;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x, turn ^= 1) {
    const float mean = stats[r], rstd = stats[rows + r];
    double sum = 0., across = 0.;  // (see the forward kernel)
    for (int c = c0; c < cols; c += step) {
      const LongPiece<T> p(x + r * xs, dy + r * dys, gamma, beta, mean, rstd, act, c, cols);
      float a = 0.f, b = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float t = p.t[0][j] * p.g[0][j];
        a += t;
        b = fmaf(t, p.xh[0][j], b);
      }
      sum += a;
      across += b;
    }
    float s[2] = {(float)sum, (float)across};
    waves_sum(s, waves, sh[turn]);
    const float ma = s[0] / n, mq = s[1] / n;
    for (int c = c0; c < cols; c += step) {
      const LongPiece<T> p(x + r * xs, dy + r * dys, gamma, beta, mean, rstd, act, c, cols);
      float d[V];
#pragma unroll
      for (int j = 0; j < V; ++j) d[j] = rstd * fmaf(-mq, p.xh[0][j], p.t[0][j] * p.g[0][j] - ma);
      store_piece<kPlain, T, V>(dx + r * dxs + p.at.c[0], p.at.skip[0], d);
    }
  }
}

// part[0][p][c] = sum of du xhat, part[1][p][c] = sum of du over rows p, p + parts, ...
template <typename T>
__global__ __launch_bounds__(kThreads) void layer_norm_bwd_long_sums_kernel(
    const T* x, int64_t xs, const T* dy, int64_t dys, int64_t rows, int cols, const float* __restrict__ gamma,
    const float* __restrict__ beta, const float* __restrict__ stats, int act, int parts, float* __restrict__ part) {
  constexpr int V = kVec<T>;
  const int c = ((int)blockIdx.x * kThreads + (int)threadIdx.x) * V, p = blockIdx.y;
  if (c >= cols) return;
  float sg[V], sb[V];
#pragma unroll
  for (int j = 0; j < V; ++j) sg[j] = sb[j] = 0.f;
  for (int64_t r = p; r < rows; r += parts) {
    const LongPiece<T> q(x + r * xs, dy + r * dys, gamma, beta, stats[r], stats[rows + r], act, c, cols);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      sg[j] = fmaf(q.t[0][j], q.xh[0][j], sg[j]);
      sb[j] += q.t[0][j];
    }
  }
  const Pieces<T, 1> at(c, 0, cols);
  store_piece<kPlain, float, V>(part + (int64_t)p * cols + at.c[0], at.skip[0], sg);
  store_piece<kPlain, float, V>(part + (int64_t)(parts + p) * cols + at.c[0], at.skip[0], sb);
}

// dgamma (blockIdx.y = 0) and dbeta from the blocks' partial sums: 32 columns by 32 slices of the parts per block.  A
// column's slices are added up by 32 lanes, as a tree: one after the other the 32 roundings weighed more than those of all
// else on the way (8192 x 20 fp32).  Blocks walk the columns: a launch takes fewer than 2^32 threads, which 2^27 columns
// would need.
constexpr int kFinish = 32;
constexpr int kFinishBlocks = 1 << 16;  // (2^21 columns in one turn)
__global__ __launch_bounds__(kFinish* kFinish) void layer_norm_bwd_finish_kernel(const float* __restrict__ part,
                                                                                 int parts, int cols,
                                                                                 float* __restrict__ dgamma,
                                                                                 float* __restrict__ dbeta) {
  __shared__ float sh[kFinish][kFinish + 1];
  const int x = threadIdx.x, y = threadIdx.y;
  const float* p = part + (int64_t)blockIdx.y * parts * cols;
  float* out = blockIdx.y ? dbeta : dgamma;
  for (int c0 = (int)blockIdx.x * kFinish;;) {
    float s = 0.f;
    if (c0 + x < cols) {
#pragma unroll 8
      for (int k = y; k < parts; k += kFinish) s += p[(int64_t)k * cols + c0 + x];
    }
    sh[y][x] = s;
    __syncthreads();
    s = group_sum<kFinish>(sh[x][y]);
    if (x == 0 && c0 + y < cols) out[c0 + y] = s;
    c0 += (int)gridDim.x * kFinish;
    if (c0 >= cols) break;
    __syncthreads();
  }
}

// ------------------------------------------------------------------ which kernel, how many blocks
constexpr int kCus = 256;
constexpr int kMaxParts = 2 * kCus;  // backward blocks of 8 waves or more at 4 waves a SIMD: 2 at most on a CU

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// lanes per row (0: whole waves), 16-byte pieces per thread, waves per row
struct Shape {
  int group, pieces, waves;
};

// A row is held by as few lanes as one 16-byte piece each covers; from 64 lanes on by one wave with up to `alone`
// pieces a lane (its sums need no barrier); then by several waves with `wave` pieces a thread.  pieces = 0: too long
// for the registers of 16 waves.
Shape shape_of(int cols, int vec, int alone, int wave) {
  const int64_t need = ceil_div(cols, vec);
  if (need <= 8) return {8, 1, 1};
  if (need <= 16) return {16, 1, 1};
  if (need <= 32) return {32, 1, 1};
  if (need <= 64 * alone) return {64, (int)ceil_div(need, 64), 1};
  if (need <= 64 * kMaxWaves * wave) return {0, wave, (int)ceil_div(need, 64 * wave)};
  return {0, 0, kMaxWaves};
}

bool streams(int64_t rows, int cols, int passes, size_t size) { return (double)rows * cols * passes * size > 128e6; }

// blocks that are all on the chip at once (`waves` to each, `room` of them to a SIMD): with 1024 blocks on 768 places the
// last 256 took a second round (2496 x 16384 bf16 backward, 118 against 108 us).  All of those, though only some have a
// last turn: fewer blocks of equal turns leave CUs a block short (3091 x 5192 bf16 sigmoid 24.6 against 21.9 us, 512 x
// 20000 fp32 backward 25.0 and 23.5).
int64_t blocks_of(int64_t turns, int waves, int room) {
  const int64_t resident = (int64_t)kCus * (4 * room / waves);
  return turns <= resident ? turns : resident;
}

bool act_ok(int act) { return act >= XDFM_ACT_IDENTITY && act <= XDFM_ACT_ELU; }
bool dtype_ok(int t) { return t == XDFM_F32 || t == XDFM_BF16 || t == XDFM_F16; }
bool aligned(const void* p, int dtype) { return ((uintptr_t)p & (dtype == XDFM_F32 ? 3 : 1)) == 0; }

// rows * stride elements have to be addressable, and a column's number plus a block's stride an int
bool extent_ok(int64_t rows, int64_t stride, int cols) {
  return rows >= 0 && cols > 0 && cols <= 1 << 30 && stride >= cols && rows <= (INT64_MAX / 8) / stride;
}

template <typename T, int MODE>
void fwd_as(const void* x, int64_t xs, int64_t rows, int cols, const float* gamma, const float* beta, float eps, int act,
         void* y, int64_t ys, float* stats, hipStream_t st) {
  // 16 elements a thread, up to 24 where they hold the row without company (1536 x 16384 bf16 17.5 against 19.2 us, 1100
  // columns 17.3 and 20.0).  Many longer rows of 16 bits, and rows too long for 16: 16, 24 or 40 elements a thread,
  // whichever leaves the fewest of a CU's lanes empty, in the row and behind the last row that fits (2496 x 16384 bf16 31.0
  // against 32.3 us; 10240 x 5192 38.7 and 50.4; 6144 x 16384 sigmoid 81 and 110; 18000 x 5192 75 and 117, fp32 138 and 210;
  // but 9000 x 300 7.1 and 6.0, fp32 9000 x 5192 68.5 and 65).
  constexpr int kWave = 16 / kVec<T>, kMore = 24 / kVec<T>, kMost = 40 / kVec<T>;
  Shape s = shape_of(cols, kVec<T>, kMore, kWave);
  const int64_t need = ceil_div(cols, 64 * kVec<T>);
  if (s.pieces == 0 || (sizeof(T) == 2 && need > kMore && rows >= 4096)) {
    double best = 0.;
    for (const int each : {kWave, kMore, kMost}) {
      const int64_t at = places(each * kVec<T>), waves = ceil_div(need, each);
      const double filled = (double)(need * (at / waves)) / (double)(each * at);  // 0: the row does not fit
      if (filled > best && (sizeof(T) == 2 || each != kMost)) best = filled, s = {waves == 1 ? 64 : 0, each, (int)waves};
    }
  }
  const dim3 block(s.group ? kThreads : 64 * s.waves);
  const int64_t turns = s.group ? ceil_div(rows, kThreads / s.group) : rows;
  const int each = s.pieces * kVec<T>;
  const int room = each > 16 ? places(each) / 4 : each > 8 ? (sizeof(T) == 2 && s.group ? 5 : 4) : each ? 7 : 8;
  const dim3 grid((unsigned)blocks_of(turns, (int)block.x / 64, room));
#define CASE(G, NV)                                                                                              \
  if (s.group == G && s.pieces == NV) {                                                                          \
    XDFM_LAUNCH("layer_norm_fwd_kernel", st, (layer_norm_fwd_kernel<T, G, NV, MODE>), grid, block, 0, (const T*)x, \
                xs, rows, cols, gamma, beta, eps, act, (T*)y, ys, stats);                                        \
    return;                                                                                                      \
  }
  CASE(8, 1) CASE(16, 1) CASE(32, 1) CASE(64, 1) CASE(64, 2)
  if constexpr (kWave == 4) {
    CASE(64, 3) CASE(64, 4) CASE(64, 5) CASE(64, kMore) CASE(0, kWave) CASE(0, kMore)
  } else {
    CASE(64, kMore) CASE(64, kMost) CASE(0, kWave) CASE(0, kMore) CASE(0, kMost)
  }
#undef CASE
  XDFM_LAUNCH("layer_norm_fwd_long_kernel", st, layer_norm_fwd_long_kernel<T>, grid, block, 0, (const T*)x, xs, rows,
              cols, gamma, beta, eps, act, (T*)y, ys, stats);
}

// Waves of a backward block, whose row groups share one partial sum.  16 leave 256 partial sums on a full chip (with 4
// waves a block 1024; 512 columns of bf16 by 16384 rows: 14.6 against 16.6 us; 2496 columns, 5 waves a row: 56 against
// 108).  Where that would leave CUs without a block, 8 (20 x 8192 fp32: 7.3 against 8.2 us; 65536 rows: 9.0 and 8.9).
constexpr int kBwdWaves = kMaxWaves;
// Turns up to which one block takes all rows and writes dgamma and dbeta itself, without a second launch: 128 x 20 fp32
// 4.8 against 7.1 us, two turns 16 x 1024 7.05 against 7.6, four turns 32 x 1024 10.7 against 7.6.
constexpr int kTurnsOfOne = 2;

// the number of partial sums that lie in ws afterwards (0: dgamma and dbeta are written)
template <typename T, int MODE>
int bwd_as(const void* x, int64_t xs, const void* dy, int64_t dys, int64_t rows, int cols, const float* gamma,
           const float* beta, const float* stats, int act, void* dx, int64_t dxs, float* dgamma, float* dbeta, float* ws,
           hipStream_t st) {
  // Rows in waves of many registers, see there, if they are enough to give most CUs a block (16-bit 2496 x 256 9.5 against
  // 8.9 us, x 1024 11.1 and 12.3; four waves a row need two rounds: 8192 x 600 21 and 18, x 1024 20 and 19.6).  fp32, of
  // which the other kernel has twice the bytes under way, only where the pass stays in the caches, or is too long for it.
  const int need = (int)ceil_div(cols, 64 * kVec<T>);
  const auto go = [&](auto kernel, int w, int each) {
    const int64_t blocks = blocks_of(ceil_div(rows, kRowWaves / w), kRowWaves, each <= (act ? 12 : 16) ? 4 : 2);
    XDFM_LAUNCH("layer_norm_bwd_wave_kernel", st, kernel, dim3((unsigned)blocks), dim3(64 * kRowWaves), 0, (const T*)x,
                xs, (const T*)dy, dys, rows, cols, gamma, beta, stats, act, (T*)dx, dxs, ws, ws + blocks * cols);
    return (int)blocks;
  };
  const auto fits = [&](int w, int most) {
    return need <= most * w && ceil_div(rows, kRowWaves / w) >= (w == 4 ? 2 * kCus : kCus / 2);
  };
#define CASE(W, NV)                                                               \
  if (need <= W * NV)                                                             \
    return go(act ? layer_norm_bwd_wave_kernel<T, W, NV, MODE, true>              \
                  : layer_norm_bwd_wave_kernel<T, W, NV, MODE, false>, W, NV * kVec<T>);
  static_assert(XDFM_ACT_IDENTITY == 0, "");
  if constexpr (sizeof(T) == 2) {
    if (need >= 2 && fits(1, 5)) {
      CASE(1, 2) CASE(1, 3) CASE(1, 4) CASE(1, 5)
    }
    if (need > 5 && fits(2, 5)) {
      CASE(2, 3) CASE(2, 4) CASE(2, 5)
    }
    if (need > 10 && fits(4, 5)) {
      CASE(4, 3) CASE(4, 4) CASE(4, 5)
    }
    if (need > 16) {
      CASE(8, 3) CASE(8, 4)
    }
  } else {
    if constexpr (MODE == kPlain)
      if (need >= 3 && fits(1, 6)) {
        CASE(1, 3) CASE(1, 4) CASE(1, 5) CASE(1, 6)
      }
    if (need > 32) {
      CASE(8, 5) CASE(8, 6) CASE(8, 7) CASE(8, 8)
    }
  }
#undef CASE
  // 8 elements a thread: with their weights and the weights' gradients they take 6 registers each
  constexpr int kWave = 8 / kVec<T>;
  const Shape s = shape_of(cols, kVec<T>, kWave, kWave);
  const int per_row = s.group ? s.group : 64 * s.waves;
  const int at_most = kBwdWaves * 64 / per_row;
  const bool one = ceil_div(rows, at_most) <= kTurnsOfOne;
  const int at_once = !one && s.group && ceil_div(rows, at_most) < kCus ? at_most / 2 : at_most;
  const int threads = at_once * per_row;
  const int64_t blocks = one ? 1 : blocks_of(ceil_div(rows, at_once), threads / 64, 4);
  float *part_g = one ? dgamma : ws, *part_b = one ? dbeta : ws + blocks * cols;
#define CASE(G, NV)                                                                                                \
  if (s.group == G && s.pieces == NV) {                                                                            \
    XDFM_LAUNCH("layer_norm_bwd_kernel", st, (layer_norm_bwd_kernel<T, G, NV, MODE>), dim3((unsigned)blocks),      \
                dim3((unsigned)threads), (size_t)threads* NV* kVec<T> * sizeof(float), (const T*)x, xs,            \
                (const T*)dy, dys, rows, cols, gamma, beta, stats, act, (T*)dx, dxs, part_g, part_b, s.waves);     \
    return one ? 0 : (int)blocks;                                                                                  \
  }
  CASE(8, 1) CASE(16, 1) CASE(32, 1) CASE(64, 1)
  if constexpr (kWave == 2) {
    CASE(64, 2) CASE(0, 2)
  } else {
    CASE(0, 1)
  }
#undef CASE
  // (the sums first: dx may be dy or x; 16 rows a part where there are few: 256 x 16384 fp32 26 us, with 64 rows 46)
  const int parts = (int)(rows < 16 ? 1 : rows < 16 * kCus ? rows / 16 : kCus);
  XDFM_LAUNCH("layer_norm_bwd_long_sums_kernel", st, layer_norm_bwd_long_sums_kernel<T>,
              dim3((unsigned)ceil_div(cols, kThreads * kVec<T>), (unsigned)parts), dim3(kThreads), 0, (const T*)x, xs,
              (const T*)dy, dys, rows, cols, gamma, beta, stats, act, parts, ws);
  XDFM_LAUNCH("layer_norm_bwd_long_kernel", st, layer_norm_bwd_long_kernel<T>, dim3((unsigned)blocks_of(rows, kMaxWaves, 8)),
              dim3(64 * kMaxWaves), 0, (const T*)x, xs, (const T*)dy, dys, rows, cols, gamma, beta, stats, act, (T*)dx,
              dxs);
  return parts;
}

template <typename T>
void fwd(const void* x, int64_t xs, int64_t rows, int cols, const float* gamma, const float* beta, float eps, int act,
         void* y, int64_t ys, float* stats, hipStream_t st) {
  (streams(rows, cols, 2, sizeof(T)) ? fwd_as<T, kStream> : fwd_as<T, kPlain>)(x, xs, rows, cols, gamma, beta, eps, act,
                                                                               y, ys, stats, st);
}

template <typename T>
int bwd(const void* x, int64_t xs, const void* dy, int64_t dys, int64_t rows, int cols, const float* gamma,
        const float* beta, const float* stats, int act, void* dx, int64_t dxs, float* dgamma, float* dbeta, float* ws,
        hipStream_t st) {
  return (streams(rows, cols, 3, sizeof(T)) ? bwd_as<T, kStream> : bwd_as<T, kPlain>)(
      x, xs, dy, dys, rows, cols, gamma, beta, stats, act, dx, dxs, dgamma, dbeta, ws, st);
}

}  // namespace

extern "C" int xdfm_layer_norm_fwd(const void* x, int64_t x_stride, int32_t dtype, int64_t rows, int32_t cols,
                                   const float* gamma, const float* beta, float eps, int32_t act, void* y,
                                   int64_t y_stride, float* stats, void* stream) {
  XDFM_REQUIRE(dtype_ok(dtype), "xdfm_layer_norm_fwd: unknown element type %d", dtype);
  XDFM_REQUIRE(act_ok(act), "xdfm_layer_norm_fwd: unknown activation %d", act);
  XDFM_REQUIRE(extent_ok(rows, x_stride, cols) && extent_ok(rows, y_stride, cols),
               "xdfm_layer_norm_fwd: bad sizes (rows %lld, cols %d, strides %lld, %lld)", (long long)rows, cols,
               (long long)x_stride, (long long)y_stride);
  XDFM_REQUIRE(eps > 0.f && eps < 1e30f, "xdfm_layer_norm_fwd: eps has to be positive");
  if (rows == 0) return XDFM_OK;
  XDFM_REQUIRE(x && y && gamma && beta, "xdfm_layer_norm_fwd: null argument");
  XDFM_REQUIRE(aligned(x, dtype) && aligned(y, dtype), "xdfm_layer_norm_fwd: misaligned x or y");
  XDFM_REQUIRE(x != y || x_stride == y_stride, "xdfm_layer_norm_fwd: y on x needs the same stride");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == XDFM_F32)
    fwd<float>(x, x_stride, rows, cols, gamma, beta, eps, act, y, y_stride, stats, st);
  else if (dtype == XDFM_BF16)
    fwd<__bf16>(x, x_stride, rows, cols, gamma, beta, eps, act, y, y_stride, stats, st);
  else
    fwd<_Float16>(x, x_stride, rows, cols, gamma, beta, eps, act, y, y_stride, stats, st);
  XDFM_LAUNCH_CHECK();
  return XDFM_OK;
}

extern "C" int xdfm_layer_norm_bwd_workspace_floats(int64_t rows, int32_t cols, size_t* floats) {
  XDFM_REQUIRE(floats && rows >= 0 && cols > 0 && cols <= 1 << 30,
               "xdfm_layer_norm_bwd_workspace_floats: bad argument");
  *floats = (size_t)2 * (rows < 1 ? 1 : rows < kMaxParts ? rows : kMaxParts) * cols;
  return XDFM_OK;
}

extern "C" int xdfm_layer_norm_bwd(const void* x, int64_t x_stride, const void* dy, int64_t dy_stride, int32_t dtype,
                                   int64_t rows, int32_t cols, const float* gamma, const float* beta,
                                   const float* stats, int32_t act, void* dx, int64_t dx_stride, float* dgamma,
                                   float* dbeta, float* workspace, void* stream) {
  XDFM_REQUIRE(dtype_ok(dtype), "xdfm_layer_norm_bwd: unknown element type %d", dtype);
  XDFM_REQUIRE(act_ok(act), "xdfm_layer_norm_bwd: unknown activation %d", act);
  XDFM_REQUIRE(extent_ok(rows, x_stride, cols) && extent_ok(rows, dy_stride, cols) && extent_ok(rows, dx_stride, cols),
               "xdfm_layer_norm_bwd: bad sizes (rows %lld, cols %d, strides %lld, %lld, %lld)", (long long)rows, cols,
               (long long)x_stride, (long long)dy_stride, (long long)dx_stride);
  XDFM_REQUIRE(gamma && beta && dgamma && dbeta && workspace, "xdfm_layer_norm_bwd: null argument");
  XDFM_REQUIRE(rows == 0 || (x && dy && dx && stats), "xdfm_layer_norm_bwd: null argument");
  XDFM_REQUIRE(aligned(x, dtype) && aligned(dy, dtype) && aligned(dx, dtype) && ((uintptr_t)workspace & 15) == 0,
               "xdfm_layer_norm_bwd: misaligned x, dy, dx or workspace");
  XDFM_REQUIRE((dx != dy || dx_stride == dy_stride) && (dx != x || dx_stride == x_stride),
               "xdfm_layer_norm_bwd: dx on dy or x needs the same stride");
  hipStream_t st = (hipStream_t)stream;
  int parts = 0;
  if (rows == 0)
    ;  // sums of nothing
  else if (dtype == XDFM_F32)
    parts = bwd<float>(x, x_stride, dy, dy_stride, rows, cols, gamma, beta, stats, act, dx, dx_stride, dgamma, dbeta,
                       workspace, st);
  else if (dtype == XDFM_BF16)
    parts = bwd<__bf16>(x, x_stride, dy, dy_stride, rows, cols, gamma, beta, stats, act, dx, dx_stride, dgamma, dbeta,
                        workspace, st);
  else
    parts = bwd<_Float16>(x, x_stride, dy, dy_stride, rows, cols, gamma, beta, stats, act, dx, dx_stride, dgamma, dbeta,
                          workspace, st);
  if (parts || rows == 0)
    XDFM_LAUNCH("layer_norm_bwd_finish_kernel", st, layer_norm_bwd_finish_kernel,
                dim3((unsigned)std::min<int64_t>(ceil_div(cols, kFinish), kFinishBlocks), 2), dim3(kFinish, kFinish), 0,
                workspace, parts, cols, dgamma, dbeta);
  XDFM_LAUNCH_CHECK();
  return XDFM_OK;
}
