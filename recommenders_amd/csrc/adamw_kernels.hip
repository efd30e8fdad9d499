// AdamW over many tensors at once, states in 32 or in 8 bits (xdfm_adamw_*, include/xdfm.h).
//
//   m <- b1 m + (1 - b1) g,  v <- b2 v + (1 - b2) g^2
//   p <- p - lr wd p - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound by memory: 28 bytes an element with fp32 gradients and 32-bit states, 16 with 8-bit ones (and a hash, two
// roundings and the packing: ~85 operations, of ~105 that fit beside the bytes).
//   25.3 M elements (a table of 2.3 M rows of 10 and its linear weights)   32-bit 118 us, 6.0 TB/s; 8-bit 65 us, 6.2 TB/s
//   6.0 M elements in 16 tensors (the wide model's dense variables)        32-bit 29 us, 5.8 TB/s
//   47 k elements in 17 tensors                                            5 us: the launch
//
// The plan is an array of chunks: runs of at most chunk_elems elements of one tensor with their addresses, so that
// a block needs one record and no search, and tensors of one element and of 10^8 share a launch.
// The codes of the 8-bit states: a value scaled by a power of two so that the largest of its block has the
// exponent field 14 (m) or 30 (v) as a float; the float's bits from the third mantissa bit up are then the code, and
// what lies below is cut off after random bits were added to it.  Values under 2^-126 of that scale are denormal
// floats, whose bits go on being the value in units: the same shift codes them too.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include "xdfm_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 64;  // elements that share a scale
// Elements of a chunk, two pieces of a thread: 40 bytes of record for 32 KB and more.  8-bit table with read-out 98 us,
// with 4096 elements 100, with 8192 105; the wide model 28.9, 28.8, 31.0.
constexpr int kChunk = 2048;
// of a plan: a launch takes fewer than 2^32 threads
constexpr int64_t kMostChunks = ((int64_t)1 << 32) / kThreads - 1;
constexpr int kScaleMin = 48;  // units stay normal floats: 2^(48 - 159)
constexpr uint32_t kMul1 = 0x9E3779B1u;  // 2^32 / golden ratio
constexpr uint32_t kMul2 = 0x6A09E667u;  // the fraction of sqrt(2)

struct Chunk {
  float* p;
  const void* g;
  void* m;
  void* v;
  uint8_t* sm;
  uint8_t* sv;
  int64_t start;  // of the chunk in its tensor (a multiple of kBlock)
  int64_t out;    // of the chunk in the tensors laid one behind the other
  int32_t count;
  int32_t tensor;
  float wd;
  int32_t gtype;
};
static_assert(sizeof(Chunk) == 80, "the plan's record");

struct Args {
  float lr, b1, omb1, b2, omb2, eps;
  float log_b1, log_b2;     // for t from the device
  float step, inv_root;     // lr / (1 - b1^t), 1 / sqrt(1 - b2^t) for t from the host
  const float* state;
  uint32_t seed_lo, seed_hi, t;
};

struct Step {
  float size, inv_root;
  uint32_t t;
  bool past;  // t is a float that has come to stand still
};

__device__ __forceinline__ Step step_of(const Args& a) {
  if (!a.state) return {a.step, a.inv_root, a.t, false};
  const float t = fmaxf(a.state[3], 1.f);  // (a state that was not advanced yet: the first step)
  return {a.lr / -expm1f(t * a.log_b1), 1.f / sqrtf(-expm1f(t * a.log_b2)), (uint32_t)t,
          __builtin_amdgcn_readfirstlane(t >= 0x1p24f) != 0};
}

// (multiplications and additions are not contracted in this build: m and v are the two products' sum.  Root and
// reciprocal are the hardware's, good to one unit of the last place; the root takes no denormal numbers.)
__device__ __forceinline__ float root(float v) {
  const bool small = v < 0x1p-96f;
  const float r = __builtin_amdgcn_sqrtf(small ? v * 0x1p64f : v);
  return small ? r * 0x1p-32f : r;
}
__device__ __forceinline__ float update(float p, float g, float& m, float& v, const Args& a, const Step& s, float wd) {
  m = m * a.b1 + g * a.omb1;
  v = v * a.b2 + (g * g) * a.omb2;
  return (p - wd * p) - s.size * m * __builtin_amdgcn_rcpf(fmaf(root(v), s.inv_root, a.eps));
}

__device__ __forceinline__ uint32_t mix(uint32_t a, uint32_t b) { return (a ^ (a >> 15)) * kMul1 + b; }

// keys of a tensor's random bits at a step
__device__ __forceinline__ uint2 keys_of(const Args& a, uint32_t t, int tensor, int64_t i) {
  const uint32_t k = mix(mix(mix(a.seed_lo, a.seed_hi), t), (uint32_t)tensor);
  return make_uint2(mix(k, 1u), mix(k, 2u + (uint32_t)(i >> 32)));
}

__device__ __forceinline__ uint32_t random_bits(uint2 k, uint32_t i) {
  uint32_t a = (i + k.x) * kMul1;
  a = (a ^ (a >> 15) ^ k.y) * kMul2;
  return a ^ (a >> 16);
}

// What sets an element's random bits apart from those of other steps once the step count does not: a float stays at 2^24,
// and with the same bits every step a v that decays by a thousandth of itself would stay where it is (98 of 100 do).
__device__ __forceinline__ uint32_t salt_of(float p, float g) { return __float_as_uint(p) * kMul1 ^ __float_as_uint(g); }

// largest magnitude of a block (as bits: NaN above infinity above the rest) -> its scale byte
__device__ __forceinline__ int scale_of(uint32_t top) {
  const int e = (int)(top >> 23);
  return e < kScaleMin ? kScaleMin : e;
}
// the largest over the 16 lanes that hold a block
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t x) {
  return max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ uint32_t block_max(uint32_t x) {
  x = dpp_max<0xB1>(x);   // lane ^ 1
  x = dpp_max<0x4E>(x);   // lane ^ 2
  x = dpp_max<0x141>(x);  // 7 - lane of 8
  return dpp_max<0x140>(x);  // 15 - lane of 16
}

__device__ __forceinline__ uint32_t code_of(float size, int shift, uint32_t r20) {
  return (__float_as_uint(ldexpf(size, shift)) + r20) >> 20;
}
__device__ __forceinline__ uint32_t code_m(float x, int s, uint32_t r20) {
  return code_of(fabsf(x), 14 - s, r20) | (__float_as_uint(x) >> 24 & 0x80u);
}
__device__ __forceinline__ uint32_t code_v(float x, int s, uint32_t r20) {
  const uint32_t c = code_of(x, 30 - s, r20);
  return c ? c : x > 0.f;
}
__device__ __forceinline__ float value_m(uint32_t c, int s) {
  const float x = __uint_as_float((c & 0x7Fu) << 20 | (c & 0x80u) << 24);
  return s == 255 ? __uint_as_float(0x7FC00000u) : ldexpf(x, s - 14);
}
__device__ __forceinline__ float value_v(uint32_t c, int s) {
  return s == 255 ? __uint_as_float(0x7FC00000u) : ldexpf(__uint_as_float(c << 20), s - 30);
}

// ------------------------------------------------------------------ four elements of a thread
constexpr int kEach = 4;                               // elements of a piece
constexpr int kPieces = kChunk / (kThreads * kEach);   // of a thread in a whole chunk
static_assert(kBlock == 16 * kEach && kPieces * kThreads * kEach == kChunk, "16 lanes hold a block");

// pieces of the tensors at any address of their type
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32_any __attribute__((aligned(1)));

template <typename T>
struct Four;  // T x 4 as they are loaded
template <>
struct Four<float> {
  f32x4 w;
};
template <>
struct Four<__bf16> {
  u32x2 w;
};
template <>
struct Four<_Float16> {
  u32x2 w;
};
template <>
struct Four<uint8_t> {
  uint32_t w;
};

// elements i .. i + 3 of p (EDGE: those before n, 0 behind)
template <bool EDGE, bool STREAM, typename T>
__device__ __forceinline__ Four<T> get(const T* p, int i, int n) {
  Four<T> r;
  if (!EDGE || i + kEach <= n) {
    if constexpr (sizeof(T) == 4)
      r.w = STREAM ? __builtin_nontemporal_load((const f32x4_any*)(p + i)) : *(const f32x4_any*)(p + i);
    else if constexpr (sizeof(T) == 2)
      r.w = STREAM ? __builtin_nontemporal_load((const u32x2_any*)(p + i)) : *(const u32x2_any*)(p + i);
    else
      r.w = STREAM ? __builtin_nontemporal_load((const u32_any*)(p + i)) : *(const u32_any*)(p + i);
  } else {
    T e[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) e[j] = i + j < n ? p[i + j] : (T)0;
    __builtin_memcpy(&r.w, e, sizeof(e));
  }
  return r;
}

template <bool EDGE, bool STREAM, typename T>
__device__ __forceinline__ void put(T* p, int i, int n, const Four<T>& r) {
  if (!EDGE || i + kEach <= n) {
    if constexpr (sizeof(T) == 4) {
      if (STREAM)
        __builtin_nontemporal_store(r.w, (f32x4_any*)(p + i));
      else
        *(f32x4_any*)(p + i) = r.w;
    } else if constexpr (sizeof(T) == 2) {
      *(u32x2_any*)(p + i) = r.w;
    } else {
      *(u32_any*)(p + i) = r.w;  // (codes: a quarter of the bytes of what they stand for may stay in the cache)
    }
  } else {
    T e[kEach];
    __builtin_memcpy(e, &r.w, sizeof(e));
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (i + j < n) p[i + j] = e[j];
  }
}

template <typename T>
__device__ __forceinline__ void as_floats(const Four<T>& r, float (&v)[kEach]) {
  T e[kEach];
  __builtin_memcpy(e, &r.w, sizeof(e));
#pragma unroll
  for (int j = 0; j < kEach; ++j) v[j] = (float)e[j];
}

// four codes -> values and back
__device__ __forceinline__ void decode(uint32_t cm, uint32_t cv, int sm, int sv, float (&m)[kEach], float (&v)[kEach]) {
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    m[j] = value_m(cm >> (8 * j) & 0xFFu, sm);
    v[j] = value_v(cv >> (8 * j) & 0xFFu, sv);
  }
}

// (a whole block's 16 lanes call it; what lies behind a tensor's end is 0 and raises no scale)
template <bool RANDOM>
__device__ __forceinline__ void encode(const float (&m)[kEach], const float (&v)[kEach], uint2 key,
                                       const uint32_t (&index)[kEach], Four<uint8_t>& cm, Four<uint8_t>& cv, int& sm,
                                       int& sv) {
  uint32_t am = 0, av = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    am = max(am, __float_as_uint(m[j]) & 0x7FFFFFFFu);
    av = max(av, __float_as_uint(v[j]) & 0x7FFFFFFFu);
  }
  sm = scale_of(block_max(am));
  sv = scale_of(block_max(av));
  cm.w = cv.w = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    uint32_t rm = 1u << 19, rv = 1u << 19;
    if (RANDOM) {
      const uint32_t r = random_bits(key, index[j]);
      rm = ((r & 0xFFFFu) << 4) + 8u;
      rv = ((r >> 16) << 4) + 8u;
    }
    cm.w |= (code_m(m[j], sm, rm) & 0xFFu) << (8 * j);
    cv.w |= (code_v(v[j], sv, rv) & 0xFFu) << (8 * j);
  }
}

// ------------------------------------------------------------------ the step
// The pieces of a thread are loaded first, all of them, then worked on one by one: with 8 blocks on a CU that keeps
// the memory busy.  EDGE: a tensor's last chunk.
template <typename T, int N, bool EDGE, bool STREAM>
__device__ __forceinline__ void step32(const Chunk& c, const Args& a, const Step& s, int first) {
  const float wd = a.lr * c.wd;
  float *m = (float*)c.m, *v = (float*)c.v;
  Four<float> p4[N], m4[N], v4[N];
  Four<T> g4[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int i = first + k * kThreads * kEach;
    p4[k] = get<EDGE, STREAM>(c.p, i, c.count);
    g4[k] = get<EDGE, STREAM>((const T*)c.g, i, c.count);
    m4[k] = get<EDGE, STREAM>(m, i, c.count);
    v4[k] = get<EDGE, STREAM>(v, i, c.count);
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int i = first + k * kThreads * kEach;
    float g[kEach];
    as_floats(g4[k], g);
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      float mj = m4[k].w[j], vj = v4[k].w[j];
      p4[k].w[j] = update(p4[k].w[j], g[j], mj, vj, a, s, wd);
      m4[k].w[j] = mj;
      v4[k].w[j] = vj;
    }
    put<EDGE, STREAM>(c.p, i, c.count, p4[k]);
    put<EDGE, STREAM>(m, i, c.count, m4[k]);
    put<EDGE, STREAM>(v, i, c.count, v4[k]);
  }
}

template <typename T, int N, bool EDGE, bool STREAM>
__device__ __forceinline__ void step8(const Chunk& c, const Args& a, const Step& s, int first) {
  const float wd = a.lr * c.wd;
  const uint2 key = keys_of(a, s.t, c.tensor, c.start);
  uint8_t *m = (uint8_t*)c.m, *v = (uint8_t*)c.v;
  Four<float> p4[N];
  Four<T> g4[N];
  Four<uint8_t> m4[N], v4[N];
  int sm[N], sv[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int i = first + k * kThreads * kEach;
    p4[k] = get<EDGE, STREAM>(c.p, i, c.count);
    g4[k] = get<EDGE, STREAM>((const T*)c.g, i, c.count);
    m4[k] = get<EDGE, STREAM>(m, i, c.count);
    v4[k] = get<EDGE, STREAM>(v, i, c.count);
    const bool in = !EDGE || i < c.count;  // (its block lies in the tensor)
    sm[k] = in ? c.sm[i / kBlock] : 0;
    sv[k] = in ? c.sv[i / kBlock] : 0;
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int i = first + k * kThreads * kEach;
    float g[kEach], mj[kEach], vj[kEach];
    uint32_t index[kEach];
    as_floats(g4[k], g);
    decode(m4[k].w, v4[k].w, sm[k], sv[k], mj, vj);
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      p4[k].w[j] = update(p4[k].w[j], g[j], mj[j], vj[j], a, s, wd);
      index[j] = (uint32_t)(c.start + i + j);
      if (EDGE && i + j >= c.count) mj[j] = vj[j] = 0.f;  // (a block of NaN is NaN behind the end too)
    }
    if (s.past) {
#pragma unroll
      for (int j = 0; j < kEach; ++j) index[j] ^= salt_of(p4[k].w[j], g[j]);
    }
    put<EDGE, STREAM>(c.p, i, c.count, p4[k]);
    encode<true>(mj, vj, key, index, m4[k], v4[k], sm[k], sv[k]);
    put<EDGE, STREAM>(m, i, c.count, m4[k]);
    put<EDGE, STREAM>(v, i, c.count, v4[k]);
    if ((threadIdx.x & 15) == 0 && (!EDGE || i < c.count)) {
      c.sm[i / kBlock] = (uint8_t)sm[k];
      c.sv[i / kBlock] = (uint8_t)sv[k];
    }
  }
}

template <typename T, int BITS, bool STREAM>
__device__ __forceinline__ void step_chunk(const Chunk& c, const Args& a, const Step& s) {
  const int mine = (int)threadIdx.x * kEach;
  if (c.count == kChunk) {
    if constexpr (BITS == 32)
      step32<T, kPieces, false, STREAM>(c, a, s, mine);
    else
      step8<T, kPieces, false, STREAM>(c, a, s, mine);
  } else {
    if constexpr (BITS == 32)
      step32<T, kPieces, true, STREAM>(c, a, s, mine);
    else
      step8<T, kPieces, true, STREAM>(c, a, s, mine);
  }
}

template <int BITS, bool STREAM>
__global__ __launch_bounds__(kThreads) void adamw_kernel(const Chunk* __restrict__ chunks, Args a) {
  const Chunk c = chunks[blockIdx.x];
  const Step s = step_of(a);
  if (c.gtype == XDFM_F32)
    step_chunk<float, BITS, STREAM>(c, a, s);
  else if (c.gtype == XDFM_BF16)
    step_chunk<__bf16, BITS, STREAM>(c, a, s);
  else
    step_chunk<_Float16, BITS, STREAM>(c, a, s);
}

// Eight elements a thread: 16 bytes of each output, past the caches (it goes to a checkpoint; a table of 25.3 M, step
// and read-out: 98 -> 91 us).
template <bool EDGE, int N>
__device__ __forceinline__ void read_pieces(const Chunk& c, __bf16* out_m, __bf16* out_v, int first) {
  constexpr int kStep = 2 * kThreads * kEach;
  Four<uint8_t> m4[N][2], v4[N][2];
  int sm[N], sv[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int i = first + k * kStep;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      m4[k][h] = get<EDGE, false>((const uint8_t*)c.m, i + h * kEach, c.count);
      v4[k][h] = get<EDGE, false>((const uint8_t*)c.v, i + h * kEach, c.count);
    }
    sm[k] = c.sm[i / kBlock];
    sv[k] = c.sv[i / kBlock];
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int i = first + k * kStep;
    __bf16 em[2 * kEach], ev[2 * kEach];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float m[kEach], v[kEach];
      decode(m4[k][h].w, v4[k][h].w, sm[k], sv[k], m, v);
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        em[h * kEach + j] = (__bf16)m[j];
        ev[h * kEach + j] = (__bf16)v[j];
      }
    }
    if (!EDGE || i + 2 * kEach <= c.count) {
      u32x4 wm, wv;
      __builtin_memcpy(&wm, em, sizeof(em));
      __builtin_memcpy(&wv, ev, sizeof(ev));
      __builtin_nontemporal_store(wm, (u32x4_any*)(out_m + i));
      __builtin_nontemporal_store(wv, (u32x4_any*)(out_v + i));
    } else {
#pragma unroll
      for (int j = 0; j < 2 * kEach; ++j)
        if (i + j < c.count) {
          out_m[i + j] = em[j];
          out_v[i + j] = ev[j];
        }
    }
  }
}

__global__ __launch_bounds__(kThreads) void adamw_state_read_kernel(const Chunk* __restrict__ chunks, __bf16* out_m,
                                                                    __bf16* out_v) {
  const Chunk c = chunks[blockIdx.x];
  const int mine = (int)threadIdx.x * 2 * kEach;
  out_m += c.out;
  out_v += c.out;
  if (c.count == kChunk)
    read_pieces<false, kPieces / 2>(c, out_m, out_v, mine);
  else
    for (int i = mine; i < c.count; i += 2 * kThreads * kEach) read_pieces<true, 1>(c, out_m, out_v, i);
}

__global__ __launch_bounds__(kThreads) void adamw_state_write_kernel(const Chunk* __restrict__ chunks,
                                                                     const float* __restrict__ in_m,
                                                                     const float* __restrict__ in_v) {
  const Chunk c = chunks[blockIdx.x];
  for (int first = 0; first < c.count; first += kThreads * kEach) {
    const int i = first + (int)threadIdx.x * kEach;
    float m[kEach], v[kEach];
    as_floats(get<true, false>(in_m + c.out, i, c.count), m);
    as_floats(get<true, false>(in_v + c.out, i, c.count), v);
    Four<uint8_t> m4, v4;
    int sm, sv;
    encode<false>(m, v, make_uint2(0, 0), {0u, 0u, 0u, 0u}, m4, v4, sm, sv);
    put<true, false>((uint8_t*)c.m, i, c.count, m4);
    put<true, false>((uint8_t*)c.v, i, c.count, v4);
    if ((threadIdx.x & 15) == 0 && i < c.count) {
      c.sm[i / kBlock] = (uint8_t)sm;
      c.sv[i / kBlock] = (uint8_t)sv;
    }
  }
}

struct Range {
  uintptr_t beg, end;
  int tensor;
};

// every range that is written lies apart from every other one, and from those that are read
int check_apart(const xdfm_adamw_tensor* t, int n, int bits) {
  std::vector<Range> written, read;
  const size_t size = bits == 32 ? 4 : 1;
  auto put = [](std::vector<Range>& to, const void* p, size_t bytes, int k) {
    to.push_back({(uintptr_t)p, (uintptr_t)p + bytes, k});
  };
  for (int k = 0; k < n; ++k) {
    if (t[k].n == 0) continue;
    const size_t e = (size_t)t[k].n, blocks = (e + kBlock - 1) / kBlock;
    put(written, t[k].param, 4 * e, k);
    put(written, t[k].slot_m, size * e, k);
    put(written, t[k].slot_v, size * e, k);
    if (bits == 8) {
      put(written, t[k].scale_m, blocks, k);
      put(written, t[k].scale_v, blocks, k);
    }
    put(read, t[k].grad, (t[k].grad_dtype == XDFM_F32 ? 4 : 2) * e, k);
  }
  auto before = [](const Range& x, const Range& y) { return x.beg < y.beg; };
  std::sort(written.begin(), written.end(), before);
  for (size_t i = 1; i < written.size(); ++i)
    XDFM_REQUIRE(written[i - 1].end <= written[i].beg, "xdfm_adamw_plan: tensors %d and %d overlap where they are written",
                 written[i - 1].tensor, written[i].tensor);
  for (const Range& r : read) {
    auto after = std::lower_bound(written.begin(), written.end(), r, before);
    XDFM_REQUIRE(after == written.end() || r.end <= after->beg, "xdfm_adamw_plan: the gradient of tensor %d lies in what "
                 "the step writes of tensor %d", r.tensor, after->tensor);
    XDFM_REQUIRE(after == written.begin() || (after - 1)->end <= r.beg, "xdfm_adamw_plan: the gradient of tensor %d lies "
                 "in what the step writes of tensor %d", r.tensor, (after - 1)->tensor);
  }
  return XDFM_OK;
}

int make_plan(const xdfm_adamw_tensor* t, int n, int bits, Chunk* image, xdfm_adamw_plan_info* info) {
  int64_t chunks = 0, out = 0;
  for (int k = 0; k < n; ++k) {
    const xdfm_adamw_tensor& x = t[k];
    XDFM_REQUIRE(x.n >= 0 && x.n <= (int64_t)1 << 44, "xdfm_adamw_plan: tensor %d has %lld elements", k, (long long)x.n);
    XDFM_REQUIRE(x.grad_dtype == XDFM_F32 || x.grad_dtype == XDFM_BF16 || x.grad_dtype == XDFM_F16,
                 "xdfm_adamw_plan: tensor %d: unknown gradient type %d", k, x.grad_dtype);
    XDFM_REQUIRE(x.weight_decay >= 0.f && std::isfinite(x.weight_decay),
                 "xdfm_adamw_plan: tensor %d: weight_decay has to be finite and not negative", k);
    if (x.n == 0) continue;
    XDFM_REQUIRE(x.param && x.grad && x.slot_m && x.slot_v, "xdfm_adamw_plan: tensor %d: null argument", k);
    XDFM_REQUIRE(bits == 32 || (x.scale_m && x.scale_v), "xdfm_adamw_plan: tensor %d: 8-bit states need their scales", k);
    XDFM_REQUIRE(bits == 8 || (!x.scale_m && !x.scale_v), "xdfm_adamw_plan: tensor %d: 32-bit states have no scales", k);
    XDFM_REQUIRE(((uintptr_t)x.param & 3) == 0 && ((uintptr_t)x.grad & (x.grad_dtype == XDFM_F32 ? 3 : 1)) == 0 &&
                     (bits == 8 || (((uintptr_t)x.slot_m | (uintptr_t)x.slot_v) & 3) == 0),
                 "xdfm_adamw_plan: tensor %d: misaligned pointer", k);
    const int gsize = x.grad_dtype == XDFM_F32 ? 4 : 2, ssize = bits == 32 ? 4 : 1;
    for (int64_t at = 0; at < x.n; at += kChunk, ++chunks) {
      if (!image) {
        const int64_t more = (x.n - 1) / kChunk;  // counted, not walked
        chunks += more;
        at += more * kChunk;
        continue;
      }
      Chunk& c = image[chunks];
      c.p = x.param + at;
      c.g = (const char*)x.grad + at * gsize;
      c.m = (char*)x.slot_m + at * ssize;
      c.v = (char*)x.slot_v + at * ssize;
      c.sm = x.scale_m ? x.scale_m + at / kBlock : nullptr;
      c.sv = x.scale_v ? x.scale_v + at / kBlock : nullptr;
      c.start = at;
      c.out = out + at;
      c.count = (int32_t)std::min<int64_t>(kChunk, x.n - at);
      c.tensor = k;
      c.wd = x.weight_decay;
      c.gtype = x.grad_dtype;
    }
    out += x.n;
    XDFM_REQUIRE(chunks <= kMostChunks, "xdfm_adamw_plan: too many elements (more than %lld chunks of %d)",
                 (long long)kMostChunks, kChunk);
  }
  info->bytes = chunks * (int64_t)sizeof(Chunk);
  info->chunks = chunks;
  info->elements = out;
  info->state_bits = bits;
  info->chunk_elems = kChunk;
  return XDFM_OK;
}

int check_plan(const char* who, const void* plan, const xdfm_adamw_plan_info* info) {
  XDFM_REQUIRE(info, "%s: null argument", who);
  XDFM_REQUIRE((info->state_bits == 32 || info->state_bits == 8) && info->chunk_elems == kChunk && info->chunks >= 0 &&
                   info->chunks <= kMostChunks && info->bytes == info->chunks * (int64_t)sizeof(Chunk),
               "%s: *info is not what xdfm_adamw_plan gave", who);
  XDFM_REQUIRE(info->chunks == 0 || plan, "%s: null argument", who);
  XDFM_REQUIRE(((uintptr_t)plan & 7) == 0, "%s: misaligned plan", who);
  return XDFM_OK;
}

}  // namespace

extern "C" int xdfm_adamw_plan(const xdfm_adamw_tensor* tensors, int32_t n_tensors, int32_t state_bits, void* image,
                               size_t image_bytes, xdfm_adamw_plan_info* info) {
  XDFM_REQUIRE(info && n_tensors >= 0 && (tensors || n_tensors == 0), "xdfm_adamw_plan: bad argument");
  XDFM_REQUIRE(state_bits == 32 || state_bits == 8, "xdfm_adamw_plan: states have 32 or 8 bits, not %d", state_bits);
  XDFM_REQUIRE(((uintptr_t)image & 7) == 0, "xdfm_adamw_plan: misaligned image");
  try {
    int rc = make_plan(tensors, n_tensors, state_bits, nullptr, info);
    if (!rc) rc = check_apart(tensors, n_tensors, state_bits);
    if (rc || !image) return rc;
    if (image_bytes < (size_t)info->bytes)
      return xdfm::fail(XDFM_E_WORKSPACE, "xdfm_adamw_plan: the image takes %lld bytes", (long long)info->bytes);
    return make_plan(tensors, n_tensors, state_bits, (Chunk*)image, info);
  } catch (const std::exception& e) {
    return xdfm::fail(XDFM_E_INVALID, "xdfm_adamw_plan: %s", e.what());
  }
}

extern "C" int xdfm_adamw_step(const void* plan, const xdfm_adamw_plan_info* info, const xdfm_adamw_args* args,
                               void* stream) {
  const int rc = check_plan("xdfm_adamw_step", plan, info);
  if (rc) return rc;
  XDFM_REQUIRE(args, "xdfm_adamw_step: null argument");
  // (lr / (1 - beta1^t) stays finite in 32 bits: 1 - beta1 is 2^-53 at least)
  XDFM_REQUIRE(args->lr >= 0 && args->lr <= 1e20, "xdfm_adamw_step: lr has to lie in [0, 1e20]");
  XDFM_REQUIRE(args->beta1 >= 0 && args->beta1 < 1 && args->beta2 >= 0 && args->beta2 < 1,
               "xdfm_adamw_step: beta1 and beta2 have to lie in [0, 1)");
  XDFM_REQUIRE(args->eps >= 1e-30 && args->eps <= 1e30, "xdfm_adamw_step: eps has to lie in [1e-30, 1e30]");
  XDFM_REQUIRE(args->opt_state || args->step >= 1, "xdfm_adamw_step: steps count from 1");
  if (info->chunks == 0) return XDFM_OK;
  Args a;
  a.lr = (float)args->lr;
  a.b1 = (float)args->beta1;
  a.omb1 = (float)(1.0 - args->beta1);
  a.b2 = (float)args->beta2;
  a.omb2 = (float)(1.0 - args->beta2);
  a.eps = (float)args->eps;
  a.log_b1 = (float)std::log(args->beta1);
  a.log_b2 = (float)std::log(args->beta2);
  a.state = args->opt_state;
  a.step = a.inv_root = 0.f;
  a.t = 0;
  if (!a.state) {
    const double t = (double)args->step;
    a.step = (float)(args->lr / (1.0 - std::pow(args->beta1, t)));
    a.inv_root = (float)(1.0 / std::sqrt(1.0 - std::pow(args->beta2, t)));
    a.t = (uint32_t)args->step;
  }
  a.seed_lo = (uint32_t)args->seed;
  a.seed_hi = (uint32_t)(args->seed >> 32);
  const dim3 grid((unsigned)info->chunks);
  // past the caches (kept codes apart) where a step moves more than the Infinity Cache holds: table of 25.3 M 119 against
  // 135 us; the next step of 6.0 M elements (169 MB) still finds some of it there, 28.9 against 31.7
  const bool stream_by = (double)info->elements * (info->state_bits == 32 ? 28 : 16) > 256e6;
  if (info->state_bits == 32 && stream_by)
    XDFM_LAUNCH("adamw_kernel", stream, (adamw_kernel<32, true>), grid, dim3(kThreads), 0, (const Chunk*)plan, a);
  else if (info->state_bits == 32)
    XDFM_LAUNCH("adamw_kernel", stream, (adamw_kernel<32, false>), grid, dim3(kThreads), 0, (const Chunk*)plan, a);
  else if (stream_by)
    XDFM_LAUNCH("adamw8_kernel", stream, (adamw_kernel<8, true>), grid, dim3(kThreads), 0, (const Chunk*)plan, a);
  else
    XDFM_LAUNCH("adamw8_kernel", stream, (adamw_kernel<8, false>), grid, dim3(kThreads), 0, (const Chunk*)plan, a);
  XDFM_LAUNCH_CHECK();
  return XDFM_OK;
}

extern "C" int xdfm_adamw_state_read(const void* plan, const xdfm_adamw_plan_info* info, uint16_t* m, uint16_t* v,
                                     void* stream) {
  const int rc = check_plan("xdfm_adamw_state_read", plan, info);
  if (rc) return rc;
  XDFM_REQUIRE(info->state_bits == 8, "xdfm_adamw_state_read: 32-bit states are values as they stand");
  if (info->chunks == 0) return XDFM_OK;
  XDFM_REQUIRE(m && v && (((uintptr_t)m | (uintptr_t)v) & 1) == 0, "xdfm_adamw_state_read: null or misaligned output");
  XDFM_LAUNCH("adamw_state_read_kernel", stream, adamw_state_read_kernel, dim3((unsigned)info->chunks), dim3(kThreads),
              0, (const Chunk*)plan, (__bf16*)m, (__bf16*)v);
  XDFM_LAUNCH_CHECK();
  return XDFM_OK;
}

extern "C" int xdfm_adamw_state_write(const void* plan, const xdfm_adamw_plan_info* info, const float* m,
                                      const float* v, void* stream) {
  const int rc = check_plan("xdfm_adamw_state_write", plan, info);
  if (rc) return rc;
  XDFM_REQUIRE(info->state_bits == 8, "xdfm_adamw_state_write: 32-bit states are values as they stand");
  if (info->chunks == 0) return XDFM_OK;
  XDFM_REQUIRE(m && v && (((uintptr_t)m | (uintptr_t)v) & 3) == 0, "xdfm_adamw_state_write: null or misaligned input");
  XDFM_LAUNCH("adamw_state_write_kernel", stream, adamw_state_write_kernel, dim3((unsigned)info->chunks),
              dim3(kThreads), 0, (const Chunk*)plan, m, v);
  XDFM_LAUNCH_CHECK();
  return XDFM_OK;
}
