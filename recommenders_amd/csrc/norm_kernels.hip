// Layer norm of matrix rows with the activation behind it, forward and backward (enable_LN branch of the DNN tower).
//
//   xhat = (x - mean) rstd,  u = gamma xhat + beta,  y = act(u)
//   du = dy act'(u),  t = du gamma,  dx = rstd (t - mean(t) - xhat mean(t xhat)),
//   dgamma = sum_rows du xhat,  dbeta = sum_rows du
#include <hip/hip_runtime.h>

#include "act.h"
#include "xdfm_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// sum over the block, the same in every thread, in an order that does not depend on timing
__device__ __forceinline__ float block_total(float v, float* sh) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) s += sh[w];
  return s;
}

// act'(u).  relu: 32 bits lose the sign of u where gamma xhat and beta nearly cancel (three roundings of
// 2^-24 of |beta|); there it is taken from 64 bits.
__device__ __forceinline__ float slope(float u, int act, float x, float mean, float rstd, float g, float b) {
  switch (act) {
    case XDFM_ACT_RELU:
      if (fabsf(u) <= 6e-7f * fabsf(b))
        return ((double)x - (double)mean) * (double)rstd * (double)g + (double)b > 0.0 ? 1.f : 0.f;
      return u > 0.f ? 1.f : 0.f;
    case XDFM_ACT_SIGMOID: {
      const float s = 1.f / (1.f + expf(-u));
      return s * (1.f - s);
    }
    case XDFM_ACT_TANH: {
      const float t = tanhf(u);
      return 1.f - t * t;
    }
    case XDFM_ACT_ELU: return u > 0.f ? 1.f : expf(u);
    default: return 1.f;
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void layer_norm_fwd_kernel(const T* x, int64_t xs, int64_t rows, int cols,
                                                                  const float* __restrict__ gamma,
                                                                  const float* __restrict__ beta, float eps, int act,
                                                                  T* y, int64_t ys, float* __restrict__ stats) {
  __shared__ float sh[kWaves];
  const float n = (float)cols;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * xs;
    T* yr = y + r * ys;
    float s = 0.f;
    for (int c = threadIdx.x; c < cols; c += kThreads) s += (float)xr[c];
    const float mean = block_total(s, sh) / n;
    float q = 0.f;
    for (int c = threadIdx.x; c < cols; c += kThreads) {
      const float d = (float)xr[c] - mean;
      q += d * d;
    }
    const float rstd = 1.f / sqrtf(block_total(q, sh) / n + eps);
    for (int c = threadIdx.x; c < cols; c += kThreads) {
      const float xhat = ((float)xr[c] - mean) * rstd;
      yr[c] = (T)activate(xhat * gamma[c] + beta[c], act);
    }
    if (stats && threadIdx.x == 0) {
      stats[r] = mean;
      stats[rows + r] = rstd;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void layer_norm_bwd_dx_kernel(const T* x, int64_t xs, const T* dy, int64_t dys,
                                                                     int64_t rows, int cols,
                                                                     const float* __restrict__ gamma,
                                                                     const float* __restrict__ beta,
                                                                     const float* __restrict__ stats, int act, T* dx,
                                                                     int64_t dxs) {
  __shared__ float sh[kWaves];
  const float n = (float)cols;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float mean = stats[r], rstd = stats[rows + r];
    float a = 0.f, b = 0.f;
    for (int c = threadIdx.x; c < cols; c += kThreads) {
      const float xv = (float)x[r * xs + c], xhat = (xv - mean) * rstd;
      const float du = (float)dy[r * dys + c] *
                       slope(xhat * gamma[c] + beta[c], act, xv, mean, rstd, gamma[c], beta[c]);
      a += du * gamma[c];
      b += du * gamma[c] * xhat;
    }
    a = block_total(a, sh) / n;
    b = block_total(b, sh) / n;
    for (int c = threadIdx.x; c < cols; c += kThreads) {
      const float xv = (float)x[r * xs + c], xhat = (xv - mean) * rstd;
      const float du = (float)dy[r * dys + c] *
                       slope(xhat * gamma[c] + beta[c], act, xv, mean, rstd, gamma[c], beta[c]);
      dx[r * dxs + c] = (T)(rstd * (du * gamma[c] - a - xhat * b));
    }
  }
}

// part[0][p][c] = sum of du xhat, part[1][p][c] = sum of du over rows p, p + parts, ...
template <typename T>
__global__ __launch_bounds__(kThreads) void layer_norm_bwd_sums_kernel(const T* x, int64_t xs, const T* dy, int64_t dys,
                                                                       int64_t rows, int cols,
                                                                       const float* __restrict__ gamma,
                                                                       const float* __restrict__ beta,
                                                                       const float* __restrict__ stats, int act,
                                                                       int parts, float* __restrict__ part) {
  const int c = blockIdx.x * kThreads + threadIdx.x, p = blockIdx.y;
  if (c >= cols) return;
  const float g = gamma[c], b = beta[c];
  float sg = 0.f, sb = 0.f;
  for (int64_t r = p; r < rows; r += parts) {
    const float mean = stats[r], rstd = stats[rows + r];
    const float xv = (float)x[r * xs + c], xhat = (xv - mean) * rstd;
    const float du = (float)dy[r * dys + c] * slope(xhat * g + b, act, xv, mean, rstd, g, b);
    sg += du * xhat;
    sb += du;
  }
  part[(int64_t)p * cols + c] = sg;
  part[(int64_t)(parts + p) * cols + c] = sb;
}

__global__ __launch_bounds__(kThreads) void layer_norm_bwd_finish_kernel(const float* __restrict__ part, int parts,
                                                                         int cols, float* __restrict__ dgamma,
                                                                         float* __restrict__ dbeta) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= cols) return;
  float sg = 0.f, sb = 0.f;
  for (int p = 0; p < parts; ++p) {
    sg += part[(int64_t)p * cols + c];
    sb += part[(int64_t)(parts + p) * cols + c];
  }
  dgamma[c] = sg;
  dbeta[c] = sb;
}

int bwd_parts(int64_t rows) { return (int)(rows < 64 ? 1 : rows < 16384 ? rows / 64 : 256); }

bool act_ok(int act) { return act >= XDFM_ACT_IDENTITY && act <= XDFM_ACT_ELU; }
bool dtype_ok(int t) { return t == XDFM_F32 || t == XDFM_BF16 || t == XDFM_F16; }
bool aligned(const void* p, int dtype) { return ((uintptr_t)p & (dtype == XDFM_F32 ? 3 : 1)) == 0; }

// rows * stride elements have to be addressable
bool extent_ok(int64_t rows, int64_t stride, int cols) {
  return rows >= 0 && cols > 0 && stride >= cols && rows <= (INT64_MAX / 8) / stride;
}

unsigned row_grid(int64_t rows) { return (unsigned)(rows < (1 << 16) ? rows : (1 << 16)); }

template <typename T>
void fwd(const void* x, int64_t xs, int64_t rows, int cols, const float* gamma, const float* beta, float eps, int act,
         void* y, int64_t ys, float* stats, hipStream_t st) {
  XDFM_LAUNCH("layer_norm_fwd_kernel", st, layer_norm_fwd_kernel<T>, dim3(row_grid(rows)), dim3(kThreads), 0,
              (const T*)x, xs, rows, cols, gamma, beta, eps, act, (T*)y, ys, stats);
}

template <typename T>
void bwd(const void* x, int64_t xs, const void* dy, int64_t dys, int64_t rows, int cols, const float* gamma,
         const float* beta, const float* stats, int act, void* dx, int64_t dxs, float* ws, hipStream_t st) {
  const int parts = bwd_parts(rows);
  // (the sums first: dx may be dy)
  XDFM_LAUNCH("layer_norm_bwd_sums_kernel", st, layer_norm_bwd_sums_kernel<T>,
              dim3((unsigned)((cols + kThreads - 1) / kThreads), (unsigned)parts), dim3(kThreads), 0, (const T*)x, xs,
              (const T*)dy, dys, rows, cols, gamma, beta, stats, act, parts, ws);
  if (rows)
    XDFM_LAUNCH("layer_norm_bwd_dx_kernel", st, layer_norm_bwd_dx_kernel<T>, dim3(row_grid(rows)), dim3(kThreads), 0,
                (const T*)x, xs, (const T*)dy, dys, rows, cols, gamma, beta, stats, act, (T*)dx, dxs);
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
  XDFM_REQUIRE(floats && rows >= 0 && cols > 0, "xdfm_layer_norm_bwd_workspace_floats: bad argument");
  *floats = (size_t)2 * bwd_parts(rows) * cols;
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
  if (dtype == XDFM_F32)
    bwd<float>(x, x_stride, dy, dy_stride, rows, cols, gamma, beta, stats, act, dx, dx_stride, workspace, st);
  else if (dtype == XDFM_BF16)
    bwd<__bf16>(x, x_stride, dy, dy_stride, rows, cols, gamma, beta, stats, act, dx, dx_stride, workspace, st);
  else
    bwd<_Float16>(x, x_stride, dy, dy_stride, rows, cols, gamma, beta, stats, act, dx, dx_stride, workspace, st);
  XDFM_LAUNCH("layer_norm_bwd_finish_kernel", st, layer_norm_bwd_finish_kernel,
              dim3((unsigned)((cols + kThreads - 1) / kThreads)), dim3(kThreads), 0, workspace, bwd_parts(rows), cols,
              dgamma, dbeta);
  XDFM_LAUNCH_CHECK();
  return XDFM_OK;
}
