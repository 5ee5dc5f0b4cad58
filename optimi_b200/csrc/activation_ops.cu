// Activations kept in 8 bits (format: activation_common.cuh) and the RMS norm that writes and reads them.
#include "activation_common.cuh"

namespace optimi {
namespace act {

// ---------------------------------------------------------------------------------------------
// store and restore
// ---------------------------------------------------------------------------------------------
// One warp per group: a lane holds one value, the group's largest magnitude is a warp maximum.
template <typename T>
__global__ void compress_kernel(const T* __restrict__ x, int64_t rows, int64_t cols, int64_t stride, int8_t* __restrict__ codes,
                                int64_t pitch, uint8_t* __restrict__ exponents, int64_t epitch) {
  const int lane = threadIdx.x % 32;
  const int64_t groups = (cols + kGroup - 1) / kGroup;
  for (int64_t item = (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32; item < rows * groups;
       item += (int64_t)gridDim.x * (blockDim.x / 32)) {
    const int64_t row = item / groups, group = item % groups, col = group * kGroup + lane;
    const float v = col < cols ? to_f32(x[row * stride + col]) : 0.0f;
    const int e = group_exponent<T>(__reduce_max_sync(~0u, magnitude(v)));
    codes[row * pitch + col] = (int8_t)encode(v, e);
    if (lane == 0) exponents[row * epitch + group] = (uint8_t)e;
  }
}

template <typename T>
__global__ void decompress_kernel(const int8_t* __restrict__ codes, int64_t pitch, const uint8_t* __restrict__ exponents,
                                  int64_t epitch, const T* __restrict__ channel_scale, int64_t rows, int64_t cols,
                                  T* __restrict__ out) {
  const int lane = threadIdx.x % 32;
  const int64_t groups = (cols + kGroup - 1) / kGroup;
  for (int64_t item = (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32; item < rows * groups;
       item += (int64_t)gridDim.x * (blockDim.x / 32)) {
    const int64_t row = item / groups, group = item % groups, col = group * kGroup + lane;
    if (col >= cols) continue;
    float v = __fmul_rn((float)codes[row * pitch + col], power_of(exponents[row * epitch + group]));
    if (channel_scale) v = __fmul_rn(v, to_f32(channel_scale[col]));
    out[row * cols + col] = from_f32<T>(v);
  }
}

// ---------------------------------------------------------------------------------------------
// residual addition + RMS norm
// ---------------------------------------------------------------------------------------------
//     h = round(x + r)      rstd = (mean(h^2) + eps)^-1/2      xn = h * rstd      y = round(xn * w)
// and the 8-bit form of xn (without w, so that one checkpoint serves this norm's backward pass and, with w applied to the
// columns of its result, the weight gradient of every linear layer that reads y).
template <typename F>
static __device__ __forceinline__ F block_sum(F v) {
  __shared__ F part[32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
  for (int d = 16; d > 0; d /= 2) v += __shfl_xor_sync(~0u, v, d);
  __syncthreads();  // `part` may still be read by an earlier call
  if (lane == 0) part[warp] = v;
  __syncthreads();
  v = lane < warps ? part[lane] : F(0);
  for (int d = 16; d > 0; d /= 2) v += __shfl_xor_sync(~0u, v, d);
  return v;
}

// The normalised value is held in F: fp32, and 64 bits for fp32 activations, whose gradients would show a code that a
// last-bit difference of rstd tips over.
template <typename T> struct Wide { using type = float; };
template <> struct Wide<float> { using type = double; };

template <typename T>
__global__ void rms_norm_kernel(const T* __restrict__ x, int64_t xs, const T* __restrict__ residual, int64_t rs,
                                const T* __restrict__ weight, int64_t rows, int64_t cols, double eps, T* __restrict__ y,
                                T* sum, int8_t* __restrict__ codes, int64_t pitch, uint8_t* __restrict__ exponents,
                                int64_t epitch, float* __restrict__ rstd_out) {
  using F = typename Wide<T>::type;
  const int64_t padded = (cols + kGroup - 1) / kGroup * kGroup;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    F ss = 0;
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
      float v = to_f32(x[row * xs + c]);
      if (residual) {
        const T h = from_f32<T>(__fadd_rn(v, to_f32(residual[row * rs + c])));
        sum[row * cols + c] = h;
        v = to_f32(h);
      }
      ss += (F)v * (F)v;
    }
    ss = block_sum<F>(ss);
    const F rstd = F(1) / sqrt(ss / (F)cols + (F)eps);
    if (rstd_out && threadIdx.x == 0) rstd_out[row] = (float)rstd;
    for (int64_t c = threadIdx.x; c < padded; c += blockDim.x) {
      const float h = c >= cols ? 0.0f : to_f32(residual ? sum[row * cols + c] : x[row * xs + c]);
      const F n = (F)h * rstd;
      if (c < cols) y[row * cols + c] = from_f32<T>((float)(weight ? n * (F)to_f32(weight[c]) : n));
      if (codes) {
        // whole warps walk whole groups: lane i holds column i of a group
        const F held = c >= cols ? F(0) : n;
        const int e = exponent_of<T, F>(__reduce_max_sync(~0u, magnitude(held)));
        codes[row * pitch + c] = (int8_t)encode(held, e);
        if (threadIdx.x % 32 == 0) exponents[row * epitch + c / kGroup] = (uint8_t)e;
      }
    }
  }
}

// Backward, from the 8-bit xn:  g = dy * w    m = mean(g * xn)    dx = rstd * (g - xn * m) + dsum    dw = sum over rows of dy * xn
// dw: a block adds up its rows in order into its line of the workspace, a second kernel adds up the lines in order.
template <typename T>
__global__ void rms_norm_backward_kernel(const T* __restrict__ grad, int64_t gs, const T* __restrict__ grad_sum, int64_t hs,
                                         const int8_t* __restrict__ codes, int64_t pitch, const uint8_t* __restrict__ exponents,
                                         int64_t epitch, const float* __restrict__ rstd, const T* __restrict__ weight,
                                         int64_t rows, int64_t cols, T* __restrict__ dx, float* __restrict__ lines) {
  float* line = lines ? lines + (int64_t)blockIdx.x * cols : nullptr;
  if (line)
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) line[c] = 0.0f;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    float m = 0;
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
      const float n = (float)codes[row * pitch + c] * power_of(exponents[row * epitch + c / kGroup]);
      const float g = to_f32(grad[row * gs + c]);
      m += (weight ? g * to_f32(weight[c]) : g) * n;
      if (line) line[c] = __fmaf_rn(g, n, line[c]);
    }
    if (!dx) continue;
    m = block_sum<float>(m) / (float)cols;
    const float r = rstd[row];
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
      const float n = (float)codes[row * pitch + c] * power_of(exponents[row * epitch + c / kGroup]);
      const float g = to_f32(grad[row * gs + c]) * (weight ? to_f32(weight[c]) : 1.0f);
      float d = r * (g - n * m);
      if (grad_sum) d += to_f32(grad_sum[row * hs + c]);
      dx[row * cols + c] = from_f32<T>(d);
    }
  }
}

template <typename T>
__global__ void line_sum_kernel(const float* __restrict__ lines, int n_lines, int64_t cols, T* __restrict__ out) {
  const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= cols) return;
  float s = 0;
  for (int i = 0; i < n_lines; i++) s += lines[(int64_t)i * cols + c];
  out[c] = from_f32<T>(s);
}

static inline unsigned grid_of(int64_t items, int64_t most) { return (unsigned)(items < most ? items : most); }
constexpr int kBackwardBlocks = 148 * 4;

}  // namespace act
}  // namespace optimi

using namespace optimi;
using namespace optimi::act;

#define FOR_DTYPE(dtype, call)                                  \
  do {                                                          \
    if ((dtype) == OPTIMI_F32) { using T = float; call; }       \
    else if ((dtype) == OPTIMI_BF16) { using T = __nv_bfloat16; call; } \
    else { using T = __half; call; }                            \
  } while (0)

static int check_shape(const char* fn, int64_t rows, int64_t cols, int dtype) {
  if (!known_dtype(dtype)) return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", fn, dtype);
  if (rows < 0 || cols < 0 || rows > INT32_MAX || cols > INT32_MAX)
    return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: %lld rows of %lld values are outside 0..2^31-1", fn, (long long)rows, (long long)cols);
  return OPTIMI_OK;
}

extern "C" {

int optimi_b200_compress(const void* x, int64_t x_stride, int64_t rows, int64_t cols, int dtype, void* codes, int64_t code_pitch,
                         void* exponents, int64_t exponent_pitch, void* stream) {
  const char* fn = "optimi_b200_compress";
  int rc = check_shape(fn, rows, cols, dtype);
  if (rc != OPTIMI_OK || rows == 0 || cols == 0) return rc;
  if (!x) return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: x is NULL", fn);
  rc = check_codes(fn, codes, code_pitch, exponents, exponent_pitch, cols);
  if (rc != OPTIMI_OK) return rc;
  const int64_t items = rows * (round_up(cols, kGroup) / kGroup);
  FOR_DTYPE(dtype, (compress_kernel<T><<<grid_of((items + 7) / 8, 148 * 64), 256, 0, (cudaStream_t)stream>>>(
                       (const T*)x, rows, cols, x_stride, (int8_t*)codes, code_pitch, (uint8_t*)exponents, exponent_pitch)));
  return launched(fn);
}

int optimi_b200_decompress(const void* codes, int64_t code_pitch, const void* exponents, int64_t exponent_pitch,
                           const void* channel_scale, int64_t rows, int64_t cols, int dtype, void* out, void* stream) {
  const char* fn = "optimi_b200_decompress";
  int rc = check_shape(fn, rows, cols, dtype);
  if (rc != OPTIMI_OK || rows == 0 || cols == 0) return rc;
  if (!out) return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: out is NULL", fn);
  rc = check_codes(fn, codes, code_pitch, exponents, exponent_pitch, cols);
  if (rc != OPTIMI_OK) return rc;
  const int64_t items = rows * (round_up(cols, kGroup) / kGroup);
  FOR_DTYPE(dtype, (decompress_kernel<T><<<grid_of((items + 7) / 8, 148 * 64), 256, 0, (cudaStream_t)stream>>>(
                       (const int8_t*)codes, code_pitch, (const uint8_t*)exponents, exponent_pitch, (const T*)channel_scale, rows,
                       cols, (T*)out)));
  return launched(fn);
}

int optimi_b200_rms_norm(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, const void* weight,
                         int64_t rows, int64_t cols, double eps, int dtype, void* y, void* sum, void* codes, int64_t code_pitch,
                         void* exponents, int64_t exponent_pitch, float* rstd, void* stream) {
  const char* fn = "optimi_b200_rms_norm";
  int rc = check_shape(fn, rows, cols, dtype);
  if (rc != OPTIMI_OK || rows == 0 || cols == 0) return rc;
  if (!x || !y) return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: x or y is NULL", fn);
  if ((residual != nullptr) != (sum != nullptr)) return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: residual and sum go together", fn);
  if (!(eps >= 0)) return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: eps=%g must not be negative", fn, eps);
  if (codes || exponents || rstd) {
    rc = check_codes(fn, codes, code_pitch, exponents, exponent_pitch, cols);
    if (rc != OPTIMI_OK) return rc;
    if (!rstd) return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: codes, exponents and rstd go together", fn);
  }
  FOR_DTYPE(dtype, (rms_norm_kernel<T><<<grid_of(rows, 1 << 20), 256, 0, (cudaStream_t)stream>>>(
                       (const T*)x, x_stride, (const T*)residual, residual_stride, (const T*)weight, rows, cols, eps, (T*)y, (T*)sum,
                       (int8_t*)codes, code_pitch, (uint8_t*)exponents, exponent_pitch, rstd)));
  return launched(fn);
}

size_t optimi_b200_rms_norm_backward_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return (size_t)grid_of(rows, kBackwardBlocks) * (size_t)cols * sizeof(float);
}

int optimi_b200_rms_norm_backward(const void* grad, int64_t grad_stride, const void* grad_sum, int64_t grad_sum_stride,
                                  const void* codes, int64_t code_pitch, const void* exponents, int64_t exponent_pitch,
                                  const float* rstd, const void* weight, int64_t rows, int64_t cols, int dtype, void* grad_input,
                                  void* grad_weight, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "optimi_b200_rms_norm_backward";
  int rc = check_shape(fn, rows, cols, dtype);
  if (rc != OPTIMI_OK || cols == 0) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  if (rows == 0) {
    if (!grad_weight) return OPTIMI_OK;
    cudaError_t e = cudaMemsetAsync(grad_weight, 0, (size_t)cols * (dtype == OPTIMI_F32 ? 4 : 2), s);
    return e == cudaSuccess ? OPTIMI_OK : fail(OPTIMI_ERR_CUDA, "%s: %s", fn, cudaGetErrorString(e));
  }
  if (!grad || !rstd) return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: grad or rstd is NULL", fn);
  if (!grad_input && !grad_weight) return OPTIMI_OK;
  rc = check_codes(fn, codes, code_pitch, exponents, exponent_pitch, cols);
  if (rc != OPTIMI_OK) return rc;
  const size_t need = optimi_b200_rms_norm_backward_workspace_bytes(rows, cols);
  if (grad_weight && (!workspace || workspace_bytes < need))
    return fail(OPTIMI_ERR_WORKSPACE_TOO_SMALL, "%s: workspace has %zu bytes, %zu are needed", fn, workspace ? workspace_bytes : (size_t)0, need);
  const unsigned blocks = grid_of(rows, kBackwardBlocks);
  FOR_DTYPE(dtype, (rms_norm_backward_kernel<T><<<blocks, 256, 0, s>>>(
                       (const T*)grad, grad_stride, (const T*)grad_sum, grad_sum_stride, (const int8_t*)codes, code_pitch,
                       (const uint8_t*)exponents, exponent_pitch, rstd, (const T*)weight, rows, cols, (T*)grad_input,
                       grad_weight ? (float*)workspace : nullptr)));
  rc = launched(fn);
  if (rc != OPTIMI_OK || !grad_weight) return rc;
  FOR_DTYPE(dtype, (line_sum_kernel<T><<<(unsigned)((cols + 127) / 128), 128, 0, s>>>((const float*)workspace, (int)blocks, cols, (T*)grad_weight)));
  return launched(fn);
}

}  // extern "C"
