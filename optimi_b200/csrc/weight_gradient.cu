// The weight gradient of a linear layer whose input is held in 8 bits:
//     dW[o, c] = w[c] * sum_t dY[t, o] * X[t, c]        X = code * 2^(e - 127)  (format: activation_common.cuh)
#include "activation_common.cuh"

namespace optimi {
namespace act {

constexpr int kTile = 64, kTokens = 16;

template <typename T>
__global__ void __launch_bounds__(256) weight_gradient_kernel(const T* __restrict__ grad, int64_t gs, const int8_t* __restrict__ codes,
                                                              int64_t pitch, const uint8_t* __restrict__ exponents, int64_t epitch,
                                                              const T* __restrict__ channel_scale, int64_t rows, int64_t outputs,
                                                              int64_t channels, T* __restrict__ dw) {
  __shared__ float a[kTokens][kTile], b[kTokens][kTile];
  const int64_t o0 = (int64_t)blockIdx.x * kTile, c0 = (int64_t)blockIdx.y * kTile;
  const int to = threadIdx.x / 16 * 4, tc = threadIdx.x % 16 * 4;
  float acc[4][4] = {};
  for (int64_t t0 = 0; t0 < rows; t0 += kTokens) {
    __syncthreads();
    for (int i = threadIdx.x; i < kTokens * kTile; i += 256) {
      const int64_t t = t0 + i / kTile, o = o0 + i % kTile, c = c0 + i % kTile;
      a[i / kTile][i % kTile] = t < rows && o < outputs ? to_f32(grad[t * gs + o]) : 0.0f;
      b[i / kTile][i % kTile] = t < rows && c < channels ? (float)codes[t * pitch + c] * power_of(exponents[t * epitch + c / kGroup]) : 0.0f;
    }
    __syncthreads();
    for (int t = 0; t < kTokens; t++)
      for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) acc[i][j] = __fmaf_rn(a[t][to + i], b[t][tc + j], acc[i][j]);
  }
  for (int i = 0; i < 4; i++)
    for (int j = 0; j < 4; j++)
      if (o0 + to + i < outputs && c0 + tc + j < channels) {
        const float scale = channel_scale ? to_f32(channel_scale[c0 + tc + j]) : 1.0f;
        dw[(o0 + to + i) * channels + c0 + tc + j] = from_f32<T>(acc[i][j] * scale);
      }
}

}  // namespace act
}  // namespace optimi

using namespace optimi;
using namespace optimi::act;

extern "C" {

size_t optimi_b200_weight_gradient_workspace_bytes(int64_t rows, int64_t outputs, int64_t channels) {
  (void)rows, (void)outputs, (void)channels;
  return 0;
}

int optimi_b200_weight_gradient(const void* grad, int64_t grad_stride, const void* codes, int64_t code_pitch, const void* exponents,
                                int64_t exponent_pitch, const void* channel_scale, int64_t rows, int64_t outputs, int64_t channels,
                                int dtype, void* grad_weight, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "optimi_b200_weight_gradient";
  (void)workspace, (void)workspace_bytes;
  if (dtype != OPTIMI_BF16 && dtype != OPTIMI_F16)
    return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: dtype %d is neither bfloat16 nor float16", fn, dtype);
  if (rows < 0 || outputs < 0 || channels < 0 || rows > INT32_MAX || outputs > INT32_MAX || channels > INT32_MAX)
    return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: %lld tokens, %lld outputs, %lld channels are outside 0..2^31-1", fn, (long long)rows,
                (long long)outputs, (long long)channels);
  if (outputs == 0 || channels == 0) return OPTIMI_OK;
  if (!grad_weight) return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: grad_weight is NULL", fn);
  cudaStream_t s = (cudaStream_t)stream;
  if (rows > 0) {
    if (!grad) return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: grad is NULL", fn);
    int rc = check_codes(fn, codes, code_pitch, exponents, exponent_pitch, channels);
    if (rc != OPTIMI_OK) return rc;
  }
  const dim3 grid((unsigned)((outputs + kTile - 1) / kTile), (unsigned)((channels + kTile - 1) / kTile));
  if (grid.y > 65535) return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: %lld channels are too many", fn, (long long)channels);
  if (dtype == OPTIMI_BF16)
    weight_gradient_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>((const __nv_bfloat16*)grad, grad_stride, (const int8_t*)codes, code_pitch,
                                                               (const uint8_t*)exponents, exponent_pitch, (const __nv_bfloat16*)channel_scale,
                                                               rows, outputs, channels, (__nv_bfloat16*)grad_weight);
  else
    weight_gradient_kernel<__half><<<grid, 256, 0, s>>>((const __half*)grad, grad_stride, (const int8_t*)codes, code_pitch,
                                                        (const uint8_t*)exponents, exponent_pitch, (const __half*)channel_scale, rows, outputs,
                                                        channels, (__half*)grad_weight);
  return launched(fn);
}

}  // extern "C"
