// What the activation kernels share: the 8-bit group format, typed loads and stores, errors and launches.
//
// Format.  The last dimension of an activation is cut into groups of 32.  A group has one exponent byte e, and its
// values are code * 2^(e - 127) with int8 codes in -127..127.  e = 0 is a group of zeros; e = 255 a group that held an
// infinity or a NaN and reads back as 32 NaNs (code 0, and 0 * 2^128 = 0 * inf = NaN needs no special case: the byte is
// the exponent field of an fp32).  2^k is the smallest power of two of which the group's largest magnitude, rounded, is
// at most 127:
//     amax = m * 2^E (1 <= m < 2)    k = E - 6, one more from m = 127.5 / 64 on (127.5 rounds to 128)
// and that condition is a carry: (bits(amax) + 0x10000) >> 23 is E + 127, plus one from that m on.  k is kept in a range
// per type in which code * 2^k neither overflows nor loses bits, so a restored value is exact in the type it came from.
#pragma once
#include "../../include/optimi_b200.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <type_traits>

namespace optimi {

extern thread_local char g_error[512];                // owned by optimi_b200.cu
extern std::atomic<unsigned long long> g_launches;    // owned by optimi_b200.cu

namespace act {

constexpr int kGroup = 32;
constexpr uint32_t kCarry = 0x10000u;    // 2 - 127.5 / 64 in units of 2^-23
constexpr float kToInt = 12582912.0f;    // 1.5 * 2^23: adding it rounds to a whole number, ties to even, in the low bits

static inline int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_error, sizeof(g_error), fmt, ap);
  va_end(ap);
  return code;
}

static inline int launched(const char* fn) {
  g_launches.fetch_add(1, std::memory_order_relaxed);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? OPTIMI_OK : fail(OPTIMI_ERR_CUDA, "%s: %s", fn, cudaGetErrorString(e));
}

static inline bool known_dtype(int dtype) { return dtype == OPTIMI_F32 || dtype == OPTIMI_BF16 || dtype == OPTIMI_F16; }
static inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
static inline int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

static inline int check_codes(const char* fn, const void* codes, int64_t pitch, const void* exponents, int64_t epitch, int64_t cols) {
  if (!codes || !exponents) return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: codes or exponents is NULL", fn);
  const int64_t padded = round_up(cols, kGroup);
  if (pitch < padded || pitch % kGroup || !aligned(codes, 16))
    return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: codes need 16-byte alignment and a pitch that is a multiple of 32 and at least %lld (got %lld)",
                fn, (long long)padded, (long long)pitch);
  if (epitch < padded / kGroup)
    return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: the exponent pitch %lld is below the %lld groups of a row", fn, (long long)epitch,
                (long long)(padded / kGroup));
  return OPTIMI_OK;
}

// Smallest and largest exponent byte of a group that is neither empty nor NaN.
template <typename T> struct Range { static constexpr int low = 1, high = 248; };        // fp32, bf16: k -126..121
template <> struct Range<__half> { static constexpr int low = 103, high = 136; };         // fp16: k -24..9

static __device__ __forceinline__ float to_f32(float x) { return x; }
static __device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
static __device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <typename T> static __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

static __device__ __forceinline__ float power_of(int e) { return __uint_as_float((uint32_t)e << 23); }  // 2^(e - 127)

// The exponent byte for a group whose largest magnitude has these fp32 bits.
template <typename T>
static __device__ __forceinline__ int group_exponent(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return 255;
  if (amax_bits == 0) return 0;
  const int e = (int)((amax_bits + kCarry) >> 23) - 6;
  return min(max(e, Range<T>::low), Range<T>::high);
}

// The same for magnitudes held in 64 bits, of which the high words' maximum is given: exponent and threshold lie there.
template <typename T>
static __device__ __forceinline__ int group_exponent_f64(uint32_t amax_high) {
  if (amax_high >= 0x7ff00000u) return 255;
  if (amax_high == 0) return 0;
  const int e = (int)((amax_high + (kCarry >> 3)) >> 20) - (1023 - 127) - 6;
  return min(max(e, Range<T>::low), Range<T>::high);
}

// What the maximum over a group is taken of, and the group's exponent byte from that maximum.
static __device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
static __device__ __forceinline__ uint32_t magnitude(double x) { return (uint32_t)__double2hiint(x) & 0x7fffffffu; }
template <typename T, typename F>
static __device__ __forceinline__ int exponent_of(uint32_t amax) {
  if constexpr (sizeof(F) == 8) return group_exponent_f64<T>(amax);
  else return group_exponent<T>(amax);
}

// The code of x in a group with exponent byte e.  The product with a power of two is exact and so is the rounding
// (to nearest, ties to even); the clamp only acts where the exponent was held at its largest.
static __device__ __forceinline__ int encode(float x, int e) {
  if (e == 0 || e == 255) return 0;
  const float v = fminf(fmaxf(__fmul_rn(x, power_of(254 - e)), -127.0f), 127.0f);
  return __float_as_int(__fadd_rn(v, kToInt)) << 24 >> 24;
}

static __device__ __forceinline__ int encode(double x, int e) {
  if (e == 0 || e == 255) return 0;
  return __double2int_rn(fmin(fmax(x * (double)power_of(254 - e), -127.0), 127.0));
}

}  // namespace act
}  // namespace optimi
