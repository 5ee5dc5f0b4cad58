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

// ---------------------------------------------------------------------------------------------
// chunks: 16 bytes of neighbouring values of a row in one thread
// ---------------------------------------------------------------------------------------------
// Rows need not begin on 16 bytes (an odd width, a slice).  Fetched<T, true> and store_any move such a chunk all the same: a
// row's chunks lie between 16-byte blocks at one distance, so a load takes the one or two blocks around it and shifts, and a
// store gets the head of its block from the lane before.  A block is only read where a byte of it belongs to the row, and
// no byte outside the row is written.
template <typename T>
struct Chunk {
  static constexpr int C = 16 / (int)sizeof(T);
  static constexpr int kLanes = kGroup / C;  // neighbouring lanes that hold a group
  uint32_t w[4];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = 0;
  }
  __device__ __forceinline__ void load(const T* p) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]); }

  __device__ __forceinline__ void store_value(T* p, int i) const {
    if constexpr (sizeof(T) == 4) p[i] = __uint_as_float(w[i]);
    else reinterpret_cast<unsigned short*>(p)[i] = (unsigned short)(w[i / 2] >> (i % 2 * 16));
  }
  // The first n values to p.  All lanes of a warp call it, with neighbouring chunks of one row: lane l's p is lane 0's + l * C, n is
  // C up to some lane and 0 after the next.  n may be negative: nothing.
  __device__ __forceinline__ void store_any(T* p, int n) const {
    const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(p) & 15u;  // the same in all lanes
    n = max(0, min(n, C));
    if (off == 0) {
      if (n == C) {
        store(p);
      } else {
#pragma unroll
        for (int i = 0; i < C; i++)
          if (i < n) store_value(p, i);
      }
      return;
    }
    const int lane = threadIdx.x % 32, head = (16 - (int)off) / (int)sizeof(T);  // values of a chunk that lie in its first block
    const uint32_t skip = 16 - off;                                                // their bytes
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 4; i++) u[i] = __shfl_up_sync(~0u, w[i], 1), u[4 + i] = w[i];
    const int n_before = __shfl_up_sync(~0u, n, 1);
    if (lane > 0 && n >= head) {  // then the chunk before is whole, and the block is bytes skip .. skip + 15 of the two
      shift(u, skip);
      *reinterpret_cast<uint4*>(reinterpret_cast<uintptr_t>(p) - off) = make_uint4(u[0], u[1], u[2], u[3]);
    } else if (lane == 0 && n == C) {  // the head alone, up to the next block: 2, 4 and 8 bytes of it
      uint32_t a[8] = {w[0], w[1], w[2], w[3], 0, 0, 0, 0};
      char* at = reinterpret_cast<char*>(p);
      if (sizeof(T) == 2 && (skip & 2)) *reinterpret_cast<unsigned short*>(at) = (unsigned short)a[0], at += 2, shift(a, 2);
      if (skip & 4) *reinterpret_cast<uint32_t*>(at) = a[0], at += 4, shift(a, 4);
      if (skip & 8) *reinterpret_cast<uint2*>(at) = make_uint2(a[0], a[1]);
    } else {
      Chunk before;
#pragma unroll
      for (int i = 0; i < 4; i++) before.w[i] = u[i];
#pragma unroll
      for (int i = 0; i < C; i++) {
        if (lane > 0 && i >= head && i < n_before) before.store_value(p - C, i);
        if (i < head && i < n) store_value(p, i);
      }
    }
    if (lane == 31 && n > head) {  // the tail, which no lane after this one takes along
      if (n == C) {
        uint32_t a[8] = {w[0], w[1], w[2], w[3], 0, 0, 0, 0};
        shift(a, skip);
        char* at = reinterpret_cast<char*>(reinterpret_cast<uintptr_t>(p) + skip);
        if (off & 8) *reinterpret_cast<uint2*>(at) = make_uint2(a[0], a[1]), at += 8, shift(a, 8);
        if (off & 4) *reinterpret_cast<uint32_t*>(at) = a[0], at += 4, shift(a, 4);
        if (sizeof(T) == 2 && (off & 2)) *reinterpret_cast<unsigned short*>(at) = (unsigned short)a[0];
      } else {
#pragma unroll
        for (int i = 0; i < C; i++)
          if (i >= head && i < n) store_value(p, i);
      }
    }
  }
  // The first 16 of 32 bytes, from byte `by` (below 16) on.
  static __device__ __forceinline__ void shift(uint32_t (&u)[8], uint32_t by) {
    if (by & 8) {
#pragma unroll
      for (int i = 0; i < 6; i++) u[i] = u[i + 2];
    }
    if (by & 4) {
#pragma unroll
      for (int i = 0; i < 5; i++) u[i] = u[i + 1];
    }
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 4; i++) u[i] = __funnelshift_r(u[i], u[i + 1], (by & 2) * 8);
    }
  }

  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    else if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)(w[i / 2] >> (i % 2 * 16))));
    else return __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  }
  // v[0..C-1], rounded to T
  __device__ __forceinline__ void set(const float* v) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(v[i]);
      else if constexpr (std::is_same<T, __half>::value) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
      else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
    }
  }
  // The largest magnitude, as fp32 bits: magnitudes compare as whole numbers, NaNs above infinity.
  __device__ __forceinline__ uint32_t amax() const {
    uint32_t m = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; i++) m = max(m, w[i] & 0x7fffffffu);
      return m;
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
      m = max(m & 0xffffu, m >> 16);
      if constexpr (std::is_same<T, __half>::value) return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
      else return m << 16;
    }
  }
};

// A chunk on its way from memory: fetch() asks for it, settle() (same arguments) is the first to need it, so that many can be under
// way at once.  The first n values at p, zeros behind them; n may be more than a chunk or negative.
template <typename T, bool kAny>
struct Fetched {
  static constexpr int C = Chunk<T>::C;
  uint32_t u[kAny ? 8 : 4];

  __device__ __forceinline__ void fetch(const T* p, int n) {
    uint4 a = make_uint4(0, 0, 0, 0), b = make_uint4(0, 0, 0, 0);
    if constexpr (!kAny) {
      if (n > 0) a = *reinterpret_cast<const uint4*>(p);
    } else {
      const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(p) & 15u;
      const uint4* block = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) - off);
      if (n > 0) a = block[0];
      if (n > 0 && off + (uint32_t)min(n, C) * (uint32_t)sizeof(T) > 16) b = block[1];
      u[4] = b.x, u[5] = b.y, u[6] = b.z, u[7] = b.w;
    }
    u[0] = a.x, u[1] = a.y, u[2] = a.z, u[3] = a.w;
  }
  __device__ __forceinline__ Chunk<T> settle(const T* p, int n) const {
    Chunk<T> v;
    if constexpr (!kAny) {
#pragma unroll
      for (int i = 0; i < 4; i++) v.w[i] = u[i];
    } else {
      uint32_t s[8];
#pragma unroll
      for (int i = 0; i < 8; i++) s[i] = u[i];
      Chunk<T>::shift(s, (uint32_t)reinterpret_cast<uintptr_t>(p) & 15u);
#pragma unroll
      for (int i = 0; i < 4; i++) v.w[i] = s[i];
      if (n < C) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          if constexpr (sizeof(T) == 4) v.w[i] = i < n ? v.w[i] : 0;
          else v.w[i] = 2 * i + 1 < n ? v.w[i] : 2 * i < n ? v.w[i] & 0xffffu : 0;
        }
      }
    }
    return v;
  }
};

// The largest of a group's magnitudes, in all its lanes.
template <int kLanes>
static __device__ __forceinline__ uint32_t group_max(uint32_t m) {
#pragma unroll
  for (int d = 1; d < kLanes; d *= 2) m = max(m, __shfl_xor_sync(~0u, m, d));
  return m;
}

// C (8 or 4) codes.
template <int C>
struct CodeChunk {
  static constexpr int kWords = C / 4;
  uint32_t w[kWords];

  // From values in fp32 that are at most 127.5 in a unit of 2^(e - 127), or more where e was held at its largest.  One fused
  // multiply-add gives product, rounding and code: the product is exact, and the sum with 1.5 * 2^23 rounds to a whole number.
  template <typename T>
  __device__ __forceinline__ void encode(const float* v, int e) {
    const float inverse = power_of(254 - e);
    uint32_t c[C];
    if (e >= Range<T>::high) {  // the top of the range, or a NaN group: rare
#pragma unroll
      for (int i = 0; i < C; i++) c[i] = (uint32_t)act::encode(v[i], e);
    } else {
#pragma unroll
      for (int i = 0; i < C; i++) c[i] = __float_as_uint(__fmaf_rn(v[i], inverse, kToInt));
    }
    set(c);
  }
  template <typename T>
  __device__ __forceinline__ void encode(const double* v, int e) {
    uint32_t c[C];
#pragma unroll
    for (int i = 0; i < C; i++) c[i] = (uint32_t)act::encode(v[i], e);
    set(c);
  }
  __device__ __forceinline__ void set(const uint32_t* c) {
#pragma unroll
    for (int i = 0; i < kWords; i++)
      w[i] = __byte_perm(__byte_perm(c[4 * i], c[4 * i + 1], 0x0040), __byte_perm(c[4 * i + 2], c[4 * i + 3], 0x0040), 0x5410);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; i++) w[i] = 0;
  }
  __device__ __forceinline__ void load(const int8_t* p) {
    if constexpr (C == 8) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x, w[1] = v.y;
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
  }
  __device__ __forceinline__ void store(int8_t* p) const {
    if constexpr (C == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
  }
  // Code i times a unit of at most 2^100, given the unit and scaled_offset(unit): exact, so one fused operation does for both.
  static __device__ __forceinline__ float scaled_offset(float unit) { return __fmul_rn(-8388736.0f, unit); }
  __device__ __forceinline__ float get_scaled(int i, float unit, float offset) const { return __fmaf_rn(raw(i), unit, offset); }
  // Code i as fp32: the byte with its sign bit flipped, set into the low bits of 2^23, is 2^23 + 128 + code.
  __device__ __forceinline__ float raw(int i) const { return __uint_as_float(__byte_perm(w[i / 4] ^ 0x80808080u, 0x4b000000u, 0x7440 + i % 4)); }
  __device__ __forceinline__ float get(int i) const { return raw(i) - 8388736.0f; }
};

// 2^(e - 127) for two exponent bytes, as a pair of T.  bf16: the byte is the exponent field (255 gives an infinity, which
// makes the zero codes of its group NaN).  fp16: through fp32, exact down to the subnormal 2^-24.
template <typename T> static __device__ __forceinline__ uint32_t scale_pair(uint32_t bytes, uint32_t select);
template <> __device__ __forceinline__ uint32_t scale_pair<__nv_bfloat16>(uint32_t bytes, uint32_t select) {
  return __byte_perm(bytes, 0, select) << 7;
}
template <> __device__ __forceinline__ uint32_t scale_pair<__half>(uint32_t bytes, uint32_t select) {
  const uint32_t p = __byte_perm(bytes, 0, select);
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(__uint_as_float((p >> 16) << 23)), "f"(__uint_as_float((p & 0xff) << 23)));
  return r;
}

// Two codes (bytes picked by `select`) times two scales, exactly.  A byte set into the low mantissa bits of a constant is a
// whole number plus that constant, which a subtraction takes off again.
// bf16 has 7 such bits: 0x43 << 8 is 128, so the low 7 bits give 128 + b & 127 and the sign bit, in the exponent, tells 128 from 256.
template <typename T> static __device__ __forceinline__ uint32_t code_pair(uint32_t codes, uint32_t select, uint32_t scale);
template <> __device__ __forceinline__ uint32_t code_pair<__nv_bfloat16>(uint32_t codes, uint32_t select, uint32_t scale) {
  const uint32_t p = __byte_perm(codes, 0x43, select), with = p & 0xff7fff7fu, without = p & 0xff80ff80u;
  uint32_t r;
  asm("{\n.reg .b32 t;\nsub.rn.bf16x2 t, %1, %2;\nmul.rn.bf16x2 %0, t, %3;\n}" : "=r"(r) : "r"(with), "r"(without), "r"(scale));
  return r;
}
// fp16 has 10: 0x64 << 8 is 1024, and the byte with its sign bit flipped is code + 128.
template <> __device__ __forceinline__ uint32_t code_pair<__half>(uint32_t codes, uint32_t select, uint32_t scale) {
  const uint32_t p = __byte_perm(codes ^ 0x80808080u, 0x64, select);
  uint32_t r;
  asm("{\n.reg .b32 t;\nsub.rn.f16x2 t, %1, %2;\nmul.rn.f16x2 %0, t, %3;\n}" : "=r"(r) : "r"(p), "r"(0x64806480u), "r"(scale));
  return r;
}

}  // namespace act
}  // namespace optimi
