// The weight gradient of a linear layer whose input is held in 8 bits:
//     dW[o, c] = w[c] * sum_t dY[t, o] * X[t, c]        X = code * 2^(e - 127)  (format: activation_common.cuh)
//
// On the tensor cores as D[c, o] = X^T dY with M = channels, N = outputs, K = tokens.  Both operands have the token as
// their slow dimension in memory.  dY goes by TMA into shared memory and is read there with the token as the strided
// (MN-major) dimension.  X^T has to be made from codes, and the result goes to tensor memory, as the left operand of the
// instruction may lie there: a row per channel, tokens along the columns.  That costs shared memory only the codes' own
// bytes (one read of 8 bits a value) where a 16-bit copy beside dY would be written and then read again.
// code * 2^k has 7 bits and fits bf16 and fp16 exactly, so the products are those of the restored activation.
#include "activation_common.cuh"

#include <cuda.h>

namespace optimi {
namespace act {

// A pair of blocks on two neighbouring SMs works on one tile of 256 channels x 256 outputs, 64 tokens at a time.  Each holds
// the codes, X^T and the results of its 128 channels, and the gradients of its 128 outputs; the instruction reads the other
// half of the gradients from the partner's shared memory.
constexpr int kM = 128, kN = 256, kK = 64;           // channels of a block, outputs of the pair, tokens of a step
constexpr int kStages = 8;
constexpr int kGradBytes = kK * (kN / 2) * 2, kCodeBytes = kK * kM, kStageBytes = kGradBytes + kCodeBytes;
constexpr int kSmemBytes = kStages * kStageBytes + 1024;
constexpr int kAColumns = kK / 2;                    // 32-bit columns of tensor memory of one block of X^T
constexpr int kMakers = 8;                           // warps that convert, in two sets that take turns, and write results
constexpr int kLoader = kMakers, kIssuer = kMakers + 1;
constexpr int kThreads = 32 * (kMakers + 2);
constexpr int kWaitLimit = 1 << 22;                  // polls after which a wait gives up

// Set by a kernel whose wait gave up (its results are NaN); read by optimi_b200_weight_gradient_status.
static __device__ int g_gave_up;

static __device__ __forceinline__ uint32_t smem_of(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

static __device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
// The same barrier of the pair's first block.
static __device__ __forceinline__ uint32_t in_first(uint32_t bar) {
  uint32_t at;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(bar));
  return at;
}
// Relaxed: what it announces lies in tensor memory, which tcgen05.wait::st and the fences around the barrier order; a release
// over the cluster would wait for the loads under way too (measured: half the kernel's time).
static __device__ __forceinline__ void barrier_arrive(uint32_t remote) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote) : "memory");
}
static __device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// False if the phase did not complete within the limit.
static __device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity) {
  for (int n = 0; n < kWaitLimit; n++) {
    uint32_t done;
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\nselp.b32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
  }
  return false;
}

static __device__ __forceinline__ void pair_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The barrier is arrived at in both blocks once all the multiplications issued so far are done.
static __device__ __forceinline__ void commit_to_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3)
               : "memory");
}

// `bar` may be a barrier of either block of the pair.
static __device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
               "l"(map), "r"(x), "r"(y), "r"(bar)
               : "memory");
}

// Shared memory as the right operand, token-strided, in the 128-byte swizzle: rows of 64 outputs (128 bytes) per token; 1024
// bytes from one group of 8 tokens to the next, kK * 128 from one block of 64 outputs to the next.
static __device__ __forceinline__ uint64_t grad_descriptor(uint32_t addr) {
  return (uint64_t)((addr & 0x3ffff) >> 4) | (uint64_t)(kK * 128 >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

// D in fp32; A and B in T; A as it lies in tensor memory, B transposed (its outputs are contiguous); N and M of the pair.
template <typename T>
static __device__ __forceinline__ constexpr uint32_t instruction_descriptor() {
  constexpr uint32_t kind = sizeof(T) == 2 && !std::is_same<T, __half>::value ? 1 : 0;
  return 1u << 4 | kind << 7 | kind << 10 | 1u << 16 | (uint32_t)(kN >> 3) << 17 | (uint32_t)(2 * kM >> 4) << 24;
}

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    weight_gradient_kernel(const __grid_constant__ CUtensorMap grad_map, const __grid_constant__ CUtensorMap code_map,
                           const uint8_t* __restrict__ exponents, int64_t epitch, const T* __restrict__ channel_scale, int rows,
                           int outputs, int channels, T* __restrict__ dw) {
  extern __shared__ uint8_t dynamic[];
  __shared__ __align__(8) uint64_t bars[4 * kStages + 1];
  __shared__ __align__(4) uint8_t bytes[kMakers][2][kK];
  __shared__ uint32_t tmem_base;
  __shared__ int gave_up;
  const uint32_t tiles = (smem_of(dynamic) + 1023) & ~1023u;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int half = blockIdx.x % 2;  // which block of the pair
  // codes: this block's codes are there.  grads, made (the first block's): both blocks' gradients, both halves of X^T are there.
  // empty: the multiplications that read a stage are done.
  const uint32_t codes_in = smem_of(bars), grads_in = codes_in + 8 * kStages, made = grads_in + 8 * kStages, empty = made + 8 * kStages,
                 done = empty + 8 * kStages;
  const int c0 = blockIdx.x * kM, o0 = blockIdx.y * kN;
  const int blocks = (rows + kK - 1) / kK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; s++) {
      barrier_init(codes_in + 8 * s, 1);
      barrier_init(grads_in + 8 * s, 1);
      barrier_init(made + 8 * s, 2 * 4);  // four warps of each block
      barrier_init(empty + 8 * s, 1);
    }
    barrier_init(done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    gave_up = 0;
  }
  if (warp == kIssuer) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_of(&tmem_base)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  pair_sync();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_base, tmem_a = tmem + kN;
  bool ok = true;

  if (warp == kLoader) {
    if (lane == 0) {
      int b = 0;
      for (; b < blocks; b++) {
        const int s = b % kStages;
        if (b >= kStages && !barrier_wait(empty + 8 * s, (b / kStages - 1) & 1)) break;
        const uint32_t at = tiles + s * kStageBytes, grads = in_first(grads_in + 8 * s);
        barrier_expect(codes_in + 8 * s, kCodeBytes);
        load_tile(at + kGradBytes, &code_map, c0, b * kK, codes_in + 8 * s);
        if (half == 0) barrier_expect(grads_in + 8 * s, 2 * kGradBytes);
        for (int j = 0; j < kN / 2 / 64; j++) load_tile(at + j * kK * 128, &grad_map, o0 + half * (kN / 2) + j * 64, b * kK, grads);
      }
      ok = b == blocks;
      // Nothing of a block's shared memory is given back while a copy into it is under way: both blocks wait for the codes they
      // asked for, the first for the gradients of both.  (The partner stays until the first block is here too.)
      for (int n = b > kStages ? b - kStages : 0; n < b; n++) {
        ok &= barrier_wait(codes_in + 8 * (n % kStages), (n / kStages) & 1);
        if (half == 0) ok &= barrier_wait(grads_in + 8 * (n % kStages), (n / kStages) & 1);
      }
    }
  } else if (warp == kIssuer) {
    if (lane == 0 && half == 0) {
      for (int b = 0; b < blocks; b++) {
        const int s = b % kStages;
        ok = barrier_wait(grads_in + 8 * s, (b / kStages) & 1) && barrier_wait(made + 8 * s, (b / kStages) & 1);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t desc = grad_descriptor(tiles + s * kStageBytes);
#pragma unroll
        for (int k = 0; k < kK / 16; k++) {
          const uint32_t accumulate = b > 0 || k > 0;
          asm volatile(
              "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
              "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(tmem),
              "r"(tmem_a + s * kAColumns + k * 8), "l"(desc + (uint64_t)(k * 2048 >> 4)), "r"(instruction_descriptor<T>()), "r"(accumulate)
              : "memory");
        }
        commit_to_pair(empty + 8 * s);
      }
      commit_to_pair(done);
    }
  } else {
    // channels 32 * (warp % 4) .. + 31 of the block are this warp's rows of tensor memory, and one group of the format
    const int part = warp % 4, set = warp / 4;
    const int group = c0 / kGroup + part, quad = lane % 4;
    const bool live = group * kGroup < channels;
    const auto exponent = [&](int t) -> uint32_t { return live && t < rows ? exponents[(int64_t)t * epitch + group] : 0; };
    uint32_t e0 = exponent(set * kK + lane), e1 = exponent(set * kK + lane + 32);
    for (int b = set; b < blocks; b += kMakers / 4) {
      const int s = b % kStages, parity = (b / kStages) & 1;
      uint8_t* mine = bytes[warp][b / (kMakers / 4) & 1];
      mine[lane] = (uint8_t)e0, mine[lane + 32] = (uint8_t)e1;
      __syncwarp();
      const int next = (b + kMakers / 4) * kK + lane;
      e0 = exponent(next), e1 = exponent(next + 32);
      ok = barrier_wait(codes_in + 8 * s, parity);
      if (!ok) break;
      const uint32_t codes = tiles + s * kStageBytes + kGradBytes;
      uint32_t low[16], high[16];
#pragma unroll
      for (int j = 0; j < kK / 16; j++) {
        // two 16 x 16 byte transposes: thread l gets channel l / 4 (and + 8), tokens 4 * (l % 4) .. + 3 of each
        const int t = j * 16 + lane % 16, chunk = 2 * part + lane / 16;
        uint32_t r[4];
        asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(codes + t * 128 + ((chunk ^ (t & 7)) << 4)));
        const uint32_t four = reinterpret_cast<const uint32_t*>(mine)[j * 4 + quad];
        const uint32_t s01 = scale_pair<T>(four, 0x4140), s23 = scale_pair<T>(four, 0x4342);
#pragma unroll
        for (int i = 0; i < 2; i++) {
          low[4 * j + 2 * i] = code_pair<T>(r[i], 0x4140, s01), low[4 * j + 2 * i + 1] = code_pair<T>(r[i], 0x4342, s23);
          high[4 * j + 2 * i] = code_pair<T>(r[2 + i], 0x4140, s01), high[4 * j + 2 * i + 1] = code_pair<T>(r[2 + i], 0x4342, s23);
        }
      }
      const uint32_t to = tmem_a + s * kAColumns + ((uint32_t)(part * 32) << 16);
#define STORE16(addr, v)                                                                                                            \
  asm volatile("tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" \
               ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),       \
               "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])                                     \
               : "memory")
      STORE16(to, low);
      STORE16(to + (16u << 16), high);
#undef STORE16
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) barrier_arrive(in_first(made + 8 * s));
    }
    ok = barrier_wait(done, 0) && ok;
  }
  if (!ok) gave_up = 1;
  __syncwarp();
  __syncthreads();
  if (gave_up && threadIdx.x == 0) g_gave_up = 1;

  if (warp < kMakers) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const int part = warp % 4;
    const int c = c0 + part * 32 + lane;
    const float scale = channel_scale && c < channels ? to_f32(channel_scale[c]) : 1.0f;
    const bool lost = gave_up;
    const int first = warp / 4 * (kN / (kMakers / 4));
    for (int n = first; n < first + kN / (kMakers / 4) && o0 + n < outputs; n += 16) {
      uint32_t v[16];
      asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                   : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
                     "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                   : "r"(tmem + n + ((uint32_t)(part * 32) << 16)));
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const float d = lost ? __int_as_float(0x7fffffff) : __uint_as_float(v[i]);
        if (o0 + n + i < outputs && c < channels) dw[(int64_t)(o0 + n + i) * channels + c] = from_f32<T>(__fmul_rn(d, scale));
      }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }
  __syncwarp();
  pair_sync();  // the partner may still read this block's gradients or arrive at its barriers
  if (warp == kIssuer) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      p = nullptr;
    }
    return (EncodeTiled)p;
  }();
  return fn;
}

// A matrix of rows whose tiles of `width` x `height` elements (128 bytes wide) are loaded in the 128-byte swizzle; zeros outside.
static int make_map(const char* fn, CUtensorMap* map, CUtensorMapDataType type, const void* base, int64_t cols, int64_t rows,
                    int64_t pitch_bytes, int width, int height) {
  const EncodeTiled encode = encode_tiled();
  if (!encode) return fail(OPTIMI_ERR_CUDA, "%s: the driver has no cuTensorMapEncodeTiled", fn);
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)pitch_bytes};
  const cuuint32_t box[2] = {(cuuint32_t)width, (cuuint32_t)height}, steps[2] = {1, 1};
  const CUresult r = encode(map, type, 2, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? OPTIMI_OK : fail(OPTIMI_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed with %d", fn, (int)r);
}

template <typename T>
static int launch_weight_gradient(const char* fn, const CUtensorMap& grad_map, const CUtensorMap& code_map, const void* exponents,
                                  int64_t epitch, const void* channel_scale, int rows, int outputs, int channels, void* dw, cudaStream_t s) {
  cudaError_t e = cudaFuncSetAttribute(weight_gradient_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
  if (e != cudaSuccess) return fail(OPTIMI_ERR_CUDA, "%s: %s", fn, cudaGetErrorString(e));
  const dim3 grid((channels + 2 * kM - 1) / (2 * kM) * 2, (outputs + kN - 1) / kN);
  weight_gradient_kernel<T><<<grid, kThreads, kSmemBytes, s>>>(grad_map, code_map, (const uint8_t*)exponents, epitch,
                                                              (const T*)channel_scale, rows, outputs, channels, (T*)dw);
  return launched(fn);
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

int optimi_b200_weight_gradient_status(int* gave_up) {
  const char* fn = "optimi_b200_weight_gradient_status";
  if (!gave_up) return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: gave_up is NULL", fn);
  cudaError_t e = cudaMemcpyFromSymbol(gave_up, g_gave_up, sizeof(int));
  return e == cudaSuccess ? OPTIMI_OK : fail(OPTIMI_ERR_CUDA, "%s: %s", fn, cudaGetErrorString(e));
}

int optimi_b200_weight_gradient(const void* grad, int64_t grad_stride, const void* codes, int64_t code_pitch, const void* exponents,
                                int64_t exponent_pitch, const void* channel_scale, int64_t rows, int64_t outputs, int64_t channels,
                                int dtype, void* grad_weight, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "optimi_b200_weight_gradient";
  (void)workspace, (void)workspace_bytes;
  if (dtype != OPTIMI_BF16 && dtype != OPTIMI_F16)
    return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: dtype %d is neither bfloat16 nor float16", fn, dtype);
  // token and output coordinates are 32-bit and run past the end by less than a block
  const int64_t most = INT32_MAX - 4096;
  if (rows < 0 || outputs < 0 || channels < 0 || rows > most || outputs > most || channels > most)
    return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: %lld tokens, %lld outputs, %lld channels are outside 0..%lld", fn, (long long)rows,
                (long long)outputs, (long long)channels, (long long)most);
  if (outputs == 0 || channels == 0) return OPTIMI_OK;
  if (!grad_weight) return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: grad_weight is NULL", fn);
  cudaStream_t s = (cudaStream_t)stream;
  if (rows == 0) {
    cudaError_t e = cudaMemsetAsync(grad_weight, 0, (size_t)outputs * (size_t)channels * 2, s);
    return e == cudaSuccess ? OPTIMI_OK : fail(OPTIMI_ERR_CUDA, "%s: %s", fn, cudaGetErrorString(e));
  }
  if (!grad) return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: grad is NULL", fn);
  int rc = check_codes(fn, codes, code_pitch, exponents, exponent_pitch, channels);
  if (rc != OPTIMI_OK) return rc;
  if (grad_stride < outputs || grad_stride % 8 || !aligned(grad, 16))
    return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: rows of grad must begin on 16 bytes: stride %lld is no multiple of 8 of at least %lld, or the base is unaligned",
                fn, (long long)grad_stride, (long long)outputs);
  if ((outputs + kN - 1) / kN > 65535) return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: %lld outputs are too many", fn, (long long)outputs);
  CUtensorMap grad_map, code_map;
  rc = make_map(fn, &grad_map, dtype == OPTIMI_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, grad, outputs, rows,
                grad_stride * 2, 64, kK);
  if (rc != OPTIMI_OK) return rc;
  rc = make_map(fn, &code_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, channels, rows, code_pitch, kM, kK);
  if (rc != OPTIMI_OK) return rc;
  if (dtype == OPTIMI_BF16)
    return launch_weight_gradient<__nv_bfloat16>(fn, grad_map, code_map, exponents, exponent_pitch, channel_scale, (int)rows, (int)outputs,
                                                 (int)channels, grad_weight, s);
  return launch_weight_gradient<__half>(fn, grad_map, code_map, exponents, exponent_pitch, channel_scale, (int)rows, (int)outputs,
                                        (int)channels, grad_weight, s);
}

}  // extern "C"
