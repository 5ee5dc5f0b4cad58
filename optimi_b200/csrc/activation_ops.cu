// Activations kept in 8 bits (format: activation_common.cuh) and the RMS norm that writes and reads them.
#include "activation_common.cuh"

namespace optimi {
namespace act {

// ---------------------------------------------------------------------------------------------
// store and restore
// ---------------------------------------------------------------------------------------------
// Both stream: an item is a chunk of C values in one thread (the neighbouring lanes of a group find its largest magnitude
// together), kUnroll items a thread are loaded before the first is used, and nothing is read or written twice.
constexpr int kBlock = 256, kUnroll = 4;

// Where chunk `item` lies: rows of `chunks` chunks, the last group of a row filled up.  With kFlat rows follow one another without
// a gap and are whole groups, so that a tensor is one long row and nothing is divided.
template <int C, bool kFlat>
struct Place {
  int64_t row, col;
  __device__ __forceinline__ Place(int64_t item, int64_t chunks) {
    if constexpr (kFlat) {
      row = 0, col = item * C;
    } else if (item < (1ll << 31) && chunks < (1ll << 31)) {
      row = (uint32_t)item / (uint32_t)chunks, col = ((uint32_t)item - (uint32_t)row * (uint32_t)chunks) * (int64_t)C;
    } else {
      row = item / chunks, col = (item - row * chunks) * C;
    }
  }
};

template <typename T, int C, bool kFlat>
__global__ void __launch_bounds__(kBlock) compress_kernel(const T* __restrict__ x, int64_t items, int64_t chunks, int64_t cols, int64_t stride,
                                                          int8_t* __restrict__ codes, int64_t pitch, uint8_t* __restrict__ exponents,
                                                          int64_t epitch) {
  constexpr int kLanes = Chunk<T, C>::kLanes;
  const int64_t first = (int64_t)blockIdx.x * (kBlock * kUnroll) + threadIdx.x;
  Chunk<T, C> v[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; u++) {
    const int64_t item = first + u * kBlock;
    v[u].clear();
    if (item < items) {
      const Place<C, kFlat> at(item, chunks);
      if (kFlat || at.col < cols) v[u].load(x + at.row * stride + at.col);
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; u++) {
    const int64_t item = first + u * kBlock;
    const int e = group_exponent<T>(group_max<kLanes>(v[u].amax()));
    float f[C];
#pragma unroll
    for (int i = 0; i < C; i++) f[i] = v[u].get(i);
    CodeChunk<C> c;
    c.template encode<T>(f, e);
    if (item < items) {
      const Place<C, kFlat> at(item, chunks);
      c.store(codes + at.row * pitch + at.col);
      if (threadIdx.x % kLanes == 0) exponents[at.row * epitch + at.col / kGroup] = (uint8_t)e;
    }
  }
}

template <typename T, int C, bool kFlat, bool kScaled>
__global__ void __launch_bounds__(kBlock) decompress_kernel(const int8_t* __restrict__ codes, int64_t pitch, const uint8_t* __restrict__ exponents,
                                                            int64_t epitch, const T* __restrict__ channel_scale, int64_t items,
                                                            int64_t chunks, int64_t cols, T* __restrict__ out) {
  const int64_t first = (int64_t)blockIdx.x * (kBlock * kUnroll) + threadIdx.x;
  CodeChunk<C> c[kUnroll];
  uint32_t e[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; u++) {
    const int64_t item = first + u * kBlock;
    c[u].clear(), e[u] = 0;
    if (item < items) {
      const Place<C, kFlat> at(item, chunks);
      c[u].load(codes + at.row * pitch + at.col);
      e[u] = exponents[at.row * epitch + at.col / kGroup];
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; u++) {
    const int64_t item = first + u * kBlock;
    if (item >= items) return;
    const Place<C, kFlat> at(item, chunks);
    if (!kFlat && at.col >= cols) continue;
    Chunk<T, C> v;
    if constexpr (sizeof(T) == 2 && C == 8 && !kScaled) {
      const uint32_t s = scale_pair<T>(e[u], 0x4040);
#pragma unroll
      for (int i = 0; i < 4; i++) v.w[i] = code_pair<T>(c[u].w[i / 2], i % 2 ? 0x4342 : 0x4140, s);
    } else {
      float f[C];
      const float s = power_of((int)e[u]);
#pragma unroll
      for (int i = 0; i < C; i++) {
        f[i] = __fmul_rn(c[u].get(i), s);
        if (kScaled) f[i] = __fmul_rn(f[i], to_f32(channel_scale[(kFlat ? at.col % cols : at.col) + i]));
      }
      v.set(f);
    }
    v.store(out + at.row * cols + at.col);
  }
}

// ---------------------------------------------------------------------------------------------
// residual addition + RMS norm
// ---------------------------------------------------------------------------------------------
//     h = round(x + r)      rstd = (mean(h^2) + eps)^-1/2      xn = h * rstd      y = round(xn * w)
// and the 8-bit form of xn (without w, so that one checkpoint serves this norm's backward pass and, with w applied to the
// columns of its result, the weight gradient of every linear layer that reads y).
//
// A row belongs to P threads, each with K chunks of it in registers from the first load to the last store.
//
// The normalised value is held in F: fp32, and 64 bits for fp32 activations, whose gradients would show a code that a
// last-bit difference of rstd tips over.
template <typename T> struct Wide { using type = float; };
template <> struct Wide<float> { using type = double; };

// Sum over the P threads of a row, in all of them, added up in a fixed order.  `part` is this row's scratch; consecutive calls
// alternate between two of them (turn), so that one barrier a call is enough.
template <int P, typename F>
static __device__ __forceinline__ F row_sum(F v, F (*part)[P / 32], int turn, int group) {
#pragma unroll
  for (int d = 16; d > 0; d /= 2) v += __shfl_xor_sync(~0u, v, d);
  if constexpr (P > 32) {
    F* mine = part[turn & 1];
    const int warp = threadIdx.x % P / 32;
    if (threadIdx.x % 32 == 0) mine[warp] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(P) : "memory");
    v = mine[0];
#pragma unroll
    for (int i = 1; i < P / 32; i++) v += mine[i];
  }
  return v;
}

template <typename T, int C, int P, int K, bool kKeep>
__global__ void __launch_bounds__(P < 128 ? 128 : P)
    rms_norm_kernel(const T* __restrict__ x, int64_t xs, const T* __restrict__ residual, int64_t rs, const T* __restrict__ weight,
                    int64_t rows, int cols, double eps, T* __restrict__ y, T* __restrict__ sum, int8_t* __restrict__ codes, int64_t pitch,
                    uint8_t* __restrict__ exponents, int64_t epitch, float* __restrict__ rstd_out) {
  using F = typename Wide<T>::type;
  using Values = Chunk<T, C>;
  constexpr int kGroups = (P < 128 ? 128 : P) / P;
  __shared__ F part[kGroups][2][P / 32];
  const int group = threadIdx.x / P, t = threadIdx.x % P;
  const int padded = (cols + kGroup - 1) / kGroup * kGroup;
  Values w[K];
#pragma unroll
  for (int k = 0; k < K; k++) {
    const int c = (k * P + t) * C;
    if (weight && c < cols) w[k].load(weight + c);
  }
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * kGroups + group; row < rows; row += (int64_t)gridDim.x * kGroups, turn++) {
    Values h[K];
    F ss = 0;
#pragma unroll
    for (int k = 0; k < K; k++) {
      const int c = (k * P + t) * C;
      h[k].clear();
      if (c < cols) h[k].load(x + row * xs + c);
    }
    if (residual) {
      Values r[K];
#pragma unroll
      for (int k = 0; k < K; k++) {
        const int c = (k * P + t) * C;
        r[k].clear();
        if (c < cols) r[k].load(residual + row * rs + c);
      }
#pragma unroll
      for (int k = 0; k < K; k++) {
        const int c = (k * P + t) * C;
        float f[C];
#pragma unroll
        for (int i = 0; i < C; i++) f[i] = __fadd_rn(h[k].get(i), r[k].get(i));
        h[k].set(f);
        if (c < cols) h[k].store(sum + row * cols + c);
      }
    }
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
      for (int i = 0; i < C; i++) {
        const F v = (F)h[k].get(i);
        if constexpr (sizeof(F) == 4) ss = __fmaf_rn(v, v, ss);
        else ss = __fma_rn(v, v, ss);
      }
    ss = row_sum<P, F>(ss, part[group], turn, group);
    const F rstd = F(1) / sqrt(ss / (F)cols + (F)eps);
    if (kKeep && t == 0) rstd_out[row] = (float)rstd;
#pragma unroll
    for (int k = 0; k < K; k++) {
      const int c = (k * P + t) * C;
      F n[C];
      float f[C];
#pragma unroll
      for (int i = 0; i < C; i++) {
        n[i] = (F)h[k].get(i) * rstd;
        f[i] = (float)(weight ? n[i] * (F)w[k].get(i) : n[i]);
      }
      Values out;
      out.set(f);
      if (c < cols) out.store(y + row * cols + c);
      if constexpr (kKeep) {
        // rounding keeps the order of magnitudes, so the largest |h| times rstd is the largest |xn|
        const F top = (F)__uint_as_float(h[k].amax()) * rstd;
        const int e = exponent_of<T, F>(group_max<Values::kLanes>(magnitude(top)));
        CodeChunk<C> code;
        code.template encode<T>(n, e);
        if (c < padded) {
          code.store(codes + row * pitch + c);
          if (t % Values::kLanes == 0) exponents[row * epitch + c / kGroup] = (uint8_t)e;
        }
      }
    }
  }
}

// Rows too long for registers: the same, reading the row a second time.
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

template <typename T>
__global__ void long_rms_norm_kernel(const T* __restrict__ x, int64_t xs, const T* __restrict__ residual, int64_t rs,
                                     const T* __restrict__ weight, int64_t rows, int64_t cols, double eps, T* __restrict__ y, T* sum,
                                     int8_t* __restrict__ codes, int64_t pitch, uint8_t* __restrict__ exponents, int64_t epitch,
                                     float* __restrict__ rstd_out) {
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
//
// A block keeps its threads' columns of dw in registers over all its rows, and leaves one line of partial sums in the workspace
// (its row groups added up in order in shared memory); a second kernel adds up the lines in order.  Few blocks, so few lines.
template <typename T, int C, int P, int K, int kThreads>
__global__ void __launch_bounds__(kThreads)
    rms_norm_backward_kernel(const T* __restrict__ grad, int64_t gs, const T* __restrict__ grad_sum, int64_t hs, const int8_t* __restrict__ codes,
                             int64_t pitch, const uint8_t* __restrict__ exponents, int64_t epitch, const float* __restrict__ rstd,
                             const T* __restrict__ weight, int64_t rows, int cols, T* __restrict__ dx, float* __restrict__ lines) {
  using Values = Chunk<T, C>;
  constexpr int kGroups = kThreads / P;
  __shared__ float part[kGroups][2][P / 32];
  extern __shared__ float line[];
  const int group = threadIdx.x / P, t = threadIdx.x % P;
  Values w[K];
  float dw[K][C];
#pragma unroll
  for (int k = 0; k < K; k++) {
    const int c = (k * P + t) * C;
    w[k].clear();
    if (weight && c < cols) w[k].load(weight + c);
#pragma unroll
    for (int i = 0; i < C; i++) dw[k][i] = 0.0f;
  }
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * kGroups + group; row < rows; row += (int64_t)gridDim.x * kGroups, turn++) {
    Values g[K], s[K];
    CodeChunk<C> code[K];
    uint32_t e[K];
    const float r = rstd[row];
#pragma unroll
    for (int k = 0; k < K; k++) {
      const int c = (k * P + t) * C;
      g[k].clear(), code[k].clear(), e[k] = 0;
      if (c < cols) {
        g[k].load(grad + row * gs + c);
        code[k].load(codes + row * pitch + c);
        e[k] = exponents[row * epitch + c / kGroup];
      }
    }
    if (grad_sum && dx) {
#pragma unroll
      for (int k = 0; k < K; k++) {
        const int c = (k * P + t) * C;
        if (c < cols) s[k].load(grad_sum + row * hs + c);
      }
    }
    float m = 0;
#pragma unroll
    for (int k = 0; k < K; k++) {
      const float unit = power_of((int)e[k]);
#pragma unroll
      for (int i = 0; i < C; i++) {
        const float n = __fmul_rn(code[k].get(i), unit), v = g[k].get(i);
        dw[k][i] = __fmaf_rn(v, n, dw[k][i]);
        m = __fmaf_rn(weight ? __fmul_rn(v, w[k].get(i)) : v, n, m);
      }
    }
    if (!dx) continue;
    m = row_sum<P, float>(m, part[group], turn, group) / (float)cols;
#pragma unroll
    for (int k = 0; k < K; k++) {
      const int c = (k * P + t) * C;
      const float unit = power_of((int)e[k]);
      float f[C];
#pragma unroll
      for (int i = 0; i < C; i++) {
        const float n = __fmul_rn(code[k].get(i), unit), v = g[k].get(i);
        f[i] = __fmul_rn(r, __fmaf_rn(-n, m, weight ? __fmul_rn(v, w[k].get(i)) : v));
        if (grad_sum) f[i] = __fadd_rn(f[i], s[k].get(i));
      }
      Values out;
      out.set(f);
      if (c < cols) out.store(dx + row * cols + c);
    }
  }
  if (!lines) return;
  if constexpr (kGroups == 1) {
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
      for (int i = 0; i < C; i++) {
        const int c = (k * P + t) * C + i;
        if (c < cols) lines[(int64_t)blockIdx.x * cols + c] = dw[k][i];
      }
    return;
  }
  for (int j = 0; j < kGroups; j++) {
    if (j == group) {
#pragma unroll
      for (int k = 0; k < K; k++)
#pragma unroll
        for (int i = 0; i < C; i++) {
          const int c = (k * P + t) * C + i;
          if (c < cols) line[c] = j ? line[c] + dw[k][i] : dw[k][i];
        }
    }
    __syncthreads();
  }
  for (int c = threadIdx.x; c < cols; c += kThreads) lines[(int64_t)blockIdx.x * cols + c] = line[c];
}

template <typename T>
__global__ void long_rms_norm_backward_kernel(const T* __restrict__ grad, int64_t gs, const T* __restrict__ grad_sum, int64_t hs,
                                              const int8_t* __restrict__ codes, int64_t pitch, const uint8_t* __restrict__ exponents,
                                              int64_t epitch, const float* __restrict__ rstd, const T* __restrict__ weight, int64_t rows,
                                              int64_t cols, T* __restrict__ dx, float* __restrict__ lines) {
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

// A warp of columns, 16 lines at a time; the 16 sums are added up in order.
template <typename T>
__global__ void __launch_bounds__(512) line_sum_kernel(const float* __restrict__ lines, int n_lines, int64_t cols, T* __restrict__ out) {
  __shared__ float part[16][32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float s = 0;
  if (c < cols)
    for (int i = warp; i < n_lines; i += 16) s += lines[(int64_t)i * cols + c];
  part[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || c >= cols) return;
  for (int i = 1; i < 16; i++) s += part[i][lane];
  out[c] = from_f32<T>(s);
}

static inline unsigned grid_of(int64_t items, int64_t most) { return (unsigned)(items < most ? items : most); }
constexpr int kBackwardBlocks = 148;   // one a multiprocessor
constexpr int kLongBlocks = 148 * 4;

// Whether rows from `p` on, `stride` apart, begin on 16 bytes.
static bool rows_aligned(const void* p, int64_t stride, int64_t rows, int size) { return aligned(p, 16) && (rows <= 1 || stride * size % 16 == 0); }

// How a row is dealt out: P threads with K chunks of C values each.  K = 0: too long for registers.
struct Deal {
  int C, P, K;
};

static Deal deal_of(int64_t cols, int size, bool vectors) {
  Deal d;
  d.C = vectors && cols % (16 / size) == 0 ? 16 / size : 1;
  const int64_t chunks = round_up(cols, kGroup) / d.C;
  const int most = d.C == 1 ? 16 : 4;
  d.P = chunks <= 32 * most ? 32 : chunks <= 128 * most ? 128 : chunks <= 256 * most ? 256 : chunks <= 512 * most ? 512 : 1024;
  const int64_t k = (chunks + d.P - 1) / d.P;
  d.K = k > most ? 0 : d.C == 1 ? (k <= 4 ? 4 : 16) : k <= 1 ? 1 : k <= 2 ? 2 : 4;
  return d;
}

// Calls f with C, P and K as constants, for every deal that deal_of makes.
template <typename T, typename F>
static void with_deal(const Deal& d, F f) {
  constexpr int V = 16 / (int)sizeof(T);
#define CASE(c, p, k) \
  if (d.C == c && d.P == p && d.K == k) return f(std::integral_constant<int, c>(), std::integral_constant<int, p>(), std::integral_constant<int, k>())
  CASE(V, 32, 1);
  CASE(V, 32, 2);
  CASE(V, 32, 4);
  CASE(V, 128, 2);
  CASE(V, 128, 4);
  CASE(V, 256, 4);
  CASE(V, 512, 4);
  CASE(V, 1024, 4);
  CASE(1, 32, 4);
  CASE(1, 32, 16);
  CASE(1, 128, 16);
  CASE(1, 256, 16);
  CASE(1, 512, 16);
  CASE(1, 1024, 16);
#undef CASE
}

}  // namespace act
}  // namespace optimi

using namespace optimi;
using namespace optimi::act;

#define FOR_DTYPE(dtype, ...)                                          \
  do {                                                                 \
    if ((dtype) == OPTIMI_F32) { using T = float; __VA_ARGS__; }       \
    else if ((dtype) == OPTIMI_BF16) { using T = __nv_bfloat16; __VA_ARGS__; } \
    else { using T = __half; __VA_ARGS__; }                            \
  } while (0)

static int check_shape(const char* fn, int64_t rows, int64_t cols, int dtype) {
  if (!known_dtype(dtype)) return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", fn, dtype);
  if (rows < 0 || cols < 0 || rows > INT32_MAX || cols > INT32_MAX)
    return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: %lld rows of %lld values are outside 0..2^31-1", fn, (long long)rows, (long long)cols);
  return OPTIMI_OK;
}

template <typename T, int C>
static void launch_compress(const void* x, int64_t stride, int64_t rows, int64_t cols, void* codes, int64_t pitch, void* exponents,
                            int64_t epitch, cudaStream_t s) {
  const int64_t chunks = round_up(cols, kGroup) / C, items = rows * chunks;
  const bool flat = rows == 1 ? cols % kGroup == 0 : cols % kGroup == 0 && stride == cols && pitch == cols && epitch * kGroup == cols;
  const unsigned blocks = (unsigned)((items + kBlock * kUnroll - 1) / (kBlock * kUnroll));
  if (flat)
    compress_kernel<T, C, true><<<blocks, kBlock, 0, s>>>((const T*)x, items, chunks, cols, stride, (int8_t*)codes, pitch, (uint8_t*)exponents, epitch);
  else
    compress_kernel<T, C, false><<<blocks, kBlock, 0, s>>>((const T*)x, items, chunks, cols, stride, (int8_t*)codes, pitch, (uint8_t*)exponents, epitch);
}

template <typename T, int C>
static void launch_decompress(const void* codes, int64_t pitch, const void* exponents, int64_t epitch, const void* scale, int64_t rows,
                              int64_t cols, void* out, cudaStream_t s) {
  const int64_t chunks = round_up(cols, kGroup) / C, items = rows * chunks;
  const bool flat = rows == 1 ? cols % kGroup == 0 : cols % kGroup == 0 && pitch == cols && epitch * kGroup == cols;
  const unsigned blocks = (unsigned)((items + kBlock * kUnroll - 1) / (kBlock * kUnroll));
#define LAUNCH(is_flat, is_scaled)                                                                                                       \
  decompress_kernel<T, C, is_flat, is_scaled><<<blocks, kBlock, 0, s>>>((const int8_t*)codes, pitch, (const uint8_t*)exponents, epitch, \
                                                                        (const T*)scale, items, chunks, cols, (T*)out)
  if (flat) {
    if (scale) LAUNCH(true, true);
    else LAUNCH(true, false);
  } else {
    if (scale) LAUNCH(false, true);
    else LAUNCH(false, false);
  }
#undef LAUNCH
}

// Items of the largest launch: a grid has at most 2^31 - 1 blocks.
static int check_items(const char* fn, int64_t rows, int64_t cols) {
  if (rows * round_up(cols, kGroup) / (kBlock * kUnroll) >= INT32_MAX)
    return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: %lld rows of %lld values are too many for one call", fn, (long long)rows, (long long)cols);
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
  if (rc == OPTIMI_OK) rc = check_items(fn, rows, cols);
  if (rc != OPTIMI_OK) return rc;
  FOR_DTYPE(dtype, {
    constexpr int V = 16 / (int)sizeof(T);
    if (cols % V == 0 && rows_aligned(x, x_stride, rows, sizeof(T)))
      launch_compress<T, V>(x, x_stride, rows, cols, codes, code_pitch, exponents, exponent_pitch, (cudaStream_t)stream);
    else
      launch_compress<T, 1>(x, x_stride, rows, cols, codes, code_pitch, exponents, exponent_pitch, (cudaStream_t)stream);
  });
  return launched(fn);
}

int optimi_b200_decompress(const void* codes, int64_t code_pitch, const void* exponents, int64_t exponent_pitch,
                           const void* channel_scale, int64_t rows, int64_t cols, int dtype, void* out, void* stream) {
  const char* fn = "optimi_b200_decompress";
  int rc = check_shape(fn, rows, cols, dtype);
  if (rc != OPTIMI_OK || rows == 0 || cols == 0) return rc;
  if (!out) return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: out is NULL", fn);
  rc = check_codes(fn, codes, code_pitch, exponents, exponent_pitch, cols);
  if (rc == OPTIMI_OK) rc = check_items(fn, rows, cols);
  if (rc != OPTIMI_OK) return rc;
  FOR_DTYPE(dtype, {
    constexpr int V = 16 / (int)sizeof(T);
    if (cols % V == 0 && aligned(out, 16))
      launch_decompress<T, V>(codes, code_pitch, exponents, exponent_pitch, channel_scale, rows, cols, out, (cudaStream_t)stream);
    else
      launch_decompress<T, 1>(codes, code_pitch, exponents, exponent_pitch, channel_scale, rows, cols, out, (cudaStream_t)stream);
  });
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
  const bool keep = codes || exponents || rstd;
  if (keep) {
    rc = check_codes(fn, codes, code_pitch, exponents, exponent_pitch, cols);
    if (rc != OPTIMI_OK) return rc;
    if (!rstd) return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: codes, exponents and rstd go together", fn);
  }
  cudaStream_t s = (cudaStream_t)stream;
  const int size = dtype == OPTIMI_F32 ? 4 : 2;
  const bool vectors = rows_aligned(x, x_stride, rows, size) && (!residual || rows_aligned(residual, residual_stride, rows, size)) &&
                       (!weight || aligned(weight, 16)) && aligned(y, 16) && (!sum || aligned(sum, 16));
  const Deal d = deal_of(cols, size, vectors);
  FOR_DTYPE(dtype, {
    if (d.K == 0) {
      long_rms_norm_kernel<T><<<grid_of(rows, 1 << 20), 512, 0, s>>>((const T*)x, x_stride, (const T*)residual, residual_stride, (const T*)weight,
                                                                    rows, cols, eps, (T*)y, (T*)sum, (int8_t*)codes, code_pitch,
                                                                    (uint8_t*)exponents, exponent_pitch, rstd);
    } else {
      with_deal<T>(d, [&](auto c, auto p, auto k) {
        constexpr int C = decltype(c)::value, P = decltype(p)::value, K = decltype(k)::value, kThreads = P < 128 ? 128 : P;
        const unsigned blocks = grid_of((rows + kThreads / P - 1) / (kThreads / P), 1 << 20);
        if (keep)
          rms_norm_kernel<T, C, P, K, true><<<blocks, kThreads, 0, s>>>((const T*)x, x_stride, (const T*)residual, residual_stride, (const T*)weight,
                                                                       rows, (int)cols, eps, (T*)y, (T*)sum, (int8_t*)codes, code_pitch,
                                                                       (uint8_t*)exponents, exponent_pitch, rstd);
        else
          rms_norm_kernel<T, C, P, K, false><<<blocks, kThreads, 0, s>>>((const T*)x, x_stride, (const T*)residual, residual_stride, (const T*)weight,
                                                                        rows, (int)cols, eps, (T*)y, (T*)sum, nullptr, 0, nullptr, 0, nullptr);
      });
    }
  });
  return launched(fn);
}

// Blocks of the backward pass, and so lines of its workspace: the kernels for rows in registers take at most 148 blocks, the one
// for long rows four times as many.
static unsigned backward_blocks(int64_t rows) { return grid_of(rows, kLongBlocks); }

size_t optimi_b200_rms_norm_backward_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return (size_t)backward_blocks(rows) * (size_t)cols * sizeof(float);
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
  const int size = dtype == OPTIMI_F32 ? 4 : 2;
  const bool vectors = rows_aligned(grad, grad_stride, rows, size) && (!grad_sum || rows_aligned(grad_sum, grad_sum_stride, rows, size)) &&
                       (!weight || aligned(weight, 16)) && (!grad_input || aligned(grad_input, 16));
  const Deal d = deal_of(cols, size, vectors);
  float* lines = grad_weight ? (float*)workspace : nullptr;
  unsigned blocks = 0;
  FOR_DTYPE(dtype, {
    if (d.K == 0 || d.P > 512) {
      blocks = backward_blocks(rows);
      long_rms_norm_backward_kernel<T><<<blocks, 512, 0, s>>>((const T*)grad, grad_stride, (const T*)grad_sum, grad_sum_stride, (const int8_t*)codes,
                                                              code_pitch, (const uint8_t*)exponents, exponent_pitch, rstd, (const T*)weight,
                                                              rows, cols, (T*)grad_input, lines);
    } else {
      with_deal<T>(d, [&](auto c, auto p, auto k) {
        constexpr int C = decltype(c)::value, P = decltype(p)::value, K = decltype(k)::value, kThreads = 512;
        if constexpr (P <= 512) {
          blocks = grid_of((rows + kThreads / P - 1) / (kThreads / P), kBackwardBlocks);
          rms_norm_backward_kernel<T, C, P, K, kThreads><<<blocks, kThreads, kThreads > P ? (size_t)cols * sizeof(float) : 0, s>>>(
              (const T*)grad, grad_stride, (const T*)grad_sum, grad_sum_stride, (const int8_t*)codes, code_pitch, (const uint8_t*)exponents,
              exponent_pitch, rstd, (const T*)weight, rows, (int)cols, (T*)grad_input, lines);
        }
      });
    }
  });
  rc = launched(fn);
  if (rc != OPTIMI_OK || !grad_weight) return rc;
  FOR_DTYPE(dtype, (line_sum_kernel<T><<<(unsigned)((cols + 31) / 32), 512, 0, s>>>(lines, (int)blocks, cols, (T*)grad_weight)));
  return launched(fn);
}

}  // extern "C"
