// Activations kept in 8 bits (format: activation_common.cuh) and the RMS norm that writes and reads them.
#include "activation_common.cuh"
#include "activation_offsets.h"

namespace optimi {
namespace act {

// ---------------------------------------------------------------------------------------------
// store and restore
// ---------------------------------------------------------------------------------------------
// Both stream: an item is a chunk of C values in one thread (the neighbouring lanes of a group find its largest magnitude
// together), kUnroll items a thread are loaded before the first is used, and nothing is read or written twice.  Bound by HBM:
// 8192 x 14336 bf16 stored and restored in 112 us, 6.3 TB/s (0.98 of the measured copy rate); a warp to a group with one value a lane
// took 688 us.  Rows of odd width spend their time on shifting: 4096 x 4095 bf16 19 us each way, 4096 x 4096 under 13 (76 % of the
// issue slots used in storing, 82 % in restoring, 38 to 45 % of the memory's rate).
constexpr int kBlock = 256, kUnroll = 4;

static __device__ __forceinline__ void divide(int a, int b, int* quotient, int* rest) {
  *quotient = (uint32_t)a / (uint32_t)b;
  *rest = (uint32_t)a % (uint32_t)b;
}
static __device__ __forceinline__ void divide(int64_t a, int64_t b, int64_t* quotient, int64_t* rest) {
  if (((a | b) >> 31) == 0) {
    *quotient = (uint32_t)a / (uint32_t)b;
    *rest = (uint32_t)a % (uint32_t)b;
  } else {
    *quotient = a / b;
    *rest = a % b;
  }
}

// The rows and columns (in units of `per_row` a row) of the items that a thread takes: one division, then steps of kBlock items.  I:
// int where all offsets fit, else 64 bits (4096 x 4095 bf16 restored: 18.5 us, 26.7 with 64 bits).
template <typename I>
struct Walk {
  I row, col;
  I rows_on, cols_on, per_row;
  __device__ __forceinline__ Walk(I item, I step, I units_per_row) : per_row(units_per_row) {
    divide(item, per_row, &row, &col);
    divide(step, per_row, &rows_on, &cols_on);
  }
  __device__ __forceinline__ void on() {
    row += rows_on, col += cols_on;
    if (col >= per_row) col -= per_row, row++;
  }
};

// How the rows of the 16-bit or 32-bit tensor lie.  kFlat: whole groups, one row after another without a gap, so that it is one
// long row and nothing is divided.  kRows: every row begins on 16 bytes and is whole chunks.  kAny: neither.
enum Lie : int { kFlat, kRows, kAny };

template <typename T, int kLie, typename I>
__global__ void __launch_bounds__(kBlock) compress_kernel(const T* __restrict__ x, I items, I chunks, I cols, I stride, int8_t* __restrict__ codes,
                                                          I pitch, uint8_t* __restrict__ exponents, I epitch) {
  constexpr int C = Chunk<T>::C, kLanes = Chunk<T>::kLanes;
  const I first = (I)blockIdx.x * (kBlock * kUnroll) + threadIdx.x;
  Fetched<T, kLie == kAny> in[kUnroll];
  I row[kUnroll], col[kUnroll];
  int n[kUnroll];
  Walk<I> walk(kLie == kFlat ? 0 : first, kBlock, kLie == kFlat ? 1 : chunks);
#pragma unroll
  for (int u = 0; u < kUnroll; u++) {
    const I item = first + u * kBlock;
    row[u] = kLie == kFlat ? 0 : walk.row, col[u] = (kLie == kFlat ? item : walk.col) * C;
    if (kLie != kFlat) walk.on();
    n[u] = item >= items ? 0 : kLie == kFlat ? C : (int)min((I)C, cols - col[u]);
    in[u].fetch(x + row[u] * stride + col[u], n[u]);
  }
#pragma unroll
  for (int u = 0; u < kUnroll; u++) {
    const Chunk<T> v = in[u].settle(x + row[u] * stride + col[u], n[u]);
    const int e = group_exponent<T>(group_max<kLanes>(v.amax()));
    float f[C];
#pragma unroll
    for (int i = 0; i < C; i++) f[i] = v.get(i);
    CodeChunk<C> c;
    c.template encode<T>(f, e);
    if (first + u * kBlock < items) {
      c.store(codes + row[u] * pitch + col[u]);
      if (threadIdx.x % kLanes == 0) exponents[row[u] * epitch + col[u] / kGroup] = (uint8_t)e;
    }
  }
}

template <typename T, int kLie, bool kScaled>
__global__ void __launch_bounds__(kBlock) decompress_kernel(const int8_t* __restrict__ codes, int64_t pitch, const uint8_t* __restrict__ exponents,
                                                            int64_t epitch, const T* __restrict__ channel_scale, int64_t items,
                                                            int64_t chunks, int64_t cols, T* __restrict__ out) {
  constexpr int C = Chunk<T>::C;
  const int64_t first = (int64_t)blockIdx.x * (kBlock * kUnroll) + threadIdx.x;
  CodeChunk<C> c[kUnroll];
  uint32_t e[kUnroll];
  int64_t row[kUnroll], col[kUnroll];
  Walk<int64_t> walk(kLie == kFlat ? 0 : first, kBlock, kLie == kFlat ? 1 : chunks);
#pragma unroll
  for (int u = 0; u < kUnroll; u++) {
    const int64_t item = first + u * kBlock;
    row[u] = kLie == kFlat ? 0 : walk.row, col[u] = (kLie == kFlat ? item : walk.col) * C;
    if (kLie != kFlat) walk.on();
    c[u].clear(), e[u] = 0;
    if (item < items) {
      c[u].load(codes + row[u] * pitch + col[u]);
      e[u] = exponents[row[u] * epitch + col[u] / kGroup];
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; u++) {
    if (first + u * kBlock >= items) return;
    if (kLie != kFlat && col[u] >= cols) continue;
    Chunk<T> v;
    if constexpr (sizeof(T) == 2 && !kScaled) {
      const uint32_t s = scale_pair<T>(e[u], 0x4040);
#pragma unroll
      for (int i = 0; i < 4; i++) v.w[i] = code_pair<T>(c[u].w[i / 2], i % 2 ? 0x4342 : 0x4140, s);
    } else {
      float f[C];
      const float s = power_of((int)e[u]);
#pragma unroll
      for (int i = 0; i < C; i++) {
        f[i] = __fmul_rn(c[u].get(i), s);
        if (kScaled) f[i] = __fmul_rn(f[i], to_f32(channel_scale[(kLie == kFlat ? col[u] % cols : col[u]) + i]));
      }
      v.set(f);
    }
    v.store(out + row[u] * cols + col[u]);
  }
}

// Rows that begin anywhere, copied to rows that begin on 16 bytes (zeros up to the pitch): the tensor copy engine, which feeds the
// weight gradient, loads nothing else.
template <typename T>
__global__ void __launch_bounds__(kBlock) align_rows_kernel(const T* __restrict__ x, int64_t items, int64_t chunks, int64_t cols, int64_t stride,
                                                            T* __restrict__ out) {
  constexpr int C = Chunk<T>::C;
  const int64_t first = (int64_t)blockIdx.x * (kBlock * kUnroll) + threadIdx.x;
  Fetched<T, true> in[kUnroll];
  const T* from[kUnroll];
  int n[kUnroll];
  Walk<int64_t> walk(first, kBlock, chunks);
#pragma unroll
  for (int u = 0; u < kUnroll; u++, walk.on()) {
    from[u] = x + walk.row * stride + walk.col * C;
    n[u] = first + u * kBlock < items ? (int)min((int64_t)C, cols - walk.col * C) : 0;
    in[u].fetch(from[u], n[u]);
  }
#pragma unroll
  for (int u = 0; u < kUnroll; u++)
    if (first + u * kBlock < items) in[u].settle(from[u], n[u]).store(out + (first + u * kBlock) * C);
}

// decompress for rows that begin anywhere.  The result has no gaps, so an item is one 16-byte block of it as a whole; its codes lie at
// any byte of a row (whose pitch is a multiple of 32), and a block that reaches into the next row takes them one by one.
template <typename T, bool kScaled, typename I>
__global__ void __launch_bounds__(kBlock) decompress_any_kernel(const int8_t* __restrict__ codes, I pitch, const uint8_t* __restrict__ exponents,
                                                                I epitch, const T* __restrict__ channel_scale, I values, I cols,
                                                                T* __restrict__ out) {
  constexpr int C = Chunk<T>::C;
  const I first = (I)blockIdx.x * (kBlock * kUnroll) + threadIdx.x;
  uint32_t w[kUnroll][C / 4 + 1];
  uint32_t low[kUnroll], high[kUnroll];
  I col[kUnroll];
  Walk<I> walk(first * C, kBlock * C, cols);
#pragma unroll
  for (int u = 0; u < kUnroll; u++, walk.on()) {
    col[u] = walk.col;
#pragma unroll
    for (int i = 0; i <= C / 4; i++) w[u][i] = 0;
    low[u] = high[u] = 0;
    if ((first + u * kBlock) * C < values && walk.col + C <= cols) {
      const uint32_t* words = reinterpret_cast<const uint32_t*>(codes + walk.row * pitch + (walk.col & ~(I)3));
#pragma unroll
      for (int i = 0; i < C / 4; i++) w[u][i] = words[i];
      if (walk.col & 3) w[u][C / 4] = words[C / 4];  // the last code asked for lies there
      const uint8_t* group = exponents + walk.row * epitch + walk.col / kGroup;
      low[u] = group[0], high[u] = group[((int)(walk.col % kGroup) + C - 1) / kGroup];
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; u++) {
    const I at = (first + u * kBlock) * C;
    if (at >= values) return;
    float f[C];
    if (col[u] + C <= cols) {
      CodeChunk<C> c;
#pragma unroll
      for (int i = 0; i < C / 4; i++) c.w[i] = __funnelshift_r(w[u][i], w[u][i + 1], (uint32_t)(col[u] & 3) * 8);
      const int in = (int)(col[u] % kGroup);
#pragma unroll
      for (int i = 0; i < C; i++) f[i] = __fmul_rn(c.get(i), power_of((int)(in + i < kGroup ? low[u] : high[u])));
    } else {
#pragma unroll
      for (int i = 0; i < C; i++) {
        I r, k;
        divide(min(at + i, values - 1), cols, &r, &k);
        f[i] = __fmul_rn((float)codes[r * pitch + k], power_of(exponents[r * epitch + k / kGroup]));
      }
    }
    if constexpr (kScaled) {
#pragma unroll
      for (int i = 0; i < C; i++) f[i] = __fmul_rn(f[i], to_f32(channel_scale[(col[u] + i) % cols]));
    }
    Chunk<T> v;
    v.set(f);
    if (at + C <= values) {
      v.store(out + at);
    } else {
#pragma unroll
      for (int i = 0; i < C; i++)
        if (at + i < values) v.store_value(out + at, i);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// residual addition + RMS norm
// ---------------------------------------------------------------------------------------------
//     h = round(x + r)      rstd = (mean(h^2) + eps)^-1/2      xn = h * rstd      y = round(xn * w)
// and the 8-bit form of xn (without w, so that one checkpoint serves this norm's backward pass and, with w applied to the
// columns of its result, the weight gradient of every linear layer that reads y).
//
// A row belongs to P threads, each with K chunks of it in registers from the first load to the last store, so that every value is read
// once.  Bound by HBM: 16384 x 4096 bf16 with residual 82 us without the 8-bit form (6.6 TB/s), 97 to 102 us with it.
//
// The normalised value is held in F: fp32, and 64 bits for fp32 activations, whose gradients would show a code that a
// last-bit difference of rstd tips over.
template <typename T> struct Wide { using type = float; };
template <> struct Wide<float> { using type = double; };

// What the weight's gradient, a sum over all tokens, is added up in: for fp32 results 64 bits, as 60,000 terms of either sign leave
// little more than five digits of a 32-bit sum.
template <typename T> struct Total { using type = float; };
template <> struct Total<float> { using type = double; };
static __device__ __forceinline__ float add_product(float a, float b, float sum) { return __fmaf_rn(a, b, sum); }
static __device__ __forceinline__ double add_product(float a, float b, double sum) { return __fma_rn((double)a, (double)b, sum); }

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

template <typename T, bool kAny>
static __device__ __forceinline__ void store_chunk(const Chunk<T>& v, T* row, int c, int cols) {
  if constexpr (kAny) v.store_any(row + c, cols - c);
  else if (c < cols) v.store(row + c);
}

// A chunk of the weight; ones where there is none, so that the loops over values ask nothing.
template <typename T, bool kAny>
static __device__ __forceinline__ Chunk<T> weight_chunk(const T* weight, int c, int cols) {
  Chunk<T> v;
  if (weight) {
    Fetched<T, kAny> in;
    in.fetch(weight + c, cols - c);
    v = in.settle(weight + c, cols - c);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) v.w[i] = std::is_same<T, float>::value ? 0x3f800000u : std::is_same<T, __half>::value ? 0x3c003c00u : 0x3f803f80u;
  }
  return v;
}

template <typename T, int P, int K, bool kAny, bool kKeep>
__global__ void __launch_bounds__(P < 128 ? 128 : P, kAny && K <= 2 ? 1024 / (P < 128 ? 128 : P) : 0)
    rms_norm_kernel(const T* __restrict__ x, int64_t xs, const T* __restrict__ residual, int64_t rs, const T* __restrict__ weight,
                    int64_t rows, int cols, double eps, T* __restrict__ y, T* __restrict__ sum, int8_t* __restrict__ codes, int64_t pitch,
                    uint8_t* __restrict__ exponents, int64_t epitch, float* __restrict__ rstd_out) {
  using F = typename Wide<T>::type;
  using Values = Chunk<T>;
  constexpr int C = Values::C, kGroups = (P < 128 ? 128 : P) / P;
  __shared__ F part[kGroups][2][P / 32];
  const int group = threadIdx.x / P, t = threadIdx.x % P;
  const int padded = (cols + kGroup - 1) / kGroup * kGroup;
  Values w[K];
#pragma unroll
  for (int k = 0; k < K; k++) w[k] = weight_chunk<T, kAny>(weight, (k * P + t) * C, cols);
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * kGroups + group; row < rows; row += (int64_t)gridDim.x * kGroups, turn++) {
    Values h[K];
    F ss = 0;
    const auto add = [&](int k, const Values& r) {
      float f[C];
#pragma unroll
      for (int i = 0; i < C; i++) f[i] = __fadd_rn(h[k].get(i), r.get(i));
      h[k].set(f);
      store_chunk<T, kAny>(h[k], sum + row * cols, (k * P + t) * C, cols);
    };
    if constexpr (kAny) {
      Fetched<T, true> in[K], more[K];
#pragma unroll
      for (int k = 0; k < K; k++) {
        const int c = (k * P + t) * C;
        in[k].fetch(x + row * xs + c, cols - c);
        more[k].fetch(residual + row * rs + c, residual ? cols - c : 0);
      }
#pragma unroll
      for (int k = 0; k < K; k++) {
        const int c = (k * P + t) * C;
        h[k] = in[k].settle(x + row * xs + c, cols - c);
        if (residual) add(k, more[k].settle(residual + row * rs + c, cols - c));
      }
    } else {
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
        for (int k = 0; k < K; k++) add(k, r[k]);
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
        f[i] = (float)(n[i] * (F)w[k].get(i));
      }
      Values out;
      out.set(f);
      store_chunk<T, kAny>(out, y + row * cols, c, cols);
      if constexpr (kKeep) {
        // rounding keeps the order of magnitudes, so the largest |h| times rstd is the largest |xn|
        const F top = (F)__uint_as_float(group_max<Values::kLanes>(h[k].amax())) * rstd;
        const int e = exponent_of<T, F>(magnitude(top));
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
// (its row groups added up in order in shared memory); a second kernel adds up the lines in order.  Few blocks, so few lines; with
// few rows one block takes them all and writes dw itself (`direct`): the second launch costs more than up to four rows in turn.
// 16384 x 4096 bf16: 83 to 92 us, 0.8 of the copy rate; 72 % of the issue slots are used, the rest waits at the row's barrier.
// The next row is asked for before this one is reduced (kAhead), so that loads are always under way.  Long rows (K > 2) have no
// registers for that, nor for the weight, which they read again for every row, nor for dsum, asked for after the first pass.
template <typename T, int K, bool kAny>
struct BackwardRow {
  Fetched<T, kAny> g[K], s[K];
  CodeChunk<Chunk<T>::C> code[K];
  uint32_t e[K];
  float r;
};

template <typename T, int P, int K, bool kAny>
__global__ void __launch_bounds__(512, 1)
    rms_norm_backward_kernel(const T* __restrict__ grad, int64_t gs, const T* __restrict__ grad_sum, int64_t hs, const int8_t* __restrict__ codes,
                             int64_t pitch, const uint8_t* __restrict__ exponents, int64_t epitch, const float* __restrict__ rstd,
                             const T* __restrict__ weight, int64_t rows, int cols, T* __restrict__ dx,
                             typename Total<T>::type* __restrict__ lines, T* __restrict__ direct) {
  using Values = Chunk<T>;
  using A = typename Total<T>::type;
  constexpr bool kAhead = K <= 2;
  constexpr int C = Values::C, kThreads = 512, kGroups = kThreads / P;
  __shared__ float part[kGroups][2][P / 32];
  __shared__ A sums[kGroups > 1 ? kGroups : 1][kGroups > 1 ? P * K * C + 4 : 1];
  const int group = threadIdx.x / P, t = threadIdx.x % P;
  Values w[K];
  A dw[K][C];
  const auto weights = [&](int k) { return weight_chunk<T, kAny>(weight, (k * P + t) * C, cols); };
#pragma unroll
  for (int k = 0; k < K; k++) {
    if constexpr (kAhead) w[k] = weights(k);
#pragma unroll
    for (int i = 0; i < C; i++) dw[k][i] = 0;
  }
  const int64_t step = (int64_t)gridDim.x * kGroups;
  const auto ask_sum = [&](int64_t row, BackwardRow<T, K, kAny>& v) {
#pragma unroll
    for (int k = 0; k < K; k++) {
      const int c = (k * P + t) * C;
      v.s[k].fetch(grad_sum + row * hs + c, grad_sum && dx ? cols - c : 0);
    }
  };
  const auto ask = [&](int64_t row, BackwardRow<T, K, kAny>& v) {
    if (row >= rows) return;
    v.r = rstd[row];
#pragma unroll
    for (int k = 0; k < K; k++) {
      const int c = (k * P + t) * C;
      v.g[k].fetch(grad + row * gs + c, cols - c);
      v.code[k].clear(), v.e[k] = 0;
      if (c < cols) {
        v.code[k].load(codes + row * pitch + c);
        v.e[k] = exponents[row * epitch + c / kGroup];
      }
    }
    if constexpr (kAhead) ask_sum(row, v);
  };
  int turn = 0;
  BackwardRow<T, K, kAny> v, next;
  int64_t row = (int64_t)blockIdx.x * kGroups + group;
  ask(row, v);
  for (; row < rows; row += step, turn++) {
    if constexpr (kAhead) ask(row + step, next);
    Values g[K];
    float m = 0;
#pragma unroll
    for (int k = 0; k < K; k++) {
      const int c = (k * P + t) * C;
      g[k] = v.g[k].settle(grad + row * gs + c, cols - c);
      // |xn| is below sqrt(cols), so a unit is far below 2^100 (or infinite, of a NaN group, which stays NaN)
      const float unit = power_of((int)v.e[k]), offset = v.code[k].scaled_offset(unit);
      Values wk;
      if constexpr (kAhead) wk = w[k];
      else wk = weights(k);
#pragma unroll
      for (int i = 0; i < C; i++) {
        const float n = v.code[k].get_scaled(i, unit, offset), d = g[k].get(i);
        dw[k][i] = add_product(d, n, dw[k][i]);
        m = __fmaf_rn(__fmul_rn(d, wk.get(i)), n, m);
      }
    }
    if (dx) {
      if constexpr (!kAhead) ask_sum(row, v);
      m = row_sum<P, float>(m, part[group], turn, group) / (float)cols;
      const float mr = -__fmul_rn(m, v.r);
#pragma unroll
      for (int k = 0; k < K; k++) {
        const int c = (k * P + t) * C;
        const float unit = power_of((int)v.e[k]), offset = v.code[k].scaled_offset(unit);
        Values wk;
        if constexpr (kAhead) wk = w[k];
        else wk = weights(k);
        const Values s = v.s[k].settle(grad_sum + row * hs + c, cols - c);  // zeros where there is none
        float f[C];
#pragma unroll
        for (int i = 0; i < C; i++) {  // rstd * g + dsum, then - xn * (m * rstd)
          f[i] = __fmaf_rn(v.r, __fmul_rn(g[k].get(i), wk.get(i)), s.get(i));
          f[i] = __fmaf_rn(v.code[k].get_scaled(i, unit, offset), mr, f[i]);
        }
        Values out;
        out.set(f);
        store_chunk<T, kAny>(out, dx + row * cols, c, cols);
      }
    }
    if constexpr (kAhead) v = next;
    else ask(row + step, v);
  }
  if (!lines && !direct) return;
  if constexpr (kGroups == 1) {
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
      for (int i = 0; i < C; i++) {
        const int c = (k * P + t) * C + i;
        if (c >= cols) continue;
        if (direct) direct[c] = from_f32<T>((float)dw[k][i]);
        else lines[(int64_t)blockIdx.x * cols + c] = dw[k][i];
      }
  } else {
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
      for (int i = 0; i < C; i++) sums[group][(k * P + t) * C + i] = dw[k][i];
    __syncthreads();
    for (int c = threadIdx.x; c < cols; c += kThreads) {
      A s = sums[0][c];
#pragma unroll
      for (int j = 1; j < kGroups; j++) s += sums[j][c];
      if (direct) direct[c] = from_f32<T>((float)s);
      else lines[(int64_t)blockIdx.x * cols + c] = s;
    }
  }
}

template <typename T>
__global__ void long_rms_norm_backward_kernel(const T* __restrict__ grad, int64_t gs, const T* __restrict__ grad_sum, int64_t hs,
                                              const int8_t* __restrict__ codes, int64_t pitch, const uint8_t* __restrict__ exponents,
                                              int64_t epitch, const float* __restrict__ rstd, const T* __restrict__ weight, int64_t rows,
                                              int64_t cols, T* __restrict__ dx, typename Total<T>::type* __restrict__ lines) {
  typename Total<T>::type* line = lines ? lines + (int64_t)blockIdx.x * cols : nullptr;
  if (line)
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) line[c] = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    float m = 0;
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
      const float n = (float)codes[row * pitch + c] * power_of(exponents[row * epitch + c / kGroup]);
      const float g = to_f32(grad[row * gs + c]);
      m += (weight ? g * to_f32(weight[c]) : g) * n;
      if (line) line[c] = add_product(g, n, line[c]);
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
__global__ void __launch_bounds__(512) line_sum_kernel(const typename Total<T>::type* __restrict__ lines, int n_lines, int64_t cols,
                                                       T* __restrict__ out) {
  using A = typename Total<T>::type;
  __shared__ A part[16][32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  A s = 0;
  if (c < cols)
    for (int i = warp; i < n_lines; i += 16) s += lines[(int64_t)i * cols + c];
  part[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || c >= cols) return;
  for (int i = 1; i < 16; i++) s += part[i][lane];
  out[c] = from_f32<T>((float)s);
}

static inline unsigned grid_of(int64_t items, int64_t most) { return (unsigned)(items < most ? items : most); }
constexpr int kBackwardBlocks = 148;   // one a multiprocessor
constexpr int kLongBlocks = 148 * 4;

// Whether rows from `p` on, `stride` apart, begin on 16 bytes.
static bool rows_aligned(const void* p, int64_t stride, int64_t rows, int size) { return aligned(p, 16) && (rows <= 1 || stride * size % 16 == 0); }

// How a row is dealt out: P threads with K chunks each, K at most `most` as long as 512 threads are enough.  K = 0: too long for
// registers.  16384 x 4096 bf16, K = 1, 2, 4: forward 141, 108, 100 us; backward 113, 90, 136 us (for 4 there are no registers to
// ask ahead).  Rows that begin anywhere, 4096 x 4095, K = 1, 2, 4: forward 59, 51, 61 us; backward, K = 1, 2: 60, 77 us (two chunks
// and the next row's two do not fit into registers; with fewer operations a value, and K = 1, now 50 us).
constexpr int kForwardChunks = 4, kForwardAnyChunks = 2, kBackwardChunks = 2, kBackwardAnyChunks = 1;

struct Deal {
  int P, K;
};

static Deal deal_of(int64_t cols, int size, int most) {
  const int64_t chunks = round_up(cols, kGroup) * size / 16;
  Deal d;
  d.P = chunks <= 32 * most ? 32 : chunks <= 64 * most ? 64 : chunks <= 128 * most ? 128 : chunks <= 256 * most ? 256 : 512;
  const int64_t k = (chunks + d.P - 1) / d.P;
  d.K = k <= 2 ? (int)k : k <= 4 ? 4 : k <= 8 && size == 4 ? 8 : 0;
  return d;
}

// Calls f with P and K as constants, for every deal that deal_of makes.
template <typename T, int most, typename F>
static void with_deal(const Deal& d, F f) {
#define CASE(p, k) \
  if (d.P == p && d.K == k) return f(std::integral_constant<int, p>(), std::integral_constant<int, k>())
  CASE(32, 1);
  if constexpr (most >= 2) CASE(32, 2);
  if constexpr (most == 4) CASE(32, 4);
  CASE(64, most);
  CASE(128, most);
  CASE(256, most);
  if constexpr (most < 2) CASE(512, 1);
  if constexpr (most <= 2) CASE(512, 2);
  CASE(512, 4);
  if constexpr (sizeof(T) == 4) CASE(512, 8);
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

template <typename T>
static void launch_compress(const void* x, int64_t stride, int64_t rows, int64_t cols, void* codes, int64_t pitch, void* exponents,
                            int64_t epitch, cudaStream_t s) {
  constexpr int C = Chunk<T>::C;
  const int64_t chunks = round_up(cols, kGroup) / C, items = rows * chunks;
  const bool regular = cols % C == 0 && rows_aligned(x, stride, rows, sizeof(T));
  const bool flat = regular && cols % kGroup == 0 && (rows == 1 || (stride == cols && pitch == cols && epitch * kGroup == cols));
  const unsigned blocks = (unsigned)((items + kBlock * kUnroll - 1) / (kBlock * kUnroll));
#define LAUNCH(lie, I)                                                                                                             \
  compress_kernel<T, lie, I><<<blocks, kBlock, 0, s>>>((const T*)x, (I)items, (I)chunks, (I)cols, (I)stride, (int8_t*)codes, (I)pitch, \
                                                       (uint8_t*)exponents, (I)epitch)
  if (flat) LAUNCH(kFlat, int64_t);
  else if (regular) LAUNCH(kRows, int64_t);
  else if (small_offsets(rows, stride, pitch, epitch)) LAUNCH(kAny, int);
  else LAUNCH(kAny, int64_t);
#undef LAUNCH
}

template <typename T, bool kScaled>
static void launch_decompress(const void* codes, int64_t pitch, const void* exponents, int64_t epitch, const void* scale, int64_t rows,
                              int64_t cols, void* out, cudaStream_t s) {
  constexpr int C = Chunk<T>::C;
  const bool regular = cols % C == 0;
  const bool flat = regular && cols % kGroup == 0 && (rows == 1 || (pitch == cols && epitch * kGroup == cols));
  const int64_t chunks = round_up(cols, kGroup) / C, items = regular ? rows * chunks : (rows * cols + C - 1) / C;
  const unsigned blocks = (unsigned)((items + kBlock * kUnroll - 1) / (kBlock * kUnroll));
#define LAUNCH(lie)                                                                                                             \
  decompress_kernel<T, lie, kScaled><<<blocks, kBlock, 0, s>>>((const int8_t*)codes, pitch, (const uint8_t*)exponents, epitch,      \
                                                               (const T*)scale, items, chunks, cols, (T*)out)
  if (flat) LAUNCH(kFlat);
  else if (regular) LAUNCH(kRows);
  else if (small_offsets(rows, cols, pitch, epitch))
    decompress_any_kernel<T, kScaled, int><<<blocks, kBlock, 0, s>>>((const int8_t*)codes, (int)pitch, (const uint8_t*)exponents, (int)epitch,
                                                                     (const T*)scale, (int)(rows * cols), (int)cols, (T*)out);
  else
    decompress_any_kernel<T, kScaled, int64_t><<<blocks, kBlock, 0, s>>>((const int8_t*)codes, pitch, (const uint8_t*)exponents, epitch,
                                                                         (const T*)scale, rows * cols, cols, (T*)out);
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
  FOR_DTYPE(dtype, launch_compress<T>(x, x_stride, rows, cols, codes, code_pitch, exponents, exponent_pitch, (cudaStream_t)stream));
  return launched(fn);
}

int optimi_b200_decompress(const void* codes, int64_t code_pitch, const void* exponents, int64_t exponent_pitch,
                           const void* channel_scale, int64_t rows, int64_t cols, int dtype, void* out, void* stream) {
  const char* fn = "optimi_b200_decompress";
  int rc = check_shape(fn, rows, cols, dtype);
  if (rc != OPTIMI_OK || rows == 0 || cols == 0) return rc;
  if (!out || !aligned(out, 16)) return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: out is NULL or not 16-byte aligned", fn);
  rc = check_codes(fn, codes, code_pitch, exponents, exponent_pitch, cols);
  if (rc == OPTIMI_OK) rc = check_items(fn, rows, cols);
  if (rc != OPTIMI_OK) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  if (channel_scale)
    FOR_DTYPE(dtype, launch_decompress<T, true>(codes, code_pitch, exponents, exponent_pitch, channel_scale, rows, cols, out, s));
  else
    FOR_DTYPE(dtype, launch_decompress<T, false>(codes, code_pitch, exponents, exponent_pitch, nullptr, rows, cols, out, s));
  return launched(fn);
}

int optimi_b200_align_rows(const void* x, int64_t x_stride, int64_t rows, int64_t cols, int dtype, void* out, int64_t out_stride, void* stream) {
  const char* fn = "optimi_b200_align_rows";
  int rc = check_shape(fn, rows, cols, dtype);
  if (rc != OPTIMI_OK || rows == 0 || cols == 0) return rc;
  const int64_t values = dtype == OPTIMI_F32 ? 4 : 8, chunks = (cols + values - 1) / values;
  if (!x || !out || !aligned(out, 16)) return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: x or out is NULL, or out is not 16-byte aligned", fn);
  if (out_stride != chunks * values)
    return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: out_stride is %lld, not %lld (cols up to the next 16 bytes)", fn, (long long)out_stride,
                (long long)(chunks * values));
  rc = check_items(fn, rows, cols);
  if (rc != OPTIMI_OK) return rc;
  const unsigned blocks = (unsigned)((rows * chunks + kBlock * kUnroll - 1) / (kBlock * kUnroll));
  FOR_DTYPE(dtype, (align_rows_kernel<T><<<blocks, kBlock, 0, (cudaStream_t)stream>>>((const T*)x, rows * chunks, chunks, cols, x_stride, (T*)out)));
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
  const bool any = cols * size % 16 || !rows_aligned(x, x_stride, rows, size) || (residual && !rows_aligned(residual, residual_stride, rows, size)) ||
                   !aligned(weight, 16) || !aligned(y, 16) || !aligned(sum, 16);
  const Deal d = deal_of(cols, size, any ? kForwardAnyChunks : kForwardChunks);
  FOR_DTYPE(dtype, {
    if (d.K == 0) {
      long_rms_norm_kernel<T><<<grid_of(rows, 1 << 20), 512, 0, s>>>((const T*)x, x_stride, (const T*)residual, residual_stride, (const T*)weight,
                                                                    rows, cols, eps, (T*)y, (T*)sum, (int8_t*)codes, code_pitch,
                                                                    (uint8_t*)exponents, exponent_pitch, rstd);
    } else {
      const auto with_constants = [&](auto p, auto k, auto is_any) {
        constexpr int P = decltype(p)::value, K = decltype(k)::value, kThreads = P < 128 ? 128 : P;
        constexpr bool kIsAny = decltype(is_any)::value;
        const unsigned blocks = grid_of((rows + kThreads / P - 1) / (kThreads / P), 1 << 20);
        const auto launch = [&](auto kernel) {
          kernel<<<blocks, kThreads, 0, s>>>((const T*)x, x_stride, (const T*)residual, residual_stride, (const T*)weight, rows, (int)cols, eps,
                                             (T*)y, (T*)sum, (int8_t*)codes, code_pitch, (uint8_t*)exponents, exponent_pitch, rstd);
        };
        keep ? launch(rms_norm_kernel<T, P, K, kIsAny, true>) : launch(rms_norm_kernel<T, P, K, kIsAny, false>);
      };
      if (any) with_deal<T, kForwardAnyChunks>(d, [&](auto p, auto k) { with_constants(p, k, std::true_type()); });
      else with_deal<T, kForwardChunks>(d, [&](auto p, auto k) { with_constants(p, k, std::false_type()); });
    }
  });
  return launched(fn);
}

// Whether one block takes all rows of the backward pass.
static bool one_block(int64_t rows, int64_t cols, int size) {
  const Deal d = deal_of(cols, size, kBackwardAnyChunks);
  return d.K > 0 && rows <= 4 * (512 / d.P);
}

// Lines of the backward pass's workspace: the kernels for rows in registers take at most 148 blocks, the one for long rows four times
// as many.
static unsigned backward_blocks(int64_t rows) { return grid_of(rows, kLongBlocks); }

size_t optimi_b200_rms_norm_backward_workspace_bytes(int64_t rows, int64_t cols, int dtype) {
  if (rows <= 0 || cols <= 0 || !known_dtype(dtype) || one_block(rows, cols, dtype == OPTIMI_F32 ? 4 : 2)) return 0;
  return (size_t)backward_blocks(rows) * (size_t)cols * (dtype == OPTIMI_F32 ? sizeof(double) : sizeof(float));
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
  const size_t need = optimi_b200_rms_norm_backward_workspace_bytes(rows, cols, dtype);
  if (grad_weight && need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(OPTIMI_ERR_WORKSPACE_TOO_SMALL, "%s: workspace has %zu bytes, %zu are needed, 16-byte aligned", fn,
                workspace ? workspace_bytes : (size_t)0, need);
  const int size = dtype == OPTIMI_F32 ? 4 : 2;
  const bool any = cols * size % 16 || !rows_aligned(grad, grad_stride, rows, size) || (grad_sum && !rows_aligned(grad_sum, grad_sum_stride, rows, size)) ||
                   !aligned(weight, 16) || !aligned(grad_input, 16);
  const Deal d = deal_of(cols, size, any ? kBackwardAnyChunks : kBackwardChunks);
  const bool alone = one_block(rows, cols, size);
  void* lines = grad_weight && !alone ? workspace : nullptr;
  unsigned blocks = 0;
  FOR_DTYPE(dtype, {
    if (d.K == 0) {
      blocks = backward_blocks(rows);
      long_rms_norm_backward_kernel<T><<<blocks, 512, 0, s>>>((const T*)grad, grad_stride, (const T*)grad_sum, grad_sum_stride, (const int8_t*)codes,
                                                              code_pitch, (const uint8_t*)exponents, exponent_pitch, rstd, (const T*)weight,
                                                              rows, cols, (T*)grad_input, (Total<T>::type*)lines);
    } else {
      const auto with_constants = [&](auto p, auto k, auto is_any) {
        constexpr int P = decltype(p)::value, K = decltype(k)::value;
        constexpr bool kIsAny = decltype(is_any)::value;
        blocks = alone ? 1 : grid_of((rows + 512 / P - 1) / (512 / P), kBackwardBlocks);
        rms_norm_backward_kernel<T, P, K, kIsAny><<<blocks, 512, 0, s>>>(
            (const T*)grad, grad_stride, (const T*)grad_sum, grad_sum_stride, (const int8_t*)codes, code_pitch, (const uint8_t*)exponents,
            exponent_pitch, rstd, (const T*)weight, rows, (int)cols, (T*)grad_input, (typename Total<T>::type*)lines, alone ? (T*)grad_weight : nullptr);
      };
      if (any) with_deal<T, kBackwardAnyChunks>(d, [&](auto p, auto k) { with_constants(p, k, std::true_type()); });
      else with_deal<T, kBackwardChunks>(d, [&](auto p, auto k) { with_constants(p, k, std::false_type()); });
    }
  });
  rc = launched(fn);
  if (rc != OPTIMI_OK || !lines) return rc;
  FOR_DTYPE(dtype, (line_sum_kernel<T><<<(unsigned)((cols + 31) / 32), 512, 0, s>>>((const Total<T>::type*)lines, (int)blocks, cols, (T*)grad_weight)));
  return launched(fn);
}

}  // extern "C"
