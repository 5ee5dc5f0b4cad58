// The weight gradient of a linear layer whose input is held in 8 bits:
//     dW[o, c] = w[c] * sum_t dY[t, o] * X[t, c]        X = code * 2^(e - 127)  (format: activation_common.cuh)
//
// On the tensor cores as D[c, o] = X^T dY with M = channels, N = outputs, K = tokens.  Both operands have the token as
// their slow dimension in memory.  dY goes by TMA into shared memory and is read there with the token as the strided
// (MN-major) dimension.  X^T has to be made from codes, and the result goes to tensor memory, as the left operand of the
// instruction may lie there: a row per channel, tokens along the columns.  That costs shared memory only the codes' own
// bytes (one read of 8 bits a value) where a 16-bit copy beside dY would be written and then read again.
// code * 2^k has 7 bits and fits bf16 and fp16 exactly, so the products are those of the restored activation.
//
// What bounds it: the tensor cores and the card's power.  8192 tokens, 14336 outputs x 4096 channels, bf16: 615 to 625 us alone
// (1540 to 1564 TFLOP/s, 0.93 to 0.94 of the measured product rate) and 735 to 755 us in a long run, where the clock falls to 1.3 GHz
// (a 16-bit product of the same sizes by the vendor's library: 612 to 618 and 716 to 723 us there).  4096 x 1024: 58 to 60 us, 64 tiles on 74 pairs, the
// tensor cores of those 94 % busy.  With few tokens it is the results' way to memory (64 tokens, 4096 x 4096: 23 us).
#include "activation_common.cuh"

#include <cuda.h>

namespace optimi {
namespace act {

// A pair of blocks on two neighbouring SMs works on one tile of 256 channels x 384 outputs (or 256), 64 tokens at a time.  Each
// holds the codes, X^T and the results of its 128 channels, and the gradients of half of the outputs; the instruction reads
// the other half from the partner's shared memory (one block with 128 x 256 of its own loaded twice the gradients: 1175 us for the
// call above, where the pair at first took 768).  A tile is that wide because the conversion of codes, done once a tile and step,
// competes with the multiplications for issue slots and power: 384 outputs 615 us, 256 outputs 670 us.  Seven stages, eight slots or
// a third set of converting warps gained nothing.
constexpr int kM = 128, kN = 384, kK = 64;           // channels of a block, most outputs of the pair, tokens of a step
constexpr int kNarrow = 256;                         // outputs of the first instruction; the second takes the others
constexpr int kStages = 6;                           // of gradients and codes, in shared memory
constexpr int kSlots = 4;                            // of X^T, in tensor memory beside the results
constexpr int kBlockBytes = kK * 128;                // 64 outputs of a step
constexpr int kGradBytes = kN / 2 / 64 * kBlockBytes, kCodeBytes = kK * kM, kStageBytes = kGradBytes + kCodeBytes;
constexpr int kSmemBytes = kStages * kStageBytes + 1024;
constexpr int kAColumns = kK / 2;                    // 32-bit columns of tensor memory of one block of X^T
static_assert(kN + kSlots * kAColumns <= 512, "tensor memory");
constexpr int kMakers = 8, kWriters = 4;             // warps that convert, in two sets that take turns, and warps that write results
constexpr int kLoader = kMakers + kWriters, kIssuer = kLoader + 1;
constexpr int kThreads = 32 * (kIssuer + 1);
constexpr int kSets = kMakers / 4;
constexpr int kBand = 8;                             // tiles of channels that are walked together
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
// False if the phase did not complete within the limit.  For whole warps, and the same in all lanes.
static __device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity) {
  uint32_t done = 0;
  for (int n = 0; n < kWaitLimit && !done; n++)
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\nselp.b32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
  return __all_sync(~0u, done);
}

// True in one lane.  The warps that issue copies and multiplications run their loops with all lanes and branch only around the
// instructions themselves, so that loop counters and descriptors stay in uniform registers: with one lane in a divergent loop, four
// multiplications took 570 to 640 cycles to issue instead of 516.
static __device__ __forceinline__ bool elected() {
  uint32_t e;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.b32 %0, 1, 0, p;\n}" : "=r"(e));
  return e != 0;
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
// bytes from one group of 8 tokens to the next, kBlockBytes from one block of 64 outputs to the next.
static __device__ __forceinline__ uint64_t grad_descriptor(uint32_t addr) {
  return (uint64_t)((addr & 0x3ffff) >> 4) | (uint64_t)(kBlockBytes >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

// D in fp32; A and B in T; A as it lies in tensor memory, B transposed (its outputs are contiguous); N and M of the pair.
template <typename T>
static __device__ __forceinline__ constexpr uint32_t instruction_descriptor(int n) {
  constexpr uint32_t kind = sizeof(T) == 2 && !std::is_same<T, __half>::value ? 1 : 0;
  return 1u << 4 | kind << 7 | kind << 10 | 1u << 16 | (uint32_t)(n >> 3) << 17 | (uint32_t)(2 * kM >> 4) << 24;
}

static __device__ __forceinline__ void multiply(uint32_t d, uint32_t a, uint64_t b, uint32_t instruction, uint32_t accumulate) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a), "l"(b),
               "r"(instruction), "r"(accumulate)
               : "memory");
}

// What the pairs of blocks do.  (A block per tile, started anew for each, lost 9 us a tile to its start and to storing results: the
// pairs stay, and results are stored while the next tile is multiplied.)  `whole` tiles are dealt out in turns, all their
// tokens at once, so that the pairs of one turn read the same tokens at the same time (from L2); the tiles that would not
// fill another turn are cut into `slices` along the tokens, whose sums go to the workspace in fp32 and are added up in order
// by a second kernel.
struct Plan {
  int rows, outputs, channels;
  int steps;         // of kK tokens
  int width;         // outputs of a tile: kN or kNarrow
  int channel_tiles, output_tiles;
  int whole;         // tiles without slices
  int cut, slices;   // the tiles after those, and slices of each
  int slice_steps;
};

struct Item {
  int channel_tile, output_tile, first, last;  // steps first..last - 1
  int piece;                                   // of the workspace; -1: a result
};

static __host__ __device__ __forceinline__ void tile_at(const Plan& p, int tile, int* channel_tile, int* output_tile) {
  const int band = tile / (kBand * p.output_tiles), width = min(kBand, p.channel_tiles - band * kBand);
  const int at = tile - band * kBand * p.output_tiles;
  *channel_tile = band * kBand + at % width;
  *output_tile = at / width;
}

// The n-th item of a pair; false after the last.
static __device__ __forceinline__ bool item_at(const Plan& p, int pair, int pairs, int n, Item* it) {
  const int64_t w = pair + (int64_t)n * pairs;
  if (w < p.whole) {
    tile_at(p, (int)w, &it->channel_tile, &it->output_tile);
    it->first = 0, it->last = p.steps, it->piece = -1;
    return true;
  }
  // `whole` fills whole turns unless there are no others, so the slices are dealt out from the first pair on
  const int64_t piece = w - p.whole;
  if (piece >= (int64_t)p.cut * p.slices) return false;
  tile_at(p, p.whole + (int)(piece / p.slices), &it->channel_tile, &it->output_tile);
  it->first = (int)(piece % p.slices) * p.slice_steps;
  it->last = min(p.steps, it->first + p.slice_steps);
  it->piece = (int)piece;
  return true;
}

template <typename T> static __device__ __forceinline__ uint32_t pack(float low, float high);
template <> __device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float low, float high) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(high), "f"(low));
  return r;
}
template <> __device__ __forceinline__ uint32_t pack<__half>(float low, float high) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(high), "f"(low));
  return r;
}

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    weight_gradient_kernel(const __grid_constant__ CUtensorMap grad_map, const __grid_constant__ CUtensorMap code_map,
                           const uint8_t* __restrict__ exponents, int64_t epitch, const T* __restrict__ channel_scale,
                           const __grid_constant__ Plan plan, T* __restrict__ dw, float* __restrict__ pieces) {
  extern __shared__ uint8_t dynamic[];
  __shared__ __align__(8) uint64_t bars[4 * kStages + 3];
  __shared__ __align__(4) uint8_t bytes[kMakers][2][kK];
  __shared__ uint32_t tmem_base;
  const uint32_t tiles = (smem_of(dynamic) + 1023) & ~1023u;
  const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;  // warp: known to be uniform
  const int half = blockIdx.x % 2, pair = blockIdx.x / 2, pairs = gridDim.x / 2;  // half: which block of the pair
  // codes_in: this block's codes are there.  grads_in, made (the first block's): both blocks' gradients, both halves of X^T are
  // there.  empty: the multiplications that read a stage are done.  summed: those of an item are.  taken (the first block's): both
  // blocks' sums have been read.  drained: all multiplications are done.
  const uint32_t codes_in = smem_of(bars), grads_in = codes_in + 8 * kStages, made = grads_in + 8 * kStages, empty = made + 8 * kStages,
                 summed = empty + 8 * kStages, taken = summed + 8, drained = taken + 8;

  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&grad_map));
    asm volatile("prefetch.tensormap [%0];" ::"l"(&code_map));
    for (int s = 0; s < kStages; s++) {
      barrier_init(codes_in + 8 * s, 1);
      barrier_init(grads_in + 8 * s, 1);
      barrier_init(made + 8 * s, 2 * 4);  // four warps of each block
      barrier_init(empty + 8 * s, 1);
    }
    barrier_init(summed, 1);
    barrier_init(taken, 2 * kWriters);
    barrier_init(drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
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
  Item it;

  if (warp == kLoader) {
    const bool mine = elected();
    int g = 0;  // steps of all items so far
    for (int n = 0; ok && item_at(plan, pair, pairs, n, &it); n++) {
      const int c0 = it.channel_tile * 2 * kM + half * kM, o0 = it.output_tile * plan.width;
      const bool wide = plan.width > kNarrow && o0 + kNarrow < plan.outputs;
      for (int b = it.first; b < it.last; b++, g++) {
        const int s = g % kStages;
        if (g >= kStages && !barrier_wait(empty + 8 * s, (g / kStages - 1) & 1)) {
          ok = false;
          break;
        }
        if (mine) {
          const uint32_t at = tiles + s * kStageBytes, grads = in_first(grads_in + 8 * s);
          barrier_expect(codes_in + 8 * s, kCodeBytes);
          load_tile(at + kGradBytes, &code_map, c0, b * kK, codes_in + 8 * s);
          if (half == 0) barrier_expect(grads_in + 8 * s, (wide ? 6 : 4) * kBlockBytes);
          // this block's 64-output blocks: 0, 1 and 4 or 2, 3 and 5, so that a column of the results is an output
          load_tile(at, &grad_map, o0 + half * 128, b * kK, grads);
          load_tile(at + kBlockBytes, &grad_map, o0 + half * 128 + 64, b * kK, grads);
          if (wide) load_tile(at + 2 * kBlockBytes, &grad_map, o0 + kNarrow + half * 64, b * kK, grads);
        }
        __syncwarp();
      }
    }
    // Nothing of a block's shared memory is given back while a copy into it or an arrival there is under way: both blocks wait for the
    // codes they asked for, the first for the gradients of both (the partner stays until the first block is here too), and both for
    // the multiplications' arrivals at their own barriers, which the barrier of the pair does not order.
    for (int n = g > kStages ? g - kStages : 0; n < g; n++) {
      ok &= barrier_wait(codes_in + 8 * (n % kStages), (n / kStages) & 1);
      if (half == 0) ok &= barrier_wait(grads_in + 8 * (n % kStages), (n / kStages) & 1);
      ok = ok && barrier_wait(empty + 8 * (n % kStages), (n / kStages) & 1);
    }
  } else if (warp == kIssuer) {
    if (half == 0) {
      const bool mine = elected();
      int g = 0;
      for (int n = 0; ok && item_at(plan, pair, pairs, n, &it); n++) {
        const bool wide = plan.width > kNarrow && it.output_tile * plan.width + kNarrow < plan.outputs;
        ok = n == 0 || barrier_wait(taken, (n - 1) & 1);
        for (int b = it.first; ok && b < it.last; b++, g++) {
          const int s = g % kStages;
          ok = barrier_wait(grads_in + 8 * s, (g / kStages) & 1) && barrier_wait(made + 8 * s, (g / kStages) & 1);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t desc = grad_descriptor(tiles + s * kStageBytes);
          const uint32_t a = tmem_a + g % kSlots * kAColumns;
          if (mine) {
#pragma unroll
            for (int k = 0; k < kK / 16; k++) {
              const uint32_t accumulate = b > it.first || k > 0;
              multiply(tmem, a + k * 8, desc + (uint64_t)(k * 2048 >> 4), instruction_descriptor<T>(kNarrow), accumulate);
              if (wide)
                multiply(tmem + kNarrow, a + k * 8, desc + (uint64_t)((2 * kBlockBytes + k * 2048) >> 4),
                         instruction_descriptor<T>(kN - kNarrow), accumulate);
            }
            commit_to_pair(empty + 8 * s);
          }
          __syncwarp();
        }
        if (ok && mine) commit_to_pair(summed);
        __syncwarp();
      }
      if (mine) commit_to_pair(drained);
      __syncwarp();
      ok &= barrier_wait(drained, 0);
    }
  } else if (warp < kMakers) {
    // channels 32 * (warp % 4) .. + 31 of the block are this warp's rows of tensor memory, and one group of the format
    const int part = warp % 4, quad = lane % 4, set = warp / 4;
    const int64_t stride = (int64_t)kSets * kK * epitch;
    int g0 = 0;  // steps of the items before this one
    for (int n = 0; ok && item_at(plan, pair, pairs, n, &it); n++) {
      const int group = (it.channel_tile * 2 + half) * (kM / kGroup) + part;
      const int turn = (g0 ^ set) & (kSets - 1);  // the sets take turns over the steps of all items
      int b = it.first + turn;
      // This lane's exponent bytes of a step: tokens lane and lane + 32.  `left` tokens from the first on; none in a group past the end.
      int left = group * kGroup < plan.channels ? plan.rows - b * kK - lane : 0;
      const uint8_t* from = exponents + (int64_t)(b * kK + lane) * epitch + group;
      uint32_t e0 = left > 0 && b < it.last ? from[0] : 0, e1 = left > 32 && b < it.last ? from[32 * epitch] : 0;
      for (; b < it.last; b += kSets) {
        const int g = g0 + b - it.first, s = g % kStages, parity = (g / kStages) & 1;
        uint8_t* mine = bytes[warp][g / kSets & 1];
        mine[lane] = (uint8_t)e0, mine[lane + 32] = (uint8_t)e1;
        __syncwarp();
        left -= kSets * kK, from += stride;
        const bool again = b + kSets < it.last;
        e0 = again && left > 0 ? from[0] : 0, e1 = again && left > 32 ? from[32 * epitch] : 0;
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
        if (g >= kSlots) {  // the multiplications of the step that had this slot before
          ok = barrier_wait(empty + 8 * ((g - kSlots) % kStages), ((g - kSlots) / kStages) & 1);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        }
        const uint32_t to = tmem_a + g % kSlots * kAColumns + ((uint32_t)(part * 32) << 16);
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
      g0 += it.last - it.first;
    }
  } else {
    // Lane = channel.  128 outputs at a time are rounded into registers; after the last of them the tensor memory is given back,
    // before those are stored: the next item's multiplications run meanwhile.
    const int part = warp % 4;
    const uint32_t from = tmem + ((uint32_t)(part * 32) << 16);
    const bool even_rows = plan.channels % 2 == 0 && reinterpret_cast<uintptr_t>(dw) % 4 == 0;
    for (int n = 0; item_at(plan, pair, pairs, n, &it); n++) {
      const int c = (it.channel_tile * 2 + half) * kM + part * 32 + lane;
      ok = ok && barrier_wait(summed, n & 1);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      // a wait that gave up makes NaNs of the results
      const float scale = !ok ? __int_as_float(0x7fffffff) : it.piece < 0 && channel_scale && c < plan.channels ? to_f32(channel_scale[c]) : 1.0f;
#define LOAD16(v, addr)                                                                                                                  \
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"  \
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), \
                 "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])                                            \
               : "r"(addr))
      constexpr int kPart = 128;
      const int last = it.output_tile * plan.width + kNarrow < plan.outputs ? plan.width - kPart : kNarrow - kPart;
      for (int first = 0; first <= last; first += kPart) {
        const int o0 = it.output_tile * plan.width + first;
        if (it.piece < 0) {
          uint32_t held[kPart / 2];
#pragma unroll
          for (int i = 0; i < kPart; i += 16) {
            uint32_t v[16];
            LOAD16(v, from + first + i);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int k = 0; k < 8; k++)
              held[i / 2 + k] = pack<T>(__fmul_rn(__uint_as_float(v[2 * k]), scale), __fmul_rn(__uint_as_float(v[2 * k + 1]), scale));
          }
          if (first == last) {
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) barrier_arrive(in_first(taken));
          }
          T* out = dw + (int64_t)o0 * plan.channels + c;
          if (even_rows) {
            // neighbouring lanes swap, so that a lane stores two channels of one output: even lanes the first, odd ones the second
            const int odd = lane & 1;
            uint32_t* at = reinterpret_cast<uint32_t*>(out - odd + (int64_t)odd * plan.channels);
#pragma unroll
            for (int k = 0; k < kPart / 2; k++) {
              const uint32_t other = __shfl_xor_sync(~0u, held[k], 1);
              const uint32_t both = odd ? __byte_perm(other, held[k], 0x7632) : __byte_perm(held[k], other, 0x5410);
              if (o0 + 2 * k + odd < plan.outputs && c < plan.channels) *at = both;
              at += plan.channels;
            }
          } else if (c < plan.channels) {
            unsigned short* at = reinterpret_cast<unsigned short*>(out);
#pragma unroll
            for (int k = 0; k < kPart / 2; k++) {
              if (o0 + 2 * k < plan.outputs) at[0] = (unsigned short)held[k];
              if (o0 + 2 * k + 1 < plan.outputs) at[plan.channels] = (unsigned short)(held[k] >> 16);
              at += 2 * (int64_t)plan.channels;
            }
          }
        } else {
          float* out = pieces + (((int64_t)it.piece * 2 + half) * kN + first) * kM + part * 32 + lane;
          for (int i = 0; i < kPart; i += 16) {
            uint32_t v[16];
            LOAD16(v, from + first + i);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int k = 0; k < 16; k++) out[(i + k) * kM] = __fmul_rn(__uint_as_float(v[k]), scale);
          }
          if (first == last) {
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) barrier_arrive(in_first(taken));
          }
        }
      }
#undef LOAD16
    }
    ok &= barrier_wait(drained, 0);  // the last arrival in this block, as above
  }
  if (!ok) g_gave_up = 1;
  __syncwarp();
  pair_sync();  // the partner may still read this block's gradients or arrive at its barriers
  if (warp == kIssuer) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// Adds up the slices of the tiles that were cut, always in the same order.  A warp takes one output and the 128 channels of a half
// tile; with many slices the eight warps of a block share them (kShared), and their sums are added up in order.
template <typename T, bool kShared>
__global__ void __launch_bounds__(256) join_slices_kernel(const float4* __restrict__ pieces, const __grid_constant__ Plan plan,
                                                          const T* __restrict__ channel_scale, T* __restrict__ dw) {
  __shared__ float4 part[8][32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, half = blockIdx.y;
  int channel_tile, output_tile;
  tile_at(plan, plan.whole + blockIdx.z, &channel_tile, &output_tile);
  const int n = kShared ? blockIdx.x : blockIdx.x * 8 + warp, o = output_tile * plan.width + n;
  const int c = (channel_tile * 2 + half) * kM + lane * 4;
  if (o < plan.outputs && (channel_tile * 2 + half) * kM < plan.channels) {  // the same for a block where its warps share
    float4 sum = make_float4(0, 0, 0, 0);
    const float4* at = pieces + (((int64_t)blockIdx.z * plan.slices * 2 + half) * kN + n) * (kM / 4) + lane;
    const int64_t stride = (int64_t)2 * kN * kM / 4;
#pragma unroll 4
    for (int s = kShared ? warp : 0; s < plan.slices; s += kShared ? 8 : 1) {
      const float4 v = at[s * stride];
      sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    }
    if constexpr (kShared) {
      part[warp][lane] = sum;
      __syncthreads();
      if (warp > 0) return;
#pragma unroll
      for (int w = 1; w < 8; w++) {
        const float4 v = part[w][lane];
        sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
      }
    }
    const float f[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (c + i < plan.channels)
        dw[(int64_t)o * plan.channels + c + i] = from_f32<T>(__fmul_rn(f[i], channel_scale ? to_f32(channel_scale[c + i]) : 1.0f));
  }
}

// What a call costs, in steps of a tile of 256 outputs (0.38 us): a step of 384 outputs is kWideStep of them (0.47 to 0.58 us); slices
// cost a launch and, each, a trip of its sums through L2.  Of the two widths the cheaper is taken, and slices only where they are
// cheaper.  8192 tokens: 14336 x 4096 615 us wide, 666 narrow; 4096 x 1024 74 wide, 58 narrow; 16384 tokens, 256 x 256: 20 us in
// 74 slices, about 100 in one.
constexpr float kWideStep = 1.4f, kJoin = 10.0f, kPiece = 0.1f;

static Plan plan_of_width(int64_t rows, int64_t outputs, int64_t channels, int pairs, int width, float* cost) {
  Plan p;
  p.rows = (int)rows, p.outputs = (int)outputs, p.channels = (int)channels, p.width = width;
  p.steps = (int)((rows + kK - 1) / kK);
  p.channel_tiles = (int)((channels + 2 * kM - 1) / (2 * kM)), p.output_tiles = (int)((outputs + width - 1) / width);
  const int64_t tiles = (int64_t)p.channel_tiles * p.output_tiles;
  const int rest = (int)(tiles % pairs);
  const float step = width > kNarrow ? kWideStep : 1.0f;
  p.whole = (int)tiles, p.cut = 0, p.slices = 0, p.slice_steps = 0;
  *cost = (float)(tiles / pairs) * (float)p.steps * step;
  if (rest == 0) return p;
  const int slices = pairs / rest, each = (p.steps + slices - 1) / slices;
  const float uncut = (float)p.steps * step, cut = (float)each * step + kJoin + kPiece * (float)(rest * slices);
  if (slices > 1 && cut < uncut) {
    p.whole -= rest, p.cut = rest, p.slice_steps = each;
    p.slices = (p.steps + each - 1) / each;
  }
  *cost += cut < uncut && slices > 1 ? cut : uncut;
  return p;
}

static Plan plan_of(int64_t rows, int64_t outputs, int64_t channels, int pairs) {
  float narrow_cost, wide_cost;
  const Plan narrow = plan_of_width(rows, outputs, channels, pairs, kNarrow, &narrow_cost);
  const Plan wide = plan_of_width(rows, outputs, channels, pairs, kN, &wide_cost);
  return wide_cost < narrow_cost ? wide : narrow;
}

static int pairs_of_device() {
  int device = 0, sms = 0;
  if (cudaGetDevice(&device) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
    cudaGetLastError();
    return 74;
  }
  return sms / 2;
}

constexpr int64_t kMostSize = INT32_MAX - 4096;  // coordinates are 32-bit and run past the end by less than a block

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
static int launch_weight_gradient(const char* fn, const void* grad, int64_t grad_stride, const void* codes, int64_t pitch, const void* exponents,
                                  int64_t epitch, const void* channel_scale, const Plan& plan, int pairs, void* dw, void* workspace,
                                  cudaStream_t s) {
  // First a call of the runtime: it makes the device's context current, which a thread without any CUDA call so far (autograd's,
  // for one) lacks, and which the driver's encoder of tensor maps asks for.
  cudaError_t e = cudaFuncSetAttribute(weight_gradient_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
  if (e != cudaSuccess) return fail(OPTIMI_ERR_CUDA, "%s: %s", fn, cudaGetErrorString(e));
  CUtensorMap grad_map, code_map;
  constexpr CUtensorMapDataType kType = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  int rc = make_map(fn, &grad_map, kType, grad, plan.outputs, plan.rows, grad_stride * 2, 64, kK);
  if (rc == OPTIMI_OK) rc = make_map(fn, &code_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, plan.channels, plan.rows, pitch, kM, kK);
  if (rc != OPTIMI_OK) return rc;
  const int64_t items = (int64_t)plan.whole + (int64_t)plan.cut * plan.slices;
  weight_gradient_kernel<T><<<(unsigned)(2 * (items < pairs ? items : pairs)), kThreads, kSmemBytes, s>>>(
      grad_map, code_map, (const uint8_t*)exponents, epitch, (const T*)channel_scale, plan, (T*)dw, (float*)workspace);
  rc = launched(fn);
  if (rc != OPTIMI_OK || plan.cut == 0) return rc;
  if (plan.slices > 8)
    join_slices_kernel<T, true><<<dim3(plan.width, 2, plan.cut), 256, 0, s>>>((const float4*)workspace, plan, (const T*)channel_scale, (T*)dw);
  else
    join_slices_kernel<T, false><<<dim3(plan.width / 8, 2, plan.cut), 256, 0, s>>>((const float4*)workspace, plan, (const T*)channel_scale, (T*)dw);
  return launched(fn);
}

}  // namespace act
}  // namespace optimi

using namespace optimi;
using namespace optimi::act;

extern "C" {

size_t optimi_b200_weight_gradient_workspace_bytes(int64_t rows, int64_t outputs, int64_t channels) {
  if (rows <= 0 || outputs <= 0 || channels <= 0 || rows > kMostSize || outputs > kMostSize || channels > kMostSize) return 0;
  const Plan p = plan_of(rows, outputs, channels, pairs_of_device());
  return (size_t)p.cut * p.slices * 2 * kM * kN * sizeof(float);
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
  if (dtype != OPTIMI_BF16 && dtype != OPTIMI_F16)
    return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: dtype %d is neither bfloat16 nor float16", fn, dtype);
  if (rows < 0 || outputs < 0 || channels < 0 || rows > kMostSize || outputs > kMostSize || channels > kMostSize)
    return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: %lld tokens, %lld outputs, %lld channels are outside 0..%lld", fn, (long long)rows,
                (long long)outputs, (long long)channels, (long long)kMostSize);
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
  const int pairs = pairs_of_device();
  if ((channels + 2 * kM - 1) / (2 * kM) * ((outputs + kNarrow - 1) / kNarrow) > INT32_MAX)
    return fail(OPTIMI_ERR_INVALID_ARGUMENT, "%s: %lld x %lld results are too many", fn, (long long)outputs, (long long)channels);
  const Plan plan = plan_of(rows, outputs, channels, pairs);
  const size_t need = (size_t)plan.cut * plan.slices * 2 * kM * kN * sizeof(float);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(OPTIMI_ERR_WORKSPACE_TOO_SMALL, "%s: workspace has %zu bytes, %zu are needed, 16-byte aligned", fn,
                workspace ? workspace_bytes : (size_t)0, need);
  if (dtype == OPTIMI_BF16)
    return launch_weight_gradient<__nv_bfloat16>(fn, grad, grad_stride, codes, code_pitch, exponents, exponent_pitch, channel_scale, plan, pairs,
                                                 grad_weight, workspace, s);
  return launch_weight_gradient<__half>(fn, grad, grad_stride, codes, code_pitch, exponents, exponent_pitch, channel_scale, plan, pairs,
                                        grad_weight, workspace, s);
}

}  // extern "C"
