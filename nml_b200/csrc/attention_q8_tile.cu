// Attention over the 8-bit paged K/V cache for runs of tokens (prompts, chunks of them, drafted
// tokens) on the tcgen05 tensor cores; the mathematics is that of attention_q8.cu.
//
// A CTA takes 128 query rows of one kv head: 128 / group consecutive tokens of a sequence times
// the group's query heads, so that every key and value is widened once for all of them, and walks
// the visible pages in steps of 64 tokens.  Two CTAs share an SM (half of tensor memory each): one
// computes exponentials while the other's matrix products, prologue or epilogue run.  Roles:
//   warps 0-3  softmax, one thread for each row: q into tensor memory (F16, a power of two for the
//              row), then for every step the scores out of tensor memory, maximum, weights back
//              into tensor memory over the scores; rescales the accumulator when needed
//   warps 4-7  widen the codes: 16-byte loads, E4M3 to F16 (exact, the block scales stay out),
//              128-byte swizzled stores; the next step's loads are in flight meanwhile, page
//              table entries and scales are fetched for 32 pages at a time, 32 pages ahead
//   warp 8     issues the products: S = Q K^T (A: q in tensor memory, B: keys, K-major) and
//              O += W V (A: weights in tensor memory, B: values, MN-major: tokens are rows)
// Registers move from the last two warpgroups to the softmax, which holds a row's 64 scores.
//
// The running maximum M only stabilises: weights above one are as good as those below as long as
// F16 holds them (sums are f32).  So a step is weighted against the maximum of the steps before it,
// and only when a page's weights sum to more than 2^14 is its own maximum formed, the accumulator
// in tensor memory rescaled and the step repeated: once or twice for a row.  A value row of NaN codes (stored whole by the append) becomes zeros in the
// product and NaN scores for the rows that see it, so that it does not reach the rows that do not.
//
// What bounds it: one exponential for each score.  A step of 128 x 64 takes 512 clocks of the SM's
// 16 exponentials per clock and 256 (head_dim 64) of the tensor cores.
#include <type_traits>

#include "attention_q8.cuh"
#include "sm100_primitives.cuh"

namespace nml_sm100 {
namespace {

constexpr int kStepTokens = 64;
constexpr int kStepPages = kStepTokens / kCachePage;
constexpr int kSoftmaxThreads = 128;
constexpr int kWidenThreads = 128;
constexpr int kWidenWarp = 4;
constexpr int kMmaWarp = 8;
constexpr int kThreads = 384;  // the last three warps only give their registers
constexpr int kLaunchRegisters = 80;  // of a thread: two CTAs fill an SM
// Sum of a page's 16 weights up to which the maximum so far still serves: F16 holds each of them.
constexpr float kLargestSum = 16384.0f;
constexpr int kTmemColumns = 256;

// Bits 8 + site of the status word say which wait ran out.
constexpr int kSiteScores = 16, kSiteWeights = 17, kSiteTiles = 18, kSiteProduct = 19,
              kSiteFree = 20;

// What the softmax needs to know of a page: score factor, exponent of the values, its inverse
// power for the denominator, first token.
struct alignas(16) PageInfo {
  float key_scale, value_exponent, unscale;
  int token;
};

template <int D>
struct Shape {
  static constexpr int kTileBytes = kStepTokens * D * 2;
  static constexpr int kStages = D == 64 ? 4 : 3;
  static constexpr int kBuffers = D == 64 ? 2 : 1;  // score buffers in tensor memory
  static constexpr int kOut = 0, kQuery = D, kScores = D + D / 2;
  static constexpr int kSharedBytes = kStages * 2 * kTileBytes + 1024;
  // The three warpgroups' shares of the CTA's registers at launch.
  static constexpr int kSoftmaxRegisters = D == 64 ? 144 : 136;
  static constexpr int kWidenRegisters = D == 64 ? 72 : 80;
  static constexpr int kMmaRegisters = 24;
  static_assert(kSoftmaxRegisters + kWidenRegisters + kMmaRegisters == 3 * kLaunchRegisters,
                "a share that the launch does not cover would be waited for without end");
  static_assert(kScores + kBuffers * kStepTokens <= kTmemColumns, "tensor memory");
};

template <int D>
struct Control {
  uint64_t tiles_full[Shape<D>::kStages], tiles_free[Shape<D>::kStages];
  uint64_t scores_full[Shape<D>::kBuffers];
  // one for each buffer: a warp may run ahead of the others by as many steps as there are buffers
  uint64_t weights_full[Shape<D>::kBuffers], product_done[Shape<D>::kBuffers];
  uint64_t query_full, drained;
  uint32_t tmem;
  int abort_flag;
  int sequence, tile;
  PageInfo pages[Shape<D>::kStages][kStepPages];
  alignas(16) uint32_t any_nan[Shape<D>::kStages][4];  // read 16 bytes at a time
  uint8_t row_nan[Shape<D>::kStages][kStepTokens];
};

template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Two f32 at a time.
__device__ __forceinline__ uint64_t pack_f32x2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack_f32x2(uint64_t x, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x));
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2)
tile_kernel(const AttentionParams p) {
  using S = Shape<D>;
  extern __shared__ uint8_t raw_shared[];
  uint8_t* const shared = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(raw_shared) + 1023) & ~static_cast<uintptr_t>(1023));
  __shared__ __align__(16) Control<D> control;
  volatile int* const abort_flag = &control.abort_flag;

  // through a shuffle: the compiler then knows the roles' branches and loops to be warp-uniform
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int kv_head = blockIdx.x % p.cache.kv_heads;
  const int item = blockIdx.x / p.cache.kv_heads / p.splits;
  const int split = blockIdx.x / p.cache.kv_heads % p.splits;
  const int per_tile = kTileRows / p.group;

  // ---- which sequence, which of its tiles: the last tile (the longest walk) comes first ----
  if (warp == 0) {
    int sequence = -1, tile = 0, passed = 0;
    for (int base = 0; base < p.cache.batch && sequence < 0; base += 32) {
      const int b = base + lane;
      int tiles = 0;
      if (b < p.cache.batch) {
        const int rows = min(p.offsets[b + 1], p.tokens) - max(p.offsets[b], 0);
        tiles = rows > 0 ? (rows + per_tile - 1) / per_tile : 0;
      }
      int upto = tiles;
#pragma unroll
      for (int offset = 1; offset < 32; offset <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, upto, offset);
        if (lane >= offset) upto += other;
      }
      const uint32_t holds = __ballot_sync(0xffffffffu, item - passed < upto);
      if (holds != 0) {
        const int at = __ffs(holds) - 1;
        sequence = base + at;
        tile = __shfl_sync(0xffffffffu, upto, at) - 1 - (item - passed);
      }
      passed += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) {
      control.sequence = sequence;
      control.tile = tile;
    }
  }
  if (threadIdx.x == kMmaWarp * 32) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&control.tiles_full[i], kWidenThreads);
      mbar_init(&control.tiles_free[i], 1);
    }
    for (int i = 0; i < S::kBuffers; ++i) {
      mbar_init(&control.scores_full[i], 1);
      mbar_init(&control.weights_full[i], kSoftmaxThreads);
      mbar_init(&control.product_done[i], 1);
    }
    mbar_init(&control.query_full, kSoftmaxThreads);
    mbar_init(&control.drained, 1);
    control.abort_flag = 0;
    mbar_fence_init();
  }
  __syncthreads();
  const int sequence = control.sequence;
  if (sequence < 0) return;  // more work items than tiles

  const int begin = max(p.offsets[sequence], 0);
  const int end = min(p.offsets[sequence + 1], p.tokens);
  const int first_row = begin + control.tile * per_tile;
  const int rows = min(per_tile, end - first_row);
  const int first_position =
      sequence_length(p.cache, sequence, p.status) - p.offsets[sequence + 1] + first_row;
  const Visible v = visible_pages(first_position + rows,
                                  p.window > 0 ? first_position + 1 - p.window : 0, p.first);
  const int all_steps = (v.pages + kStepPages - 1) / kStepPages;
  const int per_split = (all_steps + p.splits - 1) / p.splits;
  const int step_begin = min(all_steps, split * per_split);
  const int steps = __shfl_sync(0xffffffffu, min(all_steps - step_begin, per_split), 0);

  if (warp == kMmaWarp) {
    tmem_alloc(&control.tmem, kTmemColumns);
    tmem_relinquish_alloc_permit();
  }
  tcgen05_fence_before_sync();
  __syncthreads();
  tcgen05_fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, control.tmem, 0);

  auto wait = [&](uint64_t* bar, int phase, int site) {
    mbar_wait_or_abort(bar, static_cast<uint32_t>(phase) & 1u, abort_flag, p.status, site);
    __syncwarp();
  };

  // The product of step j.  Whoever has step j's scores knows that the product kBuffers steps
  // back is complete, and no product passes a step that this warp has not handed over: with a
  // barrier for each buffer a parity names one phase only.
  auto wait_product = [&](int j) {
    wait(&control.product_done[j % S::kBuffers], j / S::kBuffers, kSiteProduct);
  };

  if (warp < kWidenWarp) {
    // ------------------------------------------------------------------ softmax
    more_registers<S::kSoftmaxRegisters>();
    const int row = threadIdx.x;
    const int token = row / p.group;
    const int head = kv_head * p.group + row - token * p.group;
    const bool live = token < rows;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    // rows of nobody walk like the last row, so that they do not ask for masks
    const int length = first_position + 1 + (live ? token : rows - 1);
    const int start = p.window > 0 ? max(0, length - p.window) : 0;

    // q: largest magnitude, then F16 into tensor memory, column c holding elements 2c and 2c + 1
    float factor = p.scale_log2;
    {
      const T* source = static_cast<const T*>(p.query) +
                        static_cast<int64_t>(first_row + token) * p.query_token_stride +
                        head * p.query_head_stride;
      uint32_t largest = 0;
      if constexpr (!std::is_same<T, __half>::value) {
        if (live) {
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            const uint4 x = reinterpret_cast<const uint4*>(source)[i];
            const uint32_t words[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              largest = max(largest, max((words[w] & 0x7fffu) << 16, words[w] & 0x7fff0000u));
            }
          }
        }
      }
      const int shift = std::is_same<T, __half>::value ? 0 : query_shift(largest);
      const float up = exp2_int(shift);
      factor *= exp2_int(-shift);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        uint32_t packed[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint4 x = make_uint4(0, 0, 0, 0);
          if (live) x = reinterpret_cast<const uint4*>(source)[2 * i + h];
          const uint32_t words[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            if constexpr (std::is_same<T, __half>::value) {
              packed[4 * h + w] = words[w];
            } else {
              packed[4 * h + w] = Elem<__half>::pack2(Elem<T>::from_bits(words[w] & 0xffffu) * up,
                                                      Elem<T>::from_bits(words[w] >> 16) * up);
            }
          }
        }
        __syncwarp();
        tmem_store_32x8(lanes + S::kQuery + 8 * i, packed);
      }
      tmem_store_wait();
      tcgen05_fence_before_sync();
      mbar_arrive(&control.query_full);
    }

    // steps whose tokens every row of the tile sees: behind the last row's window start, in front
    // of the first row's own token
    const int last_start = p.window > 0 ? max(0, first_position + rows - p.window) : 0;
    const int first_whole = last_start == 0 ? 0 : v.front + (last_start + kCachePage - 1) /
                                                                kCachePage - v.back;
    const int whole_pages = v.front + max(first_position + 1, 0) / kCachePage - v.back;
    const int whole_begin = (first_whole + kStepPages - 1) / kStepPages - step_begin;
    const int whole_end = max(whole_pages, 0) / kStepPages - step_begin;

    float running_max = -INFINITY, running_sum = 0.0f;
    for (int j = 0; j < steps; ++j) {
      const int buffer = j % S::kBuffers, stage = j % S::kStages;
      const uint32_t columns = lanes + S::kScores + buffer * kStepTokens;
      wait(&control.tiles_full[stage], j / S::kStages, kSiteTiles);  // for the page data
      float page_factor[kStepPages], value_exponent[kStepPages], unscale[kStepPages];
#pragma unroll
      for (int q = 0; q < kStepPages; ++q) {
        const float4 info = *reinterpret_cast<const float4*>(&control.pages[stage][q]);
        page_factor[q] = factor * info.x;
        value_exponent[q] = info.y;
        unscale[q] = info.z;
      }
      const uint4 nan_words = *reinterpret_cast<const uint4*>(control.any_nan[stage]);
      const bool nans = (nan_words.x | nan_words.y | nan_words.z | nan_words.w) != 0;
      wait(&control.scores_full[buffer], j / S::kBuffers, kSiteScores);
      tcgen05_fence_after_sync();

      // Weights against the maximum so far; their sum tells whether it still serves.  Only when it
      // does not (or there is none yet) is the step's maximum formed and the step done again.
      uint32_t packed[kStepTokens / 2];
      float step_sum;
      bool with_maximum = __any_sync(0xffffffffu, running_max == -INFINITY);
      while (true) {
        uint32_t scores_lo[32], scores_hi[32];
        tmem_load_32x32(columns, scores_lo);
        tmem_load_32x32(columns + 32, scores_hi);
        tmem_load_wait();
        float s[kStepTokens];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          s[i] = __uint_as_float(scores_lo[i]);
          s[32 + i] = __uint_as_float(scores_hi[i]);
        }
        if (j < whole_begin || j >= whole_end || nans) {
          // bit i: token i of the step is seen, its value row is NaN; loops, so that the steps
          // without masks branch over all of this
          uint32_t seen[2] = {0, 0}, nan[2] = {0, 0};
#pragma unroll 1
          for (int q = 0; q < kStepPages; ++q) {
            const int t = control.pages[stage][q].token;
            auto below = [&](int limit) {  // bits of the page's tokens in front of `limit`
              return (1u << min(max(limit - t, 0), kCachePage)) - 1u;
            };
            const uint32_t bits = below(length) & (~below(start) | below(p.first));
            uint32_t nan_bits = 0;
            if (nans) {
#pragma unroll 1
              for (int i = 0; i < kCachePage; ++i) {
                nan_bits |= static_cast<uint32_t>(control.row_nan[stage][q * kCachePage + i]) << i;
              }
            }
            const int shift = q * kCachePage & 31;
            seen[0] |= q < 2 ? bits << shift : 0u;
            seen[1] |= q < 2 ? 0u : bits << shift;
            nan[0] |= q < 2 ? nan_bits << shift : 0u;
            nan[1] |= q < 2 ? 0u : nan_bits << shift;
          }
#pragma unroll
          for (int i = 0; i < kStepTokens; ++i) {
            if ((nan[i / 32] >> (i % 32) & 1u) != 0) s[i] = __uint_as_float(0x7fc00000u);
            if ((seen[i / 32] >> (i % 32) & 1u) == 0) s[i] = -INFINITY;
          }
        }
        if (with_maximum) {
          float top = -INFINITY;
#pragma unroll
          for (int q = 0; q < kStepPages; ++q) {
            float m = fmaxf(s[q * kCachePage], s[q * kCachePage + 1]);
#pragma unroll
            for (int i = 2; i < kCachePage; i += 2) {
              m = fmaxf(fmaxf(m, s[q * kCachePage + i]), s[q * kCachePage + i + 1]);
            }
            top = fmaxf(top, fmaf(m, page_factor[q], value_exponent[q]));
          }
          const bool raise = top > running_max;  // also from -infinity
          const float next = raise ? top : running_max;
          const float rescale = raise ? exp2_fast(running_max - next) : 1.0f;
          if (j > 0) {
            wait_product(j - 1);
            tcgen05_fence_after_sync();
#pragma unroll
            for (int c = 0; c < D; c += 16) {
              uint32_t x[16], y[8], z[8];
              tmem_load_32x16(lanes + S::kOut + c, x);
              tmem_load_wait();
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                y[i] = __float_as_uint(__uint_as_float(x[i]) * rescale);
                z[i] = __float_as_uint(__uint_as_float(x[i + 8]) * rescale);
              }
              tmem_store_32x8(lanes + S::kOut + c, y);
              tmem_store_32x8(lanes + S::kOut + c + 8, z);
            }
          }
          running_sum *= rescale;
          running_max = next;
        }
        const float base = running_max == -INFINITY ? 0.0f : running_max;
        step_sum = 0.0f;
        float largest_sum = 0.0f;
#pragma unroll
        for (int q = 0; q < kStepPages; ++q) {
          const float offset = value_exponent[q] - base;
          const uint64_t factor2 = pack_f32x2(page_factor[q], page_factor[q]);
          const uint64_t offset2 = pack_f32x2(offset, offset);
          uint64_t sum2 = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float a, b;
            unpack_f32x2(fma_f32x2(pack_f32x2(s[q * kCachePage + 2 * i],
                                              s[q * kCachePage + 2 * i + 1]),
                                   factor2, offset2),
                         a, b);
            a = exp2_fast(a);
            b = exp2_fast(b);
            sum2 = add_f32x2(sum2, pack_f32x2(a, b));
            packed[8 * q + i] = Elem<__half>::pack2(a, b);
          }
          float sum_even, sum_odd;
          unpack_f32x2(sum2, sum_even, sum_odd);
          const float sum = sum_even + sum_odd;
          largest_sum = fmaxf(largest_sum, sum);
          step_sum = fmaf(sum, unscale[q], step_sum);
        }
        if (with_maximum || !__any_sync(0xffffffffu, largest_sum > kLargestSum)) break;
        with_maximum = true;
      }
      running_sum += step_sum;
#pragma unroll
      for (int q = 0; q < kStepPages; ++q) {
        const uint32_t(&page)[8] = *reinterpret_cast<const uint32_t(*)[8]>(&packed[8 * q]);
        tmem_store_32x8(columns + 8 * q, page);
      }
      tmem_store_wait();
      tcgen05_fence_before_sync();
      mbar_arrive(&control.weights_full[buffer]);
    }

    // ---- the rows' results ----
    if (steps > 0) {
      wait_product(steps - 1);
      tcgen05_fence_after_sync();
    }
    const int64_t query_head = static_cast<int64_t>(first_row + token) * p.query_heads + head;
    float denominator = running_sum;
    if (p.sinks != nullptr && live) {
      denominator += exp2f(p.sinks[head] * kLog2e - running_max);
    }
    // only a row that sees nothing has a sum of exactly zero; its output is zero
    const float inverse = running_sum == 0.0f ? 0.0f : 1.0f / denominator;
    float* partial = p.partial + (query_head * p.splits + split) * (D + 2);
    T* out = static_cast<T*>(p.output) + query_head * D;
#pragma unroll
    for (int c = 0; c < D; c += 16) {
      uint32_t x[16];
      if (steps > 0) {
        tmem_load_32x16(lanes + S::kOut + c, x);
        tmem_load_wait();
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = 0;
      }
      if (live && p.splits > 1) {
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          *reinterpret_cast<uint2*>(partial + c + i) = make_uint2(x[i], x[i + 1]);
        }
      } else if (live) {
        uint32_t packed[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          packed[i] = Elem<T>::pack2(__uint_as_float(x[2 * i]) * inverse,
                                     __uint_as_float(x[2 * i + 1]) * inverse);
        }
        reinterpret_cast<uint4*>(out + c)[0] =
            make_uint4(packed[0], packed[1], packed[2], packed[3]);
        reinterpret_cast<uint4*>(out + c)[1] =
            make_uint4(packed[4], packed[5], packed[6], packed[7]);
      }
      __syncwarp();
    }
    if (live && p.splits > 1) {
      *reinterpret_cast<float2*>(partial + D) = make_float2(running_max, running_sum);
    }
  } else if (warp >= kMmaWarp) {
    // ------------------------------------------------------------------ matrix products
    fewer_registers<S::kMmaRegisters>();
    if (warp == kMmaWarp) {
      constexpr uint64_t desc_hi = static_cast<uint64_t>(kUmmaDescHiSw128) << 32;
      constexpr uint32_t score_idesc = umma_idesc_f16(kUmmaF16, kUmmaF16, kTileRows, kStepTokens);
      constexpr uint32_t product_idesc =
          umma_idesc_f16(kUmmaF16, kUmmaF16, kTileRows, D) | (1u << 16);  // B is MN-major
      auto scores = [&](int j) {
        const int stage = j % S::kStages, buffer = j % S::kBuffers;
        wait(&control.tiles_full[stage], j / S::kStages, kSiteTiles);
        tcgen05_fence_after_sync();
        const uint32_t keys = smem_u32(shared + stage * 2 * S::kTileBytes);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          // 64-element halves of the head are tiles of their own, 16 elements are 32 bytes of a row
          const uint32_t address = keys + (k / 4) * (kStepTokens * 128) + (k % 4) * 32;
          umma_f16_tmem_a_elect(tmem + S::kScores + buffer * kStepTokens, tmem + S::kQuery + 8 * k,
                                desc_hi | umma_desc_lo(address), score_idesc, k > 0 ? 1u : 0u);
        }
        umma_commit_elect(&control.scores_full[buffer]);
      };
      if (steps > 0) {
        wait(&control.query_full, 0, kSiteWeights);
        tcgen05_fence_after_sync();
        for (int j = 0; j < min(steps, S::kBuffers); ++j) scores(j);
      }
      for (int j = 0; j < steps; ++j) {
        const int stage = j % S::kStages, buffer = j % S::kBuffers;
        wait(&control.weights_full[buffer], j / S::kBuffers, kSiteWeights);
        tcgen05_fence_after_sync();
        const uint32_t values = smem_u32(shared + stage * 2 * S::kTileBytes + S::kTileBytes);
#pragma unroll
        for (int k = 0; k < kStepTokens / 16; ++k) {
          // 16 tokens are 2 KB of 128-byte rows; the leading offset is the next 64 dimensions' tile
          const uint32_t address = values + k * 2048;
          const uint32_t low = ((address & 0x3ffffu) >> 4) | ((kStepTokens * 128 >> 4) << 16);
          umma_f16_tmem_a_elect(tmem + S::kOut, tmem + S::kScores + buffer * kStepTokens + 8 * k,
                                desc_hi | low, product_idesc, j > 0 || k > 0 ? 1u : 0u);
        }
        umma_commit_elect(&control.tiles_free[stage]);
        umma_commit_elect(&control.product_done[buffer]);
        if (j + S::kBuffers < steps) {
          // the scores go over the weights that this product reads
          wait_product(j);
          scores(j + S::kBuffers);
        }
      }
      umma_commit_elect(&control.drained);
      if (!mbar_wait(&control.drained, 0)) {
        *abort_flag = 1;
        atomicOr(p.status, NML_SM100_STATUS_BARRIER_TIMEOUT | (0x100 << kSiteProduct));
      }
    }
  } else {
    // ------------------------------------------------------------------ codes to F16 tiles
    fewer_registers<S::kWidenRegisters>();
    constexpr int kParts = D / 16;                          // pieces of 16 codes of a token's row
    constexpr int kTokens = kWidenThreads / kParts;         // tokens of one load of the group
    constexpr int kRounds = kStepTokens / kTokens;          // loads for the keys of a step
    constexpr int kGroup = 32;                              // pages looked up at once
    const int thread = threadIdx.x - kWidenWarp * 32;
    const int part = thread % kParts, first_token = thread / kParts;
    // page of round r's token: r * (kTokens / 16) + lane_page
    const int lane_page = first_token / kCachePage;
    const uint32_t head_bytes = kCachePage * D;
    const int64_t page_bytes = static_cast<int64_t>(p.cache.kv_heads) * head_bytes;
    const int64_t thread_bytes = static_cast<int64_t>(kv_head) * head_bytes +
                                 (first_token % kCachePage) * D + part * 16;
    const uint8_t* const key_codes = p.cache.codes[0] + thread_bytes;
    const uint8_t* const value_codes = p.cache.codes[1] + thread_bytes;
    uint8_t* const own_tile = shared + (part / 4) * (kStepTokens * 128) + first_token * 128;
    // 16-byte chunks 2 part and 2 part + 1 of a 128-byte row, swizzled by the token
    const int chunk_lo = ((2 * (part % 4)) ^ (first_token & 7)) * 16;
    const int chunk_hi = ((2 * (part % 4) + 1) ^ (first_token & 7)) * 16;

    // lane i holds page (-1: nothing there) and scale bytes of entry i of a group of 32
    auto look_up = [&](int group, int& page, uint32_t& bytes) {
      page = -1;
      bytes = 0;
      const int i = group * kGroup + lane;
      if (i >= step_begin * kStepPages && i < min(v.pages, (step_begin + steps) * kStepPages)) {
        page = physical_page(p.cache, sequence, i < v.front ? i : i - v.front + v.back, p.status);
        if (page >= 0) {
          const int64_t block = static_cast<int64_t>(page) * p.cache.kv_heads + kv_head;
          bytes = p.cache.scales[0][block] | static_cast<uint32_t>(p.cache.scales[1][block]) << 8;
        }
      }
    };
    constexpr int kSteps = kGroup / kStepPages;  // steps of a group of pages
    int group = step_begin / kSteps;
    int page, next_page;          // of this group and of the one behind it
    uint32_t bytes, next_bytes;
    look_up(group, page, bytes);
    look_up(group + 1, next_page, next_bytes);

    auto load = [&](int j, uint4 (&keys)[kRounds], uint4 (&values)[kRounds]) {
      const int step = step_begin + j;
      const int held = step / kSteps == group ? page : next_page;
      const int at = step % kSteps * kStepPages + lane_page;
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        const int q = __shfl_sync(0xffffffffu, held, at + r * (kTokens / kCachePage));
        keys[r] = values[r] = make_uint4(0, 0, 0, 0);
        if (q >= 0) {
          keys[r] = *reinterpret_cast<const uint4*>(key_codes + q * page_bytes);
          values[r] = *reinterpret_cast<const uint4*>(value_codes + q * page_bytes);
        }
      }
    };
    auto widen = [](uint8_t* row, int lo, int hi, const uint4& x) {
      *reinterpret_cast<uint4*>(row + lo) =
          make_uint4(e4m3x2_to_f16x2(x.x & 0xffffu), e4m3x2_to_f16x2(x.x >> 16),
                     e4m3x2_to_f16x2(x.y & 0xffffu), e4m3x2_to_f16x2(x.y >> 16));
      *reinterpret_cast<uint4*>(row + hi) =
          make_uint4(e4m3x2_to_f16x2(x.z & 0xffffu), e4m3x2_to_f16x2(x.z >> 16),
                     e4m3x2_to_f16x2(x.w & 0xffffu), e4m3x2_to_f16x2(x.w >> 16));
    };
    auto put = [&](int j, const uint4 (&keys)[kRounds], const uint4 (&values)[kRounds]) {
      const int stage = j % S::kStages;
      const int step = step_begin + j;
      const int entry = step * kStepPages;
      if (j >= S::kStages) wait(&control.tiles_free[stage], j / S::kStages - 1, kSiteFree);
      uint8_t* const tile = own_tile + stage * 2 * S::kTileBytes;
      bool any_nan = false;
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        const int token = r * kTokens + first_token;
        const int i = entry + r * (kTokens / kCachePage) + lane_page;
        const int position = (i < v.front ? i : i - v.front + v.back) * kCachePage +
                             first_token % kCachePage;
        // values that no row sees, or that are NaN (the whole row then), must not meet the product
        const bool unseen = position >= v.length;
        const bool nan = (values[r].x & 0x7fu) == 0x7fu && !unseen;
        any_nan = any_nan || nan;
        if (part == 0) control.row_nan[stage][token] = nan ? 1 : 0;
        widen(tile + r * kTokens * 128, chunk_lo, chunk_hi, keys[r]);
        widen(tile + S::kTileBytes + r * kTokens * 128, chunk_lo, chunk_hi,
              nan || unseen ? make_uint4(0, 0, 0, 0) : values[r]);
      }
      any_nan = __any_sync(0xffffffffu, any_nan);
      if (lane == 0) control.any_nan[stage][warp - kWidenWarp] = any_nan ? 1u : 0u;
      if (warp == kWidenWarp) {
        const int at = step % kSteps * kStepPages + (lane & (kStepPages - 1));
        const int held = __shfl_sync(0xffffffffu, page, at);
        const uint32_t scales = __shfl_sync(0xffffffffu, bytes, at);
        if (lane < kStepPages) {
          // a page of nobody gives weights of zero and asks for no masks
          PageInfo info{0.0f, -INFINITY, 0.0f, -kStepTokens};
          if (held >= 0) {
            const int i = entry + lane;
            const int e = scale_exponent(scales >> 8);
            info = PageInfo{exp2_int(scale_exponent(scales & 0xffu)), static_cast<float>(e),
                            exp2_int(-e), (i < v.front ? i : i - v.front + v.back) * kCachePage};
          }
          control.pages[stage][lane] = info;
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&control.tiles_full[stage]);
      if ((step + 1) % kSteps == 0) {  // on to the next group of pages
        ++group;
        page = next_page;
        bytes = next_bytes;
        look_up(group + 1, next_page, next_bytes);
      }
    };
    uint4 keys_a[kRounds], values_a[kRounds], keys_b[kRounds], values_b[kRounds];
    if (steps > 0) load(0, keys_a, values_a);
    for (int j = 0; j < steps; j += 2) {
      if (j + 1 < steps) load(j + 1, keys_b, values_b);
      put(j, keys_a, values_a);
      if (j + 1 < steps) {
        if (j + 2 < steps) load(j + 2, keys_a, values_a);
        put(j + 1, keys_b, values_b);
      }
    }
  }

  tcgen05_fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    tcgen05_fence_after_sync();
    tmem_dealloc(tmem, kTmemColumns);
  }
}

}  // namespace

template <typename T, int D>
int32_t launch_tiles(const AttentionParams& p, cudaStream_t stream, char* message,
                     size_t capacity) {
  if (cudaFuncSetAttribute(tile_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           Shape<D>::kSharedBytes) != cudaSuccess ||
      cudaFuncSetAttribute(tile_kernel<T, D>, cudaFuncAttributePreferredSharedMemoryCarveout,
                           cudaSharedmemCarveoutMaxShared) != cudaSuccess) {
    return fail(NML_SM100_LAUNCH_FAILURE, "cannot configure shared memory", message, capacity);
  }
  // the shares above count on what the compiler gave every thread
  cudaFuncAttributes attributes;
  if (cudaFuncGetAttributes(&attributes, tile_kernel<T, D>) != cudaSuccess ||
      attributes.numRegs != kLaunchRegisters) {
    return fail(NML_SM100_LAUNCH_FAILURE, "tile kernel built with another register count", message,
                capacity);
  }
  const int64_t items = query_tiles(p.tokens, p.cache.batch, p.group);
  tile_kernel<T, D><<<static_cast<unsigned>(items * p.splits * p.cache.kv_heads), kThreads,
                      Shape<D>::kSharedBytes, stream>>>(p);
  return NML_SM100_OK;
}

template int32_t launch_tiles<__half, 64>(const AttentionParams&, cudaStream_t, char*, size_t);
template int32_t launch_tiles<__half, 128>(const AttentionParams&, cudaStream_t, char*, size_t);
template int32_t launch_tiles<__nv_bfloat16, 64>(const AttentionParams&, cudaStream_t, char*,
                                                 size_t);
template int32_t launch_tiles<__nv_bfloat16, 128>(const AttentionParams&, cudaStream_t, char*,
                                                  size_t);

}  // namespace nml_sm100
