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
//   warps 4-7  widen the codes: E4M3 to F16 (exact, the block scales stay out), from where they are
//              staged into 128-byte swizzled tiles
//   warp 8     issues the products: S = Q K^T (A: q in tensor memory, B: keys, K-major) and
//              O += W V (A: weights in tensor memory, B: values, MN-major: tokens are rows)
//   warp 9     brings in the blocks of codes by bulk copies some steps ahead; page table entries
//              and scales are fetched for 32 pages at a time, 32 pages ahead
//   warps 10-11  find the range of the pages' value exponents while the others prepare
// Registers move from the last two warpgroups to the softmax, which holds a row's 64 scores.
//
// F16 weights carry the exponents of their values, which costs them bits where these lie far apart.
// Where the walk's pages lie within 2^6 of each other, as those of one head do, that is bounded (a
// probability is good to 2^-11 of itself and to 2^-19 of the row's largest); other walks take their
// values whole, as BF16 (a code times a power of two is exact there), and their weights as the sum
// of two BF16 terms with a product each.  The ragged prompts below take 379 us with both forms in the
// kernel, 366 with the first alone, 459 when they need the second; choosing step by step cost 393.
//
// The running maximum M only stabilises: weights above one are as good as those below as long as
// F16 holds them (sums are f32).  So a step is weighted against the maximum of the steps before it,
// and only when a page's weights sum to more than 2^14 is its own maximum formed, the accumulator
// in tensor memory rescaled and the step repeated: once or twice for a row.  A key or value row of
// NaN codes (stored whole by the append) enters the products as zeros and marks the rows that see
// it, whose results become NaN; it does not reach the rows that do not.
//
// What bounds it: one exponential for each score.  A step of 128 x 64 takes 512 clocks of the SM's
// 16 exponentials per clock and 256 (head_dim 64) of the tensor cores.  Measured on B200: four ragged
// prompts (1200 to 2000 tokens behind up to 2000, 64 query and 8 kv heads of 64, 197 GFLOP) 379 us,
// 520 TFLOP/s, 0.45 of the exponentials' rate.  With the first form alone a CTA's step takes 1490
// clocks beside another CTA and 1265 alone: score barrier 100, page data 110, scores 90, exponentials
// 900 (605 with nothing else on the SM), weights back 120; finding the tile, queries and first codes
// cost a CTA about 8000, its results 2500.  Tried and slower: polynomial exponentials on the
// multiply-add units for a quarter or half of the scores (two f32 at a time run there at no more than
// the rate of one), two threads for a row (437 us where one took 368), three CTAs with the queries in
// shared memory (446), one CTA of two tiles that share the widened codes and take the exponentials in
// turn (392), a short loop over pages for the second form (373, but 757 where it is needed).
#include <type_traits>

#include "attention_q8.cuh"
#include "sm100_primitives.cuh"

namespace nml_sm100 {
namespace {

constexpr int kStepTokens = 64;
constexpr int kStepPages = kStepTokens / kCachePage;
constexpr int kSoftmaxThreads = 128;
constexpr int kWidenThreads = 128;
constexpr int kWidenWarp = 4, kMmaWarp = 8, kLoadWarp = 9;
constexpr int kThreads = 384;
constexpr int kRangeWarp = 10, kRangeThreads = 64;
// named barriers: tensor memory, and the range of exponents for each of the roles that ask for it
constexpr int kBarrierTmem = 1, kBarrierSoftmax = 2, kBarrierWiden = 3, kBarrierMma = 4;
constexpr int kLaunchRegisters = 80;  // of a thread: two CTAs fill an SM
constexpr int kTmemColumns = 256;

// Bits 8 + site of the status word say which wait ran out.
constexpr int kSiteScores = 16, kSiteWeights = 17, kSiteTiles = 18, kSiteProduct = 19,
              kSiteFree = 20, kSiteStaged = 21;

// What the softmax needs to know of a page: score factor, exponent of the values, its inverse
// power for the denominator, first token.
struct alignas(16) PageInfo {
  float key_scale, value_exponent, unscale;
  int token;
};

template <int D>
struct Shape {
  static constexpr int kTileBytes = kStepTokens * D * 2;
  static constexpr int kStages = D == 64 ? 3 : 2;       // F16 tiles
  static constexpr int kCodeBytes = kStepTokens * D;    // of a step's keys, then of its values
  static constexpr int kStaged = D == 64 ? 6 : 2;       // steps of codes on their way
  static constexpr int kBuffers = D == 64 ? 2 : 1;  // score buffers in tensor memory
  static constexpr int kOut = 0, kQuery = D, kScores = D + D / 2;
  static constexpr int kStagedOffset = kStages * 2 * kTileBytes;
  static constexpr int kSharedBytes = kStagedOffset + kStaged * 2 * kCodeBytes + 1024;
  // The three warpgroups' shares of the CTA's registers at launch.
  static constexpr int kSoftmaxRegisters = D == 64 ? 144 : 128;
  static constexpr int kWidenRegisters = D == 64 ? 56 : 72;
  static constexpr int kMmaRegisters = 40;
  static_assert(kSoftmaxRegisters + kWidenRegisters + kMmaRegisters == 3 * kLaunchRegisters,
                "a share that the launch does not cover would be waited for without end");
  static_assert(kStaged + kStages < 16, "page data");
  static_assert(kScores + kBuffers * kStepTokens <= kTmemColumns, "tensor memory");
};

// Steps whose page data is kept: more than the staged and the widened ones together.
constexpr int kInfoSteps = 16;

template <int D>
struct Control {
  uint64_t staged_full[Shape<D>::kStaged], staged_free[Shape<D>::kStaged];
  uint64_t tiles_full[Shape<D>::kStages], tiles_free[Shape<D>::kStages];
  uint64_t scores_full[Shape<D>::kBuffers];
  // one for each buffer: a warp may run ahead of the others by as many steps as there are buffers
  uint64_t weights_full[Shape<D>::kBuffers], product_done[Shape<D>::kBuffers];
  uint64_t query_full, drained;
  uint32_t tmem;
  int abort_flag;
  int sequence, first_row, rows, first_position;
  int largest_exponent[kRangeThreads / 32], least_exponent[kRangeThreads / 32];
  PageInfo pages[kInfoSteps][kStepPages];
  alignas(16) uint32_t any_nan[Shape<D>::kStages][4];  // read 16 bytes at a time
  uint8_t row_nan[Shape<D>::kStages][kStepTokens];
};

// The warpgroup's share of the CTA's registers; a larger one waits for others to give theirs.
template <int N>
__device__ __forceinline__ void take_registers() {
  if constexpr (N > kLaunchRegisters) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
  }
}

template <int kBarrier, int kCount>
__device__ __forceinline__ void named_barrier_sync() {
  asm volatile("barrier.cta.sync.aligned %0, %1;" ::"n"(kBarrier), "n"(kCount) : "memory");
}
template <int kBarrier, int kCount>
__device__ __forceinline__ void named_barrier_arrive() {
  asm volatile("barrier.cta.arrive.aligned %0, %1;" ::"n"(kBarrier), "n"(kCount) : "memory");
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

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // through a shuffle: the compiler then knows the roles' branches and loops to be warp-uniform
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int kv_head = blockIdx.x % p.cache.kv_heads;
  const int item = blockIdx.x / p.cache.kv_heads / p.splits;
  const int split = blockIdx.x / p.cache.kv_heads % p.splits;
  const int per_tile = kTileRows / p.group;

  // ---- which sequence, which of its tiles: the last tile (the longest walk) comes first ----
  if (warp == 0) {
    int sequence = -1, tile = 0, passed = 0, begin = 0, end = 0, given_end = 0, length = 0;
    for (int base = 0; base < p.cache.batch && sequence < 0; base += 32) {
      const int b = base + lane;
      int tiles = 0;
      if (b < p.cache.batch) {
        begin = max(p.offsets[b], 0);
        given_end = p.offsets[b + 1];
        length = max(p.cache.lengths[b], 0);
        end = min(given_end, p.tokens);
        tiles = end > begin ? (end - begin + per_tile - 1) / per_tile : 0;
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
        begin = __shfl_sync(0xffffffffu, begin, at);
        end = __shfl_sync(0xffffffffu, end, at);
        given_end = __shfl_sync(0xffffffffu, given_end, at);
        length = __shfl_sync(0xffffffffu, length, at);
      }
      passed += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) {
      if (sequence >= 0 && length > p.cache.table_width * kCachePage) {
        atomicOr(p.status, NML_SM100_STATUS_INDEX_RANGE);
      }
      control.sequence = sequence;
      control.first_row = begin + tile * per_tile;
      control.rows = min(per_tile, end - control.first_row);
      control.first_position = length - given_end + control.first_row;
    }
  }
  if (threadIdx.x == kMmaWarp * 32) {
    for (int i = 0; i < S::kStaged; ++i) {
      mbar_init(&control.staged_full[i], 1);
      mbar_init(&control.staged_free[i], kWidenThreads);
    }
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&control.tiles_full[i], kWidenThreads);
      mbar_init(&control.tiles_free[i], 1);
    }
    for (int i = 0; i < S::kBuffers; ++i) {
      mbar_init(&control.scores_full[i], 2);
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

  const int first_row = control.first_row, rows = control.rows;
  const int first_position = control.first_position;
  const int most = p.cache.table_width * kCachePage;
  const Visible v = visible_pages(first_position + rows,
                                  p.window > 0 ? first_position + 1 - p.window : 0, p.first, most);
  const int all_steps = (v.pages + kStepPages - 1) / kStepPages;
  const int per_split = (all_steps + p.splits - 1) / p.splits;
  const int step_begin = min(all_steps, split * per_split);
  const int steps = __shfl_sync(0xffffffffu, min(all_steps - step_begin, per_split), 0);

  if (warp == kMmaWarp) {
    tmem_alloc(&control.tmem, kTmemColumns);
    tmem_relinquish_alloc_permit();
  }
  // A softmax thread's row; its queries (and sink) are on their way before tensor memory is waited
  // for, which the loads of codes need not do at all.
  const int token = threadIdx.x / p.group;
  const int head = kv_head * p.group + threadIdx.x - token * p.group;
  const bool live = warp < kWidenWarp && token < rows;
  uint4 query[D / 8];
  float sink = 0.0f;
  uint32_t tmem = 0;
  if (warp < kWidenWarp || warp == kMmaWarp) {
    if (warp < kWidenWarp) {
      const uint4* const source = reinterpret_cast<const uint4*>(
          static_cast<const T*>(p.query) +
          static_cast<int64_t>(first_row + token) * p.query_token_stride +
          head * p.query_head_stride);
#pragma unroll
      for (int i = 0; i < D / 8; ++i) query[i] = live ? source[i] : make_uint4(0, 0, 0, 0);
      if (p.sinks != nullptr && live) sink = p.sinks[head] * kLog2e;
    }
    tcgen05_fence_before_sync();
    named_barrier_sync<kBarrierTmem, kSoftmaxThreads + 32>();
    tcgen05_fence_after_sync();
    tmem = __shfl_sync(0xffffffffu, control.tmem, 0);
  }

  auto wait = [&](uint64_t* bar, int phase, int site) {
    mbar_wait_or_abort(bar, static_cast<uint32_t>(phase) & 1u, abort_flag, p.status, site);
    __syncwarp();
  };

  // Whether the walk's values lie too far apart for weights in F16, behind the role's barrier.
  auto values_far_apart = [&]() {
    const int range = max(control.largest_exponent[0], control.largest_exponent[1]) -
                      min(control.least_exponent[0], control.least_exponent[1]);
    return __any_sync(0xffffffffu, range > kExponentRange) != 0;
  };

  // The product of step j.  Whoever has step j's scores knows that the product kBuffers steps
  // back is complete, and no product passes a step that this warp has not handed over: with a
  // barrier for each buffer a parity names one phase only.
  auto wait_product = [&](int j) {
    wait(&control.product_done[j % S::kBuffers], j / S::kBuffers, kSiteProduct);
  };

  if (warp < kWidenWarp) {
    // ------------------------------------------------------------------ softmax
    take_registers<S::kSoftmaxRegisters>();
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    // rows of nobody walk like the last row, so that they do not ask for masks
    const int position = first_position + (live ? token : rows - 1);
    const int length = min(position + 1, most);
    const int start = p.window > 0 ? min(max(0, position + 1 - p.window), most) : 0;

    // q: largest magnitude, then F16 into tensor memory, column c holding elements 2c and 2c + 1
    float factor = p.scale_log2;
    bool poisoned;  // something the row sees, or the row itself, is NaN: so is its result
    {
      uint32_t largest = 0;  // magnitude bits in the upper half
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const uint32_t words[4] = {query[i].x, query[i].y, query[i].z, query[i].w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          largest = max(largest, max((words[w] & 0x7fffu) << 16, words[w] & 0x7fff0000u));
        }
      }
      // a query with an infinity or a NaN gives NaN; its scores need not be formed
      constexpr bool kHalf = std::is_same<T, __half>::value;
      poisoned = largest >= (kHalf ? 0x7c000000u : 0x7f800000u);
      const int shift = kHalf ? 0 : query_shift(largest);
      const float up = exp2_int(shift);
      factor *= exp2_int(-shift);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        uint32_t packed[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 x = poisoned ? make_uint4(0, 0, 0, 0) : query[2 * i + h];
          const uint32_t words[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            if constexpr (kHalf) {
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
    const int last_start = p.window > 0 ? min(max(0, first_position + rows - p.window), most) : 0;
    const int first_whole = last_start == 0 ? 0 : v.front + (last_start + kCachePage - 1) /
                                                                kCachePage - v.back;
    const int whole_pages = v.front + min(max(first_position + 1, 0), most) / kCachePage - v.back;
    const int whole_begin = (first_whole + kStepPages - 1) / kStepPages - step_begin;
    const int whole_end = max(whole_pages, 0) / kStepPages - step_begin;

    float running_max = -INFINITY, running_sum = 0.0f;
    // a warp none of whose rows is anybody's hands over whatever its lanes hold: a row of the
    // products depends on that row of weights only
    const bool idle = warp * 32 >= rows * p.group;
    auto walk = [&](auto whole_values) {
      constexpr bool kWide = decltype(whole_values)::value;
      for (int j = 0; j < steps; ++j) {
        const int buffer = j % S::kBuffers, stage = j % S::kStages;
        if (idle) {
          wait(&control.scores_full[buffer], j / S::kBuffers, kSiteScores);
          mbar_arrive(&control.weights_full[buffer]);
          continue;
        }
        const uint32_t columns = lanes + S::kScores + buffer * kStepTokens;
        const PageInfo* const pages = control.pages[j % kInfoSteps];
        wait(&control.scores_full[buffer], j / S::kBuffers, kSiteScores);
        tcgen05_fence_after_sync();
        float page_factor[kStepPages], value_exponent[kStepPages], unscale[kStepPages];
#pragma unroll
        for (int q = 0; q < kStepPages; ++q) {
          const float4 info = *reinterpret_cast<const float4*>(&pages[q]);
          page_factor[q] = factor * info.x;
          // (minus infinity for a page of nobody)
          value_exponent[q] = !kWide || info.y == -INFINITY ? info.y : 0.0f;
          unscale[q] = kWide ? 1.0f : info.z;
        }
        const uint4 nan_words = *reinterpret_cast<const uint4*>(control.any_nan[stage]);
        const bool nans = (nan_words.x | nan_words.y | nan_words.z | nan_words.w) != 0;

        // Weights against the maximum so far; their sum tells whether it still serves.  Only when
        // it does not (or there is none yet) is the step's maximum formed and the step done again.
        uint32_t packed[kStepTokens / 2], low[kWide ? kStepTokens / 2 : 1];
        float step_sum;
        bool with_maximum = __any_sync(0xffffffffu, running_max == -INFINITY);
        while (true) {
          uint32_t scores[2][32];
          tmem_load_32x32(columns, scores[0]);
          tmem_load_32x32(columns + 32, scores[1]);
          tmem_load_wait();
          float s[kStepTokens];
#pragma unroll
          for (int i = 0; i < kStepTokens; ++i) s[i] = __uint_as_float(scores[i / 32][i % 32]);
          if (j < whole_begin || j >= whole_end || nans) {
            // bit i: token i is seen; loops, so that steps without masks branch over all of this
            uint32_t seen[2] = {0, 0};
#pragma unroll 1
            for (int q = 0; q < kStepPages; ++q) {
              const int t = pages[q].token;
              auto below = [&](int limit) {  // bits of the page's tokens in front of `limit`
                return (1u << min(max(limit - t, 0), kCachePage)) - 1u;
              };
              const uint32_t bits = below(length) & (~below(start) | below(p.first));
              if (nans) {
                const uint8_t* const row_nan = &control.row_nan[stage][q * kCachePage];
#pragma unroll 1
                for (int i = 0; i < kCachePage; ++i) {
                  if (row_nan[i] != 0 && (bits >> i & 1u) != 0) poisoned = true;
                }
              }
              const int shift = q * kCachePage & 31;
              seen[0] |= q < 2 ? bits << shift : 0u;
              seen[1] |= q < 2 ? 0u : bits << shift;
            }
#pragma unroll
            for (int i = 0; i < kStepTokens; ++i) {
              if ((seen[i / 32] >> (i % 32) & 1u) == 0) s[i] = -INFINITY;
            }
#pragma unroll
            for (int q = 0; q < kStepPages; ++q) page_factor[q] = masked_factor(page_factor[q]);
            __syncwarp();
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
                const uint32_t out_columns = lanes + S::kOut + c;
                uint32_t x[16], y[8], z[8];
                tmem_load_32x16(out_columns, x);
                tmem_load_wait();
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  y[i] = __float_as_uint(__uint_as_float(x[i]) * rescale);
                  z[i] = __float_as_uint(__uint_as_float(x[i + 8]) * rescale);
                }
                tmem_store_32x8(out_columns, y);
                tmem_store_32x8(out_columns + 8, z);
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
              if constexpr (kWide) {
                const uint32_t high = Elem<__nv_bfloat16>::pack2(a, b);
                packed[8 * q + i] = high;
                low[8 * q + i] = Elem<__nv_bfloat16>::pack2(
                    a - __uint_as_float(high << 16), b - __uint_as_float(high & 0xffff0000u));
              } else {
                packed[8 * q + i] = Elem<__half>::pack2(a, b);
              }
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
        // over the thread's own scores
#pragma unroll
        for (int q = 0; q < kStepPages; ++q) {
          const uint32_t(&page)[8] = *reinterpret_cast<const uint32_t(*)[8]>(&packed[8 * q]);
          tmem_store_32x8(columns + 8 * q, page);
          if constexpr (kWide) {
            const uint32_t(&rest)[8] = *reinterpret_cast<const uint32_t(*)[8]>(&low[8 * q]);
            tmem_store_32x8(columns + kStepTokens / 2 + 8 * q, rest);
          }
        }
        tmem_store_wait();
        tcgen05_fence_before_sync();
        mbar_arrive(&control.weights_full[buffer]);
      }
    };
    if (steps > 0) {
      named_barrier_sync<kBarrierSoftmax, kRangeThreads + kSoftmaxThreads>();
      if (values_far_apart()) {
        walk(std::true_type{});
      } else {
        walk(std::false_type{});
      }
    }

    // ---- the rows' results ----
    if (steps > 0) {
      wait_product(steps - 1);
      tcgen05_fence_after_sync();
    }
    const int64_t query_head = static_cast<int64_t>(first_row + token) * p.query_heads + head;
    // a row that sees nothing has no maximum; its output is zero, whatever its queries hold
    if (running_max == -INFINITY) {
      running_sum = 0.0f;
    } else if (poisoned) {
      running_sum = __uint_as_float(0x7fc00000u);
    }
    float denominator = running_sum;
    if (p.sinks != nullptr && live) {
      denominator += exp2f(sink - running_max);
    }
    const float inverse = running_sum == 0.0f ? 0.0f : 1.0f / denominator;
    float* partial = p.partial + (query_head * p.splits + split) * kPartial<D>;
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
        for (int i = 0; i < 16; i += 4) {
          *reinterpret_cast<uint4*>(partial + c + i) =
              make_uint4(x[i], x[i + 1], x[i + 2], x[i + 3]);
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
      *reinterpret_cast<float4*>(partial + D) = make_float4(running_max, running_sum, 0.0f, 0.0f);
    }
  } else if (warp >= kMmaWarp) {
    // ------------------------------------------------------------------ matrix products
    take_registers<S::kMmaRegisters>();
    if (warp == kLoadWarp) {
      // Blocks of codes are contiguous: one bulk copy each.  Lane i holds page (-1: nothing there)
      // and scale bytes of entry i of a group of 32 pages, the next group's beside them.
      constexpr int kGroup = 32, kSteps = kGroup / kStepPages;
      constexpr uint32_t kBlockBytes = kCachePage * D;
      constexpr int32_t kNoEntry = -2147483647 - 1;  // past the walk, unlike a bad table entry
      auto table_entry = [&](int group) {
        const int i = group * kGroup + lane;
        return i >= step_begin * kStepPages && i < min(v.pages, (step_begin + steps) * kStepPages)
                   ? p.cache.page_table[static_cast<int64_t>(sequence) * p.cache.table_width +
                                        (i < v.front ? i : i - v.front + v.back)]
                   : kNoEntry;
      };
      auto look_up = [&](int32_t entry, int& page, uint32_t& key_byte, uint32_t& value_byte) {
        page = -1;
        key_byte = value_byte = 0;
        if (entry == kNoEntry) return;
        if (entry < 0 || entry >= p.cache.physical_pages) {
          atomicOr(p.status, NML_SM100_STATUS_INDEX_RANGE);
          return;
        }
        page = entry;
        const int64_t block = static_cast<int64_t>(page) * p.cache.kv_heads + kv_head;
        key_byte = p.cache.scales[0][block];
        value_byte = p.cache.scales[1][block];
      };
      int group = step_begin / kSteps;
      int page, next_page;
      uint32_t key_byte, value_byte, next_key, next_value;
      {
        const int32_t entry = table_entry(group), next_entry = table_entry(group + 1);
        look_up(entry, page, key_byte, value_byte);
        look_up(next_entry, next_page, next_key, next_value);
      }
      for (int j = 0; j < steps; ++j) {
        const int step = step_begin + j, slot = j % S::kStaged;
        if (j >= S::kStaged) wait(&control.staged_free[slot], j / S::kStaged - 1, kSiteFree);
        const int at = step % kSteps * kStepPages + (lane & (kStepPages - 1));
        const int held = __shfl_sync(0xffffffffu, page, at);
        const uint32_t key_scale = __shfl_sync(0xffffffffu, key_byte, at);
        const uint32_t value_scale = __shfl_sync(0xffffffffu, value_byte, at);
        const bool mine = lane < kStepPages;
        if (mine) {
          // a page of nobody gives weights of zero and asks for no masks
          PageInfo info{0.0f, -INFINITY, 0.0f, -kStepTokens};
          if (held >= 0) {
            const int i = step * kStepPages + lane;
            const int e = scale_exponent(value_scale);
            info = PageInfo{exp2_int(scale_exponent(key_scale)), static_cast<float>(e),
                            exp2_int(-e), (i < v.front ? i : i - v.front + v.back) * kCachePage};
          }
          control.pages[j % kInfoSteps][lane] = info;
        }
        __syncwarp();  // lane 0's arrival hands over the other lanes' page data too
        const uint32_t there = __ballot_sync(0xffffffffu, mine && held >= 0);
        if (lane == 0) {
          mbar_arrive_expect_tx(&control.staged_full[slot], __popc(there) * 2 * kBlockBytes);
        }
        __syncwarp();
        if (mine && held >= 0) {
          const int64_t block = static_cast<int64_t>(held) * p.cache.kv_heads + kv_head;
          uint8_t* const codes =
              shared + S::kStagedOffset + slot * 2 * S::kCodeBytes + lane * kBlockBytes;
          bulk_load(codes, p.cache.codes[0] + block * kBlockBytes, kBlockBytes,
                    &control.staged_full[slot]);
          bulk_load(codes + S::kCodeBytes, p.cache.codes[1] + block * kBlockBytes, kBlockBytes,
                    &control.staged_full[slot]);
        }
        __syncwarp();
        if ((step + 1) % kSteps == 0) {  // on to the next group of pages
          ++group;
          page = next_page;
          key_byte = next_key;
          value_byte = next_value;
          look_up(table_entry(group + 1), next_page, next_key, next_value);
        }
      }
      // whatever has happened, no copy may land after the CTA is gone
      for (int j = max(0, steps - S::kStaged); j < steps; ++j) {
        mbar_wait(&control.staged_full[j % S::kStaged], j / S::kStaged & 1);
      }
    } else if (warp == kMmaWarp) {
      constexpr uint64_t desc_hi = static_cast<uint64_t>(kUmmaDescHiSw128) << 32;
      constexpr uint32_t score_idesc = umma_idesc_f16(kUmmaF16, kUmmaF16, kTileRows, kStepTokens);
      constexpr uint32_t product_idesc =
          umma_idesc_f16(kUmmaF16, kUmmaF16, kTileRows, D) | (1u << 16);  // B is MN-major
      constexpr uint32_t wide_idesc =
          umma_idesc_f16(kUmmaBF16, kUmmaBF16, kTileRows, D) | (1u << 16);
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
        // a plain arrival too: it passes on what this warp saw at tiles_full, the page data
        if (lane == 0) mbar_arrive(&control.scores_full[buffer]);
        __syncwarp();
      };
      if (steps > 0) {
        wait(&control.query_full, 0, kSiteWeights);
        tcgen05_fence_after_sync();
        for (int j = 0; j < min(steps, S::kBuffers); ++j) scores(j);
      }
      auto walk = [&](auto whole_values) {
        constexpr bool kWide = decltype(whole_values)::value;
        for (int j = 0; j < steps; ++j) {
          const int stage = j % S::kStages, buffer = j % S::kBuffers;
          wait(&control.weights_full[buffer], j / S::kBuffers, kSiteWeights);
          tcgen05_fence_after_sync();
          const uint32_t values = smem_u32(shared + stage * 2 * S::kTileBytes + S::kTileBytes);
#pragma unroll
          for (int k = 0; k < (kWide ? 2 : 1) * kStepTokens / 16; ++k) {
            // 16 tokens are 2 KB of 128-byte rows; the leading offset is the tile of the next 64
            // dimensions
            const uint32_t address = values + k % (kStepTokens / 16) * 2048;
            const uint32_t low = ((address & 0x3ffffu) >> 4) | ((kStepTokens * 128 >> 4) << 16);
            const uint32_t weights = tmem + S::kScores + buffer * kStepTokens + 8 * k;
            umma_f16_tmem_a_elect(tmem + S::kOut, weights, desc_hi | low,
                                  kWide ? wide_idesc : product_idesc, j > 0 || k > 0 ? 1u : 0u);
          }
          umma_commit_elect(&control.tiles_free[stage]);
          umma_commit_elect(&control.product_done[buffer]);
          if (j + S::kBuffers < steps) {
            // the scores go over the weights that this product reads
            wait_product(j);
            scores(j + S::kBuffers);
          }
        }
      };
      if (steps > 0) {
        named_barrier_sync<kBarrierMma, kRangeThreads + 32>();
        if (values_far_apart()) {
          walk(std::true_type{});
        } else {
          walk(std::false_type{});
        }
      }
      umma_commit_elect(&control.drained);
      if (!mbar_wait(&control.drained, 0)) {
        *abort_flag = 1;
        atomicOr(p.status, NML_SM100_STATUS_BARRIER_TIMEOUT | (0x100 << kSiteProduct));
      }
    } else if (steps > 0) {
      // ---- the range of the walk's value exponents, eight pages of a lane under way at once ----
      constexpr int kAtOnce = 8;
      int largest = kLowestExponent, least = kHighestExponent;
      const int end = min(v.pages, (step_begin + steps) * kStepPages);
      const int32_t* const table =
          p.cache.page_table + static_cast<int64_t>(sequence) * p.cache.table_width;
      for (int i = step_begin * kStepPages + (warp - kRangeWarp) * 32 + lane; i < end;
           i += kAtOnce * kRangeThreads) {
        int32_t page[kAtOnce];
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
          const int entry = i + n * kRangeThreads;
          page[n] = entry < end ? table[entry < v.front ? entry : entry - v.front + v.back] : -1;
        }
        int exponent[kAtOnce];
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
          if (page[n] >= p.cache.physical_pages) page[n] = -1;  // (reported by the loads)
          const int64_t block = static_cast<int64_t>(page[n]) * p.cache.kv_heads + kv_head;
          exponent[n] = page[n] < 0 ? 0 : scale_exponent(p.cache.scales[1][block]);
        }
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
          if (page[n] < 0) continue;
          largest = max(largest, exponent[n]);
          least = min(least, exponent[n]);
        }
      }
      largest = __reduce_max_sync(0xffffffffu, largest);
      least = __reduce_min_sync(0xffffffffu, least);
      if (lane == 0) {
        control.largest_exponent[warp - kRangeWarp] = largest;
        control.least_exponent[warp - kRangeWarp] = least;
      }
      __syncwarp();
      named_barrier_arrive<kBarrierWiden, kRangeThreads + kWidenThreads>();
      named_barrier_arrive<kBarrierMma, kRangeThreads + 32>();
      named_barrier_arrive<kBarrierSoftmax, kRangeThreads + kSoftmaxThreads>();
    }
  } else {
    // ------------------------------------------------------------------ codes to F16 tiles
    take_registers<S::kWidenRegisters>();
    constexpr int kParts = D / 16;                          // pieces of 16 codes of a token's row
    constexpr int kTokens = kWidenThreads / kParts;         // tokens of one pass of the group
    constexpr int kRounds = kStepTokens / kTokens;
    const int thread = threadIdx.x - kWidenWarp * 32;
    const int part = thread % kParts, first_token = thread / kParts;
    const int first_page = first_token / kCachePage;
    const uint8_t* const own_codes = shared + S::kStagedOffset + thread * 16;
    uint8_t* const own_tile = shared + (part / 4) * (kStepTokens * 128) + first_token * 128;
    // 16-byte chunks 2 part and 2 part + 1 of a 128-byte row, swizzled by the token
    const int chunk_lo = ((2 * (part % 4)) ^ (first_token & 7)) * 16;
    const int chunk_hi = ((2 * (part % 4) + 1) ^ (first_token & 7)) * 16;
    auto widen = [&](uint8_t* row, const uint4& x) {
      *reinterpret_cast<uint4*>(row + chunk_lo) =
          make_uint4(e4m3x2_to_f16x2(x.x & 0xffffu), e4m3x2_to_f16x2(x.x >> 16),
                     e4m3x2_to_f16x2(x.y & 0xffffu), e4m3x2_to_f16x2(x.y >> 16));
      *reinterpret_cast<uint4*>(row + chunk_hi) =
          make_uint4(e4m3x2_to_f16x2(x.z & 0xffffu), e4m3x2_to_f16x2(x.z >> 16),
                     e4m3x2_to_f16x2(x.w & 0xffffu), e4m3x2_to_f16x2(x.w >> 16));
    };
    // a code times a power of two, exact in BF16
    auto widen_whole = [&](uint8_t* row, const uint4& x, float power) {
      const uint32_t words[4] = {x.x, x.y, x.z, x.w};
      uint32_t y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t pair = e4m3x2_to_f16x2(words[i / 2] >> (16 * (i & 1)) & 0xffffu);
        y[i] = Elem<__nv_bfloat16>::pack2(Elem<__half>::from_bits(pair & 0xffffu) * power,
                                          Elem<__half>::from_bits(pair >> 16) * power);
      }
      *reinterpret_cast<uint4*>(row + chunk_lo) = make_uint4(y[0], y[1], y[2], y[3]);
      *reinterpret_cast<uint4*>(row + chunk_hi) = make_uint4(y[4], y[5], y[6], y[7]);
    };
    auto walk = [&](auto whole_values) {
      constexpr bool kWide = decltype(whole_values)::value;
      for (int j = 0; j < steps; ++j) {
        const int stage = j % S::kStages, slot = j % S::kStaged;
        wait(&control.staged_full[slot], j / S::kStaged, kSiteStaged);
        uint4 keys[kRounds], values[kRounds];
        int token[kRounds];
        const uint8_t* const codes = own_codes + slot * 2 * S::kCodeBytes;
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
          keys[r] = *reinterpret_cast<const uint4*>(codes + r * kTokens * D);
          values[r] = *reinterpret_cast<const uint4*>(codes + S::kCodeBytes + r * kTokens * D);
          token[r] = control.pages[j % kInfoSteps][first_page + r * (kTokens / kCachePage)].token +
                     first_token % kCachePage;
        }
        mbar_arrive(&control.staged_free[slot]);
        if (j >= S::kStages) wait(&control.tiles_free[stage], j / S::kStages - 1, kSiteFree);
        uint8_t* const tile = own_tile + stage * 2 * S::kTileBytes;
        bool any_nan = false;
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
          // tokens that no row sees, or that are NaN (a whole row of codes then), become zeros; a
          // page of nobody has negative tokens
          const bool unseen = token[r] >= v.length || token[r] < 0;
          const bool nan =
              ((values[r].x & 0x7fu) == 0x7fu || (keys[r].x & 0x7fu) == 0x7fu) && !unseen;
          any_nan = any_nan || nan;
          if (part == 0) control.row_nan[stage][r * kTokens + first_token] = nan ? 1 : 0;
          if (nan || unseen) keys[r] = values[r] = make_uint4(0, 0, 0, 0);
          widen(tile + r * kTokens * 128, keys[r]);
          if constexpr (kWide) {
            const PageInfo& info =
                control.pages[j % kInfoSteps][first_page + r * (kTokens / kCachePage)];
            widen_whole(tile + S::kTileBytes + r * kTokens * 128, values[r],
                        nan || unseen ? 0.0f : exp2_int(static_cast<int>(info.value_exponent)));
          } else {
            widen(tile + S::kTileBytes + r * kTokens * 128, values[r]);
          }
        }
        any_nan = __any_sync(0xffffffffu, any_nan);
        if (lane == 0) control.any_nan[stage][warp - kWidenWarp] = any_nan ? 1u : 0u;
        fence_proxy_async_smem();
        mbar_arrive(&control.tiles_full[stage]);
      }
    };
    if (steps > 0) {
      named_barrier_sync<kBarrierWiden, kRangeThreads + kWidenThreads>();
      if (values_far_apart()) {
        walk(std::true_type{});
      } else {
        walk(std::false_type{});
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
