// Attention over the 8-bit paged K/V cache, one query row (token) at a time: the form for single
// tokens, bound by reading every visible code once.
//
//   out = sum_j p_j v_j / (sum_j p_j + exp(sink)),  p_j = exp(scale * q.k_j)
//
// With k_j = 2^a code_j and v_j = 2^b code'_j (one exponent for each block of 16 tokens) both
// products run on the bare codes, which are exact in f16.  With B the largest value exponent met so
// far (of a warp) and d = b - B:
//
//   t_j = q.code_j * (scale log2(e) 2^a),   w_j = exp2(t_j + d - M),   M = max_j (t_j + d)
//   numerator = 2^B sum_j w_j code'_j,      denominator = sum_j w_j 2^-d
//
// so a block's scales cost one factor of the scores and one addend of the exponent, and M bounds
// what enters the f16 product.  Only d from -4 to 2 goes into the f16 weights, whose bits a larger
// gap would cost: a page below that is weighted with d = 0 and its product scaled by 2^d in f32
// before it is added, a page above raises B, and the sums so far are scaled once.
//
// M is the maximum of the steps before: weights above one are as good as those below as long as F16
// holds them, so a step's own maximum is formed, and the state rescaled, only when the weights'
// sum passes 2^14 (or there is none yet).
//
// Shape of the work: one CTA of four warps per (row, kv head and up to 16 of its query heads, split
// of the visible pages); its warps take steps of two pages (one at head_dim 128) in turn.  A block
// is 16 * head_dim contiguous bytes: one bulk copy into a ring of two steps for each warp, the next
// one issued as soon as the last read is done, page table entries and scales fetched 32 pages ahead.
// Scores [16 tokens x 8 heads] = K . q^T with keys widened in registers into mma.sync fragments,
// weights transposed between lanes by movmatrix, out^T [dims x 8 heads] += V^T . w, where pairs of
// tokens are interleaved byte-wise before they are widened.  Four CTAs of 128 registers an SM (13 of
// their 16 warps on average) keep the conversions and products (about 100 instructions a page) off the
// memory's back.  Splits are joined by a second launch that starts while the first still runs.
//
// Measured on B200 (device time): 64 sequences of 4097 tokens, 64 query and 8 kv heads of 64 (269.5
// MB): 53.7 us, 5.0 TB/s (58.3 with values far apart); 3 sequences of 60000 to 100000 tokens, 32 and 8
// heads of 128 (474 MB): 89 us, 5.3 TB/s, in 24 splits; one sequence of 413 tokens: 6.8 us.
#include <type_traits>

#include "attention_q8.cuh"
#include "sm100_primitives.cuh"

namespace nml_sm100 {
namespace {

constexpr int kWarps = 4;
constexpr int kSiteRowCodes = 22;  // bit 8 + site of the status word: a wait for codes ran out

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 8x8 16-bit transpose between lanes: row r of the input is held by lanes 4r .. 4r + 3.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// Row r (of 8) of a score tile is token kTokenOrder(r) of its half page: neighbouring rows and every
// second row fall on different halves of the shared-memory banks for 64-byte rows of codes.
__device__ __forceinline__ int token_of_row(int r) { return r ^ ((r >> 1) & 1); }

// Steps of kPages pages that a warp has in shared memory or on the way, and its bytes of them
// (figures: 64 sequences of 4097 tokens, 8 kv heads of 64).
template <int D>
struct RowShape {
  static constexpr int kPages = 128 / D;
  static constexpr int kRing = 2;  // a deeper one costs resident CTAs: 53 us against 77 with four
  static constexpr int kBlockBytes = kCachePage * D;
  static constexpr int kStepBytes = 2 * kPages * kBlockBytes;  // keys, then values
  static constexpr int kSharedBytes = kWarps * kRing * kStepBytes;
};

// NT: tiles of 8 query heads of one kv head that share the loaded codes.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 4 : 2)
row_kernel(const AttentionParams p) {
  using S = RowShape<D>;
  constexpr int CP = S::kPages;
  constexpr int KW = D / 16;   // 32-bit words of keys a lane holds for each of its two tokens
  constexpr int VW = D / 32;   // words of values a lane holds for each of its four tokens
  constexpr int kStride = kPartial<D>;
  extern __shared__ __align__(128) uint8_t ring_shared[];
  __shared__ uint64_t full[kWarps][S::kRing];
  __shared__ float merged[kWarps][8 * NT][kStride];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // the heads of a page lie side by side: CTAs next to each other read them at about one time
  const int heads = p.cache.kv_heads * p.head_tiles;
  const int kv_head = blockIdx.x % heads / p.head_tiles;
  const int head_base = blockIdx.x % p.head_tiles * (8 * NT);  // within the group
  const int split = blockIdx.x / heads % p.splits;
  const int row = blockIdx.x / heads / p.splits;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;

  const int sequence =
      p.offsets == nullptr ? row : sequence_of_row(p.offsets, p.cache.batch, row);
  if (sequence < 0) return;  // a row of no sequence is left as it was
  int length = sequence_length(p.cache, sequence, p.status);
  if (p.offsets != nullptr) length += row + 1 - p.offsets[sequence + 1];
  const Visible v = visible_pages(length, p.window > 0 ? length - p.window : 0, p.first,
                                  p.cache.table_width * kCachePage);
  const int per_split = (v.pages + p.splits - 1) / p.splits;
  const int page_begin = split * per_split;
  const int page_end = min(v.pages, page_begin + per_split);
  // this warp's steps: step k holds entries page_begin + (k * kWarps + warp) * CP ..
  const int all_steps = max(0, (page_end - page_begin + CP - 1) / CP);
  const int steps = (all_steps - warp + kWarps - 1) / kWarps;

  if (lane == 0) {
    for (int i = 0; i < S::kRing; ++i) mbar_init(&full[warp][i], 1);
    mbar_fence_init();
  }
  __syncwarp();
  uint8_t* const ring = ring_shared + warp * S::kRing * S::kStepBytes;

  // Lane i holds what page i % CP of step kGroup * group + i / CP is: its block (-1: nothing
  // there), the factor of its scores and the exponent of its values; the next group's are under way.
  constexpr int kGroup = 32 / CP;
  struct Held {
    int64_t block;
    float key_scale, value_exponent;
  };
  auto entry_of = [&](int step, int i) { return page_begin + (step * kWarps + warp) * CP + i; };
  auto look_up = [&](int group) {
    Held held{-1, 1.0f, 0.0f};
    const int i = entry_of(group * kGroup + lane / CP, lane % CP);
    if (i < page_end) {
      const int page = physical_page(p.cache, sequence, i < v.front ? i : i - v.front + v.back,
                                     p.status);
      if (page >= 0) {
        held.block = static_cast<int64_t>(page) * p.cache.kv_heads + kv_head;
        held.key_scale = exp2_int(scale_exponent(p.cache.scales[0][held.block]));
        held.value_exponent =
            static_cast<float>(scale_exponent(p.cache.scales[1][held.block]));
      }
    }
    return held;
  };
  int group = 0;  // of the step worked on
  Held held = look_up(0), next_held = look_up(1);
  // Brings step k's blocks into its slot, one bulk copy each, by the lanes that hold them.
  auto fetch = [&](int k) {
    const int64_t at = k / kGroup == group ? held.block : next_held.block;
    const bool mine = lane / CP == k % kGroup && at >= 0;
    const int slot = k % S::kRing;
    const uint32_t count = __popc(__ballot_sync(0xffffffffu, mine));
    if (lane == 0) mbar_arrive_expect_tx(&full[warp][slot], count * 2 * S::kBlockBytes);
    __syncwarp();
    if (mine) {
      uint8_t* const to = ring + slot * S::kStepBytes + (lane % CP) * S::kBlockBytes;
      bulk_load(to, p.cache.codes[0] + at * S::kBlockBytes, S::kBlockBytes, &full[warp][slot]);
      bulk_load(to + CP * S::kBlockBytes, p.cache.codes[1] + at * S::kBlockBytes, S::kBlockBytes,
                &full[warp][slot]);
    }
    __syncwarp();
  };
  for (int k = 0; k < min(steps, S::kRing); ++k) fetch(k);

  // Queries as B fragments: head g of every tile, the dimensions that this lane's key words hold
  // (word w of a token: dimensions 64 (w / 4) + 16 c + 4 (w % 4) .. + 3).
  uint32_t q[NT][KW][2];
  float factor[NT][2];  // scale * log2(e) / (the row's power of two) of heads 2c and 2c + 1
  uint32_t poisoned = 0;  // bit 2n + j: head 2c + j's query holds an infinity or a NaN
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int head = head_base + 8 * n + g;
    const bool live = head < p.group;
    const T* source = static_cast<const T*>(p.query) + static_cast<int64_t>(row) * p.query_token_stride +
                      (kv_head * p.group + head) * p.query_head_stride + 16 * c;
    uint32_t words[KW][2];
#pragma unroll
    for (int w = 0; w < KW; w += 4) {
      uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
      if (live) {
        lo = *reinterpret_cast<const uint4*>(source + 64 * (w / 4));
        hi = *reinterpret_cast<const uint4*>(source + 64 * (w / 4) + 8);
      }
      words[w][0] = lo.x; words[w][1] = lo.y; words[w + 1][0] = lo.z; words[w + 1][1] = lo.w;
      words[w + 2][0] = hi.x; words[w + 2][1] = hi.y; words[w + 3][0] = hi.z;
      words[w + 3][1] = hi.w;
    }
    uint32_t largest = 0;  // magnitude bits in the upper half
#pragma unroll
    for (int w = 0; w < KW; ++w) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        largest = max(largest, max((words[w][i] & 0x7fffu) << 16, words[w][i] & 0x7fff0000u));
      }
    }
    largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
    largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
    constexpr bool kHalf = std::is_same<T, __half>::value;
    const int shift = kHalf ? 0 : query_shift(largest);
    const float up = exp2_int(shift);
    // a query with an infinity or a NaN gives NaN where it sees a token; its scores are not formed
    const bool bad = largest >= (kHalf ? 0x7c000000u : 0x7f800000u);
    const float inverse = exp2_int(-shift);
#pragma unroll
    for (int w = 0; w < KW; ++w) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (bad) words[w][i] = 0;
        q[n][w][i] = kHalf ? words[w][i]
                           : Elem<__half>::pack2(Elem<T>::from_bits(words[w][i] & 0xffffu) * up,
                                                 Elem<T>::from_bits(words[w][i] >> 16) * up);
      }
    }
    factor[n][0] = p.scale_log2 * __shfl_sync(0xffffffffu, inverse, 8 * c);
    factor[n][1] = p.scale_log2 * __shfl_sync(0xffffffffu, inverse, 8 * c + 4);
    const uint32_t bad_lanes = __ballot_sync(0xffffffffu, bad);
    poisoned |= (bad_lanes >> (8 * c) & 1u) << (2 * n) | (bad_lanes >> (8 * c + 4) & 1u) << (2 * n + 1);
  }

  float running_max[NT][2], running_sum[NT][2];
  float out[NT][2 * VW][4];  // tile i: dimensions D/8 g + 2i (registers 0, 1) and + 1 (2, 3)
  float out_exponent = kLowestExponent;  // out is in units of two to this
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    running_max[n][0] = running_max[n][1] = -INFINITY;
    running_sum[n][0] = running_sum[n][1] = 0.0f;
#pragma unroll
    for (int i = 0; i < 2 * VW; ++i) out[n][i][0] = out[n][i][1] = out[n][i][2] = out[n][i][3] = 0;
  }

  // entries whose tokens are all seen
  const int whole_begin =
      v.start == 0 ? 0 : v.front + (v.start + kCachePage - 1) / kCachePage - v.back;
  const int whole_end = min(page_end, v.front + v.length / kCachePage - v.back);
  uint32_t there = __ballot_sync(0xffffffffu, held.block >= 0);
  const int row_token = token_of_row(g);

  for (int k = 0; k < steps; ++k) {
    const int slot = k % S::kRing;
    const int entry = entry_of(k, 0);
    const int at = k % kGroup * CP;  // lane of the step's first page
    const uint32_t present = there >> at;
    const bool whole = entry >= whole_begin && entry + CP <= whole_end &&
                       (present & ((1u << CP) - 1u)) == (1u << CP) - 1u;
    float score_factor[NT][CP][2];
    float relative[CP];  // exponent of the page's values, relative to out's
    bool narrow = true;
#pragma unroll
    for (int i = 0; i < CP; ++i) {
      const float key_scale = __shfl_sync(0xffffffffu, held.key_scale, at + i);
      const float value_exponent = __shfl_sync(0xffffffffu, held.value_exponent, at + i);
      relative[i] = (present >> i & 1u) != 0 ? value_exponent - out_exponent : 0.0f;
      narrow = narrow && relative[i] >= kBelowExponent && relative[i] <= kAboveExponent;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        score_factor[n][i][0] = factor[n][0] * key_scale;
        score_factor[n][i][1] = factor[n][1] * key_scale;
      }
    }
    float page_power[CP];  // what a page's products are still to be multiplied by
    bool wide = false;     // not one for all of them
    if (__any_sync(0xffffffffu, !narrow)) {
      float raise = 0.0f;
#pragma unroll
      for (int i = 0; i < CP; ++i) {
        if (relative[i] > kAboveExponent) raise = fmaxf(raise, relative[i]);
      }
      out_exponent += raise;
      const float down = exp2_int(-static_cast<int>(raise));
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < 2 * VW; ++i) {
#pragma unroll
          for (int j = 0; j < 4; ++j) out[n][i][j] *= down;
        }
      }
#pragma unroll
      for (int i = 0; i < CP; ++i) {
        if ((present >> i & 1u) != 0) relative[i] -= raise;
        wide = wide || relative[i] < kBelowExponent;
      }
      wide = __any_sync(0xffffffffu, wide);
#pragma unroll
      for (int i = 0; i < CP; ++i) {
        page_power[i] = exp2_int(static_cast<int>(relative[i]));
        if (wide) relative[i] = 0.0f;
      }
    }
    if (!mbar_wait(&full[warp][slot], k / S::kRing & 1)) {
      if (lane == 0) {
        atomicOr(p.status, NML_SM100_STATUS_BARRIER_TIMEOUT | (0x100 << kSiteRowCodes));
      }
    }
    __syncwarp();
    const uint8_t* const codes = ring + slot * S::kStepBytes;

    float s[NT][CP][4];  // tokens of rows g (0, 1) and g + 8 (2, 3), heads 2c and 2c + 1
#pragma unroll
    for (int i = 0; i < CP; ++i) {
      uint32_t keys[2][KW];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int w = 0; w < KW; w += 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(
              codes + i * S::kBlockBytes + (row_token + 8 * h) * D + 64 * (w / 4) + 16 * c);
          keys[h][w] = x.x; keys[h][w + 1] = x.y;
          keys[h][w + 2] = x.z; keys[h][w + 3] = x.w;
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][i][0] = s[n][i][1] = s[n][i][2] = s[n][i][3] = 0.0f;
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const uint32_t a0 = e4m3x2_to_f16x2(keys[0][w] & 0xffffu);
        const uint32_t a2 = e4m3x2_to_f16x2(keys[0][w] >> 16);
        const uint32_t a1 = e4m3x2_to_f16x2(keys[1][w] & 0xffffu);
        const uint32_t a3 = e4m3x2_to_f16x2(keys[1][w] >> 16);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_f16(s[n][i], a0, a1, a2, a3, q[n][w][0], q[n][w][1]);
      }
    }
    // tokens of page i that the row does not see
    auto seen = [&](int i, int within) {
      const int e = entry + i;
      const int t = (e < v.front ? e : e - v.front + v.back) * kCachePage + within;
      return (present >> i & 1u) != 0 && t < v.length && (t >= v.start || t < p.first);
    };
    if (!whole) {
#pragma unroll
      for (int i = 0; i < CP; ++i) {
        const bool seen_g = seen(i, row_token), seen_h = seen(i, row_token + 8);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (!seen_g) s[n][i][0] = s[n][i][1] = -INFINITY;
          if (!seen_h) s[n][i][2] = s[n][i][3] = -INFINITY;
          score_factor[n][i][0] = masked_factor(score_factor[n][i][0]);
          score_factor[n][i][1] = masked_factor(score_factor[n][i][1]);
        }
      }
    }

    // Weights against the maximum so far; only when their sum says that it does not serve (or when
    // there is none) is the step's maximum formed and the step weighted again.
    uint32_t weights[NT][CP][2];
    float step_sum[NT][2];
    bool missing = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      missing = missing || running_max[n][0] == -INFINITY || running_max[n][1] == -INFINITY;
    }
    bool with_maximum = __any_sync(0xffffffffu, missing);
    while (true) {
      if (with_maximum) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float m = running_max[n][j];
#pragma unroll
            for (int i = 0; i < CP; ++i) {
              m = fmaxf(m, fmaf(fmaxf(s[n][i][j], s[n][i][j + 2]), score_factor[n][i][j],
                                relative[i]));
            }
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
            // nothing seen yet: leave the (empty) state as it is
            const float rescale = m == -INFINITY ? 1.0f : exp2_fast(running_max[n][j] - m);
            running_max[n][j] = m;
            running_sum[n][j] *= rescale;
#pragma unroll
            for (int i = 0; i < 2 * VW; ++i) {
              out[n][i][j] *= rescale;
              out[n][i][j + 2] *= rescale;
            }
          }
        }
      }
      float largest = 0.0f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float base[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          base[j] = running_max[n][j] == -INFINITY ? 0.0f : running_max[n][j];
          step_sum[n][j] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < CP; ++i) {
          const float unscale = exp2_fast(-relative[i]);
          float w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            w[j] = exp2_fast(fmaf(s[n][i][j], score_factor[n][i][j & 1],
                                  relative[i] - base[j & 1]));
          }
          largest = fmaxf(largest, fmaxf(w[0] + w[2], w[1] + w[3]));
          step_sum[n][0] = fmaf(w[0] + w[2], unscale, step_sum[n][0]);
          step_sum[n][1] = fmaf(w[1] + w[3], unscale, step_sum[n][1]);
          weights[n][i][0] = Elem<__half>::pack2(w[0], w[1]);
          weights[n][i][1] = Elem<__half>::pack2(w[2], w[3]);
        }
      }
      if (with_maximum || !__any_sync(0xffffffffu, largest > kLargestSum)) break;
      with_maximum = true;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      running_sum[n][0] += step_sum[n][0];
      running_sum[n][1] += step_sum[n][1];
    }
#pragma unroll
    for (int i = 0; i < CP; ++i) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        weights[n][i][0] = transpose8x8(weights[n][i][0]);
        weights[n][i][1] = transpose8x8(weights[n][i][1]);
      }
      uint32_t values[4][VW];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int token = token_of_row(2 * c + (t & 1)) + 8 * (t >> 1);
        const uint8_t* const source = codes + (CP + i) * S::kBlockBytes + token * D + (D / 8) * g;
        if constexpr (VW == 2) {
          const uint2 x = *reinterpret_cast<const uint2*>(source);
          values[t][0] = x.x; values[t][1] = x.y;
        } else {
          const uint4 x = *reinterpret_cast<const uint4*>(source);
          values[t][0] = x.x; values[t][1] = x.y;
          values[t][2] = x.z; values[t][3] = x.w;
        }
      }
      if (!whole) {
        // whatever an unseen slot holds must not meet the product: 0 * NaN
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          if (!seen(i, token_of_row(2 * c + (t & 1)) + 8 * (t >> 1))) {
#pragma unroll
            for (int w = 0; w < VW; ++w) values[t][w] = 0;
          }
        }
      }
      // two forms of the page's products, so that the common one has no branch in it
      auto add_products = [&](auto scaled) {
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          const uint32_t lo01 = __byte_perm(values[0][w], values[1][w], 0x5140);
          const uint32_t lo23 = __byte_perm(values[0][w], values[1][w], 0x7362);
          const uint32_t hi01 = __byte_perm(values[2][w], values[3][w], 0x5140);
          const uint32_t hi23 = __byte_perm(values[2][w], values[3][w], 0x7362);
          const uint32_t a[2][4] = {
              {e4m3x2_to_f16x2(lo01 & 0xffffu), e4m3x2_to_f16x2(lo01 >> 16),
               e4m3x2_to_f16x2(hi01 & 0xffffu), e4m3x2_to_f16x2(hi01 >> 16)},
              {e4m3x2_to_f16x2(lo23 & 0xffffu), e4m3x2_to_f16x2(lo23 >> 16),
               e4m3x2_to_f16x2(hi23 & 0xffffu), e4m3x2_to_f16x2(hi23 >> 16)}};
#pragma unroll
          for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float(&sum)[4] = out[n][2 * w + h];
              if constexpr (!decltype(scaled)::value) {
                mma_f16(sum, a[h][0], a[h][1], a[h][2], a[h][3], weights[n][i][0],
                        weights[n][i][1]);
              } else {
                float product[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                mma_f16(product, a[h][0], a[h][1], a[h][2], a[h][3], weights[n][i][0],
                        weights[n][i][1]);
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[j] = fmaf(product[j], page_power[i], sum[j]);
              }
            }
          }
        }
      };
      if (!wide) {
        add_products(std::false_type{});
      } else {
        add_products(std::true_type{});
      }
    }
    __syncwarp();  // every lane has its codes: the slot is free
    if (k + S::kRing < steps) fetch(k + S::kRing);
    if ((k + 1) % kGroup == 0) {
      ++group;
      held = next_held;
      there = __ballot_sync(0xffffffffu, held.block >= 0);
      next_held = look_up(group + 1);
    }
  }

  // ---- merge the warps ----
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float sum = running_sum[n][j];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      if ((poisoned >> (2 * n + j) & 1u) != 0 && running_max[n][j] != -INFINITY) {
        sum = __uint_as_float(0x7fc00000u);
      }
      float* state = merged[warp][8 * n + 2 * c + j];
#pragma unroll
      for (int i = 0; i < 2 * VW; ++i) {
        state[(D / 8) * g + 2 * i] = out[n][i][j];
        state[(D / 8) * g + 2 * i + 1] = out[n][i][j + 2];
      }
      if (g == 0) {
        state[D] = running_max[n][j];
        state[D + 1] = sum;
        state[D + 2] = out_exponent;
      }
    }
  }
  __syncthreads();
  for (int item = threadIdx.x; item < 8 * NT * (D / 4); item += kWarps * 32) {
    const int h = item / (D / 4), d0 = 4 * (item % (D / 4));
    const int head = head_base + h;
    if (head >= p.group) continue;
    float total_max = -INFINITY, exponent = kLowestExponent;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      total_max = fmaxf(total_max, merged[w][h][D]);
      exponent = fmaxf(exponent, merged[w][h][D + 2]);
    }
    float total_sum = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float m = merged[w][h][D];
      const float weight = m == -INFINITY ? 0.0f : exp2f(m - total_max);
      total_sum += merged[w][h][D + 1] * weight;
      const float power = weight * exp2_int(static_cast<int>(merged[w][h][D + 2] - exponent));
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = fmaf(merged[w][h][d0 + i], power, acc[i]);
    }
    const int64_t query_head = static_cast<int64_t>(row) * p.query_heads + kv_head * p.group + head;
    if (p.splits > 1) {
      float* destination = p.partial + (query_head * p.splits + split) * kStride;
      *reinterpret_cast<float4*>(destination + d0) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      if (d0 == 0) {
        *reinterpret_cast<float4*>(destination + D) =
            make_float4(total_max, total_sum, exponent, 0.0f);
      }
    } else {
      float denominator = total_sum;
      if (p.sinks != nullptr) {
        denominator += exp2f(p.sinks[kv_head * p.group + head] * kLog2e - total_max);
      }
      // only a row that sees nothing has a sum of exactly zero; its output is zero
      const float inverse =
          total_sum == 0.0f ? 0.0f : exp2_int(static_cast<int>(exponent)) / denominator;
      T* out_row = static_cast<T*>(p.output) + query_head * D + d0;
      *reinterpret_cast<uint2*>(out_row) =
          make_uint2(Elem<T>::pack2(acc[0] * inverse, acc[1] * inverse),
                     Elem<T>::pack2(acc[2] * inverse, acc[3] * inverse));
    }
  }
}

// Joins the splits of a row's query head, applies the sink, narrows: kJoinWarps warps for one, which
// take its splits in turn (one where rows are many and splits few, four where it is the other way).
template <typename T, int D, int kJoinWarps>
__global__ void __launch_bounds__(128)
join_kernel(const AttentionParams p) {
  constexpr int kStride = kPartial<D>;
  constexpr int kHeads = 4 / kJoinWarps;  // of a CTA
  __shared__ float shared_sum[4], shared_out[4][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t query_head = static_cast<int64_t>(blockIdx.x) * kHeads + warp / kJoinWarps;
  const int row = static_cast<int>(query_head / p.query_heads);
  // (a CTA of one head leaves as a whole)
  const bool nobodys = row >= p.tokens || (p.offsets != nullptr &&
                                           sequence_of_row(p.offsets, p.cache.batch, row) < 0);
  // Launched while the splits still run: everything above overlaps with them.  Every CTA waits, so
  // that this launch never ends before the one that it belongs to.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (nobodys) return;
  const float* base = p.partial + query_head * p.splits * kStride;
  float total_max = -INFINITY, exponent = kLowestExponent;
  for (int s = lane; s < p.splits; s += 32) {
    total_max = fmaxf(total_max, base[s * kStride + D]);
    exponent = fmaxf(exponent, base[s * kStride + D + 2]);
  }
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) {
    total_max = fmaxf(total_max, __shfl_xor_sync(0xffffffffu, total_max, offset));
    exponent = fmaxf(exponent, __shfl_xor_sync(0xffffffffu, exponent, offset));
  }
  float total_sum = 0.0f, acc[D / 32] = {};
#pragma unroll 4
  for (int s = warp % kJoinWarps; s < p.splits; s += kJoinWarps) {
    const float* part = base + s * kStride;
    const float4 state = *reinterpret_cast<const float4*>(part + D);
    const float weight = state.x == -INFINITY ? 0.0f : exp2f(state.x - total_max);
    total_sum += state.y * weight;
    const float power = weight * exp2_int(static_cast<int>(state.z - exponent));
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const float2 x = *reinterpret_cast<const float2*>(part + 64 * i + 2 * lane);
      acc[2 * i] = fmaf(x.x, power, acc[2 * i]);
      acc[2 * i + 1] = fmaf(x.y, power, acc[2 * i + 1]);
    }
  }
  if constexpr (kJoinWarps > 1) {
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      *reinterpret_cast<float2*>(&shared_out[warp][64 * i + 2 * lane]) =
          make_float2(acc[2 * i], acc[2 * i + 1]);
    }
    if (lane == 0) shared_sum[warp] = total_sum;
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int w = 1; w < kJoinWarps; ++w) {
      total_sum += shared_sum[w];
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        acc[2 * i] += shared_out[w][64 * i + 2 * lane];
        acc[2 * i + 1] += shared_out[w][64 * i + 2 * lane + 1];
      }
    }
  }
  float denominator = total_sum;
  if (p.sinks != nullptr) {
    denominator += exp2f(p.sinks[query_head % p.query_heads] * kLog2e - total_max);
  }
  const float inverse =
      total_sum == 0.0f ? 0.0f : exp2_int(static_cast<int>(exponent)) / denominator;
  T* out = static_cast<T*>(p.output) + query_head * D + 2 * lane;
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    *reinterpret_cast<uint32_t*>(out + 64 * i) =
        Elem<T>::pack2(acc[2 * i] * inverse, acc[2 * i + 1] * inverse);
  }
}

template <typename T, int D>
int32_t launch_attention(const AttentionParams& p, bool tiles, cudaStream_t stream, char* message,
                         size_t capacity) {
  const unsigned grid = static_cast<unsigned>(static_cast<int64_t>(p.tokens) * p.splits *
                                              p.cache.kv_heads * p.head_tiles);
  if (tiles) {
    const int32_t code = launch_tiles<T, D>(p, stream, message, capacity);
    if (code != NML_SM100_OK) return code;
  } else {
    auto kernel = p.group <= 8 ? row_kernel<T, D, 1> : row_kernel<T, D, 2>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             RowShape<D>::kSharedBytes) != cudaSuccess ||
        cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                             cudaSharedmemCarveoutMaxShared) != cudaSuccess) {
      return fail(NML_SM100_LAUNCH_FAILURE, "cannot configure shared memory", message, capacity);
    }
    kernel<<<grid, kWarps * 32, RowShape<D>::kSharedBytes, stream>>>(p);
  }
  if (p.splits > 1) {
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config = {};
    const int64_t query_heads = static_cast<int64_t>(p.tokens) * p.query_heads;
    const bool many = query_heads > 4096;
    config.gridDim = dim3(static_cast<unsigned>(many ? (query_heads + 3) / 4 : query_heads));
    config.blockDim = dim3(128);
    config.stream = stream;
    config.attrs = &early;
    config.numAttrs = 1;
    const cudaError_t status =
        cudaLaunchKernelEx(&config, many ? join_kernel<T, D, 1> : join_kernel<T, D, 4>, p);
    if (status != cudaSuccess) {
      return fail(NML_SM100_LAUNCH_FAILURE, cudaGetErrorString(status), message, capacity);
    }
  }
  return launch_result(message, capacity);
}

// Pages that a row can see at most.
int64_t most_pages(const NmlSm100PagedAttentionQ8& r) {
  if (r.sliding_window == 0) return r.cache.table_width;
  // (a tile's rows see windows that start up to 127 tokens apart)
  const int64_t pages = (r.sliding_window + kCachePage - 1) / kCachePage + 1 +
                        (r.first_tokens + kCachePage - 1) / kCachePage;
  return pages < r.cache.table_width ? pages : r.cache.table_width;
}

// Runs of tokens go to the tile kernel, single tokens, and runs of fewer than three on average, to
// the row kernel.  Measured (8 kv heads of 64, groups of 8): 16 sequences of two rows and 2000 tokens
// 19 us by rows, 22 by tiles; of four rows 26 and 25; 64 of four rows 86 and 61.
bool use_tiles(const NmlSm100PagedAttentionQ8& r) {
  return r.query_offsets != nullptr && r.tokens >= 3 * r.cache.batch;
}

// Splits of the visible pages: the number with the least estimate of the launch's time, in units of
// one page of head_dim 64 for a resident CTA of the row kernel (0.19 us): waves of CTAs, each as
// long as its pages and a fixed part, and what partial results cost to write and join.  At least
// eight pages each.  Measured on B200 (8 kv heads).  Rows: 64 sequences of 4097 tokens, 53 us
// unsplit, 59 in two; 128 of 1025, 33 unsplit, 40 in two; 16 of 4097, 19 in four, 34 unsplit; one of
// 131001, 33 in 64, 953 unsplit; 3 of 60000 to 97000 with head_dim 128, 92 in 24, 133 in 12.  Tiles
// (an SM's two CTAs take as long as one after the other): one sequence of 64 rows and 4000 tokens,
// 23 in four, 47 unsplit; 16 of 16 rows and 2000 tokens, 28 unsplit, 32 in two.
int64_t choose_splits(const NmlSm100PagedAttentionQ8& r) {
  if (r.splits > 0) return r.splits;
  const int64_t group = r.query_heads / r.cache.kv_heads;
  const bool tiles = use_tiles(r);
  const int64_t units = r.cache.kv_heads *
                        (tiles ? query_tiles(r.tokens, r.cache.batch, group)
                               : r.tokens * (group <= 8 ? 1 : (group + 15) / 16));
  // (of tiles with few rows, whose exponentials do not fill an SM, two run side by side)
  const bool few = r.tokens * group <= 64 * r.cache.batch;
  const int64_t slots = 148 * (tiles ? (few ? 2 : 1) : group <= 8 ? 4 : 2);
  const double fixed = tiles ? 25.0 : 19.0, page = tiles ? 0.85 : 1.0;
  const double join = tiles ? 20.0 : 13.0, join_split = tiles ? 0.5 : 0.3;
  const int64_t pages = most_pages(r);
  int64_t best = 1;
  double least = 0.0;
  for (int64_t s = 1; s <= 64 && (s == 1 || pages / s >= 8); ++s) {
    const double waves = static_cast<double>((units * s + slots - 1) / slots);
    const double length = page * static_cast<double>(pages * r.cache.head_dim) / (64.0 * s);
    const double cost = waves * (length + fixed) + (s > 1 ? join + join_split * s : 0.0);
    if (s == 1 || cost < least) {
      least = cost;
      best = s;
    }
  }
  return best;
}

bool valid_request(const NmlSm100PagedAttentionQ8& r) {
  return fits_i32(r.tokens) && fits_i32(r.cache.kv_heads) && r.query_heads > 0 &&
         r.query_heads % r.cache.kv_heads == 0 && r.query_heads / r.cache.kv_heads <= 128 &&
         (r.cache.head_dim == 64 || r.cache.head_dim == 128) && fits_i32(r.cache.batch) &&
         fits_i32(r.cache.table_width) && r.splits >= 0 && r.splits <= 64 &&
         r.sliding_window >= 0 && r.first_tokens >= 0 &&
         r.sliding_window <= std::numeric_limits<int32_t>::max() &&
         r.first_tokens <= std::numeric_limits<int32_t>::max() - kCachePage;
}

}  // namespace
}  // namespace nml_sm100

using namespace nml_sm100;

extern "C" size_t nml_sm100_paged_attention_q8_workspace_bytes(
    const NmlSm100PagedAttentionQ8* request) {
  if (request == nullptr || request->struct_size < sizeof(NmlSm100PagedAttentionQ8) ||
      !valid_request(*request)) {
    return 0;
  }
  const int64_t splits = choose_splits(*request);
  if (splits <= 1) return 0;
  return static_cast<size_t>(request->tokens) * request->query_heads * splits *
         (request->cache.head_dim + 4) * sizeof(float);
}

extern "C" int32_t nml_sm100_paged_attention_q8(const NmlSm100PagedAttentionQ8* request,
                                                char* error_message,
                                                size_t error_message_capacity) {
  if (request == nullptr || request->struct_size < sizeof(NmlSm100PagedAttentionQ8)) {
    return fail(NML_SM100_INVALID_ARGUMENT, "truncated paged attention request", error_message,
                error_message_capacity);
  }
  const NmlSm100PagedAttentionQ8& r = *request;
  if (!valid_cache_q8(r.cache, true) || !valid_request(r) || r.query == nullptr ||
      r.output == nullptr || r.stream == nullptr ||
      (r.query_offsets == nullptr && r.tokens != r.cache.batch) ||
      r.query_token_stride % 8 != 0 || r.query_head_stride % 8 != 0 ||
      r.query_token_stride < 0 || r.query_head_stride < 0 ||
      r.cache.kv_heads > 1024 || !(r.scale > 0.0f) ||
      r.scale > std::numeric_limits<float>::max() ||
      reinterpret_cast<uintptr_t>(r.query) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(r.output) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(r.workspace) % 16 != 0) {
    return fail(NML_SM100_INVALID_ARGUMENT,
                "invalid 8-bit paged attention request (head_dim 64 or 128, page size 16, at most "
                "128 query heads per kv head)",
                error_message, error_message_capacity);
  }
  if (r.dtype != NML_SM100_F16 && r.dtype != NML_SM100_BF16) {
    return fail(NML_SM100_INVALID_ARGUMENT, "paged attention supports F16 and BF16 only",
                error_message, error_message_capacity);
  }
  const int64_t splits = choose_splits(r);
  if ((r.tokens + r.cache.batch) * splits * r.query_heads > std::numeric_limits<int32_t>::max()) {
    return fail(NML_SM100_INVALID_ARGUMENT, "invalid 8-bit paged attention request: too many rows",
                error_message, error_message_capacity);
  }
  const size_t needed = nml_sm100_paged_attention_q8_workspace_bytes(request);
  if (needed > 0 && (r.workspace == nullptr || r.workspace_bytes < needed)) {
    return fail(NML_SM100_INVALID_ARGUMENT, "paged attention workspace is too small",
                error_message, error_message_capacity);
  }
  const DeviceInfo* device = current_device(error_message, error_message_capacity);
  if (device == nullptr) return NML_SM100_LAUNCH_FAILURE;
  AttentionParams p = {};
  p.cache = cache_params(r.cache);
  p.query = r.query;
  p.offsets = r.query_offsets;
  p.sinks = r.sinks;
  p.partial = static_cast<float*>(r.workspace);
  p.output = r.output;
  p.query_token_stride = r.query_token_stride;
  p.query_head_stride = r.query_head_stride;
  p.tokens = static_cast<int>(r.tokens);
  p.query_heads = static_cast<int>(r.query_heads);
  p.group = static_cast<int>(r.query_heads / r.cache.kv_heads);
  p.head_tiles = p.group <= 8 ? 1 : (p.group + 15) / 16;
  p.splits = static_cast<int>(splits);
  // no sequence is longer than its table
  const int64_t longest = r.cache.table_width * kCachePage;
  p.window = r.sliding_window < longest ? static_cast<int>(r.sliding_window) : 0;
  p.first = static_cast<int>(r.first_tokens < longest ? r.first_tokens : longest);
  p.scale_log2 = r.scale * kLog2e;
  p.status = device->status_word;
  cudaStream_t stream = static_cast<cudaStream_t>(r.stream);
  const bool half = r.dtype == NML_SM100_F16;
  const bool tiles = use_tiles(r);
  if (r.cache.head_dim == 64) {
    return half ? launch_attention<__half, 64>(p, tiles, stream, error_message,
                                               error_message_capacity)
                : launch_attention<__nv_bfloat16, 64>(p, tiles, stream, error_message,
                                                      error_message_capacity);
  }
  return half ? launch_attention<__half, 128>(p, tiles, stream, error_message,
                                              error_message_capacity)
              : launch_attention<__nv_bfloat16, 128>(p, tiles, stream, error_message,
                                                     error_message_capacity);
}
