// What the kernels over the paged key/value cache share.
#pragma once

#include "wq_common.h"
#include "wq_status.h"

namespace wq {

constexpr int kPagedDim = 128;            // head_dim
constexpr int kMaxSequences = 65536;      // per call
constexpr int kMaxTreeTokens = 64;        // drafted tokens of one sequence: one bit each

// Sum over the wave; every lane gets it.
__device__ __forceinline__ int64_t wave_sum_i64(int64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// The sequence of token t: the number of starts at or below t, less one (-1
// and `sequences` mean none).  Every lane of the wave counts its share of the
// starts, all of them requested at once, so the search costs one memory
// latency where a binary one costs one per step.
__device__ __forceinline__ int sequence_of(const int32_t* __restrict__ starts, int sequences, int t, int lane) {
  int n = 0;
  for (int j0 = 0; j0 <= sequences; j0 += 64) {
    const int j = j0 + lane;
    n += __popcll(__builtin_amdgcn_ballot_w64(j <= sequences && starts[min(j, sequences)] <= t));
  }
  return n - 1;
}

// What every call over a pool of pages requires of its shapes.
inline int paged_pool_check(int64_t head_dim, int64_t kv_heads, int64_t key_page_stride, int64_t value_page_stride,
                            int64_t num_pages, int64_t page_size, int64_t table_width, int64_t sequences,
                            int64_t tokens) {
  WQ_REQUIRE(head_dim == kPagedDim, WQ_ERR_UNSUPPORTED, "the paged cache is built for head_dim 128 (got %lld)",
             (long long)head_dim);
  WQ_REQUIRE(kv_heads > 0 && kv_heads <= 4096, WQ_ERR_INVALID_ARGUMENT, "kv_heads must be in [1, 4096] (got %lld)",
             (long long)kv_heads);
  WQ_REQUIRE(page_size > 0 && page_size % 16 == 0 && page_size <= 65536, WQ_ERR_INVALID_ARGUMENT,
             "page_size must be a multiple of 16 up to 65536 (got %lld)", (long long)page_size);
  WQ_REQUIRE(num_pages > 0 && num_pages <= 0x7fffffff, WQ_ERR_INVALID_ARGUMENT, "num_pages must be in [1, 2^31)");
  const int64_t page = kv_heads * page_size * kPagedDim;
  WQ_REQUIRE(key_page_stride >= page && value_page_stride >= page && key_page_stride % 8 == 0 &&
                 value_page_stride % 8 == 0 && key_page_stride <= INT64_MAX / 2 / num_pages &&
                 value_page_stride <= INT64_MAX / 2 / num_pages,
             WQ_ERR_INVALID_ARGUMENT, "page strides must be multiples of 8 and at least one page (%lld)",
             (long long)page);
  // A sequence's positions are held in 32 bits.
  WQ_REQUIRE(table_width > 0 && table_width <= 0x40000000 / page_size, WQ_ERR_INVALID_ARGUMENT,
             "table_width must be positive and table_width * page_size <= 2^30");
  WQ_REQUIRE(sequences >= 0 && sequences <= kMaxSequences, WQ_ERR_INVALID_ARGUMENT,
             "sequences must be in [0, %d] (got %lld)", kMaxSequences, (long long)sequences);
  WQ_REQUIRE(tokens >= 0 && tokens < (1 << 24), WQ_ERR_INVALID_ARGUMENT, "tokens must be in [0, 2^24) (got %lld)",
             (long long)tokens);
  return WQ_OK;
}

}  // namespace wq
