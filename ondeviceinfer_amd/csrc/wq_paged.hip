// New tokens into the paged key/value cache: per-head q/k RMSNorm, position
// rotation, k and v into their sequences' pages.
#include "ondeviceinfer_paged.h"
#include "wq_paged.h"
#include "wq_status.h"

#include <math.h>

namespace wq {
namespace {

struct AppendArgs {
  const half_t *qkv, *qn_w, *kn_w, *cos_t, *sin_t;
  const int32_t *positions, *table, *starts, *lens;
  half_t *kp, *vp, *q_out;
  int64_t k_stride, v_stride;   // elements from page to page
  float eps;
  int H, KV, table_positions, width, sequences, num_pages, page_size;
};

// grid = (tokens, parts), 256 threads.  A head's 128 elements lie in the 16
// lanes of one DPP row, eight each, so a wave loads and stores four heads with
// one 16-byte access per lane; the sum of squares is a row reduction and the
// rotation's other half, d +- 64, is the lane eight away, a row rotation.
// Wave w of part y takes the head quads 4y + w, 4 (y + parts) + w, ...  The
// projection is read once, non-temporally (34 -> 30 us for 5844 tokens of 56
// heads, 5.6 TB/s over what is read and written); q and the pages are what the
// attention reads next and stay in the caches.  Bound by memory; a single
// token by its three dependent loads (starts, page number, table row).
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = blockIdx.x;
  const int c = lane & 15, sub = lane >> 4;
  const int heads = a.H + 2 * a.KV;
  const int quads = (heads + 3) >> 2;
  const int step = 4 * gridDim.y;
  const half_t* src = a.qkv + (size_t)t * heads * kPagedDim + 8 * c;
  int quad = 4 * blockIdx.y + wave;
  // The first quad's rows are on their way while the token finds its place.
  uint4_t next = __builtin_nontemporal_load(
      reinterpret_cast<const uint4_t*>(src + (size_t)min(4 * quad + sub, heads - 1) * kPagedDim));

  const int b = sequence_of(a.starts, a.sequences, t, lane);
  if (b < 0 || b >= a.sequences) return;
  const int start = a.starts[b], end = a.starts[b + 1];
  if (start < 0 || end > (int)gridDim.x || t < start || t >= end) return;
  const int64_t index = (int64_t)a.lens[b] - (end - start) + (t - start);
  const int64_t pos = a.positions ? a.positions[t] : index;
  bool ok = index >= 0 && index < (int64_t)a.width * a.page_size && pos >= 0 && pos < a.table_positions;
  const unsigned at = ok ? (unsigned)index : 0u;   // below 2^30: the width was checked for it
  const unsigned entry = at / (unsigned)a.page_size;
  const int page = ok ? a.table[(size_t)b * a.width + entry] : -1;
  ok = ok && page >= 0 && page < a.num_pages;
  const size_t row = (size_t)(at - entry * a.page_size) * kPagedDim;
  const uint4_t cw = *reinterpret_cast<const uint4_t*>(a.cos_t + (ok ? (size_t)pos : 0) * kPagedDim + 8 * c);
  const uint4_t sw = *reinterpret_cast<const uint4_t*>(a.sin_t + (ok ? (size_t)pos : 0) * kPagedDim + 8 * c);
  const uint4_t one8 = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
  const uint4_t qw = a.qn_w ? *reinterpret_cast<const uint4_t*>(a.qn_w + 8 * c) : one8;
  const uint4_t kw = a.kn_w ? *reinterpret_cast<const uint4_t*>(a.kn_w + 8 * c) : one8;
  const half8_t ch = __builtin_bit_cast(half8_t, cw), sh = __builtin_bit_cast(half8_t, sw);

  for (; quad < quads; quad += step) {
    const uint4_t raw = next;
    if (quad + step < quads)
      next = __builtin_nontemporal_load(
          reinterpret_cast<const uint4_t*>(src + (size_t)min(4 * (quad + step) + sub, heads - 1) * kPagedDim));
    const int h = 4 * quad + sub;   // past the last head in the last quad's spare lanes: computed, not stored
    const bool is_q = h < a.H;
    const half8_t x8 = __builtin_bit_cast(half8_t, raw);
    const half8_t w8 = __builtin_bit_cast(half8_t, is_q ? qw : kw);
    float u[8];
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      u[e] = (float)x8[e];
      ss += u[e] * u[e];
    }
    ss = row_sum16(ss);
    const float r = (is_q ? a.qn_w : a.kn_w) ? rsqrtf(ss * (1.0f / kPagedDim) + a.eps) : 1.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] *= r * (float)w8[e];
    half8_t y;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float other = dpp_f<0x128>(u[e]);   // row_ror:8
      y[e] = (half_t)(u[e] * (float)ch[e] + (c < 8 ? -other : other) * (float)sh[e]);
    }
    if (is_q) {
      const uint4_t nan8 = {0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u};
      *reinterpret_cast<uint4_t*>(a.q_out + ((size_t)t * a.H + h) * kPagedDim + 8 * c) =
          ok ? __builtin_bit_cast(uint4_t, y) : nan8;
    } else if (ok && h < a.H + a.KV) {
      half_t* dst = a.kp + (size_t)page * a.k_stride + (size_t)(h - a.H) * a.page_size * kPagedDim + row + 8 * c;
      *reinterpret_cast<uint4_t*>(dst) = __builtin_bit_cast(uint4_t, y);
    } else if (ok && h < heads) {
      half_t* dst =
          a.vp + (size_t)page * a.v_stride + (size_t)(h - a.H - a.KV) * a.page_size * kPagedDim + row + 8 * c;
      *reinterpret_cast<uint4_t*>(dst) = raw;
    }
  }
}

}  // namespace
}  // namespace wq

using namespace wq;

extern "C" int wq_paged_append(const uint16_t* qkv, int64_t tokens, int64_t q_heads, int64_t kv_heads,
                               int64_t head_dim, const uint16_t* q_norm_weight, const uint16_t* k_norm_weight,
                               float eps, const uint16_t* cos_table, const uint16_t* sin_table,
                               int64_t table_positions, const int32_t* positions, const int32_t* page_table,
                               int64_t table_width, const int32_t* query_starts, const int32_t* seq_lens,
                               int64_t sequences, uint16_t* key_pages, int64_t key_page_stride,
                               uint16_t* value_pages, int64_t value_page_stride, int64_t num_pages,
                               int64_t page_size, uint16_t* q_out, void* stream) {
  const int rc = paged_pool_check(head_dim, kv_heads, key_page_stride, value_page_stride, num_pages, page_size,
                                  table_width, sequences, tokens);
  if (rc != WQ_OK) return rc;
  WQ_REQUIRE(q_heads > 0 && q_heads + 2 * kv_heads <= 65535, WQ_ERR_INVALID_ARGUMENT, "bad head counts");
  WQ_REQUIRE(table_positions > 0 && table_positions <= 0x7fffffff, WQ_ERR_INVALID_ARGUMENT,
             "the cos / sin tables need at least one row");
  if (tokens == 0 || sequences == 0) return WQ_OK;
  WQ_REQUIRE(qkv && cos_table && sin_table && page_table && query_starts && seq_lens && key_pages && value_pages && q_out,
             WQ_ERR_INVALID_ARGUMENT, "null pointer argument");
  WQ_REQUIRE(((uintptr_t)qkv | (uintptr_t)cos_table | (uintptr_t)sin_table | (uintptr_t)key_pages |
              (uintptr_t)value_pages | (uintptr_t)q_out | (uintptr_t)q_norm_weight | (uintptr_t)k_norm_weight) % 16 == 0,
             WQ_ERR_INVALID_ARGUMENT, "qkv, weights, tables, pages and q_out must be 16-byte aligned");
  WQ_REQUIRE(((uintptr_t)positions | (uintptr_t)page_table | (uintptr_t)query_starts | (uintptr_t)seq_lens) % 4 == 0,
             WQ_ERR_INVALID_ARGUMENT, "integer operands must be 4-byte aligned");
  // A workgroup writes its token's queries while others still read the projection.
  const uintptr_t in0 = (uintptr_t)qkv, in1 = in0 + (size_t)tokens * (q_heads + 2 * kv_heads) * kPagedDim * 2;
  const uintptr_t out0 = (uintptr_t)q_out, out1 = out0 + (size_t)tokens * q_heads * kPagedDim * 2;
  WQ_REQUIRE(out1 <= in0 || in1 <= out0, WQ_ERR_INVALID_ARGUMENT, "q_out must not overlap qkv");
  AppendArgs a{};
  a.qkv = reinterpret_cast<const half_t*>(qkv);
  a.qn_w = reinterpret_cast<const half_t*>(q_norm_weight);
  a.kn_w = reinterpret_cast<const half_t*>(k_norm_weight);
  a.cos_t = reinterpret_cast<const half_t*>(cos_table);
  a.sin_t = reinterpret_cast<const half_t*>(sin_table);
  a.positions = positions;
  a.table = page_table;
  a.starts = query_starts;
  a.lens = seq_lens;
  a.kp = reinterpret_cast<half_t*>(key_pages);
  a.vp = reinterpret_cast<half_t*>(value_pages);
  a.q_out = reinterpret_cast<half_t*>(q_out);
  a.k_stride = key_page_stride;
  a.v_stride = value_page_stride;
  a.eps = eps;
  a.H = (int)q_heads;
  a.KV = (int)kv_heads;
  a.table_positions = (int)table_positions;
  a.width = (int)table_width;
  a.sequences = (int)sequences;
  a.num_pages = (int)num_pages;
  a.page_size = (int)page_size;
  const int quads = (int)((q_heads + 2 * kv_heads + 3) / 4);
  // Few tokens: as many workgroups as there are quads of heads for their waves (one token 2.8 us).  Many: one
  // workgroup per token, which then looks up its sequence, page and table rows once (5844 tokens 30 us against 42).
  const int parts = tokens <= 256 ? (quads + 3) / 4 : 1;
  hipLaunchKernelGGL(paged_append_kernel, dim3((unsigned)tokens, (unsigned)parts), dim3(256), 0, as_stream(stream), a);
  return check_launch("paged_append");
}
