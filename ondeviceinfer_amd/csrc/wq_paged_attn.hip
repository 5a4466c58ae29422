// Grouped-query attention over the paged key/value cache: ragged new tokens,
// causal or a tree of drafted ones.
//
// The new tokens of a sequence times the query heads of one kv head are the
// rows that share its keys; row r of a sequence is token r / G, head r % G.
// Rows are taken in tiles of 16 (few tokens per sequence) or 128, the keys of a
// tile are cut into chunks when there are too few tiles to fill the machine,
// and every (sequence, tile, chunk, kv head) is one workgroup.
#include "ondeviceinfer_paged.h"
#include "wq_paged.h"
#include "wq_status.h"

#include <math.h>

namespace wq {
namespace {

constexpr int kKeys = 32;          // keys per step of a wave
constexpr int kWaves = 4;          // waves per workgroup
constexpr int kMaxPagedGroup = 16; // q heads per kv head

// Probabilities are rounded to fp16 for the product with the values, 2^kLift
// times as large as they are (so are their sums, and the quotient is not): the
// largest is 2^14, and what lies up to 28 octaves below it keeps its eleven
// bits, where fractions of 1 would fade from 14 octaves on and be 0 from 25.
// The sums are of the rounded ones, so that the values' weights add up to one.
constexpr float kLift = 14.f;

struct PagedArgs {
  const half_t *q, *kp, *vp;
  const int32_t *table, *starts, *lens;
  const int64_t* mask;          // nullptr: causal
  half_t* out;
  float* part_o;                // [slots][KV][R][128] unnormalized outputs of split tiles
  float2_t* part_ml;            // [slots][KV][R] (max of the raw scores, sum)
  int64_t k_stride, v_stride;   // elements from page to page
  float scale_log2;
  int sequences, tokens, H, KV, G, width, page_size, num_pages;
  int slots;                    // (tile, chunk) places the grid has per kv head
  int spare;                    // of those, beyond the largest possible number of tiles (0: nothing is split)
  int min_blocks;               // smallest chunk, in steps of kKeys keys
};

// One sequence's share of the call, from the device's starts and lengths.
struct Seq {
  int start, count, base;   // first token, tokens, positions before them (may be negative: refused by the rows)
  int keys;                 // positions that may be attended; past the table one more, which has no page
  int tiles, blocks;
};

template <int R>
__device__ __forceinline__ Seq read_seq(const PagedArgs& a, int b) {
  Seq s{};
  if (b >= a.sequences) return s;
  const int s0 = a.starts[b], s1 = a.starts[b + 1], len = a.lens[b];
  if (s0 < 0 || s1 > a.tokens || s1 <= s0) return s;
  s.start = s0;
  s.count = s1 - s0;
  s.base = (int)max((int64_t)len - s.count, -((int64_t)1 << 30));
  s.keys = min(max(len, 0), a.width * a.page_size + 1);
  s.tiles = (s.count * a.G + R - 1) / R;
  s.blocks = (s.keys + kKeys - 1) / kKeys;
  return s;
}

// Where flat place `place` of the call lies: a (tile, chunk) slot, or with
// BY_TILE a tile.  Every wave computes it for itself: two reductions and a
// scan over the sequences, 64 at a time.
//   chunk length C = max(min_blocks, ceil(sum_b tiles_b blocks_b / spare)), so
//   that sum_b tiles_b ceil(blocks_b / C) <= tiles + spare <= slots.
struct Place {
  Seq s;
  int b, tile, chunk, chunks;
  int64_t slot0;   // the sequence's first slot
  bool found;
};

// The last tiles, which see the most keys, come first.
__device__ __forceinline__ int64_t slot_of(const Place& p, int tile, int chunk) {
  return p.slot0 + chunk * p.s.tiles + (p.s.tiles - 1 - tile);
}

template <int R, bool BY_TILE>
__device__ __forceinline__ Place find_place(const PagedArgs& a, int place, int lane) {
  int chunk_blocks = 0x7fffffff;
  if (a.spare > 0) {
    int64_t work = 0;
    for (int b0 = 0; b0 < a.sequences; b0 += 64) {
      const Seq s = read_seq<R>(a, b0 + lane);
      work += (int64_t)s.tiles * s.blocks;
    }
    work = wave_sum_i64(work);
    const int64_t c = (work + a.spare - 1) / a.spare;
    chunk_blocks = (int)max(min(c, (int64_t)0x7fffffff), (int64_t)a.min_blocks);
  }
  Place p{};
  // Starts that do not follow one another could name more tiles than the grid has: 64-bit sums, and such places
  // are never found or merged.
  int64_t slots_before = 0, before = 0;
  for (int b0 = 0; b0 < a.sequences; b0 += 64) {
    const Seq s = read_seq<R>(a, b0 + lane);
    const int chunks = s.blocks > chunk_blocks ? (s.blocks + chunk_blocks - 1) / chunk_blocks : 1;
    const int slots = s.tiles * chunks;
    int upto = slots, tiles_upto = s.tiles;   // inclusive scans over the lanes
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(upto, o), v = __shfl_up(tiles_upto, o);
      if (lane >= o) {
        upto += u;
        tiles_upto += v;
      }
    }
    const int mine = BY_TILE ? s.tiles : slots;
    const int end = BY_TILE ? tiles_upto : upto;
    const int64_t want = place - before;
    const uint64_t hit = __builtin_amdgcn_ballot_w64(want >= end - mine && want < end);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      p.found = true;
      p.b = b0 + l;
      p.s.start = __builtin_amdgcn_readlane(s.start, l);
      p.s.count = __builtin_amdgcn_readlane(s.count, l);
      p.s.base = __builtin_amdgcn_readlane(s.base, l);
      p.s.keys = __builtin_amdgcn_readlane(s.keys, l);
      p.s.tiles = __builtin_amdgcn_readlane(s.tiles, l);
      p.s.blocks = __builtin_amdgcn_readlane(s.blocks, l);
      p.chunks = __builtin_amdgcn_readlane(chunks, l);
      p.slot0 = slots_before + __builtin_amdgcn_readlane(upto - slots, l);
      const int rest = (int)want - __builtin_amdgcn_readlane(end - mine, l);
      p.tile = p.s.tiles - 1 - rest % p.s.tiles;
      p.chunk = rest / p.s.tiles;
      return p;
    }
    slots_before += __builtin_amdgcn_readlane(upto, 63);
    before += __builtin_amdgcn_readlane(BY_TILE ? tiles_upto : upto, 63);
  }
  return p;
}

// The wave's 16-key groups of pages, one per lane: page number (-1: none) and
// first row of the group in its page.
struct Groups {
  int page, row;
  uint64_t bad;   // lanes whose group has no page
};

__device__ __forceinline__ Groups load_groups(const PagedArgs& a, int b, int first, int last, int lane) {
  Groups g;
  const unsigned key = 16u * (unsigned)min(first + lane, last);   // groups past the chunk's keys reread its last one
  const unsigned entry = key / (unsigned)a.page_size;
  g.row = (int)(key - entry * a.page_size);
  g.page = entry < (unsigned)a.width ? a.table[(size_t)b * a.width + entry] : -1;
  const bool ok = g.page >= 0 && g.page < a.num_pages;
  g.bad = __builtin_amdgcn_ballot_w64(!ok);
  if (!ok) {
    g.page = 0;
    g.row = 0;
  }
  return g;
}

// A hidden position's probability is 0, and 0 times a value that is infinite or
// NaN is NaN.  Where a step of keys may hide some of them, such values are
// taken as 0 and their positions' scores as NaN (before the hidden ones are
// set to -inf): a row that attends one becomes NaN, the others do not see it.
__device__ __forceinline__ bool any_not_finite(uint4_t v) {
  bool any = false;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const uint32_t u = v[w];
    any |= ((u & 0x7c00u) == 0x7c00u) | ((u & 0x7c000000u) == 0x7c000000u);
  }
  return any;
}

// What a row may attend of its sequence's positions.  Bit operations only, no
// branches: of the short-circuit form (key < keys && (tree ? ... : ...)) inside
// the unrolled score loops hipcc 7.2 loses the assignment of the hidden lanes.
struct Sight {
  int last;         // the last position attended
  int base;         // where the new tokens start
  uint64_t unseen;  // drafted ones among them that are not attended

  __device__ __forceinline__ int operator()(int key) const {
    const int j = key - base;
    return (int)(key > last) | ((int)(j >= 0) & (int)((unseen >> (j & 63)) & 1));
  }
};

__device__ __forceinline__ Sight row_sight(const PagedArgs& a, const Seq& s, int tok, int keys) {
  if (a.mask != nullptr) return Sight{keys - 1, s.base, ~(uint64_t)a.mask[s.start + tok]};
  return Sight{min(s.base + tok, keys - 1), s.base, 0};
}

// Sixteen bytes; non-temporal where every key is read by one workgroup only.
template <bool ONCE>
__device__ __forceinline__ uint4_t stream_load(const half_t* p) {
  const uint4_t* q = reinterpret_cast<const uint4_t*>(p);
  return ONCE ? __builtin_nontemporal_load(q) : *q;
}

// grid = slots * KV workgroups of four waves (flat id f: kv head f % KV, place
// f / KV; with 8 kv heads the workgroups of one head share an XCD's L2).  Wave
// w takes the w-th quarter of the chunk's 32-key steps and runs its own online
// softmax over them for the tile's 16 rows, without barriers and without LDS:
//   scores  S^T = K . Q^T on the matrix cores (16x16x32): A = 16 keys (lane
//           (i, kb) = (l % 16, l / 16) holds key i, d = 32 ks + 8 kb ..), B =
//           Q^T; lane (i, kb) receives keys 4 kb .. 4 kb + 3 of row i;
//   values  lane (i, kb) loads d = 8 i .. 8 i + 7 of the keys 4 kb + e and
//           16 + 4 kb + e: eight keys by eight d, transposed in registers (32
//           byte permutes), which makes them the A operand of O^T = V^T . P^T
//           whose m index i of tile t is d = 8 i + t and whose k slots are the
//           keys that the same lane's scores hold.  P^T needs no exchange
//           either: the lane's eight probabilities are its B operand;
//   output  lane (i, kb) holds row i, d = 8 (4 kb + v) + t in acc[t][v].
// The next step's keys are requested as soon as the scores have consumed the
// present ones, the values likewise, so that both are in flight during the
// softmax of the other.  Bound by the cache's bytes: 2.27 GB of 64 sequences in
// 374 us, 6.1 TB/s with 158 registers and three workgroups per compute unit;
// one sequence of 4101 positions (16.8 MB) by latency, 9 to 10 us and 6 for the
// merge: the starts, the page numbers, the keys, the values one after another.
template <bool ONCE>
__global__ __launch_bounds__(256, 2) void paged_attention_rows_kernel(PagedArgs a) {
  constexpr int R = 16, D = kPagedDim;
  __shared__ __attribute__((aligned(16))) float red[kWaves][R][D];
  __shared__ float2_t mlw[kWaves][R];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, kb = lane >> 4;
  const int kvh = blockIdx.x % a.KV, slot = blockIdx.x / a.KV;
  const Place p = find_place<R, false>(a, slot, lane);
  if (!p.found) return;

  // The row of this lane, its token and what it may attend.
  const int rows = p.s.count * a.G;
  const int r = p.tile * R + i;
  const int tok = min(r, rows - 1) / a.G;
  const int head = kvh * a.G + min(r, rows - 1) - tok * a.G;
  const int first_tok = (p.tile * R) / a.G;
  const int last_tok = (min(p.tile * R + R, rows) - 1) / a.G;
  const bool tree = a.mask != nullptr;
  const bool refused = tree && p.s.count > kMaxTreeTokens;
  // Keys of the tile, and the first key that not all of its rows attend.
  const int keys = refused ? 0 : tree ? p.s.keys : max(0, min(p.s.keys, p.s.base + last_tok + 1));
  const int ragged = tree ? p.s.base : p.s.base + first_tok + 1;
  const Sight hidden = row_sight(a, p.s, tok, keys);
  const int per = p.s.blocks / p.chunks, extra = p.s.blocks % p.chunks;
  const int c0 = p.chunk * per + min(p.chunk, extra), c1 = c0 + per + (p.chunk < extra ? 1 : 0);
  const int nblk = min(c1, (keys + kKeys - 1) / kKeys) - c0;   // steps of this workgroup (may be negative)
  const int w0 = nblk > 0 ? c0 + nblk * wave / kWaves : 0;
  const int w1 = nblk > 0 ? c0 + nblk * (wave + 1) / kWaves : 0;

  const half_t* qp = a.q + ((size_t)(p.s.start + tok) * a.H + head) * D + 8 * kb;
  half8_t qf[4];
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) qf[ks] = ld_h8(qp + 32 * ks);

  float4_t acc[8];
#pragma unroll
  for (int t = 0; t < 8; ++t) acc[t] = float4_t{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.f;   // of row i; l_run this lane's keys only

  if (w0 < w1) {
    const size_t head_off = (size_t)kvh * a.page_size * D;
    const half_t* kbase = a.kp + head_off + (size_t)i * D + 8 * kb;
    const half_t* vbase = a.vp + head_off + (size_t)(4 * kb) * D + 8 * i;
    const int last_group = (keys - 1) >> 4;
    int g0 = 2 * w0;
    Groups g = load_groups(a, p.b, g0, last_group, lane);
    uint4_t kr[2][4], vr[8];
    bool kbad[2];
    auto load_keys = [&](int blk) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int l = 2 * blk + h - g0;
        const half_t* src = kbase + (size_t)__builtin_amdgcn_readlane(g.page, l) * a.k_stride +
                            (size_t)__builtin_amdgcn_readlane(g.row, l) * D;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) kr[h][ks] = stream_load<ONCE>(src + 32 * ks);
        kbad[h] = (g.bad >> l) & 1;
      }
    };
    auto load_values = [&](int blk) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int l = 2 * blk + h - g0;
        const half_t* src = vbase + (size_t)__builtin_amdgcn_readlane(g.page, l) * a.v_stride +
                            (size_t)__builtin_amdgcn_readlane(g.row, l) * D;
#pragma unroll
        for (int e = 0; e < 4; ++e) vr[4 * h + e] = stream_load<ONCE>(src + (size_t)e * D);
      }
    };
    load_keys(w0);
    load_values(w0);
    for (int blk = w0; blk < w1; ++blk) {
      const int k0 = blk * kKeys;
      float4_t sc[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sc[h] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) sc[h] = mfma16(__builtin_bit_cast(half8_t, kr[h][ks]), qf[ks], sc[h]);
        if (kbad[h]) sc[h] = float4_t{NAN, NAN, NAN, NAN};
      }
      // A wave's groups run out after 32 steps; the values of this step are on their way already.
      const bool more = blk + 1 < w1;
      if (more && 2 * (blk + 1) - g0 >= 64) {
        g0 = 2 * (blk + 1);
        g = load_groups(a, p.b, g0, last_group, lane);
      }
      if (more) load_keys(blk + 1);
      if (k0 + kKeys > ragged || k0 + kKeys > keys) {
        // Lane (i, kb) looks at its eight values of the keys whose scores the lanes (.., kb) hold.
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool odd = any_not_finite(vr[e]);
          const uint64_t lanes = __builtin_amdgcn_ballot_w64(odd);
          if (lanes != 0) {
            if (odd) vr[e] = uint4_t{0u, 0u, 0u, 0u};
            if ((lanes >> (16 * kb)) & 0xffffu) sc[e >> 2][e & 3] = NAN;
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            sc[h][v] = hidden(k0 + 16 * h + 4 * kb + v) ? -INFINITY : sc[h][v];
          }
      }
      float mb = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int v = 0; v < 4; ++v) mb = fmaxf(mb, sc[h][v]);
      mb = fmaxf(mb, __shfl_xor(mb, 16));
      mb = fmaxf(mb, __shfl_xor(mb, 32));
      // Maxima are of the raw scores (scale > 0), and so are the differences: scaled first, scores of 2^24 and more
      // would be rounded by whole octaves.
      const float m_new = fmaxf(m_run, mb);
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = exp2_hw((m_run - m_use) * a.scale_log2);
      m_run = m_new;
      half8_t pb;
      float ls = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int v = 0; v < 4; ++v)
          pb[4 * h + v] = (half_t)exp2_hw(__builtin_fmaf(sc[h][v] - m_use, a.scale_log2, kLift));
#pragma unroll
      for (int e = 0; e < 8; e += 2)
        ls = __builtin_amdgcn_fdot2(half2_t{pb[e], pb[e + 1]}, half2_t{(half_t)1.f, (half_t)1.f}, ls, false);
      l_run = l_run * alpha + ls;
      if (__builtin_amdgcn_ballot_w64(alpha != 1.f) != 0) {
#pragma unroll
        for (int t = 0; t < 8; ++t)
#pragma unroll
          for (int v = 0; v < 4; ++v) acc[t][v] *= alpha;
      }
      if (k0 + kKeys > keys) {   // what lies behind the last key is not the sequence's: 0 * NaN would poison the sums
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (k0 + 16 * (e >> 2) + 4 * kb + (e & 3) >= keys) vr[e] = uint4_t{0u, 0u, 0u, 0u};
      }
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        uint4_t vt;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t lo = vr[2 * w][t >> 1], hi = vr[2 * w + 1][t >> 1];
          vt[w] = __builtin_amdgcn_perm(hi, lo, t & 1 ? 0x07060302u : 0x05040100u);
        }
        acc[t] = mfma16(__builtin_bit_cast(half8_t, vt), pb, acc[t]);
      }
      if (more) load_values(blk + 1);
    }
    l_run += __shfl_xor(l_run, 16);
    l_run += __shfl_xor(l_run, 32);
  }

  // Combine the four waves.
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    float* dst = &red[wave][i][8 * (4 * kb + v)];
    *reinterpret_cast<float4_t*>(dst) = float4_t{acc[0][v], acc[1][v], acc[2][v], acc[3][v]};
    *reinterpret_cast<float4_t*>(dst + 4) = float4_t{acc[4][v], acc[5][v], acc[6][v], acc[7][v]};
  }
  if (kb == 0) mlw[wave][i] = float2_t{m_run, l_run};
  __syncthreads();
  // Thread (row, d8): row = tid / 16, d = 8 (tid % 16) ..
  const int row = tid >> 4, d = 8 * (tid & 15);
  if (p.tile * R + row >= rows) return;
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) M = fmaxf(M, mlw[w][row].x);
  const float Mu = M == -INFINITY ? 0.f : M;
  float num[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) num[e] = 0.f;
  float den = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float wt = exp2_hw((mlw[w][row].x - Mu) * a.scale_log2);
    den += wt * mlw[w][row].y;
#pragma unroll
    for (int e = 0; e < 8; ++e) num[e] += wt * red[w][row][d + e];
  }
  if (p.chunks > 1) {
    const size_t at = ((size_t)slot * a.KV + kvh) * R + row;
    *reinterpret_cast<float4_t*>(a.part_o + at * D + d) = float4_t{num[0], num[1], num[2], num[3]};
    *reinterpret_cast<float4_t*>(a.part_o + at * D + d + 4) = float4_t{num[4], num[5], num[6], num[7]};
    if (d == 0) a.part_ml[at] = float2_t{M, den};
    return;
  }
  const int rr = p.tile * R + row, t = rr / a.G;
  half8_t o;
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = refused ? (half_t)NAN : den == 0.f ? (half_t)0.f : (half_t)(num[e] / den);
  *reinterpret_cast<half8_t*>(a.out + ((size_t)(p.s.start + t) * a.H + kvh * a.G + rr - t * a.G) * D + d) = o;
}

// Chunks of prompts and trees of many tokens: tiles of 128 rows, grid and
// places as above.  Wave w owns the rows 32 w .. 32 w + 31 of the tile; all
// four share the keys and values, 64 at a time through two stages of LDS:
//   K [key][d] in rows of 272 bytes and V^T [d][key slot] in rows of 144: the 16
//   lanes that a 16-byte read serves at once are 4 (of 64) banks apart, and every
//   fragment is one address and a constant.
// Scores are computed transposed on 32x32x16 (A = 32 keys, B = 32 rows): lane
// (l % 32, l / 32) = (ql, hh) holds in register r key 8 (r / 4) + 4 hh + r % 4
// of row ql, and the probabilities, rounded to fp16, are the B operand of O^T
// = V^T . P^T once V^T's key slots follow the same order: slot 8 h + 4 j + e
// of a 16-key step holds key 8 j + 4 h + e.  A 4096-token
// prompt takes 214 to 224 us from card to card, 0.77 to 0.80 PFLOP/s: matrix
// cores busy in 35 % of the cycles, vector instructions in 41 %, waves waiting
// in 26 % of theirs, no bank conflicts.  Neither unit is full: two waves per SIMD are not enough to overlap
// the two.  Overlapping them within a wave, the next half block's keys beside
// this half's exponentials, needs more registers than two waves leave each (242
// us with 247, 558 with spills, against 231 at the time).  Six chunks also write
// and merge 82 MB of partial results.
constexpr float kLag = 4.f;
constexpr float kTileLift = kLift - kLag + 1.f;   // of the probabilities: up to 2^(kTileLift + kLag) = 2^15
constexpr float kLarge = 4096.f;   // octaves
constexpr int kTileRows = 128;
constexpr int kTileKeys = 64;
constexpr int kKRow = kPagedDim * 2 + 16, kVRow = kTileKeys * 2 + 16;   // bytes
constexpr int kTileKBytes = kTileKeys * kKRow;
constexpr int kTileStage = kTileKBytes + kPagedDim * kVRow;   // K block, then V^T block

typedef float float16_t __attribute__((ext_vector_type(16)));

// Masks of __builtin_amdgcn_sched_group_barrier.
constexpr int kSchedMfma = 0x8, kSchedLdsRead = 0x100;

// The larger of lane l and lane l ^ 32.
__device__ __forceinline__ float max_halves(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);   // (low half twice, high half twice)
  const uint32_t lo = r[0], hi = r[1];
  return fmaxf(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
}

__global__ __launch_bounds__(256, 2) void paged_attention_tile_kernel(PagedArgs a) {
  constexpr int R = kTileRows, D = kPagedDim;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  // Per stage, for the keys 4 g + e: bit g of word e, and one such set from each wave that stored values.
  __shared__ uint32_t odd_keys[2][4][4];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ql = lane & 31, hh = lane >> 5;
  const int kvh = blockIdx.x % a.KV, slot = blockIdx.x / a.KV;
  const Place p = find_place<R, false>(a, slot, lane);
  if (!p.found) return;

  const int rows = p.s.count * a.G;
  const int r0 = p.tile * R + 32 * wave;                    // this wave's first row
  const int r = r0 + ql;
  const int tok = min(r, rows - 1) / a.G;
  const int head = kvh * a.G + min(r, rows - 1) - tok * a.G;
  const bool tree = a.mask != nullptr;
  const bool refused = tree && p.s.count > kMaxTreeTokens;
  auto keys_of = [&](int last_row) {   // positions that rows up to last_row attend
    if (refused) return 0;
    return tree ? p.s.keys : max(0, min(p.s.keys, p.s.base + min(last_row, rows - 1) / a.G + 1));
  };
  const int keys = keys_of(p.tile * R + R - 1);
  const int wave_keys = r0 < rows ? keys_of(r0 + 31) : 0;
  const int ragged = tree ? p.s.base : p.s.base + min(r0, rows - 1) / a.G + 1;   // first key that not all its rows attend
  const Sight hidden = row_sight(a, p.s, tok, keys);
  const int tile_ragged = min(keys, tree ? p.s.base : p.s.base + p.tile * R / a.G + 1);
  // Chunks are cut in steps of kKeys; here a step is two of those.
  const int blocks = (p.s.blocks + 1) >> 1;
  const int per = blocks / p.chunks, extra = blocks % p.chunks;
  const int c0 = p.chunk * per + min(p.chunk, extra);
  const int c1 = min(c0 + per + (p.chunk < extra ? 1 : 0), (keys + kTileKeys - 1) / kTileKeys);

  half8_t qf[8];
  {
    const half_t* qp = a.q + ((size_t)(p.s.start + tok) * a.H + head) * D + 8 * hh;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) qf[ks] = ld_h8(qp + 16 * ks);
  }
  float16_t acc[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[dt][e] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;

  if (c0 < c1) {
    const size_t head_off = (size_t)kvh * a.page_size * D;
    // Block loads: K rows 16 u + tid / 16, 16-byte chunk tid % 16; V keys 4 (tid
    // % 16) .., d chunk tid / 16 (the 16 lanes of a transposed write then cover
    // one whole 128-byte row).
    const half_t* kbase = a.kp + head_off + (size_t)(tid >> 4) * D + 8 * (tid & 15);
    const half_t* vbase = a.vp + head_off + (size_t)(4 * (tid & 3)) * D + 8 * (tid >> 4);
    const int vgroup = (tid & 15) >> 2;
    const int last_group = (keys - 1) >> 4;
    int g0 = 4 * c0;
    Groups g = load_groups(a, p.b, g0, last_group, lane);
    uint4_t kr[4], vr[4];
    uint32_t bad_next = 0, bad = 0;   // of the block in registers, and in the stage being read: groups without a page
    auto load_block = [&](int kb) {
      if (4 * kb - g0 >= 64) {
        g0 = 4 * kb;
        g = load_groups(a, p.b, g0, last_group, lane);
      }
      const int l = 4 * kb - g0;
      const half_t* vsrc = vbase;
      int64_t voff = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t page = __builtin_amdgcn_readlane(g.page, l + u), row = __builtin_amdgcn_readlane(g.row, l + u);
        kr[u] = *reinterpret_cast<const uint4_t*>(kbase + page * a.k_stride + row * D);
        const int64_t off = page * a.v_stride + row * D;
        voff = vgroup == u ? off : voff;
      }
      vsrc += voff;
#pragma unroll
      for (int e = 0; e < 4; ++e) vr[e] = *reinterpret_cast<const uint4_t*>(vsrc + e * D);
      bad_next = (uint32_t)(g.bad >> l) & 15;
    };
    auto store_block = [&](int st, int kb) {
      if (kb * kTileKeys + kTileKeys > keys) {   // what lies behind the last key is not the sequence's
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (kb * kTileKeys + 4 * (tid & 15) + e >= keys) vr[e] = uint4_t{0u, 0u, 0u, 0u};
      }
      if (kb * kTileKeys + kTileKeys > tile_ragged) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool odd = any_not_finite(vr[e]);
          const uint64_t lanes = __builtin_amdgcn_ballot_w64(odd);   // lane 16 c + g: key 4 g + e
          if (odd) vr[e] = uint4_t{0u, 0u, 0u, 0u};
          if (lane == 0) odd_keys[st][wave][e] = (uint32_t)(lanes | lanes >> 16 | lanes >> 32 | lanes >> 48) & 0xffffu;
        }
      }
      uint8_t* base = smem + st * kTileStage;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int row = 16 * u + (tid >> 4), c = tid & 15;
        *reinterpret_cast<uint4_t*>(base + row * kKRow + 16 * c) = kr[u];
      }
      // Keys 4 g .. 4 g + 3 (g = tid % 16) land in the slots pos .. pos + 3.
      const int gq = tid & 15, kk = (4 * gq) & 15;
      const int pos = 16 * (gq >> 2) + 8 * ((kk & 7) >> 2) + 4 * (kk >> 3);
      const int d0 = 8 * (tid >> 4);
#pragma unroll
      for (int dd = 0; dd < 8; ++dd) {
        const uint32_t sel = dd & 1 ? 0x07060302u : 0x05040100u;
        uint2_t w;
        w.x = __builtin_amdgcn_perm(vr[1][dd >> 1], vr[0][dd >> 1], sel);
        w.y = __builtin_amdgcn_perm(vr[3][dd >> 1], vr[2][dd >> 1], sel);
        *reinterpret_cast<uint2_t*>(base + kTileKBytes + (d0 + dd) * kVRow + 2 * pos) = w;
      }
    };
    auto step = [&](const uint8_t* base, int st, int k0, bool masked) {
      float16_t sc[2];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[kt][e] = 0.f;
        const int row = 32 * kt + ql;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          const half8_t ka = *reinterpret_cast<const half8_t*>(base + row * kKRow + 16 * hh + 32 * ks);
          sc[kt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, qf[ks], sc[kt], 0, 0, 0);
        }
      }
      // Six fragments ahead of the matrix cores.
      __builtin_amdgcn_sched_group_barrier(kSchedLdsRead, 6, 0);
#pragma unroll
      for (int u = 0; u < 10; ++u) {
        __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
        __builtin_amdgcn_sched_group_barrier(kSchedLdsRead, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(kSchedMfma, 6, 0);
      if (bad) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if ((bad >> (2 * kt + (e >> 3))) & 1) sc[kt][e] = NAN;
      }
      if (k0 + kTileKeys > tile_ragged) {
        uint32_t odd[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          odd[e] = __builtin_amdgcn_readfirstlane(odd_keys[st][0][e] | odd_keys[st][1][e] | odd_keys[st][2][e] |
                                                  odd_keys[st][3][e]);
        if (odd[0] | odd[1] | odd[2] | odd[3]) {
#pragma unroll
          for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              sc[kt][e] = (odd[e & 3] >> (8 * kt + 2 * (e >> 2) + hh)) & 1 ? NAN : sc[kt][e];
        }
      }
      if (masked) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            sc[kt][e] = hidden(k0 + 32 * kt + 8 * (e >> 2) + 4 * hh + (e & 3)) ? -INFINITY : sc[kt][e];
          }
      }
      float m2[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int e = 0; e < 16; ++e)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) m2[kt] = fmaxf(m2[kt], sc[kt][e]);
      const float mb = max_halves(fmaxf(m2[0], m2[1]));
      // The reference of the exponents follows the largest score only once that
      // is kLag octaves ahead in some row (of 32 rows nearly every block would
      // move one): the probabilities, so much larger than those of the
      // reference, are as exact in fp16 and the sums in fp32 have room.
      const float m_new = fmaxf(m_run, mb);   // of the raw scores, as in the kernel for small tiles
      if (__builtin_amdgcn_ballot_w64((m_new - m_run) * a.scale_log2 > kLag) != 0) {   // NaN while both are -inf
        const float alpha = exp2_hw((m_run - (m_new == -INFINITY ? 0.f : m_new)) * a.scale_log2);
        m_run = m_new;
        l_run *= alpha;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[dt][e] *= alpha;
      }
      // Large references are subtracted from the raw scores; of small ones the product with the scale is rounded by
      // less than the scores are, and it needs no instruction of its own (subtracting always: 219 us in place of 214 for
      // a 4096-token prompt).
      const float m_use = m_run == -INFINITY ? 0.f : m_run;
      float m_scaled = __builtin_fmaf(m_use, a.scale_log2, -kTileLift);
      const bool large = !(fabsf(m_scaled) < kLarge);
      if (__builtin_amdgcn_ballot_w64(large) != 0) {
        m_scaled = large ? -kTileLift : m_scaled;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int e = 0; e < 16; ++e) sc[kt][e] -= large ? m_use : 0.f;
      }
      // Sixteen keys at a time, and beside each product with the values two of the next sixteen's probabilities per
      // lane and the fragment of the next sixteen's values; the scheduler, left alone, puts every read right in front
      // of its product and waits for it.
      auto values = [&](int s4, int dt) {
        return *reinterpret_cast<const half8_t*>(base + kTileKBytes + (32 * dt + ql) * kVRow + 16 * hh + 32 * s4);
      };
      // Two at a time.  Their sum is of the probabilities as rounded: the weights of the values then add up to one.
      auto probabilities = [&](int s4, int e, half8_t& to) {
        half2_t p2;
#pragma unroll
        for (int u = 0; u < 2; ++u)
          p2[u] = (half_t)exp2_hw(__builtin_fmaf(sc[s4 >> 1][8 * (s4 & 1) + e + u], a.scale_log2, -m_scaled));
        to[e] = p2[0];
        to[e + 1] = p2[1];
        l_run = __builtin_amdgcn_fdot2(p2, half2_t{(half_t)1.f, (half_t)1.f}, l_run, false);
      };
      half8_t va[4], pb;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) va[dt] = values(0, dt);
#pragma unroll
      for (int e = 0; e < 8; e += 2) probabilities(0, e, pb);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int s4 = 0; s4 < 4; ++s4) {
        half8_t next = pb;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) {
          const half8_t v = va[dt];
          if (s4 < 3) va[dt] = values(s4 + 1, dt);
          acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pb, acc[dt], 0, 0, 0);
          if (s4 < 3) probabilities(s4 + 1, 2 * dt, next);
          __builtin_amdgcn_sched_barrier(0);
        }
        pb = next;
      }
    };

    load_block(c0);
    // The rows' q land here too: left in flight they would be waited for in every turn of the loop.
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) asm volatile("" : "+v"(qf[ks]));
    __builtin_amdgcn_s_waitcnt(0);
    store_block(0, c0);
    bad = bad_next;
    __syncthreads();
    for (int kb = c0; kb < c1; ++kb) {
      const int st = (kb - c0) & 1;
      const bool more = kb + 1 < c1;
      if (more) load_block(kb + 1);
      const int k0 = kb * kTileKeys;
      if (k0 < wave_keys) step(smem + st * kTileStage, st, k0, k0 + kTileKeys > ragged || k0 + kTileKeys > keys);
      if (more) store_block(st ^ 1, kb + 1);   // that stage was last read before the previous barrier
      bad = bad_next;
      __syncthreads();
    }
    l_run += __shfl_xor(l_run, 32);
  }

  // Lane (ql, hh) holds d = 32 dt + 8 (e / 4) + 4 hh + e % 4 of row ql.
  if (r >= rows) return;
  if (p.chunks > 1) {
    const size_t at = ((size_t)slot * a.KV + kvh) * R + 32 * wave + ql;
    float* o = a.part_o + at * D + 4 * hh;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<float4_t*>(o + 32 * dt + 8 * j) =
            float4_t{acc[dt][4 * j], acc[dt][4 * j + 1], acc[dt][4 * j + 2], acc[dt][4 * j + 3]};
    if (hh == 0) a.part_ml[at] = float2_t{m_run, l_run};
    return;
  }
  const float inv = 1.0f / l_run;
  half_t* o = a.out + ((size_t)(p.s.start + tok) * a.H + head) * D + 4 * hh;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      half4_t h;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        h[e] = refused ? (half_t)NAN : l_run == 0.f ? (half_t)0.f : (half_t)(acc[dt][4 * j + e] * inv);
      *reinterpret_cast<half4_t*>(o + 32 * dt + 8 * j) = h;
    }
}

// Over the 32 lanes of a half wave.
__device__ __forceinline__ float half_max(float v) {
  v = row_max16(v);
  return fmaxf(v, __shfl_xor(v, 16));
}
__device__ __forceinline__ float half_sum(float v) {
  v = row_sum16(v);
  return v + __shfl_xor(v, 16);
}

// The chunks of split tiles joined: grid = (tiles the call can have * KV,
// parts of R rows).  A row and turn takes a wave in small tiles, which have few
// rows and up to a hundred chunks, and half a wave in large ones, whose many
// rows of a few chunks are bound by the latency of each (one wave per row: 28
// us for 82 MB of partials, half a wave: 16).  The weights 2^(m_c - M) of as
// many chunks as there are lanes are held one per lane and read out as each
// chunk is added, in chunk order.
template <int R>
__global__ __launch_bounds__(256) void paged_attention_merge_kernel(PagedArgs a) {
  constexpr int D = kPagedDim;
  const int lane = threadIdx.x & 63;
  const int kvh = blockIdx.x % a.KV;
  const Place p = find_place<R, true>(a, blockIdx.x / a.KV, lane);
  if (!p.found || p.chunks == 1 || p.slot0 + (int64_t)p.s.tiles * p.chunks > a.slots) return;
  const int end = min(R, p.s.count * a.G - p.tile * R);
  const bool refused = a.mask != nullptr && p.s.count > kMaxTreeTokens;
  constexpr int kLanes = R == 16 ? 64 : 32, kRows = 64 / kLanes, E = D / kLanes;   // lanes of a row, rows of a wave
  typedef float vec_t __attribute__((ext_vector_type(E)));
  typedef half_t out_t __attribute__((ext_vector_type(E)));
  const int half = lane / kLanes, l = lane % kLanes;
  for (int row0 = kRows * (4 * blockIdx.y + (threadIdx.x >> 6)); row0 < end; row0 += 4 * kRows * gridDim.y) {
    const int row = min(row0 + half, end - 1);   // an odd last row: twice
    auto at = [&](int chunk) { return ((size_t)slot_of(p, p.tile, chunk) * a.KV + kvh) * R + row; };
    // The first chunks' maxima and sums and the first outputs are requested together.
    constexpr int kAhead = R == 16 ? 16 : 8;
    const int n0 = min(kLanes, p.chunks);
    float2_t ml = l < n0 ? a.part_ml[at(l)] : float2_t{-INFINITY, 0.f};
    vec_t o[kAhead];
    auto load = [&](int c) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        o[u] = *reinterpret_cast<const vec_t*>(a.part_o + at(min(c + u, p.chunks - 1)) * D + E * l);
    };
    load(0);
    float M = ml.x;
    for (int c0 = kLanes; c0 < p.chunks; c0 += kLanes)
      if (c0 + l < p.chunks) M = fmaxf(M, a.part_ml[at(c0 + l)].x);
    M = kRows == 1 ? wave_max_rl(M) : half_max(M);
    const float Mu = M == -INFINITY ? 0.f : M;
    float den = 0.f;
    vec_t num = 0.f;
    for (int c0 = 0; c0 < p.chunks; c0 += kLanes) {
      const int n = min(kLanes, p.chunks - c0);
      if (c0 > 0) ml = l < n ? a.part_ml[at(c0 + l)] : float2_t{-INFINITY, 0.f};
      const float w = exp2_hw((ml.x - Mu) * a.scale_log2);
      den += kRows == 1 ? wave_sum_rl(w * ml.y) : half_sum(w * ml.y);
      for (int c = 0; c < n; c += kAhead) {
        if (c0 + c > 0) load(c0 + c);
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          if (c + u < n) {
            const float wl = lane_f(w, min(c + u, kLanes - 1)), wh = lane_f(w, min(c + u, kLanes - 1) + 64 - kLanes);
            num += (half ? wh : wl) * o[u];
          }
      }
    }
    const int rr = p.tile * R + row, t = rr / a.G;
    out_t h;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float n = num[e];
      h[e] = refused ? (half_t)NAN : den == 0.f ? (half_t)0.f : (half_t)(n / den);
    }
    half_t* dst = a.out + ((size_t)(p.s.start + t) * a.H + kvh * a.G + rr - t * a.G) * D + E * l;
    *reinterpret_cast<out_t*>(dst) = h;
  }
}

// Which kernel a call takes, and its places of the grid per kv head: the tiles
// the call can have at most, and as many more for chunks.  Small tiles: the
// three workgroups that a compute unit holds (seven drafted tokens behind 4100:
// 22.3 us with four, 17.5 with three, 18.8 with two; the decode batches within
// 2 %), and ten per tile up to eight per unit where many tiles of unequal
// length are to end together (24 sequences 68 -> 64 us, 64 long ones 396 ->
// 380, of which two thirds more would cost 400).  Large ones: four where two are resident, since the tiles of a ragged
// batch differ in length (six chunks 120 us with two, 108 with four, 123 with
// eight; twelve trees 133, 126, 127).  Where the tiles alone give small ones
// sixteen or large ones four per compute unit nothing is split and nothing
// merged.
struct PagedPlan {
  int rows;                 // of a tile
  int64_t tiles, spare, slots;
  int min_blocks;
  size_t bytes;
};

PagedPlan paged_plan(int64_t tokens, int64_t sequences, int64_t G, int64_t KV, int64_t width, int64_t page_size) {
  PagedPlan p{};
  // On average more than 48 rows per sequence take the large tiles.  40 / 8 heads behind 4000 positions, us in small and
  // in large tiles: one sequence of 6 tokens 14.9 and 16.2, 10 tokens 18.5 and 18.4, 20 tokens 21.6 and 23.7; eight
  // sequences of 3 tokens 37.1 and 36.2, 7 tokens 51 and 42, 20 tokens 88 and 55.  One line for both costs the single
  // sequence up to 2 us above it and a batch up to 10 below.
  p.rows = tokens * G > 48 * sequences ? kTileRows : 16;
  // sum_b ceil(count_b G / R) <= ceil(tokens G / R) + sequences, and no more tiles than rows.
  p.tiles = (tokens * G + p.rows - 1) / p.rows + sequences;
  const int64_t most = tokens * ((G + p.rows - 1) / p.rows);
  if (p.tiles > most) p.tiles = most;
  const int64_t target = p.rows == 16 ? 768 : 1024;
  p.min_blocks = p.rows == 16 ? 4 : 8;
  const int64_t blocks = width * page_size / kKeys + 1;
  p.spare = blocks > p.min_blocks && p.tiles * KV < (p.rows == 16 ? 4 : 1) * target ? (target + KV - 1) / KV : 0;
  if (p.rows == 16 && p.spare > 0) {
    const int64_t many = 10 * p.tiles < 2048 / KV ? 10 * p.tiles : 2048 / KV;
    if (p.spare < many) p.spare = many;
  }
  p.slots = p.tiles + p.spare;
  p.bytes = p.spare ? (size_t)p.slots * KV * p.rows * (kPagedDim + 2) * 4 : 0;
  return p;
}

int paged_attention_check(int64_t q_heads, int64_t kv_heads) {
  WQ_REQUIRE(q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0, WQ_ERR_INVALID_ARGUMENT,
             "q_heads (%lld) must be a positive multiple of kv_heads (%lld)", (long long)q_heads, (long long)kv_heads);
  WQ_REQUIRE(q_heads / kv_heads <= kMaxPagedGroup, WQ_ERR_UNSUPPORTED, "at most %d query heads per kv head",
             kMaxPagedGroup);
  return WQ_OK;
}

}  // namespace
}  // namespace wq

using namespace wq;

extern "C" int wq_paged_attention_workspace_size(int64_t tokens, int64_t sequences, int64_t q_heads,
                                                 int64_t kv_heads, int64_t head_dim, int64_t table_width,
                                                 int64_t page_size, size_t* bytes) {
  WQ_REQUIRE(bytes, WQ_ERR_INVALID_ARGUMENT, "null pointer argument");
  int rc = paged_attention_check(q_heads, kv_heads);
  if (rc != WQ_OK) return rc;
  const int64_t page = kv_heads * page_size * head_dim;
  rc = paged_pool_check(head_dim, kv_heads, page, page, 1, page_size, table_width, sequences, tokens);
  if (rc != WQ_OK) return rc;
  *bytes = tokens && sequences
               ? paged_plan(tokens, sequences, q_heads / kv_heads, kv_heads, table_width, page_size).bytes
               : 0;
  return WQ_OK;
}

extern "C" int wq_paged_attention(const uint16_t* q, int64_t tokens, int64_t q_heads, int64_t kv_heads,
                                  int64_t head_dim, const uint16_t* key_pages, int64_t key_page_stride,
                                  const uint16_t* value_pages, int64_t value_page_stride, int64_t num_pages,
                                  int64_t page_size, const int32_t* page_table, int64_t table_width,
                                  const int32_t* query_starts, const int32_t* seq_lens, int64_t sequences,
                                  const int64_t* tree_mask, float scale, uint16_t* out, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  int rc = paged_attention_check(q_heads, kv_heads);
  if (rc != WQ_OK) return rc;
  rc = paged_pool_check(head_dim, kv_heads, key_page_stride, value_page_stride, num_pages, page_size, table_width,
                        sequences, tokens);
  if (rc != WQ_OK) return rc;
  // The maximum of the raw scores stands for the maximum of the scaled ones.
  WQ_REQUIRE(scale > 0.f && scale * kLog2e < INFINITY, WQ_ERR_INVALID_ARGUMENT, "scale must be positive and finite (got %g)",
             (double)scale);
  if (tokens == 0 || sequences == 0) return WQ_OK;
  WQ_REQUIRE(q && key_pages && value_pages && page_table && query_starts && seq_lens && out, WQ_ERR_INVALID_ARGUMENT,
             "null pointer argument");
  WQ_REQUIRE(((uintptr_t)q | (uintptr_t)key_pages | (uintptr_t)value_pages | (uintptr_t)out) % 16 == 0,
             WQ_ERR_INVALID_ARGUMENT, "q, the pages and out must be 16-byte aligned");
  WQ_REQUIRE(((uintptr_t)page_table | (uintptr_t)query_starts | (uintptr_t)seq_lens) % 4 == 0 &&
                 (uintptr_t)tree_mask % 8 == 0,
             WQ_ERR_INVALID_ARGUMENT, "integer operands must be aligned to their size");
  // A workgroup reads its rows' queries before it writes the same rows; others may not have.
  const uintptr_t in0 = (uintptr_t)q, out0 = (uintptr_t)out, bytes = (uintptr_t)(tokens * q_heads * kPagedDim * 2);
  WQ_REQUIRE(out0 == in0 || out0 + bytes <= in0 || in0 + bytes <= out0, WQ_ERR_INVALID_ARGUMENT,
             "out must be q itself or not overlap it");
  const PagedPlan plan = paged_plan(tokens, sequences, q_heads / kv_heads, kv_heads, table_width, page_size);
  WQ_REQUIRE(plan.bytes == 0 || (workspace && workspace_bytes >= plan.bytes && (uintptr_t)workspace % 16 == 0),
             WQ_ERR_WORKSPACE, "paged attention needs a 16-byte aligned workspace of %zu bytes (got %zu)", plan.bytes,
             workspace_bytes);
  WQ_REQUIRE(plan.slots * kv_heads <= 0xffffff, WQ_ERR_UNSUPPORTED,   // a grid holds 2^32 threads
             "too many tokens for one call: %lld workgroups", (long long)(plan.slots * kv_heads));
  PagedArgs a{};
  a.q = reinterpret_cast<const half_t*>(q);
  a.kp = reinterpret_cast<const half_t*>(key_pages);
  a.vp = reinterpret_cast<const half_t*>(value_pages);
  a.table = page_table;
  a.starts = query_starts;
  a.lens = seq_lens;
  a.mask = tree_mask;
  a.out = reinterpret_cast<half_t*>(out);
  a.part_o = reinterpret_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2_t*>(a.part_o + (size_t)plan.slots * kv_heads * plan.rows * kPagedDim);
  a.k_stride = key_page_stride;
  a.v_stride = value_page_stride;
  a.scale_log2 = scale * kLog2e;
  a.sequences = (int)sequences;
  a.tokens = (int)tokens;
  a.H = (int)q_heads;
  a.KV = (int)kv_heads;
  a.G = (int)(q_heads / kv_heads);
  a.width = (int)table_width;
  a.page_size = (int)page_size;
  a.num_pages = (int)num_pages;
  a.slots = (int)plan.slots;
  a.spare = (int)plan.spare;
  a.min_blocks = plan.min_blocks;
  const dim3 grid((unsigned)(plan.slots * kv_heads));
  // One tile per sequence on average: single tokens.  64 long sequences 424 us, with non-temporal loads 397 (380 with
  // more chunks too); seven drafted tokens, three tiles that share their keys through the L2, 17.5 and 18.6.
  if (plan.rows == 16 && tokens * a.G <= 16 * sequences)
    hipLaunchKernelGGL(paged_attention_rows_kernel<true>, grid, dim3(256), 0, as_stream(stream), a);
  else if (plan.rows == 16)
    hipLaunchKernelGGL(paged_attention_rows_kernel<false>, grid, dim3(256), 0, as_stream(stream), a);
  else
    hipLaunchKernelGGL(paged_attention_tile_kernel, grid, dim3(256), 2 * kTileStage, as_stream(stream), a);
  rc = check_launch("paged_attention");
  if (rc != WQ_OK || plan.spare == 0) return rc;
  const dim3 merge((unsigned)(plan.tiles * kv_heads), 4);
  if (plan.rows == 16)
    hipLaunchKernelGGL(paged_attention_merge_kernel<16>, merge, dim3(256), 0, as_stream(stream), a);
  else
    hipLaunchKernelGGL(paged_attention_merge_kernel<kTileRows>, merge, dim3(256), 0, as_stream(stream), a);
  return check_launch("paged_attention_merge");
}
