// Sampling one token per row of logits: temperature, top-k, top-p, min-p and
// the draw from a given uniform number.
//
// With y = logit log2(e) / T a token weighs 2^(y - the largest y): exactly 1 for
// the largest, so that equal ones are drawn and cut exactly.  Three launches,
// the row cut into parts of whole 16-byte chunks:
//   tally   counts every part's tokens and adds their weights in 16 bins of
//           octaves of weight, from the part's largest down;
//   gather  from the row's bins follow the ones in which top-k, top-p and
//           min-p end; their tokens, a few dozen of a peaked row and some
//           thousands of a flat one, go to a list;
//   pick    one workgroup per row finds the value at which the cut ends in the
//           list and draws: a part from the parts' remaining weights, then the
//           token in it.
// Which tokens stay comes down to one value: all above it and the first
// `ties` that equal it, by index.  Everything that decides is exact or in 64
// bits and summed in a fixed order: over 151936 normal logits a 32-bit
// sum in blocks of 512 changes the token of one to three rows in a hundred, a
// running one of a quarter to a third (numpy, 400 rows each, deviations 0.1 to 3).
// 64 rows of 151936 fp16 logits (19 MB): tally 26 to 27 us (55 vector
// instructions per token counted, 24 of them 64-bit; the vector units issue in
// 41 % of the cycles and waves wait in 41 %, so neither alone is the bound),
// gather 15, pick 24 to 29 in nine draws of twelve.  The pick's time is its
// slowest row's: 80 to 84 us where top-p ends among 44 thousand tokens of one
// bin (the weights of them all, by one workgroup), 141 where top-k of a peaked
// row ends among nearly the whole vocabulary.  One row takes 7, 9 and 17 us.
#include "ondeviceinfer_sample.h"
#include "wq_common.h"
#include "wq_status.h"

#include <limits.h>
#include <math.h>

// Every kernel has to find a token in the same octave: a product that the
// compiler keeps unrounded in one place (y - floor(y) as one fused operation)
// is another number than the rounded one it is compared with elsewhere.
#pragma clang fp contract(off)

namespace wq {
namespace {

constexpr int kBins = 16;
constexpr int kMaxParts = 64;
constexpr int kPickThreads = 1024;
constexpr int kSub = 256;              // steps of a bin, or of a byte of the key
constexpr int kBounded = 16384;        // longer lists are searched between bounds (Span)
constexpr int kMostSorted = 512;       // tokens of one step put in order at once

struct SampleArgs {
  const void* logits;
  int64_t row_stride;
  int rows, vocab, parts;
  int mass_bits;      // fraction bits of a mass as a whole number: vocab of them stay below 2^63
  int list_cap;       // entries of a row's list
  const float *uniform, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  float temperature_all, top_p_all, min_p_all;
  int32_t top_k_all;
  int64_t* tokens;
  float2_t* peak;     // [rows][parts] (largest logit, bits of its first index); NaN: the part holds one
  double* mass;       // [rows][parts][kBins], the part's largest weighs 1
  uint32_t* count;    // [rows][parts][kBins]
  float2_t* list;     // [rows][list_cap] (logit, bits of its index)
};

// One row of logits in 16-byte chunks on 16-byte boundaries: a row that starts
// off one has a first chunk that it only ends in.
template <typename T>
struct Row {
  static constexpr int E = 16 / (int)sizeof(T);
  const T* base;
  int vocab, lead;   // elements of the first chunk in front of the row
  int chunks, per_part;

  __device__ __forceinline__ Row(const SampleArgs& a, int row) {
    base = reinterpret_cast<const T*>(a.logits) + (size_t)row * a.row_stride;
    vocab = a.vocab;
    lead = (int)(((uintptr_t)base & 15) / sizeof(T));
    chunks = (lead + vocab + E - 1) / E;
    per_part = (chunks + a.parts - 1) / a.parts;
  }
  __device__ __forceinline__ int index(int chunk) const { return chunk * E - lead; }
  // The chunk's values; bit e of the result: element e is in the row.  -0 comes as +0.
  __device__ __forceinline__ uint32_t load(int chunk, float (&v)[E]) const {
    const int j = index(chunk);
    uint32_t in = 0;
    if (j >= 0 && j + E <= vocab) {
      const uint4_t raw = *reinterpret_cast<const uint4_t*>(base + j);
      unpack(raw, v);
      in = (1u << E) - 1;
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        v[e] = -INFINITY;
        if (j + e >= 0 && j + e < vocab) {
          v[e] = (float)base[j + e];
          in |= 1u << e;
        }
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] += 0.f;
    return in;
  }

 private:
  static __device__ __forceinline__ void unpack(uint4_t raw, float (&v)[8]) {
    const half8_t h = __builtin_bit_cast(half8_t, raw);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)h[e];
  }
  static __device__ __forceinline__ void unpack(uint4_t raw, float (&v)[4]) {
    const float4_t f = __builtin_bit_cast(float4_t, raw);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = f[e];
  }
};

// What a row asks for, and whether there is anything to weigh.
struct Ask {
  double to_octaves;   // log2(e) / temperature
  double top_p;        // 1: off
  double min_p;        // log2 of it; -inf: off
  int top_k;           // vocab: off
  bool greedy, none;
};

__device__ __forceinline__ Ask read_ask(const SampleArgs& a, int row) {
  const float t = a.temperature ? a.temperature[row] : a.temperature_all;
  const float p = a.top_p ? a.top_p[row] : a.top_p_all;
  const float mp = a.min_p ? a.min_p[row] : a.min_p_all;
  const int32_t k = a.top_k ? a.top_k[row] : a.top_k_all;
  const float u = a.uniform[row];
  Ask q;
  q.none = !(t >= 0.f) || t == INFINITY || p != p || mp != mp || u != u;
  q.greedy = t == 0.f || k == 1 || p <= 0.f || mp > 1.f;
  q.to_octaves = 1.4426950408889634074 / (double)t;
  q.top_p = p < 1.f ? (double)p : 1.0;
  q.min_p = mp > 0.f ? log2((double)mp) : -INFINITY;
  q.top_k = k > 0 && k < a.vocab ? k : a.vocab;
  return q;
}

// Positions against a base, the octave of the largest rounded up to one of
// 4 n + 3: the bins of a part and of the row then start whole multiples of
// four octaves apart.  Weights against the largest itself.  Infinite logits:
// where the largest is +inf only its equals weigh anything, and a part that
// holds nothing above -inf weighs nothing.
struct Scale {
  double to_octaves, base, zero;
  float top;
  bool infinite;

  __device__ __forceinline__ Scale(double per_logit, float largest)
      : to_octaves(per_logit), top(largest), infinite(isinf(largest)) {
    base = infinite ? 3.0 : 4.0 * floor(0.25 * floor((double)largest * per_logit)) + 3.0;
    zero = infinite ? 0.0 : (double)largest;
  }
  __device__ __forceinline__ double finite(float v) const {
    return (double)(infinite ? (((v == top) & (top > 0.f)) ? 0.f : -INFINITY) : v);
  }
  __device__ __forceinline__ double y(float v) const { return finite(v) * to_octaves; }
  // log2 of its weight: 0 for the largest.  The difference of two logits is exact, or as good as.
  __device__ __forceinline__ double fall(float v) const { return (finite(v) - zero) * to_octaves; }
  // Whole octaves below the base, 1100 for as many or more (2^-1100 is nothing).
  __device__ __forceinline__ int below(double y) const { return (int)fmin(base - floor(y), 1100.0); }
};

// Bins of octaves below the base: eight of one octave, seven of four, and all
// that lies 36 or more below (of 2^18 tokens less than 2^-15 of the weight:
// only top-k goes there).
__device__ __forceinline__ int bin_at(int depth) {
  return depth < 8 ? max(depth, 0) : min(8 + ((depth - 8) >> 2), kBins - 1);
}
__device__ __forceinline__ int bin_depth(int bin) { return bin < 8 ? bin : 8 + 4 * (bin - 8); }   // its first octave

// 2^d for d <= 0: its whole octaves split off, the fraction is (k + t) / 256,
// 2^(k/256) comes from a table, 2^(t/256) = e^(t ln 2 / 256) is its series to
// the fourth power (the next term is below 2e-15 of the sum).  Of a d in
// (-2^-54, 0) the fraction d + 1 rounds to 1, k is 256 and the table's last
// entry, 2, makes up for the octave that floor took off.
struct Exp2Table {
  double v[257];
};

__device__ __forceinline__ void fill_exp2(Exp2Table& t, int tid) {
  if (tid < 256) t.v[tid] = exp2((double)tid / 256.0);
  if (tid == 0) t.v[256] = 2.0;
}

__device__ __forceinline__ double exp2_64(double d, const Exp2Table& table) {
  constexpr double c = 0.69314718055994530942 / 256.0;
  const double whole = floor(d);
  const double f = 256.0 * fmax(d - whole, 0.0);   // 0 for -inf, whose difference is NaN
  const int k = (int)f;
  const double t = f - (double)k;
  double s = __builtin_fma(t, c * c * c * c / 24.0, c * c * c / 6.0);
  s = __builtin_fma(s, t, c * c / 2.0);
  s = __builtin_fma(s, t, c);
  s = __builtin_fma(s, t, 1.0);
  return ldexp(s * table.v[k], (int)fmax(whole, -1100.0));
}

// (best, at) the better of two of a row's largest: NaN first, then the larger, then the lower index.
__device__ __forceinline__ void keep_peak(float& best, int& at, float ov, int oi) {
  if (best == best && (ov != ov || ov > best || (ov == best && oi < at))) {
    best = ov;
    at = oi;
  }
}

__device__ __forceinline__ void wave_peak(float& best, int& at) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float ov = __shfl_xor(best, o);
    const int oi = __shfl_xor(at, o);
    keep_peak(best, at, ov, oi);
  }
}

// An addition in LDS that returns nothing, so that no thread waits for it.
template <typename V>
__device__ __forceinline__ void add_lds(V* at, V v) {
  __hip_atomic_fetch_add(at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}

// grid = (workgroups of 4 / W parts, rows): W = 1 wave per part, or all four
// where few rows leave waves to spare (sample_waves).  Every thread adds to its
// own column of the bins in LDS: no two lanes meet in a bank for longer than
// the access takes, and the additions happen in a fixed order.
template <typename T, int W>
__global__ __launch_bounds__(256) void sample_tally_kernel(SampleArgs a) {
  constexpr int E = Row<T>::E;
  __shared__ double mass[kBins][256];
  __shared__ uint32_t count[kBins][256];
  __shared__ Exp2Table table;
  __shared__ float sv[4];
  __shared__ int si[4];
  const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int part = blockIdx.x * (4 / W) + (W == 1 ? wave : 0);
  const int mine = W == 1 ? lane : tid;   // of the part's 64 W threads
  const Ask q = read_ask(a, row);
  const Row<T> r(a, row);
  const int c0 = min(part * r.per_part, r.chunks), c1 = min(c0 + r.per_part, r.chunks);
  fill_exp2(table, tid);
#pragma unroll
  for (int b = 0; b < kBins; ++b) {
    mass[b][tid] = 0.0;
    count[b][tid] = 0;
  }
  float best = -INFINITY;
  int at = INT_MAX;
  bool nan = false;
  for (int c = c0 + mine; c < c1; c += 64 * W) {
    float v[E];
    r.load(c, v);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      nan |= v[e] != v[e];
      if (v[e] > best) {
        best = v[e];
        at = r.index(c) + e;
      }
    }
  }
  if (nan) best = NAN;
  wave_peak(best, at);
  if (lane == 0) {
    sv[wave] = best;
    si[wave] = at;
  }
  __syncthreads();
  if (W > 1) {
    best = sv[0];
    at = si[0];
    for (int w = 1; w < W; ++w) keep_peak(best, at, sv[w], si[w]);
  }
  if (part >= a.parts) return;
  if (mine == 0) a.peak[(size_t)row * a.parts + part] = float2_t{best, __builtin_bit_cast(float, at)};
  if (q.none || q.greedy || best != best) return;   // the pick needs no weights
  const Scale s(q.to_octaves, best);
  for (int c = c0 + mine; c < c1; c += 64 * W) {
    float v[E];
    const uint32_t in = r.load(c, v);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int b = bin_at(s.below(s.y(v[e])));
      const double w = exp2_64(s.fall(v[e]), table);
      const uint32_t one = (in >> e) & 1;   // 0: not of the row
      add_lds(&mass[b][tid], one ? w : 0.0);
      add_lds(&count[b][tid], one);
    }
  }
  if (W > 1) __syncthreads();
  // 4 W threads per bin: thread (b, j) adds the columns j, j + 4 W, ...
  const int b = mine / (4 * W), j = mine % (4 * W), from = tid - mine;
  double m = 0.0;
  uint32_t n = 0;
#pragma unroll
  for (int k = 0; k < 64 * W; k += 4 * W) {
    m += mass[b][from + k + j];
    n += count[b][from + k + j];
  }
#pragma unroll
  for (int o = 2 * W; o > 0; o >>= 1) {
    m += __shfl_xor(m, o);
    n += __shfl_xor(n, o);
  }
  if (j == 0) {
    const size_t to = ((size_t)row * a.parts + part) * kBins + b;
    a.mass[to] = m;
    a.count[to] = n;
  }
}

// The row's largest logit, in every lane of every wave.
__device__ __forceinline__ float row_peak(const SampleArgs& a, int row, int lane, int& at) {
  float best = -INFINITY;
  at = INT_MAX;
  if (lane < a.parts) {
    const float2_t e = a.peak[(size_t)row * a.parts + lane];
    best = e.x;
    const float y = e.y;
    at = __builtin_bit_cast(int, y);
  }
  wave_peak(best, at);
  return best;
}

// A row's tallies against the row's own base, of each part and altogether.
struct RowTally {
  double mass[kBins];
  uint32_t count[kBins];
  double part_mass[kMaxParts][kBins];
  uint32_t part_count[kMaxParts][kBins];
  double raw_mass[kMaxParts][kBins];        // against the part's largest
  uint32_t raw_count[kMaxParts][kBins];
  int shift[kMaxParts];       // octaves from the row's base down to the part's (64: as many or more)
  double scale[kMaxParts];    // what the part's largest weighs
};

// A thread's share of the row's tallies, requested before the row's settings are known.
template <int THREADS>
struct TallyShare {
  static constexpr int N = kMaxParts * kBins / THREADS;
  double mass[N];
  uint32_t count[N];

  __device__ __forceinline__ TallyShare(const SampleArgs& a, int row, int tid) {
    const size_t from = (size_t)row * a.parts * kBins;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = min(tid + i * THREADS, a.parts * kBins - 1);
      mass[i] = a.mass[from + e];
      count[i] = a.count[from + e];
    }
  }
};

// By THREADS >= 256 threads, with barriers; the sums in a fixed order.
template <int THREADS>
__device__ __forceinline__ void read_tally(const SampleArgs& a, const Scale& s, int row, int tid,
                                           const TallyShare<THREADS>& share, RowTally& t) {
  const size_t from = (size_t)row * a.parts;
  if (tid < a.parts) {
    const float top = a.peak[from + tid].x;
    // Base against base: a part of -inf, or a finite one below +inf, is out of sight.
    const double down = isinf(s.top) || isinf(top) ? (top == s.top ? 0.0 : INFINITY)
                                                   : s.base - Scale(s.to_octaves, top).base;
    t.shift[tid] = (int)fmin(down, 64.0);
    t.scale[tid] = exp2(s.fall(top));
  }
#pragma unroll
  for (int i = 0; i < TallyShare<THREADS>::N; ++i) {   // past the last part: repeats, never read
    (&t.raw_mass[0][0])[tid + i * THREADS] = share.mass[i];
    (&t.raw_count[0][0])[tid + i * THREADS] = share.count[i];
  }
  __syncthreads();
  for (int e = tid; e < a.parts * kBins; e += THREADS) {
    const int p = e / kBins, b = e % kBins;
    double m = 0.0;
    uint32_t n = 0;
    // The part's bins that start within the row's bin b.
    const int down = t.shift[p];
    const int i1 = b == kBins - 1 ? b : bin_at(bin_depth(b + 1) - down) - 1;
    for (int i = bin_at(bin_depth(b) - down); i <= i1; ++i) {
      m += t.raw_mass[p][i];
      n += t.raw_count[p][i];
    }
    t.part_mass[p][b] = m * t.scale[p];
    t.part_count[p][b] = n;
  }
  __syncthreads();
  if (tid < 256) {
    const int b = tid >> 4;
    double m = 0.0;
    uint32_t n = 0;
    for (int p = tid & 15; p < a.parts; p += 16) {
      m += t.part_mass[p][b];
      n += t.part_count[p][b];
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      m += __shfl_xor(m, o);
      n += __shfl_xor(n, o);
    }
    if ((tid & 15) == 0) {
      t.mass[b] = m;
      t.count[b] = n;
    }
  }
  __syncthreads();
}

// The bins whose tokens decide: top-k ends in bin `by_k`, top-p (where
// top-k is off; under top-k it follows from what that leaves) in `by_p`,
// min-p in `floor`; kBins where one is off.  The list takes the bins lo ..
// hi, none if hi < lo.
struct Range {
  int by_k, by_p, floor, lo, hi;
  uint32_t want;       // tokens that top-k leaves of bin by_k
  double before;       // mass in front of bin by_k
  double whole;        // mass of all bins
  double min_y;        // the smallest y that min-p leaves
  uint32_t listed;     // tokens of the list; more than it can hold: the pick goes over the row instead
};

// The row's bins one per lane (lanes 16 .. repeat them), with the sums in
// front of each: the search for a bin costs a few lane moves instead of a
// chain of LDS reads.
struct LaneBins {
  double mass, before;
  uint32_t count, count_before;

  __device__ __forceinline__ LaneBins(const RowTally& t, int lane) {
    const int b = lane & (kBins - 1);
    mass = t.mass[b];
    count = t.count[b];
    double m = mass;
    uint32_t n = count;
#pragma unroll
    for (int o = 1; o < kBins; o <<= 1) {
      const double um = __shfl_up(m, o, kBins);
      const uint32_t un = __shfl_up(n, o, kBins);
      if (b >= o) {
        m += um;
        n += un;
      }
    }
    before = m - mass;
    count_before = n - count;
  }
  __device__ __forceinline__ uint32_t first_of(int bin) const { return __shfl(count_before, bin); }
  __device__ __forceinline__ uint32_t tokens_of(int bin) const { return __shfl(count, bin); }
  __device__ __forceinline__ double whole() const { return __shfl(before + mass, kBins - 1); }
  // The first bin up to `last` at which the mass reaches `goal`, and the mass in front of it.
  __device__ __forceinline__ int reach(double goal, int last, int lane, double& in_front) const {
    const uint64_t hit = __builtin_amdgcn_ballot_w64(lane < kBins && (lane >= last || before + mass >= goal));
    const int b = __builtin_ctzll(hit);
    in_front = __shfl(before, b);
    return b;
  }
};

__device__ __forceinline__ Range find_range(const SampleArgs& a, const Ask& q, const Scale& s, const LaneBins& bins,
                                            int lane) {
  Range g{kBins, kBins, kBins, 0, -1, 0, 0.0, bins.whole(), -INFINITY};
  if (q.min_p > -INFINITY) {
    g.min_y = s.y(s.top) + q.min_p;
    g.floor = bin_at(s.below(g.min_y));
  }
  if (q.top_k < a.vocab) {
    const uint64_t hit = __builtin_amdgcn_ballot_w64(
        lane < kBins && (lane == kBins - 1 || bins.count_before + bins.count >= (uint32_t)q.top_k));
    g.by_k = __builtin_ctzll(hit);
    g.want = (uint32_t)q.top_k - __shfl(bins.count_before, g.by_k);
    g.before = __shfl(bins.before, g.by_k);
    g.lo = 0;
    g.hi = g.by_k;
  } else if (q.top_p < 1.0) {
    double before;
    g.by_p = bins.reach(q.top_p * g.whole, kBins - 1, lane, before);
    g.lo = min(g.by_p, g.floor);
    g.hi = g.by_p;
  } else if (g.floor < kBins) {
    g.lo = g.hi = g.floor;
  }
  const uint32_t upto = bins.count_before + bins.count;
  g.listed = g.hi < g.lo ? 0 : __shfl(upto, g.hi) - __shfl(bins.count_before, g.lo);
  return g;
}

// The order of the values as unsigned numbers, in as many bytes as the type has.
template <typename T>
struct Key;
template <>
struct Key<half_t> {
  static constexpr int kBytes = 2;
  static constexpr uint32_t kLowest = 0x03ffu, kHighest = 0xfc00u;   // of -inf and +inf
  static __device__ __forceinline__ uint32_t of(float v) {
    const half_t h = (half_t)v;   // exact: v came from fp16
    const uint32_t u = __builtin_bit_cast(uint16_t, h);
    return u & 0x8000u ? (~u & 0xffffu) : (u | 0x8000u);
  }
  static __device__ __forceinline__ float value(uint32_t k) {
    const uint16_t u = (uint16_t)(k & 0x8000u ? (k & 0x7fffu) : ~k);
    return (float)__builtin_bit_cast(half_t, u);
  }
};
template <>
struct Key<float> {
  static constexpr int kBytes = 4;
  static constexpr uint32_t kLowest = 0x007fffffu, kHighest = 0xff800000u;
  static __device__ __forceinline__ uint32_t of(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    return u & 0x80000000u ? ~u : (u | 0x80000000u);
  }
  static __device__ __forceinline__ float value(uint32_t k) {
    const uint32_t u = k & 0x80000000u ? (k & 0x7fffffffu) : ~k;
    return __builtin_bit_cast(float, u);
  }
};

// The smallest value for which `holds` (which stays true as values rise), found
// by the wave 64 keys at a time; NaN, the key next above +inf, if there is none
// (the bins above that of a row's infinite logits hold nothing).
template <typename T, typename F>
__device__ __forceinline__ float lowest_where(int lane, F holds) {
  uint32_t lo = Key<T>::kLowest, n = Key<T>::kHighest - Key<T>::kLowest + 2;   // the key lies in lo .. lo + n - 1
  while (n > 1) {   // n falls to a 64th, never below 1: the last key is taken to hold, whatever it and those beyond say
    const uint32_t step = (n + 63) / 64;
    const uint32_t k = lane * step;
    const uint64_t in = __builtin_amdgcn_ballot_w64((k >= n - 1) | holds(Key<T>::value(lo + min(k, n - 1))));
    // The first probe that is in, or the stretch behind the last one.
    const int first = in ? __builtin_ctzll(in) : 64;
    if (first == 0) return Key<T>::value(lo);
    const uint32_t next = lo + (first - 1) * step + 1;
    const uint32_t end = first == 64 ? lo + n : lo + first * step + 1;
    n = min(end, lo + n) - next;
    lo = next;
  }
  return Key<T>::value(lo);
}

// The smallest value whose bin is at most `bin` (bins fall as values rise), NaN if there is none.
template <typename T>
__device__ __forceinline__ float lowest_of(const Scale& s, int bin, int lane) {
  return lowest_where<T>(lane, [&](float v) { return bin_at(s.below(s.y(v))) <= bin; });
}

// Where the parts' tokens of the bins lo .. hi lie in the list, part `lane`'s.
__device__ __forceinline__ void list_places(const RowTally& t, const Range& g, int parts, int lane, uint32_t& from,
                                            uint32_t& to) {
  uint32_t n = 0;
  if (lane < parts)
    for (int b = g.lo; b <= g.hi; ++b) n += t.part_count[lane][b];
  to = n;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t u = __shfl_up(to, o);
    if (lane >= o) to += u;
  }
  from = to - n;
}

// grid = (workgroups of 4 / W parts, rows) as for the tally: a part's tokens of
// the bins lo .. hi go to its place in the row's list, in no order.
template <typename T, int W>
__global__ __launch_bounds__(256) void sample_gather_kernel(SampleArgs a) {
  constexpr int E = Row<T>::E;
  __shared__ RowTally tally;
  __shared__ int next[4];   // W > 1: the part's next entry, in next[0]
  const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int part = blockIdx.x * (4 / W) + (W == 1 ? wave : 0);
  const TallyShare<256> share(a, row, tid);
  const Ask q = read_ask(a, row);
  int first;
  const float top = row_peak(a, row, lane, first);
  if (q.none || q.greedy || !(top > -INFINITY)) return;
  const Scale s(q.to_octaves, top);
  read_tally<256>(a, s, row, tid, share, tally);
  const Range g = find_range(a, q, s, LaneBins(tally, lane), lane);
  if (g.hi < g.lo || g.listed > (uint32_t)a.list_cap || part >= a.parts) return;
  uint32_t from, to;
  list_places(tally, g, a.parts, lane, from, to);
  int at = __builtin_amdgcn_readlane((int)from, part);
  const int end = __builtin_amdgcn_readlane((int)to, part);
  if (at == end) return;
  if (W > 1) {
    if (tid == 0) next[0] = at;
    __syncthreads();
  }
  const float least = g.hi == kBins - 1 ? -INFINITY : lowest_of<T>(s, g.hi, lane);
  const float above = g.lo == 0 ? NAN : lowest_of<T>(s, g.lo - 1, lane);   // NaN: no bound
  const Row<T> r(a, row);
  const int c0 = part * r.per_part, c1 = min(c0 + r.per_part, r.chunks);
  float2_t* list = a.list + (size_t)row * a.list_cap;
  for (int c = c0 + (W == 1 ? 0 : 64 * wave); c < c1; c += 64 * W) {
    float v[E];
    const uint32_t in = c + lane < c1 ? r.load(c + lane, v) : 0u;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool take = (bool)((in >> e) & 1) & (v[e] >= least) & !(v[e] >= above);
      const uint64_t mask = __builtin_amdgcn_ballot_w64(take);
      if (mask == 0) continue;
      const int n = __popcll(mask);
      if (W > 1) {
        int first_at = 0;
        if (lane == 0) first_at = atomicAdd(&next[0], n);
        at = __builtin_amdgcn_readfirstlane(first_at);
      }
      const int to_at = at + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                                            __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
      if (take && to_at < end) list[to_at] = float2_t{v[e], __builtin_bit_cast(float, r.index(c + lane) + e)};
      at += n;
    }
  }
  // The place was counted by the tally; an entry that came out differently here would be no token, not an old one.
  if (W > 1) {
    __syncthreads();
    at = next[0];
  }
  for (int i = at + (W == 1 ? lane : tid); i < end; i += 64 * W)
    list[i] = float2_t{0.f, __builtin_bit_cast(float, -1)};
}

// The value at which a cut ends, among the row's tokens of one bin.
struct Cut {
  int bin;          // tokens of lower bins all stay, of higher ones none (kBins: all stay)
  uint32_t key;     // of this bin: all above it stay, and the first `ties` that equal it
  uint32_t ties;
  double kept;      // mass of this bin's tokens that stay
};

// The values of a bin or of a step of it.  The position of a token, its bin and
// its step rise and fall with the value, so a token that lies outside is told
// by two comparisons in place of its position in 64 bits, which costs every pass
// about 650 cycles per 1024 tokens.  The bounds cost some 8 us to find, so only
// lists longer than kBounded are searched between them: 64 rows of which one
// lists all 151936 tokens took 198 us instead of 238 (183 now that bins of few
// tokens are sorted at once), ordinary ones 75 with bounds always and 66 without
// (now 67 to 72).
struct Span {
  float least, above;   // above NaN: no bound
  __device__ __forceinline__ bool has(float v) const { return (v >= least) & !(v >= above); }
};

struct PickShared {
  Exp2Table table;
  RowTally tally;
  uint32_t step_count[kSub];
  unsigned long long step_mass[kSub];
  uint64_t order[kMostSorted];    // (order of the value, index), the first of the order smallest
  double upto[kMostSorted];       // weights of the tokens up to each
  double part_mass[kMaxParts];
  unsigned long long part_edge[kMaxParts];
  uint32_t part_ties[kMaxParts];
  double wave_d[16];
  uint32_t wave_n[16];
  int wave_i[16];
  // what one thread found for all
  int step, n;
  int taken;   // tokens taken so far by sort(), zero between two of them
  uint32_t left, ties;
  double above, target;
  int part;
  bool part_has_ties;
};

template <typename T>
struct Picker {
  static constexpr int E = Row<T>::E;
  const SampleArgs& a;
  const Row<T>& r;
  const Scale& s;
  PickShared& sh;
  const float2_t* list;   // nullptr: the tokens come from the row
  int listed;
  int tid;

  // f(value, index) over the listed tokens, or all of the row's.
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    if (list != nullptr) {
      for (int i = tid; i < listed; i += kPickThreads) {
        const float2_t e = list[i];
        const float y = e.y;
        const int index = __builtin_bit_cast(int, y);
        if (index >= 0) f(e.x, index);
      }
    } else {
      for (int c = tid; c < r.chunks; c += kPickThreads) {
        float v[E];
        const uint32_t in = r.load(c, v);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if ((in >> e) & 1) f(v[e], r.index(c) + e);
      }
    }
  }

  __device__ __forceinline__ double weight_of(float v) const { return exp2_64(s.fall(v), sh.table); }

  // Fraction bits of masses of bin `bin` as whole numbers: the largest position lies 0 to 3 octaves below the base, and
  // a weight of the bin is at most 2^(1 - those of the bin's first octave beyond them), or 1.
  __device__ __forceinline__ int bits_of(int bin) const {
    return a.mass_bits + max(bin_depth(bin) - 1 - s.below(s.y(s.top)), 0);
  }

  __device__ __forceinline__ uint64_t order_of(float v, int index) const {
    return ((uint64_t)(~Key<T>::of(v)) << 32) | (uint32_t)index;
  }

  // One step of 256 down a bin (`byte` = kBytes), or down the values of its
  // step `sub` that share the leading bytes of the key: which step holds the
  // end, what lies above it.  The last bin, which has no end, goes in eighths
  // of an octave.  Masses are whole numbers of 2^-mass_bits of a power of two
  // that the bin's weights do not exceed, so that their sum does not depend on
  // the order.
  __device__ __forceinline__ int sub_of(int bin, double y) const {
    const double per = bin < 8 ? kSub : bin < kBins - 1 ? kSub / 4 : 8;
    return (int)fmin((s.base + 1.0 - bin_depth(bin) - y) * per, (double)(kSub - 1));
  }
  __device__ __forceinline__ void walk(int bin, bool by_mass, double before, double goal, int byte, bool bounded,
                                       Span span, int sub, uint32_t prefix) {
    const int bits = bits_of(bin);
    const double unit = ldexp(1.0, bits), per_unit = ldexp(1.0, -bits);
    for (int i = tid; i < kSub; i += kPickThreads) {
      sh.step_count[i] = 0;
      sh.step_mass[i] = 0;
    }
    __syncthreads();
    each([&](float v, int) {
      if (!span.has(v)) return;
      const double y = s.y(v);
      if (!bounded && bin_at(s.below(y)) != bin) return;
      int d = sub_of(bin, y);
      if (byte < Key<T>::kBytes) {
        const uint32_t k = Key<T>::of(v);
        if (d != sub || (byte + 1 < Key<T>::kBytes && (k >> (8 * byte + 8)) != prefix)) return;
        d = 255 - (int)((k >> (8 * byte)) & 255);
      }
      atomicAdd(&sh.step_count[d], 1u);
      atomicAdd(&sh.step_mass[d], (unsigned long long)rint(weight_of(v) * unit));
    });
    __syncthreads();
    if (tid < 64) {   // four steps per lane
      uint32_t n[4], sum_n = 0;
      unsigned long long m[4], sum_m = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        n[i] = sh.step_count[4 * tid + i];
        m[i] = sh.step_mass[4 * tid + i];
        sum_n += n[i];
        sum_m += m[i];
      }
      uint32_t run_n = sum_n;
      unsigned long long run_m = sum_m;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t un = __shfl_up(run_n, o);
        const unsigned long long um = __shfl_up(run_m, o);
        if (tid >= o) {
          run_n += un;
          run_m += um;
        }
      }
      run_n -= sum_n;
      run_m -= sum_m;
      // The first step that reaches the end; roundings can leave a mass a hair out of reach: the last with tokens then.
      const uint32_t left = sh.left;
      const double above = sh.above;
      int hit = kSub, last = -1;
      uint32_t hit_n = 0, last_n = 0;
      unsigned long long hit_m = 0, last_m = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (n[i] != 0) {
          const bool ends = by_mass ? before + above + (double)(run_m + m[i]) * per_unit >= goal : run_n + n[i] >= left;
          if (ends && hit == kSub) {
            hit = 4 * tid + i;
            hit_n = run_n;
            hit_m = run_m;
          }
          last = 4 * tid + i;
          last_n = run_n;
          last_m = run_m;
        }
        run_n += n[i];
        run_m += m[i];
      }
      const uint64_t hits = __builtin_amdgcn_ballot_w64(hit < kSub);
      const uint64_t lasts = __builtin_amdgcn_ballot_w64(last >= 0);
      const bool mine = hits ? tid == __builtin_ctzll(hits) : lasts ? tid == 63 - __builtin_clzll(lasts) : tid == 0;
      if (mine) {
        const int d = hits ? hit : max(last, 0);
        sh.step = d;
        sh.n = (int)sh.step_count[d];
        if (!by_mass) sh.left = left - (hits ? hit_n : last_n);
        sh.above = above + (double)(hits ? hit_m : last_m) * per_unit;
      }
    }
    __syncthreads();
  }

  // Puts the (at most kMostSorted, `most` expected) tokens that `take` picks in
  // order and leaves their weights beside them; their number.
  template <typename F>
  __device__ __forceinline__ int sort(F take, int most) {
    each([&](float v, int index) {
      if (!take(v)) return;
      const int to = atomicAdd(&sh.taken, 1);
      if (to < kMostSorted) sh.order[to] = order_of(v, index);
    });
    __syncthreads();
    const int n = min(sh.taken, min(most, kMostSorted));
    // Each token's rank, by as many threads as there are for it.
    int each_by = 64;
    while (each_by > 2 && n * each_by > kPickThreads) each_by >>= 1;
    const int i = tid / each_by;
    uint64_t mine = ~0ull;
    int rank = 0;
    if (i < n) {
      mine = sh.order[i];
#pragma unroll 4
      for (int j = tid & (each_by - 1); j < n; j += each_by) rank += sh.order[j] < mine;
    }
    for (int o = each_by >> 1; o > 0; o >>= 1) rank += __shfl_xor(rank, o);
    __syncthreads();
    if (i < n && (tid & (each_by - 1)) == 0) sh.order[rank] = mine;
    __syncthreads();
    const int lane = tid & 63, wave = tid >> 6;
    double x = tid < n ? weight_of(Key<T>::value(~(uint32_t)(sh.order[tid] >> 32))) : 0.0;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double u = __shfl_up(x, o);
      if (lane >= o) x += u;
    }
    if (lane == 63) sh.wave_d[wave] = x;
    __syncthreads();
    for (int w = 0; w < wave; ++w) x += sh.wave_d[w];
    if (tid < n) sh.upto[tid] = x;
    if (tid == 0) sh.taken = 0;
    __syncthreads();
    return n;
  }

  // The end among the sorted tokens first .. first + n - 1, all of them bin
  // `bin`'s from where `above` of its mass lies in front: after `left` of them,
  // or where the mass `goal` is reached; the first stays in any case.
  __device__ __forceinline__ Cut end_in(int bin, bool by_mass, double before, double goal, int first, int n, int left,
                                        double above) {
    const double front = first > 0 ? sh.upto[first - 1] : 0.0;
    int stay = min(left, n);
    if (by_mass) {   // token j > 0 stays while what lies in front of it is below the goal; the sums rise with j
      int lo = 1, hi = max(n, 1);
      while (lo < hi) {
        const int j = (lo + hi) >> 1;
        if (before + (above + (sh.upto[first + j - 1] - front)) < goal) lo = j + 1;
        else hi = j;
      }
      stay = lo;
    }
    stay = max(stay, 1);
    const uint32_t end = (uint32_t)(sh.order[first + stay - 1] >> 32);
    int lo = 0, hi = stay - 1;   // the first of the tokens that equal the last
    while (lo < hi) {
      const int j = (lo + hi) >> 1;
      if ((uint32_t)(sh.order[first + j] >> 32) == end) hi = j;
      else lo = j + 1;
    }
    return Cut{bin, ~end, (uint32_t)(stay - lo), above + (sh.upto[first + stay - 1] - front)};
  }

  // Where the count `want`, or the mass `goal` of which `before` lies in front
  // of the bin, is reached among the `tokens` tokens of bin `bin`.
  __device__ __forceinline__ Cut find_cut(int bin, uint32_t tokens, bool by_mass, uint32_t want, double before, double goal) {
    __syncthreads();   // top-p's search follows top-k's, whose end the other waves may still be reading
    if (tid == 0) {
      sh.left = want;
      sh.above = 0.0;     // mass of the bin in front of the steps found so far
      sh.ties = 0;
    }
    // The step of the bin; where many of tokens share it, most of them equal, the bytes of the key.
    const int lane = tid & 63;
    const bool bounded = listed > kBounded;
    Span span{-INFINITY, NAN};
    if (bounded && bin < kBins - 1) span.least = lowest_of<T>(s, bin, lane);
    if (bounded && bin > 0) span.above = lowest_of<T>(s, bin - 1, lane);
    int sub = -1;
    uint32_t prefix = 0;
    if (tokens <= kMostSorted) {   // the whole bin is put in order
      __syncthreads();
      const int n = sort([&](float v) { return bounded ? span.has(v) : bin_at(s.below(s.y(v))) == bin; }, (int)tokens);
      return end_in(bin, by_mass, before, goal, 0, n, (int)want, 0.0);
    }
    bool few = false;
    for (int byte = Key<T>::kBytes; byte >= 0; --byte) {
      walk(bin, by_mass, before, goal, byte, bounded, span, sub, prefix);
      if (byte == Key<T>::kBytes) {
        sub = sh.step;
        // Tokens of lower bins, of this one's first `upto` steps.
        auto above = [&](float v, int upto) {
          const double y = s.y(v);
          const int b = bin_at(s.below(y));
          return b < bin || (b == bin && sub_of(bin, y) < upto);
        };
        if (bounded && (sub < kSub - 1 || bin < kBins - 1)) {   // the last step of the last bin has no end
          const float least = lowest_where<T>(lane, [&](float v) { return above(v, sub + 1); });
          span.least = fmaxf(span.least, least);
        }
        if (bounded && sub > 0) span.above = lowest_where<T>(lane, [&](float v) { return above(v, sub); });
        few = sh.n <= kMostSorted;
        if (few) break;
      } else {
        prefix = (prefix << 8) | (uint32_t)(255 - sh.step);
      }
      __syncthreads();
    }
    Cut cut{bin, 0, 0, 0.0};
    if (few) {
      const int n = sort([&](float v) {
        if (bounded) return span.has(v);
        const double y = s.y(v);
        return bin_at(s.below(y)) == bin && sub_of(bin, y) == sub;
      }, sh.n);
      return end_in(bin, by_mass, before, goal, 0, n, (int)sh.left, sh.above);
    }
    cut.key = prefix;
    const double w = weight_of(Key<T>::value(prefix));
    if (by_mass) {
      const double need = ceil((goal - before - sh.above) / w);
      cut.ties = need >= (double)sh.n ? (uint32_t)sh.n : (uint32_t)fmax(need, 1.0);
    } else {
      cut.ties = min(sh.left, (uint32_t)sh.n);
    }
    cut.kept = sh.above + cut.ties * w;
    return cut;
  }
};

// grid = rows, 1024 threads.
template <typename T>
__global__ __launch_bounds__(kPickThreads) void sample_pick_kernel(SampleArgs a) {
  constexpr int E = Row<T>::E;
  __shared__ PickShared sh;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const TallyShare<kPickThreads> share(a, row, tid);
  const Ask q = read_ask(a, row);
  int first;
  const float top = row_peak(a, row, lane, first);
  if (q.none || q.greedy || !(top > -INFINITY)) {
    if (tid == 0) a.tokens[row] = q.none || !(top > -INFINITY) ? -1 : first;
    return;
  }
  const Row<T> r(a, row);
  const Scale s(q.to_octaves, top);
  fill_exp2(sh.table, tid);
  if (tid == 0) sh.taken = 0;
  read_tally<kPickThreads>(a, s, row, tid, share, sh.tally);
  const LaneBins bins(sh.tally, lane);
  const Range g = find_range(a, q, s, bins, lane);
  Picker<T> pick{a, r, s, sh, g.listed <= (uint32_t)a.list_cap ? a.list + (size_t)row * a.list_cap : nullptr,
                 (int)g.listed, tid};

  // Where top-k ends, then top-p of what it leaves.
  Cut cut{kBins, 0, 0, 0.0};
  double whole = g.whole;
  // A short list is put in order as a whole, for both.
  const bool cuts = g.by_k < kBins || q.top_p < 1.0;
  const bool ordered = cuts && g.listed <= (uint32_t)min(a.list_cap, kMostSorted);
  int sorted = 0;
  if (ordered) sorted = pick.sort([](float) { return true; }, (int)g.listed);
  for (int stage = 0; stage < 2; ++stage) {
    const bool by_mass = stage == 1;
    if (by_mass ? q.top_p == 1.0 : g.by_k == kBins) continue;
    const double goal = q.top_p * whole;
    double before = g.before;
    int bin = g.by_k;
    if (by_mass) bin = bins.reach(goal, min(cut.bin, kBins - 1), lane, before);
    Cut end;
    if (ordered) {
      const int from = (int)(bins.first_of(bin) - bins.first_of(g.lo));
      const int n = min((int)bins.tokens_of(bin), sorted - from);
      end = pick.end_in(bin, by_mass, before, goal, max(min(from, sorted - 1), 0), n, (int)g.want, 0.0);
    } else {
      end = pick.find_cut(bin, bins.tokens_of(bin), by_mass, g.want, before, goal);
    }
    if (!by_mass) whole = before + end.kept;
    // Both may end at one value: the fewer ties.  Otherwise top-p's is the higher one, but for roundings.
    if (end.bin < cut.bin || end.key > cut.key) cut = end;
    else if (end.key == cut.key) cut.ties = min(cut.ties, end.ties);
  }
  const int edge = min(cut.bin, g.floor);   // the only bin of which some tokens stay and some go
  // Bins, keys and y all rise with the value: 1 stays, 2 stays while there are ties left.
  const float last_value = cut.bin < kBins ? Key<T>::value(cut.key) : -INFINITY;
  const double min_y = g.min_y;
  auto stays = [&](float v, double y) -> int { return y >= min_y ? (int)(v > last_value) + 2 * (int)(v == last_value) : 0; };

  // What stays of every part: the bins in front of the edge, and its own tokens of the edge, sixteen lanes per part.
  static_assert(kPickThreads == 16 * kMaxParts, "sixteen lanes per part");
  const int bits = pick.bits_of(edge);
  const double unit = ldexp(1.0, bits), per_unit = ldexp(1.0, -bits);
  {
    uint32_t from, to;
    list_places(sh.tally, g, a.parts, lane, from, to);
    const int p = tid >> 4;
    from = __shfl(from, p);
    to = __shfl(to, p);
    unsigned long long m = 0;
    uint32_t ties = 0;
    auto add = [&](float v) {
      if (!(v >= last_value)) return;
      const double y = s.y(v);
      if (bin_at(s.below(y)) != edge) return;
      const int st = stays(v, y);
      if (st == 1) {   // what weighs anything counts for something: the last bin has no end
        const double w = pick.weight_of(v);
        m += w > 0.0 ? (unsigned long long)fmax(rint(w * unit), 1.0) : 0ull;
      }
      ties += st == 2;
    };
    if (p < a.parts && edge < kBins && sh.tally.part_count[p][edge] != 0) {
      if (pick.list != nullptr) {
        for (uint32_t i = from + (tid & 15); i < to; i += 16) {
          const float2_t e = pick.list[i];
          const float index = e.y;
          if (__builtin_bit_cast(int, index) >= 0) add(e.x);
        }
      } else {
        const int c1 = min((p + 1) * r.per_part, r.chunks);
        for (int c = p * r.per_part + (tid & 15); c < c1; c += 16) {
          float v[E];
          const uint32_t in = r.load(c, v);
#pragma unroll
          for (int e = 0; e < E; ++e)
            if ((in >> e) & 1) add(v[e]);
        }
      }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      m += __shfl_xor(m, o);
      ties += __shfl_xor(ties, o);
    }
    if ((tid & 15) == 0) {
      sh.part_edge[p] = m;
      sh.part_ties[p] = ties;
    }
  }
  __syncthreads();
  if (wave == 0) {   // a part per lane
    double m = 0.0;
    uint32_t n = 0;
    if (lane < a.parts) {
      for (int b = 0; b < edge; ++b) m += sh.tally.part_mass[lane][b];
      m += (double)sh.part_edge[lane] * per_unit;
      n = sh.part_ties[lane];
    }
    uint32_t ties = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t u = __shfl_up(ties, o);
      if (lane >= o) ties += u;
    }
    ties -= n;   // in front of the part
    // Signed on purpose: of the unsigned form, ties < cut.ties ? min(n, cut.ties - ties) : 0, hipcc 7.2 keeps a plain
    // subtraction and drops the comparison.
    const int kept = max(min((int)n, (int)cut.ties - (int)ties), 0);
    if (kept > 0) m += kept * pick.weight_of(Key<T>::value(cut.key));
    double upto = m;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double u = __shfl_up(upto, o);
      if (lane >= o) upto += u;
    }
    const double target = (double)a.uniform[row] * __shfl(upto, 63);
    const uint64_t some = __builtin_amdgcn_ballot_w64(m > 0.0);   // never none: the largest weighs 1
    const uint64_t past = __builtin_amdgcn_ballot_w64(m > 0.0 && upto > target);
    const int part = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
    if (lane == part) {
      sh.part = part;
      sh.target = target - (upto - m);
      sh.ties = ties;
      sh.part_has_ties = n > 0;
    }
  }
  __syncthreads();

  // The token inside the part: every thread a run of chunks, its mass, the sum of the threads in front of it.
  const int part = sh.part;
  const double target = sh.target;
  const int c0 = part * r.per_part, c1 = min(c0 + r.per_part, r.chunks);
  const int run = (c1 - c0 + kPickThreads - 1) / kPickThreads;
  const int t0 = min(c0 + tid * run, c1), t1 = min(t0 + run, c1);
  uint32_t ties0 = sh.ties;
  if (sh.part_has_ties) {
    uint32_t mine = 0;
    for (int c = t0; c < t1; ++c) {
      float v[E];
      const uint32_t in = r.load(c, v);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if ((in >> e) & 1) mine += stays(v[e], s.y(v[e])) == 2;
    }
    uint32_t x = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t u = __shfl_up(x, o);
      if (lane >= o) x += u;
    }
    if (lane == 63) sh.wave_n[wave] = x;
    __syncthreads();
    for (int w = 0; w < wave; ++w) ties0 += sh.wave_n[w];
    ties0 += x - mine;
  }
  double m = 0.0;
  int last = -1;
  {
    uint32_t ties = ties0;
    for (int c = t0; c < t1; ++c) {
      float v[E];
      const uint32_t in = r.load(c, v);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int st = (in >> e) & 1 ? stays(v[e], s.y(v[e])) : 0;
        const bool tie = st == 2;
        const bool in_draw = (st == 1) | (tie & (ties < cut.ties));
        ties += tie;
        if (__builtin_amdgcn_ballot_w64(in_draw) == 0) continue;   // of a filtered row most waves have nothing here
        const double w = in_draw ? pick.weight_of(v[e]) : 0.0;
        m += w;
        last = w > 0.0 ? r.index(c) + e : last;
      }
    }
  }
  double x = m;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double u = __shfl_up(x, o);
    if (lane >= o) x += u;
  }
  if (lane == 63) sh.wave_d[wave] = x;
  __syncthreads();
  double upto = 0.0;   // the mass of the threads up to this one
  for (int w = 0; w < wave; ++w) upto += sh.wave_d[w];
  upto += x;
  // The first thread at which the running weight exceeds the target, as for the parts: decided by one set of sums, so
  // that a target on the border of two runs falls into one of them.  Failing that (roundings) the last with any weight.
  const uint64_t some = __builtin_amdgcn_ballot_w64(m > 0.0);
  const uint64_t past = __builtin_amdgcn_ballot_w64((m > 0.0) & (upto > target));
  if (lane == 0) {
    sh.wave_i[wave] = past ? __builtin_ctzll(past) : INT_MAX;
    sh.wave_n[wave] = some ? 64u - (uint32_t)__builtin_clzll(some) : 0u;   // 0: none
  }
  __syncthreads();
  int owner = 0, l = -1;
  for (int w = 0; w < 16; ++w) {
    if (l < 0 && sh.wave_i[w] != INT_MAX) {
      owner = w;
      l = sh.wave_i[w];
    }
  }
  if (l < 0) {
    for (int w = 0; w < 16; ++w) {
      if (sh.wave_n[w] != 0) {
        owner = w;
        l = (int)sh.wave_n[w] - 1;
      }
    }
  }
  if (wave != owner) return;
  l = __builtin_amdgcn_readfirstlane(max(l, 0));
  // That thread's run, a token per lane of its wave: the first one past the target, or (roundings) the last that stays.
  const int f0 = __builtin_amdgcn_readlane(t0, l), f1 = __builtin_amdgcn_readlane(t1, l);
  double before = __shfl(upto - m, l);
  uint32_t ties = (uint32_t)__builtin_amdgcn_readlane((int)ties0, l);
  int hit = __builtin_amdgcn_readlane(last, l);
  const int j1 = min(r.index(f1), r.vocab);
  for (int j0 = max(r.index(f0), 0); j0 < j1; j0 += 64) {
    const int j = j0 + lane;
    const float v = j < j1 ? (float)r.base[j] + 0.f : 0.f;
    const int st = j < j1 ? stays(v, s.y(v)) : 0;
    const uint64_t tied = __builtin_amdgcn_ballot_w64(st == 2);
    const uint32_t in_front = ties + (uint32_t)__popcll(tied & ((1ull << lane) - 1));
    const double w = (st == 1) | ((st == 2) & (in_front < cut.ties)) ? pick.weight_of(v) : 0.0;
    double run_upto = w;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double u = __shfl_up(run_upto, o);
      if (lane >= o) run_upto += u;
    }
    const uint64_t hits = __builtin_amdgcn_ballot_w64((w > 0.0) & (before + run_upto > target));
    if (hits) {
      hit = j0 + __builtin_ctzll(hits);
      break;
    }
    before += __shfl(run_upto, 63);
    ties += (uint32_t)__popcll(tied);
  }
  // The tally found weight in this part; should none be left of it here (at 2^-1074), the largest is the answer.
  if (lane == 0) a.tokens[row] = hit >= 0 ? hit : first;
}

// Parts of a row, a wave each: sixteen waves per compute unit over all rows,
// and at least 1024 tokens each.
int sample_parts(int64_t rows, int64_t vocab) {
  int64_t p = (4096 + rows - 1) / rows;
  const int64_t most = (vocab + 1023) / 1024;
  if (p > most) p = most;
  if (p > kMaxParts) p = kMaxParts;
  return (int)(p < 1 ? 1 : p);
}

constexpr size_t kPartBytes = sizeof(float2_t) + kBins * (sizeof(double) + sizeof(uint32_t));

// Entries of a row's list: all of the vocabulary, or what 64 MiB of lists leave for a row.
int sample_list_cap(int64_t rows, int64_t vocab) {
  int64_t cap = (64 << 20) / (int64_t)sizeof(float2_t) / rows;
  if (cap < 4096) cap = 4096;
  return (int)(cap < vocab ? cap : vocab);
}

size_t sample_bytes(int64_t rows, int64_t vocab) {
  return (size_t)rows * (sample_parts(rows, vocab) * kPartBytes + sample_list_cap(rows, vocab) * sizeof(float2_t));
}

int sample_check(int64_t rows, int64_t vocab) {
  WQ_REQUIRE(rows >= 0 && rows <= 65535, WQ_ERR_INVALID_ARGUMENT, "rows must be in [0, 65535] (got %lld)",
             (long long)rows);
  WQ_REQUIRE(vocab > 0 && vocab <= (1 << 30), WQ_ERR_INVALID_ARGUMENT, "vocab must be in [1, 2^30] (got %lld)",
             (long long)vocab);
  return WQ_OK;
}

// Waves per part: all four of a workgroup while that leaves at most four
// workgroups per compute unit.
int sample_waves(const SampleArgs& a) { return (int64_t)a.parts * a.rows <= 1024 ? 4 : 1; }

template <typename T, int W>
int launch_sample(const SampleArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.parts * W + 3) / 4), (unsigned)a.rows);
  hipLaunchKernelGGL((sample_tally_kernel<T, W>), grid, dim3(256), 0, s, a);
  int rc = check_launch("sample_tally");
  if (rc != WQ_OK) return rc;
  hipLaunchKernelGGL((sample_gather_kernel<T, W>), grid, dim3(256), 0, s, a);
  rc = check_launch("sample_gather");
  if (rc != WQ_OK) return rc;
  hipLaunchKernelGGL(sample_pick_kernel<T>, dim3((unsigned)a.rows), dim3(kPickThreads), 0, s, a);
  return check_launch("sample_pick");
}

template <typename T>
int launch_sample(const SampleArgs& a, hipStream_t s) {
  return sample_waves(a) == 4 ? launch_sample<T, 4>(a, s) : launch_sample<T, 1>(a, s);
}

}  // namespace
}  // namespace wq

using namespace wq;

extern "C" int wq_sample_workspace_size(int64_t rows, int64_t vocab, size_t* bytes) {
  WQ_REQUIRE(bytes, WQ_ERR_INVALID_ARGUMENT, "null pointer argument");
  const int rc = sample_check(rows, vocab);
  if (rc != WQ_OK) return rc;
  *bytes = rows ? sample_bytes(rows, vocab) : 0;
  return WQ_OK;
}

extern "C" int wq_sample(const void* logits, int32_t logits_type, int64_t rows, int64_t vocab, int64_t row_stride,
                         const float* uniform, const float* temperature, float temperature_all, const int32_t* top_k,
                         int32_t top_k_all, const float* top_p, float top_p_all, const float* min_p, float min_p_all,
                         int64_t* tokens, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = sample_check(rows, vocab);
  if (rc != WQ_OK) return rc;
  WQ_REQUIRE(logits_type == WQ_LOGITS_F16 || logits_type == WQ_LOGITS_F32, WQ_ERR_INVALID_ARGUMENT,
             "unknown logits type %d", logits_type);
  if (rows == 0) return WQ_OK;
  WQ_REQUIRE(logits && uniform && tokens, WQ_ERR_INVALID_ARGUMENT, "null pointer argument");
  WQ_REQUIRE(row_stride >= vocab || (rows == 1 && row_stride >= 0), WQ_ERR_INVALID_ARGUMENT,
             "rows of %lld logits lie %lld elements apart", (long long)vocab, (long long)row_stride);
  WQ_REQUIRE(row_stride <= INT64_MAX / 8 / rows, WQ_ERR_INVALID_ARGUMENT, "row_stride out of range");
  const uintptr_t size = logits_type == WQ_LOGITS_F16 ? 2 : 4;
  WQ_REQUIRE((uintptr_t)logits % size == 0 && (uintptr_t)tokens % 8 == 0 &&
                 ((uintptr_t)uniform | (uintptr_t)temperature | (uintptr_t)top_k | (uintptr_t)top_p |
                  (uintptr_t)min_p) % 4 == 0,
             WQ_ERR_INVALID_ARGUMENT, "operands must be aligned to their size");
  SampleArgs a{};
  a.parts = sample_parts(rows, vocab);
  const size_t places = (size_t)rows * a.parts, need = sample_bytes(rows, vocab);
  WQ_REQUIRE(workspace && workspace_bytes >= need && (uintptr_t)workspace % 8 == 0, WQ_ERR_WORKSPACE,
             "sampling needs an 8-byte aligned workspace of %zu bytes (got %zu)", need, workspace_bytes);
  a.list_cap = sample_list_cap(rows, vocab);
  a.logits = logits;
  a.row_stride = row_stride;
  a.mass_bits = 63;
  while (a.mass_bits > 0 && ((int64_t)1 << (63 - a.mass_bits)) < vocab) --a.mass_bits;
  if (a.mass_bits > 50) a.mass_bits = 50;   // 2^z itself has 53
  a.rows = (int)rows;
  a.vocab = (int)vocab;
  a.uniform = uniform;
  a.temperature = temperature;
  a.temperature_all = temperature_all;
  a.top_k = top_k;
  a.top_k_all = top_k_all;
  a.top_p = top_p;
  a.top_p_all = top_p_all;
  a.min_p = min_p;
  a.min_p_all = min_p_all;
  a.tokens = tokens;
  a.peak = reinterpret_cast<float2_t*>(workspace);
  a.mass = reinterpret_cast<double*>(a.peak + places);
  a.list = reinterpret_cast<float2_t*>(a.mass + places * kBins);
  a.count = reinterpret_cast<uint32_t*>(a.list + (size_t)rows * a.list_cap);
  return logits_type == WQ_LOGITS_F16 ? launch_sample<half_t>(a, as_stream(stream))
                                      : launch_sample<float>(a, as_stream(stream));
}
