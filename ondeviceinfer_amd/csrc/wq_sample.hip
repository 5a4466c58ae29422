// Sampling one token per row of logits: temperature, top-k, top-p, min-p and
// the draw from a given uniform number.
//
// Three launches.  A row is cut into parts of whole 16-byte chunks:
//   peak    the largest logit of every part and its first index;
//   tally   with the row's largest logit m known, every token's weight
//           w = 2^z, z = (l - m) log2(e) / T <= 0, added to one of 16 bins of
//           its part, bin = min(floor(-z), 15): mass and count;
//   pick    one workgroup per row finds the bins in which top-k and top-p end,
//           the value inside them at which they do, and draws.
// Which tokens stay comes down to one value: all above it and the first
// `ties` that equal it, by index.  Everything that decides is exact or in 64
// bits and summed in a fixed order: with 32-bit sums over 151936 tokens one
// row in twenty of a flat distribution takes a neighbour of its token.
#include "ondeviceinfer_sample.h"
#include "wq_common.h"
#include "wq_status.h"

#include <limits.h>
#include <math.h>

namespace wq {
namespace {

constexpr int kBins = 16;
constexpr int kMaxParts = 64;
constexpr int kPickThreads = 1024;

struct SampleArgs {
  const void* logits;
  int64_t row_stride;
  int rows, vocab, parts;
  int mass_bits;      // fraction bits of a mass as a whole number: vocab of them stay below 2^63
  const float *uniform, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  float temperature_all, top_p_all, min_p_all;
  int32_t top_k_all;
  int64_t* tokens;
  float2_t* peak;     // [rows][parts] (largest logit, bits of its first index); NaN: the part holds one
  double* mass;       // [rows][parts][kBins]
  uint32_t* count;    // [rows][parts][kBins]
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

// What a row asks for, and what there is to say about it before its weights.
struct Ask {
  double to_octaves;   // log2(e) / temperature
  double top_p;        // 1: off
  double floor;        // smallest z (octaves) that min-p keeps; -inf: off
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
  q.floor = mp > 0.f ? log2((double)mp) : -INFINITY;
  q.top_k = k > 0 && k < a.vocab ? k : a.vocab;
  return q;
}

__device__ __forceinline__ double octaves(float v, float top, double to_octaves) {
  return v == top ? 0.0 : ((double)v - (double)top) * to_octaves;
}

// 2^z for z <= 0: z = n / 32 + r with |r| <= 1 / 64, 2^(n/32) from a table of
// 32 and an exponent, 2^r = e^(r ln 2) by its series to the fifth power (the
// next term is below 3e-15 of the sum).
struct Exp2Table {
  double v[32];
};

__device__ __forceinline__ void fill_exp2(Exp2Table& t, int tid) {
  if (tid < 32) t.v[tid] = exp2((double)tid / 32.0);
}

__device__ __forceinline__ double exp2_64(double z, const Exp2Table& t) {
  const double y = fmax(z, -1100.0);
  const double n = rint(y * 32.0);
  const double x = (y - n * (1.0 / 32.0)) * 0.69314718055994530942;
  double s = x * (1.0 / 120.0) + 1.0 / 24.0;
  s = s * x + 1.0 / 6.0;
  s = s * x + 0.5;
  s = s * x + 1.0;
  s = s * x + 1.0;
  const int k = (int)n;
  return z < -1080.0 ? 0.0 : ldexp(s * t.v[k & 31], k >> 5);
}

__device__ __forceinline__ int bin_of(double z) { return (int)fmin(-z, (double)(kBins - 1)); }

// The row's largest logit over its parts: NaN if a part holds one.  `index`
// (its first index) is valid in every lane.
__device__ __forceinline__ float row_peak(const SampleArgs& a, int row, int lane, int& index) {
  float best = -INFINITY;
  int at = INT_MAX;
  if (lane < a.parts) {
    const float2_t e = a.peak[(size_t)row * a.parts + lane];
    best = e.x;
    const float y = e.y;
    at = __builtin_bit_cast(int, y);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float ov = __shfl_xor(best, o);
    const int oi = __shfl_xor(at, o);
    if (best == best && (ov != ov || ov > best || (ov == best && oi < at))) {
      best = ov;
      at = oi;
    }
  }
  index = at;
  return best;
}

// grid = (parts, rows), 256 threads.
template <typename T>
__global__ __launch_bounds__(256) void sample_peak_kernel(SampleArgs a) {
  constexpr int E = Row<T>::E;
  __shared__ float sv[4];
  __shared__ int si[4];
  const int row = blockIdx.y, part = blockIdx.x, tid = threadIdx.x;
  const Row<T> r(a, row);
  const int c1 = min((part + 1) * r.per_part, r.chunks);
  float best = -INFINITY;
  int at = INT_MAX;
  bool nan = false;
  for (int c = part * r.per_part + tid; c < c1; c += 256) {
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
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float ov = __shfl_xor(best, o);
    const int oi = __shfl_xor(at, o);
    if (best == best && (ov != ov || ov > best || (ov == best && oi < at))) {
      best = ov;
      at = oi;
    }
  }
  if ((tid & 63) == 0) {
    sv[tid >> 6] = best;
    si[tid >> 6] = at;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < 4; ++w)
      if (best == best && (sv[w] != sv[w] || sv[w] > best || (sv[w] == best && si[w] < at))) {
        best = sv[w];
        at = si[w];
      }
    a.peak[(size_t)row * a.parts + part] = float2_t{best, __builtin_bit_cast(float, at)};
  }
}

// grid = (parts, rows), 256 threads.  Every thread keeps its own column of the
// bins in LDS, so the additions need no atomics, meet no bank conflicts
// between lanes and happen in a fixed order.
template <typename T>
__global__ __launch_bounds__(256) void sample_tally_kernel(SampleArgs a) {
  constexpr int E = Row<T>::E;
  __shared__ double mass[kBins][256];
  __shared__ uint32_t count[kBins][256];
  __shared__ Exp2Table table;
  const int row = blockIdx.y, part = blockIdx.x, tid = threadIdx.x;
  const Ask q = read_ask(a, row);
  int at;
  const float top = row_peak(a, row, tid & 63, at);
  if (q.none || q.greedy || !(top > -INFINITY)) return;   // the pick needs no weights
  fill_exp2(table, tid);
#pragma unroll
  for (int b = 0; b < kBins; ++b) {
    mass[b][tid] = 0.0;
    count[b][tid] = 0;
  }
  __syncthreads();
  const Row<T> r(a, row);
  const int c1 = min((part + 1) * r.per_part, r.chunks);
  for (int c = part * r.per_part + tid; c < c1; c += 256) {
    float v[E];
    const uint32_t in = r.load(c, v);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (!((in >> e) & 1)) continue;
      const double z = octaves(v[e], top, q.to_octaves);
      const int b = bin_of(z);
      mass[b][tid] += exp2_64(z, table);
      ++count[b][tid];
    }
  }
  __syncthreads();
  // Thread (b, j) adds the columns j, j + 16, ...; then the 16 lanes of a bin.
  const int b = tid >> 4, j = tid & 15;
  double m = 0.0;
  uint32_t n = 0;
  for (int k = j; k < 256; k += 16) {
    m += mass[b][k];
    n += count[b][k];
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    m += __shfl_xor(m, o);
    n += __shfl_xor(n, o);
  }
  if (j == 0) {
    const size_t at2 = ((size_t)row * a.parts + part) * kBins + b;
    a.mass[at2] = m;
    a.count[at2] = n;
  }
}

// The order of the values as unsigned numbers, in as many bytes as the type has.
template <typename T>
struct Key;
template <>
struct Key<half_t> {
  static constexpr int kBytes = 2;
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
  static __device__ __forceinline__ uint32_t of(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    return u & 0x80000000u ? ~u : (u | 0x80000000u);
  }
  static __device__ __forceinline__ float value(uint32_t k) {
    const uint32_t u = k & 0x80000000u ? (k & 0x7fffffffu) : ~k;
    return __builtin_bit_cast(float, u);
  }
};

struct PickShared {
  Exp2Table table;
  double mass[kBins];
  uint32_t count[kBins];
  double part_mass[kMaxParts];
  uint32_t part_ties[kMaxParts];
  uint32_t digit_count[256];
  unsigned long long digit_mass[256];
  double wave_d[16];
  uint32_t wave_n[16];
  int wave_i[16];
  // broadcasts
  uint32_t prefix, ties, ties_before;
  double above, target;
  int part;
};

// The value at which a cut ends, among the row's tokens of one bin.
struct Cut {
  int bin;          // tokens of lower bins all stay, of higher ones none
  uint32_t key;     // of this bin: all above it stay, and the first `ties` that equal it
  uint32_t ties;
  double kept;      // mass of this bin's tokens that stay
};

// Finds the key of bin `bin` at which `want` is reached counting down from the
// largest: `want` tokens (by_mass false), or the mass `goal`, of which
// `before` lies in front of the bin.  One byte of the key at a time: a pass
// over the row adds the tokens of the bin that share the bytes found so far to
// 256 counters; masses are whole numbers of 2^-mass_bits of the bin's largest
// weight (2^-45 for a vocabulary of 2^17 to 2^18), so that their sum does not
// depend on the order.
template <typename T>
__device__ Cut find_cut(const SampleArgs& a, const Row<T>& r, const Ask& q, float top, int bin, bool by_mass,
                        uint32_t want, double before, double goal, PickShared& s) {
  constexpr int E = Row<T>::E;
  const int tid = threadIdx.x;
  const double unit = ldexp(1.0, a.mass_bits + bin), per_unit = ldexp(1.0, -a.mass_bits - bin);
  if (tid == 0) {
    s.prefix = 0;
    s.ties = want;
    s.above = 0.0;     // mass of the bin above the bytes found so far
  }
  for (int byte = Key<T>::kBytes - 1; byte >= 0; --byte) {
    for (int i = tid; i < 256; i += kPickThreads) {
      s.digit_count[i] = 0;
      s.digit_mass[i] = 0;
    }
    __syncthreads();
    const uint32_t prefix = s.prefix;
    for (int c = tid; c < r.chunks; c += kPickThreads) {
      float v[E];
      const uint32_t in = r.load(c, v);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (!((in >> e) & 1)) continue;
        const double z = octaves(v[e], top, q.to_octaves);
        if (bin_of(z) != bin) continue;
        const uint32_t k = Key<T>::of(v[e]);
        if (byte + 1 < Key<T>::kBytes && (k >> (8 * byte + 8)) != prefix) continue;
        const int d = (k >> (8 * byte)) & 255;
        atomicAdd(&s.digit_count[d], 1u);
        atomicAdd(&s.digit_mass[d], (unsigned long long)rint(exp2_64(z, s.table) * unit));
      }
    }
    __syncthreads();
    if (tid == 0) {
      uint32_t left = s.ties;
      double above = s.above;
      int d = 255, last = -1;
      uint32_t last_left = 0;
      double last_above = 0.0;
      for (; d >= 0; --d) {
        const uint32_t n = s.digit_count[d];
        if (n == 0) continue;
        const double m = (double)s.digit_mass[d] * per_unit;
        last = d;
        last_left = left;
        last_above = above;
        if (by_mass ? before + above + m >= goal : n >= left) break;
        left -= n;
        above += m;
      }
      // Rounding may leave the goal a hair out of reach: the smallest value then.
      s.prefix = (prefix << 8) | (uint32_t)max(last, 0);
      s.ties = last_left;
      s.above = last_above;
      s.wave_n[0] = last >= 0 ? s.digit_count[last] : 0;
    }
    __syncthreads();
  }
  Cut cut;
  cut.bin = bin;
  cut.key = s.prefix;
  const double w = exp2_64(octaves(Key<T>::value(cut.key), top, q.to_octaves), s.table);
  const uint32_t n = s.wave_n[0];
  if (by_mass) {
    const double need = ceil((goal - before - s.above) / w);
    cut.ties = need >= (double)n ? n : (uint32_t)fmax(need, 1.0);
  } else {
    cut.ties = min(s.ties, n);
  }
  cut.kept = s.above + cut.ties * w;
  __syncthreads();
  return cut;
}

// grid = rows, 1024 threads.
template <typename T>
__global__ __launch_bounds__(kPickThreads) void sample_pick_kernel(SampleArgs a) {
  constexpr int E = Row<T>::E;
  __shared__ PickShared s;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Ask q = read_ask(a, row);
  int first;
  const float top = row_peak(a, row, lane, first);
  if (q.none || q.greedy || !(top > -INFINITY)) {
    if (tid == 0) a.tokens[row] = q.none || !(top > -INFINITY) ? -1 : first;
    return;
  }
  const Row<T> r(a, row);
  fill_exp2(s.table, tid);
  const double* mass = a.mass + (size_t)row * a.parts * kBins;
  const uint32_t* count = a.count + (size_t)row * a.parts * kBins;
  if (tid < kBins) {
    double m = 0.0;
    uint32_t n = 0;
    for (int p = 0; p < a.parts; ++p) {
      m += mass[p * kBins + tid];
      n += count[p * kBins + tid];
    }
    s.mass[tid] = m;
    s.count[tid] = n;
  }
  __syncthreads();

  // Where top-k ends, then top-p of what it leaves (every thread the same).
  Cut cut{kBins, 0, 0, 0.0};
  double whole = 0.0;
  for (int b = 0; b < kBins; ++b) whole += s.mass[b];
  if (q.top_k < a.vocab) {
    uint32_t left = (uint32_t)q.top_k;
    double before = 0.0;
    int b = 0;
    for (; b < kBins - 1 && s.count[b] < left; ++b) {
      left -= s.count[b];
      before += s.mass[b];
    }
    cut = find_cut(a, r, q, top, b, false, left, 0.0, 0.0, s);
    whole = before + cut.kept;
  }
  if (q.top_p < 1.0) {
    const double goal = q.top_p * whole;
    double before = 0.0;
    int b = 0;
    const int last = min(cut.bin, kBins - 1);
    for (; b < last && before + s.mass[b] < goal; ++b) before += s.mass[b];
    const Cut by_p = find_cut(a, r, q, top, b, true, 0, before, goal, s);
    // Both end at the same value: the fewer ties.  Otherwise top-p's is the higher one, but for roundings.
    if (by_p.bin < cut.bin || by_p.key > cut.key) cut = by_p;
    else if (by_p.key == cut.key) cut.ties = min(cut.ties, by_p.ties);
  }
  const int floor_bin = q.floor == -INFINITY ? kBins : bin_of(q.floor);
  const int edge = min(cut.bin, floor_bin);   // the only bin of which some tokens stay and some go
  // 1: stays, 2: stays while there are ties left.
  auto stays = [&](float v, double z) -> int {
    const int b = bin_of(z);
    if (b > edge) return 0;
    if (b < edge) return 1;
    if (z < q.floor) return 0;
    if (b < cut.bin) return 1;
    const uint32_t k = Key<T>::of(v);
    return k > cut.key ? 1 : k == cut.key ? 2 : 0;
  };
  const double tie_weight =
      cut.bin < kBins ? exp2_64(octaves(Key<T>::value(cut.key), top, q.to_octaves), s.table) : 0.0;

  // What stays of every part: the bins in front of the edge, and its own tokens of the edge, a wave per part.
  for (int p = wave; p < a.parts; p += 16) {
    double m = 0.0;
    uint32_t ties = 0;
    if (edge < kBins && count[p * kBins + edge] != 0) {
      const int c1 = min((p + 1) * r.per_part, r.chunks);
      for (int c = p * r.per_part + lane; c < c1; c += 64) {
        float v[E];
        const uint32_t in = r.load(c, v);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          if (!((in >> e) & 1)) continue;
          const double z = octaves(v[e], top, q.to_octaves);
          if (bin_of(z) != edge) continue;
          const int st = stays(v[e], z);
          if (st == 1) m += exp2_64(z, s.table);
          ties += st == 2;
        }
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) {
        m += __shfl_xor(m, o);
        ties += __shfl_xor(ties, o);
      }
    }
    for (int b = 0; b < min(edge, kBins); ++b) m += mass[p * kBins + b];
    if (lane == 0) {
      s.part_mass[p] = m;
      s.part_ties[p] = ties;
    }
  }
  __syncthreads();
  if (tid == 0) {
    uint32_t ties = 0;
    double all = 0.0;
    for (int p = 0; p < a.parts; ++p) {
      const uint32_t n = s.part_ties[p];
      const uint32_t kept = ties < cut.ties ? min(n, cut.ties - ties) : 0;
      s.part_ties[p] = ties;
      s.part_mass[p] += kept * tie_weight;
      ties += n;
      all += s.part_mass[p];
    }
    const double target = (double)a.uniform[row] * all;
    int part = 0;
    double run = 0.0, before = 0.0;
    for (int p = 0; p < a.parts; ++p) {
      if (!(s.part_mass[p] > 0.0)) continue;
      part = p;
      before = run;
      run += s.part_mass[p];
      if (run > target) break;
    }
    s.part = part;
    s.target = target - before;
    s.ties_before = s.part_ties[part];
  }
  __syncthreads();

  // The token inside the part: every thread a run of chunks, its mass, the sum of the threads in front of it.
  const int part = s.part;
  const double target = s.target;
  const int c0 = part * r.per_part, c1 = min(c0 + r.per_part, r.chunks);
  const int run = (c1 - c0 + kPickThreads - 1) / kPickThreads;
  const int t0 = min(c0 + tid * run, c1), t1 = min(t0 + run, c1);
  auto scan_n = [&](uint32_t n) {   // exclusive sum over the threads
    uint32_t x = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t u = __shfl_up(x, o);
      if (lane >= o) x += u;
    }
    __syncthreads();
    if (lane == 63) s.wave_n[wave] = x;
    __syncthreads();
    uint32_t base = 0;
    for (int w = 0; w < wave; ++w) base += s.wave_n[w];
    return base + x - n;
  };
  uint32_t my_ties = 0;
  if (cut.bin == edge && edge < kBins)
    for (int c = t0; c < t1; ++c) {
      float v[E];
      const uint32_t in = r.load(c, v);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if ((in >> e) & 1) my_ties += stays(v[e], octaves(v[e], top, q.to_octaves)) == 2;
    }
  const uint32_t ties0 = s.ties_before + scan_n(my_ties);
  double m = 0.0;
  uint32_t ties = ties0;
  for (int c = t0; c < t1; ++c) {
    float v[E];
    const uint32_t in = r.load(c, v);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (!((in >> e) & 1)) continue;
      const double z = octaves(v[e], top, q.to_octaves);
      const int st = stays(v[e], z);
      if (st == 1 || (st == 2 && ties++ < cut.ties)) m += exp2_64(z, s.table);
    }
  }
  double x = m;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double u = __shfl_up(x, o);
    if (lane >= o) x += u;
  }
  if (lane == 63) s.wave_d[wave] = x;
  __syncthreads();
  double base = 0.0;
  for (int w = 0; w < wave; ++w) base += s.wave_d[w];
  // The first token at which the running weight exceeds the target; failing that (roundings) the last that stays.
  double sum = base + (x - m);
  int hit = INT_MAX, last = -1;
  ties = ties0;
  for (int c = t0; c < t1; ++c) {
    float v[E];
    const uint32_t in = r.load(c, v);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (!((in >> e) & 1)) continue;
      const double z = octaves(v[e], top, q.to_octaves);
      const int st = stays(v[e], z);
      if (st == 1 || (st == 2 && ties++ < cut.ties)) {
        const double w = exp2_64(z, s.table);
        sum += w;
        if (w > 0.0) {
          last = r.index(c) + e;
          if (sum > target && hit == INT_MAX) hit = last;
        }
      }
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    hit = min(hit, __shfl_xor(hit, o));
    last = max(last, __shfl_xor(last, o));
  }
  __syncthreads();
  if (lane == 0) {
    s.wave_i[wave] = hit;
    s.wave_n[wave] = (uint32_t)last;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < 16; ++w) {
      hit = min(hit, s.wave_i[w]);
      last = max(last, (int)s.wave_n[w]);
    }
    a.tokens[row] = hit != INT_MAX ? hit : last;
  }
}

// Parts of a row: about four workgroups per compute unit over all rows, each
// with at least 4096 tokens.
int sample_parts(int64_t rows, int64_t vocab) {
  int64_t p = (1024 + rows - 1) / rows;
  const int64_t most = (vocab + 4095) / 4096;
  if (p > most) p = most;
  if (p > kMaxParts) p = kMaxParts;
  return (int)(p < 1 ? 1 : p);
}

constexpr size_t kPartBytes = sizeof(float2_t) + kBins * (sizeof(double) + sizeof(uint32_t));

int sample_check(int64_t rows, int64_t vocab) {
  WQ_REQUIRE(rows >= 0 && rows <= 65535, WQ_ERR_INVALID_ARGUMENT, "rows must be in [0, 65535] (got %lld)",
             (long long)rows);
  WQ_REQUIRE(vocab > 0 && vocab <= (1 << 30), WQ_ERR_INVALID_ARGUMENT, "vocab must be in [1, 2^30] (got %lld)",
             (long long)vocab);
  return WQ_OK;
}

template <typename T>
int launch_sample(const SampleArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)a.parts, (unsigned)a.rows);
  hipLaunchKernelGGL(sample_peak_kernel<T>, grid, dim3(256), 0, s, a);
  int rc = check_launch("sample_peak");
  if (rc != WQ_OK) return rc;
  hipLaunchKernelGGL(sample_tally_kernel<T>, grid, dim3(256), 0, s, a);
  rc = check_launch("sample_tally");
  if (rc != WQ_OK) return rc;
  hipLaunchKernelGGL(sample_pick_kernel<T>, dim3((unsigned)a.rows), dim3(kPickThreads), 0, s, a);
  return check_launch("sample_pick");
}

}  // namespace
}  // namespace wq

using namespace wq;

extern "C" int wq_sample_workspace_size(int64_t rows, int64_t vocab, size_t* bytes) {
  WQ_REQUIRE(bytes, WQ_ERR_INVALID_ARGUMENT, "null pointer argument");
  const int rc = sample_check(rows, vocab);
  if (rc != WQ_OK) return rc;
  *bytes = rows ? (size_t)rows * sample_parts(rows, vocab) * kPartBytes : 0;
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
  const size_t places = (size_t)rows * a.parts;
  WQ_REQUIRE(workspace && workspace_bytes >= places * kPartBytes && (uintptr_t)workspace % 8 == 0, WQ_ERR_WORKSPACE,
             "sampling needs an 8-byte aligned workspace of %zu bytes (got %zu)", places * kPartBytes, workspace_bytes);
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
  a.count = reinterpret_cast<uint32_t*>(a.mass + places * kBins);
  return logits_type == WQ_LOGITS_F16 ? launch_sample<half_t>(a, as_stream(stream))
                                      : launch_sample<float>(a, as_stream(stream));
}
