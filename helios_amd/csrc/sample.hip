// Drawing a token from each row of logits: temperature, top-k, top-p, min-p (gfx950).
//
// For row r with logits l, M their maximum, t the temperature, u the given number in [0, 1):
//   e_v = exp((l_v - M) / t), tokens in order of falling logit, equal ones by index
//   n_k = top_k (all without), S = sum of the first n_k weights
//   n_p = least n with  sum of the first n >= top_p S
//   n_m = number of tokens with e_v >= min_p
//   n = max(1, min(n_k, n_p, n_m)),  W = sum of the first n
//   token = the first in that order whose cumulative weight passes u W
// t <= 0: the first token in that order. The order makes every limit a prefix, and the drawn token
// a position: all are found in one histogram over the logits, without sorting the row.
//
// Weights are whole numbers round(e 2^44): their sums are exact, in any order, so no atomic's turn
// shows, and a cumulative weight next to a border is the same wherever it is computed. e comes
// from fp64 (the argument of exp loses 2^-24 of itself in fp32, more than a token's share of a flat
// row over 10^5 tokens).
//
// Two launches of many workgroups a row:
//   range  the row's largest and smallest logit, and the largest of each group of 32 tokens
//   row    rows of a small top_k: the k-th largest of the groups' maxima is a bound that the k first
//          tokens reach and few others do; the groups that reach it are read again and their tokens
//          listed. Other rows: counts and weights over 2048 bins of equal width between the extremes.
//          A row's last workgroup orders the list and draws, or finds the bins where the limits and
//          the drawn position fall, gathers their tokens and orders those.
// Bound by reading the logits from HBM, once (what is read again is in the last-level cache), and by
// the last workgroups' chain of steps. 96 rows of 151936 fp32 logits, top_k about 1000: 41 us, of
// which the first launch is 12; one bf16 row of them, top_k about 50: 18. (By the bins, in three
// launches: 115 and 31.) 96 rows without a top_k: 75 to 130 us, of which the fp64 weights of all
// tokens are 34 and each of the last workgroups' passes over its row 15.

#include "hx_common.h"

namespace {

constexpr int kBins = 2048;
constexpr int kList = 2048;      // tokens that the last launch orders at once
constexpr int kThreads = 256;    // of the first launch
constexpr int kRowThreads = 1024;  // and of the second
constexpr int kGroup = 32;       // tokens of a group
// A small top_k: of k tokens drawn at random over g groups the bound lets through about
// -g ln(1 - k / g) tokens, 1.22 k at k = g / 3; kList must hold them.
constexpr int kMostPicked = 1536;
constexpr int kFixed = 44;       // fraction bits of a weight
constexpr int kMostVocab = 1 << 18;
constexpr int kMostChunks = 64;

struct SampleArgs {
  const void* logits;
  int64_t row_stride;
  int32_t vocab;
  const float* uniforms;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int64_t* token_ids;
  float* logprobs;
  uint64_t* best;   // [rows][chunks]: the largest logit's order, and ~ of the first 16 bytes' token that hold it
  uint32_t* least;  // [rows][chunks]: the smallest finite logit's order
  uint32_t* count;  // [rows][kBins]
  uint64_t* mass;   // [rows][kBins]; or [rows][kList], the listed tokens of a row of a small top_k
  uint32_t* most;   // [rows][groups]: the order of a group's largest logit
  uint32_t* listed; // [rows][2]: tokens that a row of a small top_k lists, and its workgroups that are done
  int32_t groups;
  int32_t chunks, chunk;    // of the first launch, and their tokens
  int32_t chunks2, chunk2;  // of the second
};

template <typename T>
struct Logit {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float get(uint32_t w, int half) {
    return half ? hx::Elem<T>::hi(w) : hx::Elem<T>::lo(w);
  }
};
template <>
struct Logit<float> {
  static constexpr int kVec = 4;
};

// 16 bytes of logits, at any alignment: the hardware's loads take it.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Piece {
  uint32_t w[4];
  __device__ __forceinline__ float get(int e) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[e]);
    else return Logit<T>::get(w[e / 2], e & 1);
  }
  // No infinity or NaN: no exponent of ones, which one more would carry out of.
  __device__ __forceinline__ bool finite() const {
    constexpr uint32_t kExp = sizeof(T) == 4 ? 0x7f800000u : __is_same(T, _Float16) ? 0x7c007c00u : 0x7f807f80u;
    constexpr uint32_t kOne = sizeof(T) == 4 ? 0x00800000u : __is_same(T, _Float16) ? 0x04000400u : 0x00800080u;
    uint32_t carry = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) carry |= (w[i] & kExp) + kOne;
    return (carry & (sizeof(T) == 4 ? 0x80000000u : 0x80008000u)) == 0;
  }
  // f(logit, index from `at`) for each.
  template <typename F>
  __device__ __forceinline__ void each(int at, F f) const {
#pragma unroll
    for (int e = 0; e < Logit<T>::kVec; ++e) f(get(e), at + e);
  }
};

// Calls f(logit, index) for tokens [begin, end) of a row, spread over a workgroup's threads.
template <typename T, typename F>
__device__ __forceinline__ void each_logit(const void* row, int begin, int end, F f) {
  constexpr int kVec = Logit<T>::kVec, kAhead = 4;
  const T* const p = static_cast<const T*>(row);
  const int whole = (end - begin) / kVec;
  for (int j0 = hx::tid_x(); j0 < whole; j0 += kAhead * kRowThreads) {
    Piece<T> u[kAhead];  // in flight together
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      u[i] = *reinterpret_cast<const Piece<T>*>(p + begin + min(j0 + i * kRowThreads, whole - 1) * kVec);
    // (One copy of f's code, which is large: a workgroup's few turns cost less than fetching more.)
#pragma nounroll
    for (int j = j0; j < min(whole, j0 + kAhead * kRowThreads); j += kRowThreads) {
      u[0].each(begin + j * kVec, f);
#pragma unroll
      for (int i = 0; i + 1 < kAhead; ++i) u[i] = u[i + 1];
    }
  }
  const int v = begin + whole * kVec + hx::tid_x();
  if (v < end) f((float)p[v], v);
}

// A logit's place in the order of values: 0 and -0 alike, a NaN above all.
__device__ __forceinline__ uint32_t order_of(float l) {
  const uint32_t b = hx::raw_bits(l);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if ((b & 0x7fffffffu) == 0) return 0x80000000u;
  return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t order) {
  return __uint_as_float(order >> 31 ? order & 0x7fffffffu : ~order);
}
constexpr uint32_t kOrderInf = 0xff800000u;      // +inf; NaN above
constexpr uint32_t kOrderNegInf = 0x007fffffu;   // -inf

__device__ __forceinline__ uint64_t max_u64(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t shfl_xor_u64(uint64_t x, int m) {
  return (uint64_t)(uint32_t)__shfl_xor((int)(uint32_t)x, m) | (uint64_t)(uint32_t)__shfl_xor((int)(x >> 32), m) << 32;
}

// Whether a row goes by its groups' maxima.
__device__ __forceinline__ bool small_top_k(const SampleArgs& a, int64_t row) {
  const int k = a.top_k != nullptr ? a.top_k[row] : 0;
  return k > 0 && k <= kMostPicked && 3 * k <= a.groups;
}

// Largest of 2^n neighbouring lanes.
template <int LANES>
__device__ __forceinline__ uint32_t max_of_lanes(uint32_t x) {
  static_assert(LANES == 4 || LANES == 8);
  x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xb1, 0xf, 0xf, true));  // lane ^ 1
  x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4e, 0xf, 0xf, true));  // lane ^ 2
  if constexpr (LANES == 8) x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x141, 0xf, 0xf, true));  // 7 - lane
  return x;
}

// ---------------------------------------------------------------------------- extremes
template <typename T>
__global__ __launch_bounds__(kThreads) void sample_range_kernel(SampleArgs a) {
  __shared__ uint64_t s_best[kThreads / 64];
  __shared__ uint32_t s_least[kThreads / 64];
  const int64_t row = hx::wg_x() / a.chunks;
  const int c = hx::wg_x() % a.chunks, tid = hx::tid_x();
  if (!small_top_k(a, row)) {
    for (int b = c * kThreads + tid; b < kBins; b += a.chunks * kThreads) {
      a.count[row * kBins + b] = 0;
      a.mass[row * kBins + b] = 0;
    }
  }
  if (c == 0 && tid < 2) a.listed[2 * row + tid] = 0;
  constexpr int kVec = Logit<T>::kVec, kLanes = kGroup / kVec, kAhead = 4;
  uint32_t top = 0, at = 0;
  float least = INFINITY;
  const int begin = min(a.vocab, c * a.chunk), end = min(a.vocab, begin + a.chunk);
  const T* const p = static_cast<const T*>(a.logits) + row * a.row_stride;
  // Chunks begin with a group, and every thread of a group takes each turn. Finite pieces, most of all,
  // take a maximum and a minimum an element.
  for (int v0 = begin; v0 < end; v0 += kAhead * kThreads * kVec) {
    Piece<T> u[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int v = v0 + (i * kThreads + tid) * kVec;
      if (v + kVec <= end) u[i] = *reinterpret_cast<const Piece<T>*>(p + v);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int v = v0 + (i * kThreads + tid) * kVec;
      uint32_t here = 0;
      if (v + kVec <= end && u[i].finite()) {
        float most = u[i].get(0), fewest = most;
#pragma unroll
        for (int e = 1; e < kVec; ++e) {
          most = fmaxf(most, u[i].get(e));
          fewest = fminf(fewest, u[i].get(e));
        }
        here = order_of(most);
        least = fminf(least, fewest);
      } else {
#pragma nounroll
        for (int e = v; e < min(v + kVec, end); ++e) {
          const float l = (float)p[e];
          const uint32_t o = order_of(l);
          here = max(here, o);
          least = o > kOrderNegInf && o < kOrderInf ? fminf(least, l) : least;
        }
      }
      // Pieces come in rising order to a thread: the first of equal ones stays.
      at = here > top ? (uint32_t)v : at;
      top = max(top, here);
      here = max_of_lanes<kLanes>(here);
      if (tid % kLanes == 0 && v < end) a.most[row * a.groups + v / kGroup] = here;
    }
  }
  uint32_t low = order_of(least);
  uint64_t best = (uint64_t)top << 32 | (uint32_t)~at;
  for (int m = 1; m < 64; m <<= 1) {
    best = max_u64(best, shfl_xor_u64(best, m));
    low = min(low, (uint32_t)__shfl_xor((int)low, m));
  }
  if ((tid & 63) == 0) {
    s_best[tid >> 6] = best;
    s_least[tid >> 6] = low;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kThreads / 64; ++w) {
      best = max_u64(best, s_best[w]);
      low = min(low, s_least[w]);
    }
    a.best[row * a.chunks + c] = best;
    a.least[row * a.chunks + c] = low;
  }
}

// ----------------------------------------------------------------------- a row's measures
struct Row {
  uint64_t best;    // the largest logit's order, and ~ of the first piece's token that holds it
  float top;        // its logit
  bool drawn;       // a temperature, and a finite largest logit
  bool cut;         // the last bin's weights are all 0
  float per_bin;    // bins per unit of logit
  double scale;     // log2(e) / t
};

// By every thread of a workgroup, from the chunks' extremes.
__device__ __forceinline__ Row row_of(const SampleArgs& a, int64_t row) {
  const int lane = hx::tid_x() & 63;  // at most 64 chunks
  uint64_t best = lane < a.chunks ? a.best[row * a.chunks + lane] : 0;
  uint32_t low = lane < a.chunks ? a.least[row * a.chunks + lane] : 0xffffffffu;
  for (int m = 1; m < 64; m <<= 1) {
    best = max_u64(best, shfl_xor_u64(best, m));
    low = min(low, (uint32_t)__shfl_xor((int)low, m));
  }
  float t = a.temperature != nullptr ? a.temperature[row] : 1.f;
  const uint32_t order = (uint32_t)(best >> 32);
  Row r;
  r.best = best;
  r.top = logit_of(order);
  r.drawn = order > kOrderNegInf && order < kOrderInf && t > 0.f;
  r.cut = false;
  r.per_bin = 0.f;
  r.scale = 0.;
  if (r.drawn) {
    // Past these every weight is 0 or 1, but for logits 1e-30 apart or of 1e30: those get these temperatures.
    t = fminf(fmaxf(t, 1e-30f), 1e30f);
    // Weights below 2^-46 are 0: what lies lower is one bin.
    const float all = r.top - logit_of(low), range = fminf(all, 32.f * t);
    r.cut = all > range;
    r.per_bin = range > 0.f ? fminf((float)(kBins - 1) / range, 3e38f) : 0.f;
    r.scale = 1.4426950408889634074 / (double)t;
  }
  return r;
}

// Rises as the logit falls; kBins for -inf and where all weights are 0, whose tokens no limit and no
// drawn position needs.
__device__ __forceinline__ int bin_of(const Row& r, float l) {
  if (hx::raw_bits(l) == 0xff800000u) return kBins;
  const float x = (r.top - l) * r.per_bin;
  return x < (float)(kBins - 1) ? (int)x : r.cut ? kBins : kBins - 1;
}

// log2 of a weight, and the weight 2^y, y <= 0. The series leaves out x^12 / 12! and less, |x| <= ln 2 / 2:
// 9e-15 of the weight (2^-46.7); y's own roundings come to 2^-52 of the largest.
__device__ __forceinline__ double log_weight(const Row& r, float l) {
  return hx::raw_bits(l) == 0xff800000u ? -2000. : ((double)l - (double)r.top) * r.scale;
}
__device__ __forceinline__ double weight_of(double y) {
  if (!(y > -1000.)) return 0.;
  const double n = __builtin_rint(y), x = (y - n) * 0.69314718055994530942;
  double p = 1. / 39916800.;  // the exponential series
  p = fma(p, x, 1. / 3628800.);
  p = fma(p, x, 1. / 362880.);
  p = fma(p, x, 1. / 40320.);
  p = fma(p, x, 1. / 5040.);
  p = fma(p, x, 1. / 720.);
  p = fma(p, x, 1. / 120.);
  p = fma(p, x, 1. / 24.);
  p = fma(p, x, 1. / 6.);
  p = fma(p, x, 0.5);
  p = fma(p, x, 1.);
  p = fma(p, x, 1.);
  return __builtin_amdgcn_ldexp(p, (int)n);
}
// The weight as a whole number: e 2^44 added to 2^52 is rounded there, by at most 2^-45 of the largest.
// With the above a weight is within 2^-44.6 of the largest.
__device__ __forceinline__ uint64_t fixed_of(double e) {
  const double x = fma(e, (double)(1ull << kFixed), 4503599627370496.);
  return __builtin_bit_cast(uint64_t, x) & 0xfffffffffffffull;
}

// ------------------------------------------------------------------------ listed tokens
struct List {
  uint32_t bins[kBins];
  uint64_t list[kList];    // gathered tokens: order falling in the high half, index in the low
  uint64_t sorted[kList];
  uint64_t waves[kRowThreads / 64];
  uint32_t listed, crowd;
  // Weight up to and with a token of the sorted list: in the list's place once that is sorted.
  __device__ __forceinline__ uint64_t* cum() { return list; }
};

__device__ uint64_t block_sum(List& s, uint64_t x) {
  for (int m = 1; m < 64; m <<= 1) x += shfl_xor_u64(x, m);
  __syncthreads();
  if ((hx::tid_x() & 63) == 0) s.waves[hx::tid_x() >> 6] = x;
  __syncthreads();
  uint64_t all = 0;
#pragma unroll
  for (int w = 0; w < kRowThreads / 64; ++w) all += s.waves[w];
  return all;
}

// Sum over the threads before this one.
__device__ uint64_t block_before(List& s, uint64_t x) {
  const int lane = hx::tid_x() & 63;
  uint64_t sum = x;
  for (int m = 1; m < 64; m <<= 1) {
    const uint64_t y = (uint64_t)(uint32_t)__shfl_up((int)(uint32_t)sum, m) | (uint64_t)(uint32_t)__shfl_up((int)(sum >> 32), m) << 32;
    if (lane >= m) sum += y;
  }
  __syncthreads();
  if (lane == 63) s.waves[hx::tid_x() >> 6] = sum;
  __syncthreads();
  uint64_t before = sum - x;
#pragma unroll
  for (int w = 0; w < kRowThreads / 64; ++w) before += w < hx::tid_x() >> 6 ? s.waves[w] : 0;
  return before;
}

// First of the rising values p[0 .. n - 1] that is at least x; n if none is.
template <typename P, typename X>
__device__ __forceinline__ int first_from(const P* p, int n, X x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if ((X)p[mid] >= x) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

__device__ __forceinline__ uint64_t place_of(float l, int v) { return (uint64_t)(uint32_t)~order_of(l) << 32 | (uint32_t)v; }
__device__ __forceinline__ float place_logit(uint64_t place) { return logit_of(~(uint32_t)(place >> 32)); }

// Orders the n listed tokens and sums their weights onto `base`. By all threads. The tokens are of
// all bins, or of one bin alone.
__device__ void order_list(List& s, const Row& r, int n, uint64_t base, int one = -1) {
  constexpr int kEach = kList / kRowThreads, kBinsEach = kBins / kRowThreads;
  const int tid = hx::tid_x();
  __syncthreads();
  // Tokens to their bins' places (one bin's: parts of it), in any order; then a token's place is the
  // number of its bin's tokens before it. Lists with a crowded bin are sorted instead.
  for (int b = tid; b < kBins; b += kRowThreads) s.bins[b] = 0;
  if (tid == 0) s.crowd = 0;
  __syncthreads();
  uint64_t mine[kEach];
  int bin[kEach];
  uint32_t turn[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = tid + e * kRowThreads;
    if (i >= n) break;
    mine[e] = s.list[i];
    const float x = (r.top - place_logit(mine[e])) * r.per_bin;
    bin[e] = (int)fminf(one < 0 ? x : (x - (float)one) * (float)kBins, (float)(kBins - 1));
    turn[e] = atomicAdd(&s.bins[bin[e]], 1u);
  }
  __syncthreads();
  uint32_t here[kBinsEach], sum = 0, most = 0;
#pragma unroll
  for (int e = 0; e < kBinsEach; ++e) {
    here[e] = s.bins[kBinsEach * tid + e];
    most = max(most, here[e]);
    sum += here[e];
  }
  if (most > 256) s.crowd = 1;
  uint32_t before = (uint32_t)block_before(s, (uint64_t)sum);
#pragma unroll
  for (int e = 0; e < kBinsEach; ++e) {
    s.bins[kBinsEach * tid + e] = before;
    before += here[e];
  }
  __syncthreads();
  if (!s.crowd) {
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (tid + e * kRowThreads < n) s.list[s.bins[bin[e]] + turn[e]] = mine[e];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      if (tid + e * kRowThreads >= n) break;
      const int from = (int)s.bins[bin[e]], to = bin[e] + 1 < kBins ? (int)s.bins[bin[e] + 1] : n;
      int at = from;
      for (int i = from; i < to; ++i) at += s.list[i] < mine[e] ? 1 : 0;
      s.sorted[at] = mine[e];
    }
  } else {
    int size = 2;
    while (size < n) size <<= 1;
    for (int i = tid; i < size; i += kRowThreads) s.sorted[i] = i < n ? s.list[i] : ~0ull;
    for (int k = 2; k <= size; k <<= 1)
      for (int j = k >> 1; j > 0; j >>= 1) {
        __syncthreads();
        for (int pair = tid; pair < size / 2; pair += kRowThreads) {
          const int i = 2 * pair - (pair & (j - 1));
          const uint64_t x = s.sorted[i], y = s.sorted[i + j];
          if ((x > y) == ((i & k) == 0)) {
            s.sorted[i] = y;
            s.sorted[i + j] = x;
          }
        }
      }
  }
  __syncthreads();
  uint64_t w[kEach], all = 0;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = kEach * tid + e;
    w[e] = i < n ? fixed_of(weight_of(log_weight(r, place_logit(s.sorted[i])))) : 0;
    all += w[e];
  }
  uint64_t up_to = base + block_before(s, all);
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    up_to += w[e];
    s.cum()[kEach * tid + e] = up_to;
  }
  __syncthreads();
}

// ------------------------------------------------------------------------ a row's limits
struct Limits {
  bool limited, by_p, by_min;
  uint32_t k;
  double p, min_p, u;

  // Weights are whole: the first cumulative one above u W is the first above its whole part, which
  // rounding must not take to W. The weight to reach:
  __device__ __forceinline__ uint64_t target(uint64_t w) const {
    const uint64_t t = (uint64_t)(u * (double)w);
    return (t < w ? t : w - 1) + 1;
  }
};

__device__ __forceinline__ Limits limits_of(const SampleArgs& a, int64_t row) {
  Limits m;
  const int asked = a.top_k != nullptr ? a.top_k[row] : 0;
  m.limited = asked > 0 && asked < a.vocab;
  m.k = m.limited ? (uint32_t)asked : (uint32_t)a.vocab;
  const float top_p = a.top_p != nullptr ? a.top_p[row] : 1.f;
  m.by_p = top_p < 1.f;
  m.p = top_p > 0.f ? (double)top_p : 0.;
  m.min_p = a.min_p != nullptr ? (double)a.min_p[row] : 0.;
  m.by_min = m.min_p > 0.;
  const float given = a.uniforms[row];
  m.u = given > 0.f ? fmin((double)given, 1.) : 0.;
  return m;
}

// By one thread: the token, and its share of the kept weight.
__device__ __forceinline__ void answer(const SampleArgs& a, const Row& r, int64_t row, uint64_t place, uint64_t kept) {
  a.token_ids[row] = (int64_t)(uint32_t)place;
  if (a.logprobs != nullptr)
    a.logprobs[row] = (float)(log_weight(r, place_logit(place)) * 0.69314718055994530942 -
                              log((double)kept * (1. / (double)(1ull << kFixed))));
}

// Draws from a list that holds the row's first tokens, all that the limits can keep. `total` is the
// weight of the row where the limits need it (no top_k).
__device__ void draw_from(const SampleArgs& a, List& s, const Row& r, int64_t row, const Limits& m, int listed,
                          uint64_t total) {
  order_list(s, r, listed, 0);
  const uint64_t* const cum = s.cum();
  uint32_t n = min(m.k, (uint32_t)listed);
  if (m.by_p) {
    const uint64_t of = m.limited ? cum[n - 1] : total;
    n = min(n, (uint32_t)first_from(cum, listed, m.p * (double)of) + 1);
  }
  if (m.by_min) {
    uint64_t mine = 0;
    for (int i = hx::tid_x(); i < listed; i += kRowThreads) mine += weight_of(log_weight(r, place_logit(s.sorted[i]))) >= m.min_p ? 1 : 0;
    n = min(n, (uint32_t)block_sum(s, mine));
  }
  n = max(n, 1u);
  const uint64_t kept = !m.limited && !m.by_p && !m.by_min ? total : cum[n - 1];
  const int at = first_from(cum, listed, m.target(kept));
  if (hx::tid_x() == 0) answer(a, r, row, s.sorted[at], kept);
}

// ----------------------------------------------------------------- bounds and histograms
struct Bins {
  uint32_t count[kBins];
  unsigned long long mass[kBins];
};

// Counts and weights of a workgroup's tokens over the row's bins.
template <typename T>
__device__ void fill_bins(Bins& s, const Row& r, const void* row, int begin, int end) {
  for (int b = hx::tid_x(); b < kBins; b += kRowThreads) {
    s.count[b] = 0;
    s.mass[b] = 0;
  }
  __syncthreads();
  each_logit<T>(row, begin, end, [&](float l, int) {
    const int b = bin_of(r, l);
    if (b == kBins) return;
    atomicAdd(&s.count[b], 1u);
    const uint64_t w = fixed_of(weight_of(log_weight(r, l)));
    if (w) atomicAdd(&s.mass[b], (unsigned long long)w);
  });
  __syncthreads();
}

// The last bin of the bound: k groups have their largest logit in it or before it.
__device__ int bound_of(const SampleArgs& a, List& s, const Row& r, int64_t row, uint32_t k) {
  constexpr int kEach = kBins / kRowThreads, kAhead = 8;
  const int tid = hx::tid_x();
  for (int b = tid; b < kBins; b += kRowThreads) s.bins[b] = 0;
  if (tid == 0) s.crowd = kBins - 1;
  __syncthreads();
  for (int g0 = tid; g0 < a.groups; g0 += kAhead * kRowThreads) {
    uint32_t most[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) most[i] = g0 + i * kRowThreads < a.groups ? a.most[row * a.groups + g0 + i * kRowThreads] : kOrderNegInf;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int b = bin_of(r, logit_of(most[i]));
      if (b < kBins) atomicAdd(&s.bins[b], 1u);
    }
  }
  __syncthreads();
  uint32_t here[kEach], sum = 0;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    here[e] = s.bins[kEach * tid + e];
    sum += here[e];
  }
  uint32_t up_to = (uint32_t)block_before(s, (uint64_t)sum);
  if (up_to < k && up_to + sum >= k) {
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const bool here_it = up_to < k && up_to + here[e] >= k;
      up_to += here[e];
      if (here_it) s.crowd = kEach * tid + e;
    }
  }
  __syncthreads();
  return (int)s.crowd;
}

// Lists a workgroup's tokens within the row's bound.
template <typename T>
__device__ void pick(const SampleArgs& a, List& s, const Row& r, int64_t row, int begin, int end) {
  constexpr int kVec = Logit<T>::kVec, kLanes = kGroup / kVec;
  const int tid = hx::tid_x();
  const int bound = bound_of(a, s, r, row, (uint32_t)a.top_k[row]);
  static_assert(kMostVocab / kGroup * sizeof(uint16_t) <= sizeof(s.sorted));
  uint16_t* const reach = reinterpret_cast<uint16_t*>(s.sorted);  // the workgroup's groups that reach the bound
  __syncthreads();
  if (tid == 0) s.listed = s.crowd = 0;
  __syncthreads();
  const int g_end = (end + kGroup - 1) / kGroup;
  for (int g = begin / kGroup + tid; g < g_end; g += kRowThreads)
    if (bin_of(r, logit_of(a.most[row * a.groups + g])) <= bound) reach[atomicAdd(&s.crowd, 1u)] = (uint16_t)g;
  __syncthreads();
  const int groups = (int)s.crowd;
  const T* const p = static_cast<const T*>(a.logits) + row * a.row_stride;
  constexpr int kAhead = 4;
  for (int i0 = tid; i0 < groups * kLanes; i0 += kAhead * kRowThreads) {
    Piece<T> u[kAhead];  // in flight together
    int at[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int j = i0 + i * kRowThreads;
      at[i] = j < groups * kLanes ? reach[j / kLanes] * kGroup + j % kLanes * kVec : end;
      if (at[i] + kVec <= end) u[i] = *reinterpret_cast<const Piece<T>*>(p + at[i]);
    }
    auto take = [&](float l, int v) __attribute__((always_inline)) {
      if (bin_of(r, l) > bound) return;
      const uint32_t to = atomicAdd(&s.listed, 1u);
      if (to < (uint32_t)kList) s.list[to] = place_of(l, v);
    };
#pragma nounroll
    for (int i = 0; i < kAhead; ++i) {
      if (at[0] + kVec <= end) {
        u[0].each(at[0], take);
      } else {
#pragma nounroll
        for (int e = at[0]; e < end; ++e) take((float)p[e], e);
      }
#pragma unroll
      for (int k = 0; k + 1 < kAhead; ++k) {
        u[k] = u[k + 1];
        at[k] = at[k + 1];
      }
    }
  }
  __syncthreads();
  const uint32_t mine = s.listed;
  __syncthreads();
  if (tid == 0) s.crowd = mine ? atomicAdd(&a.listed[2 * row], mine) : 0;
  __syncthreads();
  const uint32_t base = s.crowd;
  static_assert(kList <= kBins);
  uint64_t* const list = a.mass + row * kBins;
  for (uint32_t i = tid; i < min(mine, (uint32_t)kList) && base + i < (uint32_t)kList; i += kRowThreads)
    __hip_atomic_store(&list[base + i], s.list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ---------------------------------------------------------------------------- the row
struct RowLds : List {
  Bins to;  // tokens up to and with a bin, and their weight
  uint32_t digit_count[256];
  unsigned long long digit_mass[256];
};

// Lists the row's tokens of the bins [first, last] that `take` says, at most kList. By all threads;
// their number. One test of 16 bytes' tokens comes before the tokens' own: few are of the bins.
template <typename T, typename F>
__device__ int gather(const SampleArgs& a, RowLds& s, const Row& r, const void* row, int first, int last, F take) {
  constexpr int kVec = Logit<T>::kVec, kAhead = 4;
  __syncthreads();
  if (hx::tid_x() == 0) s.listed = 0;
  __syncthreads();
  // (An infinite x, or NaN from an infinite distance and bins of no width, becomes 3.4e38: in no bin.)
  const float from = (float)first, to = last < kBins - 1 ? (float)(last + 1) : r.cut ? (float)(kBins - 1) : 3.4e38f;
  auto within = [&](float l) __attribute__((always_inline)) {
    const float x = fminf((r.top - l) * r.per_bin, 3.4e38f);
    return x >= from && x < to;
  };
  auto list = [&](float l, int v) __attribute__((always_inline)) {
    if (!within(l) || !take(place_of(l, v))) return;
    const uint32_t at = atomicAdd(&s.listed, 1u);
    if (at < (uint32_t)kList) s.list[at] = place_of(l, v);
  };
  const T* const p = static_cast<const T*>(row);
  const int whole = a.vocab / kVec;
  for (int j0 = hx::tid_x(); j0 < whole; j0 += kAhead * kRowThreads) {
    Piece<T> u[kAhead];  // in flight together
#pragma unroll
    for (int i = 0; i < kAhead; ++i) u[i] = *reinterpret_cast<const Piece<T>*>(p + min(j0 + i * kRowThreads, whole - 1) * kVec);
#pragma nounroll
    for (int j = j0; j < min(whole, j0 + kAhead * kRowThreads); j += kRowThreads) {
      bool any = false;
#pragma unroll
      for (int e = 0; e < kVec; ++e) any |= within(u[0].get(e));
      if (any) u[0].each(j * kVec, list);
#pragma unroll
      for (int i = 0; i + 1 < kAhead; ++i) u[i] = u[i + 1];
    }
  }
  const int v = whole * kVec + hx::tid_x();
  if (v < a.vocab) list((float)p[v], v);
  __syncthreads();
  return min((int)s.listed, kList);
}

// Finds, in one bin, the position where the count or the weight reaches a target (counted from the
// row's first token): fills the sorted list with tokens around it; how many, and how many tokens of
// the row come before them. A bin of more than kList tokens is narrowed down by digits of their
// places first.
struct Found {
  int n;
  uint32_t before;
};
template <typename T>
__device__ Found resolve(const SampleArgs& a, RowLds& s, const Row& r, const void* row, int bin, bool by_count, uint64_t target) {
  const int tid = hx::tid_x();
  uint32_t before = bin ? s.to.count[bin - 1] : 0;
  uint64_t mass = bin ? s.to.mass[bin - 1] : 0;
  uint32_t size = s.to.count[bin] - before;
  int shift = 64;
  uint64_t prefix = 0;
  while (size > (uint32_t)kList && shift > 0) {
    const int from = shift;
    shift -= 8;
    __syncthreads();
    if (tid < 256) {
      s.digit_count[tid] = 0;
      s.digit_mass[tid] = 0;
    }
    __syncthreads();
    each_logit<T>(row, 0, a.vocab, [&](float l, int v) {
      if (bin_of(r, l) != bin) return;
      const uint64_t p = place_of(l, v);
      if (from < 64 && (p >> from) != prefix) return;
      const int d = (int)(p >> shift) & 255;
      atomicAdd(&s.digit_count[d], 1u);
      atomicAdd(&s.digit_mass[d], (unsigned long long)fixed_of(weight_of(log_weight(r, l))));
    });
    __syncthreads();
    // The first digit that reaches the target; the last with a token if none does.
    int at = 0;
    uint32_t count_here = 0, count_before = before;
    uint64_t mass_before = mass;
    for (int d = 0; d < 256; ++d) {
      const uint32_t c = s.digit_count[d];
      if (!c) continue;
      const uint64_t m = s.digit_mass[d];
      at = d;
      count_here = c;
      if (by_count ? count_before + c >= target : mass_before + m >= target) break;
      count_before += c;
      mass_before += m;
    }
    if (count_before == before + size) {  // none reached it: the last one then
      count_before -= count_here;
      mass_before -= s.digit_mass[at];
    }
    before = count_before;
    mass = mass_before;
    size = count_here;
    prefix = from < 64 ? prefix << 8 | (uint64_t)at : (uint64_t)at;
  }
  const int n = gather<T>(a, s, r, row, bin, bin, [&](uint64_t place) { return shift == 64 || place >> shift == prefix; });
  order_list(s, r, n, mass, bin);
  return {n, before};
}

// Draws from a row by its bins: lists the tokens that the limits can keep, if a list holds them; their
// number. If not, draws, and returns 0.
template <typename T>
__device__ int draw_by_bins(const SampleArgs& a, RowLds& s, const Row& r, int64_t row, const Limits& m, bool picked) {
  const int tid = hx::tid_x();
  const void* const logits = static_cast<const T*>(a.logits) + row * a.row_stride;
  if (!picked) {
    for (int b = tid; b < kBins; b += kRowThreads) {
      s.to.count[b] = __hip_atomic_load(&a.count[row * kBins + b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      s.to.mass[b] = __hip_atomic_load(&a.mass[row * kBins + b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
  }
  {
    // Prefix sums over the bins, two a thread.
    static_assert(kBins == 2 * kRowThreads);
    const uint32_t c0 = s.to.count[2 * tid], c1 = s.to.count[2 * tid + 1];
    const uint64_t m0 = s.to.mass[2 * tid], m1 = s.to.mass[2 * tid + 1];
    const uint32_t c = (uint32_t)block_before(s, (uint64_t)c0 + c1);
    const uint64_t m = block_before(s, m0 + m1);
    s.to.count[2 * tid] = c + c0;
    s.to.count[2 * tid + 1] = c + c0 + c1;
    s.to.mass[2 * tid] = m + m0;
    s.to.mass[2 * tid + 1] = m + m0 + m1;
  }
  __syncthreads();
  const uint32_t nk = min(m.k, s.to.count[kBins - 1]);
  const int bin_k = first_from(s.to.count, kBins, nk);
  // No kept token lies in a bin past `last`.
  int last = bin_k;
  if (m.by_p) last = min(last, first_from(s.to.mass, kBins, m.p * (double)s.to.mass[bin_k]));
  if (m.by_min) {
    // How far below the largest logit the border lies, and two bins more for what is rounded.
    const float x = -logf((float)m.min_p) * (float)(1.4426950408889634074 / r.scale) * r.per_bin * 1.00001f;
    last = min(last, x < (float)(kBins - 3) ? max((int)x, 0) + 2 : kBins - 1);
  }
  const int until = m.limited && m.by_p ? bin_k : last;  // the top_k tokens' weight needs all of them
  if (s.to.count[until] <= (uint32_t)kList) return gather<T>(a, s, r, logits, 0, until, [](uint64_t) { return true; });
  uint32_t n = nk;
  uint64_t kept = s.to.mass[kBins - 1], of = kept;
  const uint64_t* const cum = s.cum();
  auto fewest = [&](uint32_t fewer, uint64_t w) __attribute__((always_inline)) {
    if (fewer < n) {
      n = fewer;
      kept = w;
    }
  };
  // The borders of top_k and of top_p, then the drawn token.
#pragma nounroll
  for (int step = m.limited ? 0 : m.by_p ? 1 : 2; step < 3; step += step == 0 && !m.by_p ? 2 : 1) {
    if (step == 2 && m.by_min) {
      uint64_t count = 0, mass = 0;
      each_logit<T>(logits, 0, a.vocab, [&](float l, int) {
        const double e = weight_of(log_weight(r, l));
        if (e >= m.min_p) {
          ++count;
          mass += fixed_of(e);
        }
      });
      count = block_sum(s, count);
      mass = block_sum(s, mass);
      // (None reaches a min_p above 1: the first token stays, whose weight is 1.)
      fewest(max((uint32_t)count, 1u), count ? mass : 1ull << kFixed);
    }
    const double border = m.p * (double)of;
    const uint64_t target = step == 0 ? nk : step == 2 ? m.target(kept) : (uint64_t)border + ((double)(uint64_t)border < border ? 1 : 0);
    const int bin = step == 0 ? bin_k : min(first_from(s.to.mass, kBins, target), kBins - 1);
    const Found f = resolve<T>(a, s, r, logits, bin, step == 0, target);
    if (step == 0) {
      kept = of = cum[nk - f.before - 1];
    } else {
      const int i = min(first_from(cum, f.n, target), f.n - 1);
      if (step == 1) fewest(f.before + (uint32_t)i + 1, cum[i]);
      else if (tid == 0) answer(a, r, row, s.sorted[i], kept);
    }
    __syncthreads();
  }
  return 0;
}

// Whether this workgroup is the row's last, which draws. What the others gave it went past the caches,
// each wave waits until it has arrived, and the last one reads it past the caches too: none need be
// written back or emptied (which took 5 us over 96 rows).
__device__ __forceinline__ bool count_done(const SampleArgs& a, RowLds& s, int64_t row) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (hx::tid_x() == 0)
    s.crowd = __hip_atomic_fetch_add(&a.listed[2 * row + 1], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  return s.crowd == (uint32_t)a.chunks2 - 1;
}

template <typename T>
__global__ __launch_bounds__(kRowThreads) void sample_row_kernel(SampleArgs a) {
  __shared__ RowLds s;
  const int64_t row = hx::wg_x() / a.chunks2;
  const int c = hx::wg_x() % a.chunks2, tid = hx::tid_x();
  const Row r = row_of(a, row);
  if (!r.drawn) {
    // The first token in order; none in a row of -inf alone.
    if (c == 0 && tid == 0) {
      const uint32_t order = (uint32_t)(r.best >> 32);
      const bool any = order > kOrderNegInf;
      const T* const p = static_cast<const T*>(a.logits) + row * a.row_stride;
      int v = (int)~(uint32_t)r.best;
      while (any && v < a.vocab - 1 && order_of((float)p[v]) != order) ++v;
      a.token_ids[row] = any ? v : -1;
      if (a.logprobs != nullptr) a.logprobs[row] = any ? 0.f : -INFINITY;
    }
    return;
  }
  const int begin = min(a.vocab, c * a.chunk2), end = min(a.vocab, begin + a.chunk2);
  const void* const logits = static_cast<const T*>(a.logits) + row * a.row_stride;
  const bool picked = small_top_k(a, row);
  uint32_t listed = 0;
  if (picked) {
    pick<T>(a, s, r, row, begin, end);
    if (!count_done(a, s, row)) return;
    listed = __hip_atomic_load(&a.listed[2 * row], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (uint32_t i = tid; i < listed && listed <= (uint32_t)kList; i += kRowThreads)
      s.list[i] = __hip_atomic_load(&a.mass[row * kBins + i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  const bool whole = listed > 0 && listed <= (uint32_t)kList;  // (a small top_k lists a token at least)
  const Limits m = limits_of(a, row);
  uint64_t total = 0;
  if (!whole) {
    fill_bins<T>(s.to, r, logits, picked ? 0 : begin, picked ? a.vocab : end);
    if (!picked) {
      for (int b = tid; b < kBins; b += kRowThreads) {
        if (!s.to.count[b]) continue;
        atomicAdd(&a.count[row * kBins + b], s.to.count[b]);
        if (s.to.mass[b]) atomicAdd(reinterpret_cast<unsigned long long*>(&a.mass[row * kBins + b]), s.to.mass[b]);
      }
      if (!count_done(a, s, row)) return;
    }
    listed = (uint32_t)draw_by_bins<T>(a, s, r, row, m, picked);
    if (!listed) return;
    total = s.to.mass[kBins - 1];
  }
  draw_from(a, s, r, row, m, (int)listed, total);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Chunks of a row, for about `wgs` workgroups in all, of at least 2048 tokens.
void cut(int64_t rows, int32_t vocab, int64_t wgs, int32_t* chunks, int32_t* chunk) {
  int64_t n = wgs / rows;
  n = n < 1 ? 1 : n > kMostChunks ? kMostChunks : n;
  int64_t each = ceil_div(ceil_div(vocab, n), 2048) * 2048;
  *chunk = (int32_t)each;
  *chunks = (int32_t)ceil_div(vocab, each);
}

template <typename T>
void launch(const SampleArgs& a, int64_t rows, hipStream_t s) {
  hipLaunchKernelGGL(sample_range_kernel<T>, dim3((unsigned)(rows * a.chunks)), dim3(kThreads), 0, s, a);
  hipLaunchKernelGGL(sample_row_kernel<T>, dim3((unsigned)(rows * a.chunks2)), dim3(kRowThreads), 0, s, a);
}

}  // namespace

extern "C" size_t hx_sample_workspace_bytes(int64_t rows, int64_t vocab) {
  if (rows < 1 || vocab < 1 || vocab > kMostVocab || rows > (1 << 20)) return 0;
  return (size_t)rows * ((kMostChunks + kBins) * (sizeof(uint64_t) + sizeof(uint32_t)) +
                         (size_t)(ceil_div(vocab, kGroup) + 2) * sizeof(uint32_t));
}

extern "C" int hx_sample_tokens(const void* logits, int64_t logits_row_stride, int64_t rows, int64_t vocab, int32_t dtype,
                                const float* uniforms, const float* temperature, const int32_t* top_k, const float* top_p,
                                const float* min_p, int64_t* token_ids, float* logprobs, void* workspace,
                                size_t workspace_bytes, void* stream) {
  if (dtype != HX_DTYPE_BF16 && dtype != HX_DTYPE_FP16 && dtype != HX_DTYPE_FP32) return HX_E_UNSUPPORTED;
  if (rows < 0 || vocab < 1 || (rows > 1 && logits_row_stride < vocab)) return HX_E_INVALID_ARG;
  if (rows == 0) return HX_OK;
  if (vocab > kMostVocab || rows > (1 << 20)) return HX_E_UNSUPPORTED;
  const uintptr_t size = dtype == HX_DTYPE_FP32 ? 4 : 2;
  if (!logits || !uniforms || !token_ids || (reinterpret_cast<uintptr_t>(logits) & (size - 1))) return HX_E_INVALID_ARG;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 7) || workspace_bytes < hx_sample_workspace_bytes(rows, vocab))
    return HX_E_WORKSPACE;
  SampleArgs a;
  a.logits = logits;
  a.row_stride = logits_row_stride;
  a.vocab = (int32_t)vocab;
  a.uniforms = uniforms;
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.token_ids = token_ids;
  a.logprobs = logprobs;
  a.best = static_cast<uint64_t*>(workspace);
  a.mass = a.best + rows * kMostChunks;
  a.least = reinterpret_cast<uint32_t*>(a.mass + rows * kBins);
  a.count = a.least + rows * kMostChunks;
  a.listed = a.count + rows * kBins;
  a.most = a.listed + rows * 2;
  a.groups = (int32_t)ceil_div(vocab, kGroup);
  cut(rows, a.vocab, 2048, &a.chunks, &a.chunk);
  cut(rows, a.vocab, 256, &a.chunks2, &a.chunk2);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == HX_DTYPE_BF16) launch<__bf16>(a, rows, s);
  else if (dtype == HX_DTYPE_FP16) launch<_Float16>(a, rows, s);
  else launch<float>(a, rows, s);
  return hx::status_from_hip(hipGetLastError());
}
