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
// Three launches: the rows' largest and smallest logits (many workgroups a row), the histogram of
// counts and weights over 2048 bins of equal width between them (many workgroups a row), and a
// workgroup a row that finds the bins where the limits and the drawn position fall, gathers their
// tokens and orders those. Bound by reading the logits three times, of which HBM sees the first.

#include "hx_common.h"

namespace {

constexpr int kBins = 2048;
constexpr int kList = 2048;      // tokens that the last launch orders at once
constexpr int kThreads = 256;    // of the first two launches
constexpr int kRowThreads = 1024;
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
  uint64_t* best;   // [rows][chunks]: the first token in order
  uint32_t* least;  // [rows][chunks]: the smallest finite logit's order
  uint32_t* count;  // [rows][kBins]
  uint64_t* mass;   // [rows][kBins]
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

// Calls f(logit, index) for tokens [begin, end) of a row, spread over a workgroup's threads, 16
// bytes at a time (at any alignment: the hardware's loads take it).
template <typename T, int THREADS, typename F>
__device__ __forceinline__ void each_logit(const void* row, int begin, int end, F f) {
  struct __attribute__((packed, aligned(sizeof(T)))) Piece {
    uint32_t w[4];
  };
  constexpr int kVec = Logit<T>::kVec;
  const T* const p = static_cast<const T*>(row);
  const int whole = (end - begin) / kVec;
  for (int j = hx::tid_x(); j < whole; j += THREADS) {
    const Piece u = *reinterpret_cast<const Piece*>(p + begin + j * kVec);
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      if constexpr (sizeof(T) == 4) f(__uint_as_float(u.w[e]), begin + j * kVec + e);
      else f(Logit<T>::get(u.w[e / 2], e & 1), begin + j * kVec + e);
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

// ---------------------------------------------------------------------------- extremes
template <typename T>
__global__ __launch_bounds__(kThreads) void sample_range_kernel(SampleArgs a) {
  __shared__ uint64_t s_best[kThreads / 64];
  __shared__ uint32_t s_least[kThreads / 64];
  const int64_t row = hx::wg_x() / a.chunks;
  const int c = hx::wg_x() % a.chunks, tid = hx::tid_x();
  for (int b = c * kThreads + tid; b < kBins; b += a.chunks * kThreads) {
    a.count[row * kBins + b] = 0;
    a.mass[row * kBins + b] = 0;
  }
  uint32_t top = 0, at = 0xffffffffu, low = 0xffffffffu;
  const int begin = min(a.vocab, c * a.chunk), end = min(a.vocab, begin + a.chunk);
  each_logit<T, kThreads>(static_cast<const T*>(a.logits) + row * a.row_stride, begin, end, [&](float l, int v) {
    const uint32_t o = order_of(l);
    // Tokens come in rising order to a thread: the first of equal ones stays.
    at = o > top ? (uint32_t)v : at;
    top = o > top ? o : top;
    low = o > kOrderNegInf && o < low ? o : low;
  });
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
  uint64_t best;    // the first token in order
  float top;        // its logit
  bool drawn;       // a temperature, and a finite largest logit
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
  r.per_bin = 0.f;
  r.scale = 0.;
  if (r.drawn) {
    t = fminf(fmaxf(t, 1e-30f), 1e30f);  // past these every weight is 0 or 1 already
    // Weights below 2^-46 are 0: what lies lower is one bin.
    const float range = fminf(r.top - logit_of(low), 32.f * t);
    r.per_bin = range > 0.f ? fminf((float)(kBins - 1) / range, 3e38f) : 0.f;
    r.scale = 1.4426950408889634074 / (double)t;
  }
  return r;
}

// Rises as the logit falls.
__device__ __forceinline__ int bin_of(const Row& r, float l) {
  const float d = r.top - l;
  const float x = d > 3e38f ? (float)kBins : d * r.per_bin;  // (-inf where all finite logits are equal: not inf * 0)
  return x < (float)(kBins - 1) ? (int)x : kBins - 1;
}

// log2 of a weight, and the weight 2^y, y <= 0, to about 1e-13 of itself.
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
// The weight as a whole number: e 2^44 added to 2^52 is rounded there.
__device__ __forceinline__ uint64_t fixed_of(double e) {
  const double x = fma(e, (double)(1ull << kFixed), 4503599627370496.);
  return __builtin_bit_cast(uint64_t, x) & 0xfffffffffffffull;
}

// --------------------------------------------------------------------------- histogram
template <typename T>
__global__ __launch_bounds__(kThreads) void sample_bins_kernel(SampleArgs a) {
  __shared__ uint32_t s_count[kBins];
  __shared__ unsigned long long s_mass[kBins];
  const int64_t row = hx::wg_x() / a.chunks2;
  const int c = hx::wg_x() % a.chunks2, tid = hx::tid_x();
  const Row r = row_of(a, row);
  if (!r.drawn) return;
  for (int b = tid; b < kBins; b += kThreads) {
    s_count[b] = 0;
    s_mass[b] = 0;
  }
  __syncthreads();
  const int begin = min(a.vocab, c * a.chunk2), end = min(a.vocab, begin + a.chunk2);
  each_logit<T, kThreads>(static_cast<const T*>(a.logits) + row * a.row_stride, begin, end, [&](float l, int) {
    const int b = bin_of(r, l);
    atomicAdd(&s_count[b], 1u);
    atomicAdd(&s_mass[b], (unsigned long long)fixed_of(weight_of(log_weight(r, l))));
  });
  __syncthreads();
  for (int b = tid; b < kBins; b += kThreads) {
    if (!s_count[b]) continue;
    atomicAdd(&a.count[row * kBins + b], s_count[b]);
    if (s_mass[b]) atomicAdd(reinterpret_cast<unsigned long long*>(&a.mass[row * kBins + b]), s_mass[b]);
  }
}

// ---------------------------------------------------------------------------- the row
struct RowLds {
  uint32_t count[kBins];  // tokens up to and with a bin
  uint64_t mass[kBins];   // their weight
  uint64_t list[kList];   // gathered tokens: order falling in the high half, index in the low
  uint64_t sorted[kList];
  uint64_t cum[kList];    // weight up to and with a token of the sorted list
  uint32_t digit_count[256];
  unsigned long long digit_mass[256];
  uint64_t waves[kRowThreads / 64];
  uint32_t listed;
};

__device__ uint64_t block_sum(RowLds& s, uint64_t x) {
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
__device__ uint64_t block_before(RowLds& s, uint64_t x) {
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
  for (int w = 0; w < hx::tid_x() >> 6; ++w) before += s.waves[w];
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

// Orders the n listed tokens and sums their weights onto `base`. By all threads.
__device__ void order_list(RowLds& s, const Row& r, int n, uint64_t base) {
  const int tid = hx::tid_x();
  __syncthreads();
  if (n <= kRowThreads) {
    // A token's place is the number of those before it.
    if (tid < n) {
      const uint64_t mine = s.list[tid];
      int before = 0;
      for (int i = 0; i < n; ++i) before += s.list[i] < mine ? 1 : 0;
      s.sorted[before] = mine;
    }
  } else {
    int size = 2 * kRowThreads;
    static_assert(kList == 2 * kRowThreads, "two of a list to a thread");
    for (int i = tid; i < size; i += kRowThreads) s.sorted[i] = i < n ? s.list[i] : ~0ull;
    for (int k = 2; k <= size; k <<= 1)
      for (int j = k >> 1; j > 0; j >>= 1) {
        __syncthreads();
        const int i = (tid / j) * 2 * j + tid % j;
        const uint64_t x = s.sorted[i], y = s.sorted[i + j];
        if ((x > y) == ((i & k) == 0)) {
          s.sorted[i] = y;
          s.sorted[i + j] = x;
        }
      }
  }
  __syncthreads();
  uint64_t w[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = 2 * tid + e;
    w[e] = i < n ? fixed_of(weight_of(log_weight(r, place_logit(s.sorted[i])))) : 0;
  }
  const uint64_t before = base + block_before(s, w[0] + w[1]);
  s.cum[2 * tid] = before + w[0];
  s.cum[2 * tid + 1] = before + w[0] + w[1];
  __syncthreads();
}

// Lists the row's tokens that `take` says, at most kList. By all threads; their number.
template <typename T, typename F>
__device__ int gather(const SampleArgs& a, RowLds& s, const void* row, F take) {
  __syncthreads();
  if (hx::tid_x() == 0) s.listed = 0;
  __syncthreads();
  each_logit<T, kRowThreads>(row, 0, a.vocab, [&](float l, int v) {
    if (take(l, v)) {
      const uint32_t at = atomicAdd(&s.listed, 1u);
      if (at < (uint32_t)kList) s.list[at] = place_of(l, v);
    }
  });
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
  uint32_t before = bin ? s.count[bin - 1] : 0;
  uint64_t mass = bin ? s.mass[bin - 1] : 0;
  uint32_t size = s.count[bin] - before;
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
    each_logit<T, kRowThreads>(row, 0, a.vocab, [&](float l, int v) {
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
  const int n = gather<T>(a, s, row, [&](float l, int v) {
    return bin_of(r, l) == bin && (shift == 64 || (place_of(l, v) >> shift) == prefix);
  });
  order_list(s, r, n, mass);
  return {n, before};
}

template <typename T>
__global__ __launch_bounds__(kRowThreads) void sample_row_kernel(SampleArgs a) {
  __shared__ RowLds s;
  const int64_t row = hx::wg_x();
  const int tid = hx::tid_x();
  const Row r = row_of(a, row);
  if (!r.drawn) {
    // The first token in order; none in a row of -inf alone.
    if (tid == 0) {
      const bool any = (uint32_t)(r.best >> 32) > kOrderNegInf;
      a.token_ids[row] = any ? (int64_t)(uint32_t)~(uint32_t)r.best : -1;
      if (a.logprobs != nullptr) a.logprobs[row] = any ? 0.f : -INFINITY;
    }
    return;
  }
  const void* const logits = static_cast<const T*>(a.logits) + row * a.row_stride;
  {
    // Prefix sums over the bins, two a thread.
    const uint32_t c0 = a.count[row * kBins + 2 * tid], c1 = a.count[row * kBins + 2 * tid + 1];
    const uint64_t m0 = a.mass[row * kBins + 2 * tid], m1 = a.mass[row * kBins + 2 * tid + 1];
    const uint32_t c = (uint32_t)block_before(s, (uint64_t)c0 + c1);
    const uint64_t m = block_before(s, m0 + m1);
    s.count[2 * tid] = c + c0;
    s.count[2 * tid + 1] = c + c0 + c1;
    s.mass[2 * tid] = m + m0;
    s.mass[2 * tid + 1] = m + m0 + m1;
  }
  __syncthreads();
  const int asked = a.top_k != nullptr ? a.top_k[row] : 0;
  const bool limited = asked > 0 && asked < a.vocab;
  const uint32_t nk = limited ? (uint32_t)asked : (uint32_t)a.vocab;
  const float top_p = a.top_p != nullptr ? a.top_p[row] : 1.f;
  const bool by_p = top_p < 1.f;
  const double p = top_p > 0.f ? (double)top_p : 0.;
  const double min_p = a.min_p != nullptr ? (double)a.min_p[row] : 0.;
  const bool by_min = min_p > 0.;
  const float given = a.uniforms[row];
  const double u = given > 0.f ? fmin((double)given, 1.) : 0.;

  const int bin_k = first_from(s.count, kBins, nk);
  // No kept token lies in a bin past `last`.
  int last = bin_k;
  if (by_p) last = min(last, first_from(s.mass, kBins, p * (double)s.mass[bin_k]));
  if (by_min) {
    // How far below the largest logit the border lies, and two bins more for what is rounded.
    const float x = -logf((float)min_p) * (float)(1.4426950408889634074 / r.scale) * r.per_bin * 1.00001f;
    last = min(last, x < (float)(kBins - 3) ? max((int)x, 0) + 2 : kBins - 1);
  }
  const int until = limited && by_p ? bin_k : last;  // the top_k tokens' weight needs all of them
  uint32_t n;
  uint64_t kept;
  int at;
  auto fewest = [&](uint32_t m, uint64_t w) __attribute__((always_inline)) {
    if (m < n) {
      n = m;
      kept = w;
    }
  };
  auto target_of = [&](uint64_t w) __attribute__((always_inline)) {
    // Weights are whole: the first cumulative one above u W is the first above its whole part,
    // which rounding must not take to W.
    const uint64_t t = (uint64_t)(u * (double)w);
    return t < w ? t : w - 1;
  };
  if (s.count[until] <= (uint32_t)kList) {
    const int listed = gather<T>(a, s, logits, [&](float l, int) { return bin_of(r, l) <= until; });
    order_list(s, r, listed, 0);
    n = min(nk, (uint32_t)listed);
    if (by_p) {
      const uint64_t of = limited ? s.cum[n - 1] : s.mass[kBins - 1];
      n = min(n, (uint32_t)first_from(s.cum, listed, p * (double)of) + 1);
    }
    if (by_min) {
      uint64_t mine = 0;
      for (int i = tid; i < listed; i += kRowThreads) mine += weight_of(log_weight(r, place_logit(s.sorted[i]))) >= min_p ? 1 : 0;
      n = min(n, (uint32_t)block_sum(s, mine));
    }
    n = max(n, 1u);
    kept = !limited && !by_p && !by_min ? s.mass[kBins - 1] : s.cum[n - 1];
    at = first_from(s.cum, listed, target_of(kept) + 1);
  } else {
    n = (uint32_t)a.vocab;
    kept = s.mass[kBins - 1];
    uint64_t of = kept;
    if (limited) {
      const Found f = resolve<T>(a, s, r, logits, bin_k, true, nk);
      of = s.cum[nk - f.before - 1];
      fewest(nk, of);
      __syncthreads();
    }
    if (by_p) {
      const double border = p * (double)of;
      const int bin = min(first_from(s.mass, kBins, border), kBins - 1);
      const uint64_t whole = (uint64_t)border + ((double)(uint64_t)border < border ? 1 : 0);
      const Found f = resolve<T>(a, s, r, logits, bin, false, whole);
      const int i = min(first_from(s.cum, f.n, border), f.n - 1);
      fewest(f.before + (uint32_t)i + 1, s.cum[i]);
      __syncthreads();
    }
    if (by_min) {
      uint64_t count = 0, mass = 0;
      each_logit<T, kRowThreads>(logits, 0, a.vocab, [&](float l, int) {
        const double e = weight_of(log_weight(r, l));
        if (e >= min_p) {
          ++count;
          mass += fixed_of(e);
        }
      });
      count = block_sum(s, count);
      mass = block_sum(s, mass);
      fewest(max((uint32_t)count, 1u), mass);
    }
    const uint64_t target = target_of(kept) + 1;
    const Found f = resolve<T>(a, s, r, logits, first_from(s.mass, kBins, target), false, target);
    at = first_from(s.cum, f.n, target);
  }
  if (tid == 0) {
    const uint64_t place = s.sorted[at];
    a.token_ids[row] = (int64_t)(uint32_t)place;
    if (a.logprobs != nullptr)
      a.logprobs[row] = (float)(log_weight(r, place_logit(place)) * 0.69314718055994530942 -
                                log((double)kept * (1. / (double)(1ull << kFixed))));
  }
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
  hipLaunchKernelGGL(sample_bins_kernel<T>, dim3((unsigned)(rows * a.chunks2)), dim3(kThreads), 0, s, a);
  hipLaunchKernelGGL(sample_row_kernel<T>, dim3((unsigned)rows), dim3(kRowThreads), 0, s, a);
}

}  // namespace

extern "C" size_t hx_sample_workspace_bytes(int64_t rows, int64_t vocab) {
  if (rows < 1 || vocab < 1 || vocab > kMostVocab || rows > (1 << 20)) return 0;
  return (size_t)rows * (kMostChunks * (sizeof(uint64_t) + sizeof(uint32_t)) + kBins * (sizeof(uint64_t) + sizeof(uint32_t)));
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
  cut(rows, a.vocab, 2048, &a.chunks, &a.chunk);
  cut(rows, a.vocab, 1024, &a.chunks2, &a.chunk2);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == HX_DTYPE_BF16) launch<__bf16>(a, rows, s);
  else if (dtype == HX_DTYPE_FP16) launch<_Float16>(a, rows, s);
  else launch<float>(a, rows, s);
  return hx::status_from_hip(hipGetLastError());
}
