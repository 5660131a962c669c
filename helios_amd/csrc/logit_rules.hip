// Penalties, biases and allowed-token masks on the logits of a tick, with the greedy ids (gfx950).
//
// For row r and token v, with l the logit in fp32 and each step rounded to fp32:
//   v among the row's known tokens (prompt or said):  l = l > 0 ? l / repetition : l * repetition
//   v said c > 0 times:                               l = l - (frequency * c + presence)
//   v in the row's bias list:                         l = l + bias (of its last entry there)
//   v not allowed by the row's mask:                  l = -inf
// then rounded to the element type; the greedy id is the smallest allowed v with the largest
// rounded result (a NaN counts as the largest), -1 in a row that nothing is allowed in.
//
// One pass over [rows, vocab], bound by memory (2 + 2 bytes a logit) until the histories are
// long: each workgroup looks through its row's whole history, from L2. A workgroup owns 4096
// logits of a row, cut at 16-byte addresses, and
//   - counts the row's tokens that fall among them in LDS, so no dense count of the vocabulary is
//     ever stored;
//   - applies the rules to the logits that a token or bias touched alone: the rules' arithmetic
//     on every logit took forty instructions and bound the kernel (97 us where it takes 35);
//   - masks all and takes the best of them on packed 16-bit integers in the values' order.
// Counts are sums of whole numbers, the bias slot and the best key maxima, so no order of the
// atomics shows. The workgroups' best keys (value, then smaller index) meet in a second launch.
//
// 129 rows of 151936 bf16 logits (78 MB in and out): 22 us without rules, 24 with a mask, 36 with
// histories of 5217 tokens in the mean too (clearing the tables 3, looking through the tokens 5,
// the touched logits 7); both launches, as the time of calls one after another.

#include "hx_common.h"

namespace {

// Four rows of 151936 bf16 logits with 1500 tokens, and 129 rows with up to 8192 tokens, 300
// biases and a mask, in us: 7.0 and 34.9; 256 threads 8.3 and 46; 256 threads on 2048 logits 6.8
// and 38.9; 512 on 8192 logits 8.5 and 40.8; 1024 on 8192 logits 7.2 and 35.6.
constexpr int kLrThreads = 512;
constexpr int kLrSlice = 4096;  // logits per workgroup

struct RuleArgs {
  const void* logits;
  int64_t row_stride;
  void* out;  // may be the logits; null: none
  int64_t out_stride;
  int64_t vocab;
  int32_t slices;
  const int32_t* tokens;  // [rows][token_stride]
  int64_t token_stride, token_cap;
  const int32_t* lengths;
  const int32_t* prompt_lens;
  const float* repetition;
  const float* presence;
  const float* frequency;
  const int32_t* bias_ids;
  const float* bias_values;
  int64_t bias_stride;
  int32_t n_bias;
  const uint32_t* allowed;
  int64_t allowed_stride;
  uint64_t* keys;  // [rows][slices]
};

template <typename T>
struct LogitElem {
  static constexpr int kVec = 8;  // elements of 16 bytes
  typedef uint16_t raw;
  static constexpr uint32_t kNegInf = __is_same(T, __bf16) ? 0xff80u : 0xfc00u;
  static constexpr uint32_t kInf = kNegInf & 0x7fffu;
  static __device__ __forceinline__ float get(raw u) { return hx::Elem<T>::lo(u); }
  static __device__ __forceinline__ raw put(float f) { return hx::Elem<T>::bits(f); }
};
template <>
struct LogitElem<float> {
  static constexpr int kVec = 4;
  typedef uint32_t raw;
  static constexpr uint32_t kNegInf = 0xff800000u, kInf = 0x7f800000u;
  static __device__ __forceinline__ float get(raw u) { return __uint_as_float(u); }
  static __device__ __forceinline__ raw put(float f) { return __float_as_uint(f); }
};

typedef short lr_s2 __attribute__((ext_vector_type(2)));

// A value's order as a signed integer: its magnitude's bits with its sign, 0 and -0 alike, a NaN
// above all; none_of lies below every value's.
template <typename T>
__device__ __forceinline__ int order_of(typename LogitElem<T>::raw u) {
  constexpr int kBits = sizeof(u) * 8;
  const uint32_t mag = u & ((1u << (kBits - 1)) - 1u);
  if (mag > LogitElem<T>::kInf) return (int)((1u << (kBits - 1)) - 1u);
  return u >> (kBits - 1) ? -(int)mag : (int)mag;
}
template <typename T>
__device__ __forceinline__ constexpr int none_of() { return sizeof(typename LogitElem<T>::raw) == 2 ? -0x8000 : (int)0x80000000; }

// A key that orders by value, then by smaller index; 0: none.
template <typename T>
__device__ __forceinline__ uint64_t key_of(int order, uint32_t v) {
  return order == none_of<T>() ? 0 : (uint64_t)((uint32_t)order ^ 0x80000000u) << 32 | (uint32_t)~v;
}

__device__ __forceinline__ uint64_t max_u64(uint64_t a, uint64_t b) { return a > b ? a : b; }

__device__ __forceinline__ uint32_t least_u32(uint32_t a, uint32_t b) { return a < b ? a : b; }

template <int CTRL>
__device__ __forceinline__ int max_dpp(int v) {
  const int x = __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, false);
  return x > v ? x : v;
}
__device__ __forceinline__ int wave_max(int v) {
  v = max_dpp<hx::kDppHalfMirror>(max_dpp<hx::kDppXor2>(max_dpp<hx::kDppXor1>(v)));
  v = max_dpp<hx::kDppMirror>(v);  // of each row of 16 lanes
  const int a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16);
  const int c = __builtin_amdgcn_readlane(v, 32), d = __builtin_amdgcn_readlane(v, 48);
  const int ab = a > b ? a : b, cd = c > d ? c : d;
  return ab > cd ? ab : cd;
}

// VEC: the rows of the logits and of the output lie alike with respect to 16 bytes.
template <typename T, bool VEC>
__global__ __launch_bounds__(kLrThreads) void logit_rules_kernel(RuleArgs a) {
  typedef LogitElem<T> L;
  typedef typename L::raw raw;
  constexpr int kVec = L::kVec, kPer = kLrSlice / kLrThreads / kVec;  // 16-byte pieces a thread
  __shared__ __attribute__((aligned(16))) uint32_t s_count[kLrSlice];  // 2 x times said + (in the prompt)
  __shared__ __attribute__((aligned(16))) uint32_t s_bias[kLrSlice];   // entry of the bias list + 1
  __shared__ uint64_t s_key[kLrThreads / 64];
  const int tid = hx::tid_x();
  const int64_t row = hx::wg_x() / a.slices;
  const raw* const logits = static_cast<const raw*>(a.logits) + row * a.row_stride;
  raw* const out = a.out != nullptr ? static_cast<raw*>(a.out) + row * a.out_stride : nullptr;
  // The slice's first element: before the row where that is what lies at a 16-byte address.
  const int lead = VEC ? (int)((reinterpret_cast<uintptr_t>(logits) & 15) / sizeof(raw)) : 0;
  const int64_t v0 = (int64_t)(hx::wg_x() % a.slices) * kLrSlice - lead;
  const int begin = v0 < 0 ? (int)-v0 : 0;
  const int end = a.vocab - v0 < kLrSlice ? (int)(a.vocab - v0) : kLrSlice;  // may lie before begin
  const bool hist = a.tokens != nullptr, biased = a.bias_ids != nullptr;

  // All that does not depend on LDS is on its way before the first wait: the row's scalars, the
  // first of its tokens (four a load, from the first 16-byte address on, and four loads at once)
  // and biases, then the logits and their mask, whose loads would hold up the tokens' otherwise.
  constexpr int kAtOnce = 4;
  const float rep = a.repetition != nullptr ? a.repetition[row] : 1.f;
  const float pres = a.presence != nullptr ? a.presence[row] : 0.f;
  const float freq = a.frequency != nullptr ? a.frequency[row] : 0.f;
  const int given = hist ? a.lengths[row] : 0;
  const int prompt = hist && a.prompt_lens != nullptr ? a.prompt_lens[row] : 0;
  const int32_t* const bias_ids = a.bias_ids + row * a.bias_stride;
  const float* const bias_values = a.bias_values + row * a.bias_stride;
  const int len = given < 0 ? 0 : given < a.token_cap ? given : (int)a.token_cap;
  const int32_t* const tokens = a.tokens + row * a.token_stride;
  const int first = (int)((16 - (reinterpret_cast<uintptr_t>(tokens) & 15)) & 15) / 4;
  const int quads = len > first ? (len - first) / 4 : 0;
  uint4 quad[kAtOnce];
  auto load_quads = [&](int q0) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k)
      if (q0 + k * kLrThreads < quads) quad[k] = reinterpret_cast<const uint4*>(tokens + first)[q0 + k * kLrThreads];
  };
  load_quads(tid);
  int32_t my_id = biased && tid < a.n_bias ? bias_ids[tid] : 0;
  uint4 piece[kPer];
  uint32_t words[kPer][2];
  const uint32_t* const mask = a.allowed != nullptr ? a.allowed + row * a.allowed_stride : nullptr;
#pragma unroll
  for (int p = 0; p < kPer; ++p) {
    const int at = (p * kLrThreads + tid) * kVec;
    const bool whole = VEC && at >= begin && at + kVec <= end;
    piece[p] = hx::zero4();
    words[p][0] = words[p][1] = 0xffffffffu;
    if (!whole) continue;
    piece[p] = hx::ld16_stream(logits + v0 + at);
    if (mask != nullptr) {
      const int64_t v = v0 + at;
      words[p][0] = mask[v >> 5];
      words[p][1] = (v & 31) + kVec > 32 ? mask[(v >> 5) + 1] : 0;
    }
  }

  if (hist || biased) {
    for (int i = tid; i < kLrSlice / 4; i += kLrThreads) {
      if (hist) reinterpret_cast<uint4*>(s_count)[i] = hx::zero4();
      if (biased) reinterpret_cast<uint4*>(s_bias)[i] = hx::zero4();
    }
    __syncthreads();
    // The slice's ids, as a range that one unsigned comparison tests.
    const uint32_t first_id = (uint32_t)(v0 + begin), ids = end > begin ? (uint32_t)(end - begin) : 0u;
    if (hist) {
      auto known = [&](int i, int32_t token) __attribute__((always_inline)) {
        const uint32_t in = (uint32_t)token - first_id;
        if (in >= ids) return;
        const int at = begin + (int)in;
        if (i >= prompt) atomicAdd(&s_count[at], 2u);
        else atomicOr(&s_count[at], 1u);
      };
      if (tid < (first < len ? first : len)) known(tid, tokens[tid]);
      for (int q0 = tid; q0 < quads; q0 += kAtOnce * kLrThreads) {
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
          if (q0 + k * kLrThreads >= quads) continue;
          const int i = first + 4 * (q0 + k * kLrThreads);
          const uint32_t id[4] = {quad[k].x, quad[k].y, quad[k].z, quad[k].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) known(i + e, (int32_t)id[e]);
        }
        load_quads(q0 + kAtOnce * kLrThreads);
      }
      const int rest = first + 4 * quads + tid;
      if (rest < len && tid < 4) known(rest, tokens[rest]);
    }
    if (biased)
      for (int i = tid; i < a.n_bias;) {
        const uint32_t in = (uint32_t)my_id - first_id;
        if (in < ids) atomicMax(&s_bias[begin + (int)in], (uint32_t)i + 1u);
        i += kLrThreads;
        if (i < a.n_bias) my_id = bias_ids[i];
      }
    __syncthreads();
  }

  auto ruled = [&](raw u, int at) __attribute__((always_inline)) -> raw {
    float x = L::get(u);
    if (hist) {
      const uint32_t c = s_count[at];
      if (c != 0) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
      if (c >> 1) x = __fsub_rn(x, __fadd_rn(__fmul_rn(freq, (float)(c >> 1)), pres));
    }
    if (biased) {
      const uint32_t b = s_bias[at];
      if (b != 0) x = __fadd_rn(x, bias_values[b - 1]);
    }
    return L::put(x);
  };
  // A thread's logits come in the order of their ids: an equal one later does not replace the best.
  int best = none_of<T>();
  uint32_t best_id = 0;
  auto better = [&](int order, uint32_t id) __attribute__((always_inline)) {
    best_id = order > best ? id : best_id;
    best = order > best ? order : best;
  };
#pragma unroll
  for (int p = 0; p < kPer; ++p) {
    const int at = (p * kLrThreads + tid) * kVec;
    if (VEC && at >= begin && at + kVec <= end) {
      const uint32_t ok = __builtin_amdgcn_alignbit(words[p][1], words[p][0], (uint32_t)(v0 + at) & 31);
      uint32_t w[4] = {piece[p].x, piece[p].y, piece[p].z, piece[p].w};
      // The touched ones, a lane's first, second, ... each in its turn.
      uint32_t touched = 0;
#pragma unroll
      for (int q = 0; q < kVec / 4; ++q) {
        uint4 any = hx::zero4();
        if (hist) any = reinterpret_cast<const uint4*>(s_count)[at / 4 + q];
        if (biased) {
          const uint4 b = reinterpret_cast<const uint4*>(s_bias)[at / 4 + q];
          any = make_uint4(any.x | b.x, any.y | b.y, any.z | b.z, any.w | b.w);
        }
        const uint32_t c[4] = {any.x, any.y, any.z, any.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) touched |= least_u32(c[e], 1u) << (4 * q + e);
      }
      touched &= ok;
      while (touched != 0) {
        const int e = __builtin_ctz(touched);
        touched &= touched - 1;
        if constexpr (kVec == 8) {
          const uint32_t pair = e & 4 ? (e & 2 ? w[3] : w[2]) : (e & 2 ? w[1] : w[0]);
          const uint32_t u = ruled((raw)(e & 1 ? pair >> 16 : pair), at + e);
          const uint32_t now = e & 1 ? (pair & 0xffffu) | u << 16 : (pair & 0xffff0000u) | u;
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = e >> 1 == k ? now : w[k];
        } else {
          const uint32_t u = ruled(e & 2 ? (e & 1 ? w[3] : w[2]) : (e & 1 ? w[1] : w[0]), at + e);
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = e == k ? u : w[k];
        }
      }
      int order[kVec], most = none_of<T>();
      if constexpr (kVec == 8) {
        lr_s2 top = {(short)-0x8000, (short)-0x8000}, ord[4], mag_top = {0, 0};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const lr_s2 x = __builtin_bit_cast(lr_s2, w[k]), sign = x >> 15, mag = x & (short)0x7fff;
          const lr_s2 o = (mag ^ sign) - sign;
          mag_top = __builtin_elementwise_max(mag_top, mag);
          const uint32_t m = (uint32_t)__builtin_amdgcn_sbfe((int)ok, 2 * k, 1) & 0xffffu |
                             (uint32_t)__builtin_amdgcn_sbfe((int)ok, 2 * k + 1, 1) << 16;
          ord[k] = __builtin_bit_cast(lr_s2, (__builtin_bit_cast(uint32_t, o) & m) | (0x80008000u & ~m));
          top = __builtin_elementwise_max(top, ord[k]);
        }
        most = max((int)top[0], (int)top[1]);
#pragma unroll
        for (int e = 0; e < 8; ++e) order[e] = ord[e / 2][e % 2];
        if (max((int)mag_top[0], (int)mag_top[1]) > (int)L::kInf) {  // a NaN among them
          most = none_of<T>();
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            order[e] = ok >> e & 1 ? order_of<T>((raw)(w[e / 2] >> (16 * (e % 2)))) : none_of<T>();
            most = max(most, order[e]);
          }
        }
        if (mask != nullptr) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t m = (uint32_t)__builtin_amdgcn_sbfe((int)ok, 2 * k, 1) & 0xffffu |
                               (uint32_t)__builtin_amdgcn_sbfe((int)ok, 2 * k + 1, 1) << 16;
            w[k] = (w[k] & m) | (L::kNegInf * 0x10001u & ~m);
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          order[e] = ok >> e & 1 ? order_of<T>((raw)w[e]) : none_of<T>();
          most = max(most, order[e]);
          if (!(ok >> e & 1)) w[e] = L::kNegInf;
        }
      }
      if (out != nullptr) hx::st16_nt(out + v0 + at, make_uint4(w[0], w[1], w[2], w[3]));
      int which = kVec - 1;
#pragma unroll
      for (int e = kVec - 2; e >= 0; --e) which = order[e] == most ? e : which;
      better(most, (uint32_t)(v0 + at + which));
      continue;
    }
    for (int e = 0; e < kVec; ++e) {  // the row's ends, or rows that lie otherwise than the output's
      const int i = at + e;
      if (i < begin || i >= end) continue;
      const int64_t v = v0 + i;
      const bool ok = mask == nullptr || mask[v >> 5] >> (v & 31) & 1u;
      raw u = (raw)L::kNegInf;
      if (ok) {
        u = logits[v];
        u = ruled(u, i);
        better(order_of<T>(u), (uint32_t)v);
      }
      if (out != nullptr) out[v] = u;
    }
  }
  const int most = wave_max(best);
  const uint32_t id = ~(uint32_t)wave_max(best == most ? (int)~best_id ^ (int)0x80000000 : (int)0x80000000) ^ 0x80000000u;
  if ((tid & 63) == 0) s_key[tid >> 6] = key_of<T>(most, id);
  __syncthreads();
  if (tid == 0) {
    uint64_t key = 0;
#pragma unroll
    for (int w = 0; w < kLrThreads / 64; ++w) key = max_u64(key, s_key[w]);
    a.keys[(int64_t)hx::wg_x()] = key;
  }
}

__global__ __launch_bounds__(64) void logit_rules_ids_kernel(const uint64_t* keys, int32_t slices, int64_t* ids) {
  const int64_t row = hx::wg_x();
  uint64_t best = 0;
  for (int i = hx::tid_x(); i < slices; i += 64) best = max_u64(best, keys[row * slices + i]);
  for (int m = 1; m < 64; m <<= 1) best = max_u64(best, __shfl_xor((unsigned long long)best, m));
  if (hx::tid_x() == 0) ids[row] = best == 0 ? -1 : (int64_t)(uint32_t)~(uint32_t)best;
}

template <typename T>
void launch_rules(const RuleArgs& a, int64_t rows, hipStream_t s) {
  constexpr int64_t kSize = sizeof(typename LogitElem<T>::raw);
  // Each row's first logit and its place in the output at the same offset from a 16-byte address.
  const bool alike = a.out == nullptr || ((reinterpret_cast<uintptr_t>(a.logits) - reinterpret_cast<uintptr_t>(a.out)) % 16 == 0 &&
                                          (a.row_stride - a.out_stride) * kSize % 16 == 0);
  const dim3 grid((unsigned)(rows * a.slices));
  if (alike) hipLaunchKernelGGL((logit_rules_kernel<T, true>), grid, dim3(kLrThreads), 0, s, a);
  else hipLaunchKernelGGL((logit_rules_kernel<T, false>), grid, dim3(kLrThreads), 0, s, a);
}

// Slices of a row, up to seven elements before it included.
int64_t slices_of(int64_t vocab) { return (vocab + 7 + kLrSlice - 1) / kLrSlice; }

}  // namespace

extern "C" size_t hx_logit_rules_workspace_bytes(int64_t rows, int64_t vocab) {
  if (rows < 1 || vocab < 1) return 0;
  return (size_t)rows * (size_t)slices_of(vocab) * sizeof(uint64_t);
}

extern "C" int hx_logit_rules(const void* logits, int64_t logits_row_stride, int64_t rows, int64_t vocab,
                              int32_t dtype, const int32_t* tokens, int64_t token_row_stride, int64_t token_cap,
                              const int32_t* lengths, const int32_t* prompt_lens, const float* repetition,
                              const float* presence, const float* frequency, const int32_t* bias_ids,
                              const float* bias_values, int64_t bias_row_stride, int32_t n_bias,
                              const uint32_t* allowed, int64_t allowed_row_stride, void* out, int64_t out_row_stride,
                              int64_t* token_ids, void* workspace, size_t workspace_bytes, void* stream) {
  if (dtype != HX_DTYPE_BF16 && dtype != HX_DTYPE_FP16 && dtype != HX_DTYPE_FP32) return HX_E_UNSUPPORTED;
  if (rows < 0 || vocab < 1 || vocab > 0x7fffffff || logits_row_stride < vocab || n_bias < 0) return HX_E_INVALID_ARG;
  if (rows == 0) return HX_OK;
  if (!logits || !token_ids || (out && out_row_stride < vocab) ||
      ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(out)) & (dtype == HX_DTYPE_FP32 ? 3 : 1)))
    return HX_E_INVALID_ARG;
  if (tokens && (!lengths || token_cap < 0 || token_cap > 0x7fffffff || token_row_stride < token_cap)) return HX_E_INVALID_ARG;
  if ((bias_ids && (!bias_values || bias_row_stride < n_bias)) ||
      (allowed && allowed_row_stride < (vocab + 31) / 32))
    return HX_E_INVALID_ARG;
  const size_t need = hx_logit_rules_workspace_bytes(rows, vocab);
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 7) || workspace_bytes < need) return HX_E_WORKSPACE;
  RuleArgs a;
  a.logits = logits;
  a.row_stride = logits_row_stride;
  a.out = out;
  a.out_stride = out_row_stride;
  a.vocab = vocab;
  a.slices = (int32_t)slices_of(vocab);
  a.tokens = tokens;
  a.token_stride = token_row_stride;
  a.token_cap = token_cap;
  a.lengths = lengths;
  a.prompt_lens = prompt_lens;
  a.repetition = repetition;
  a.presence = presence;
  a.frequency = frequency;
  a.bias_ids = n_bias > 0 ? bias_ids : nullptr;
  a.bias_values = bias_values;
  a.bias_stride = bias_row_stride;
  a.n_bias = n_bias;
  a.allowed = allowed;
  a.allowed_stride = allowed_row_stride;
  a.keys = static_cast<uint64_t*>(workspace);
  if (rows > 0xffffffffll / kLrThreads / a.slices) return HX_E_UNSUPPORTED;  // work-items of a launch: 32 bits
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == HX_DTYPE_FP32) launch_rules<float>(a, rows, s);
  else if (dtype == HX_DTYPE_BF16) launch_rules<__bf16>(a, rows, s);
  else launch_rules<_Float16>(a, rows, s);
  hipLaunchKernelGGL(logit_rules_ids_kernel, dim3((unsigned)rows), dim3(64), 0, s, a.keys, a.slices, token_ids);
  return hx::status_from_hip(hipGetLastError());
}
