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
// One pass over [rows, vocab]: HBM-bound, 2 + 2 bytes a logit. A workgroup owns 4096 logits of
// a row and counts the row's tokens that fall among them in LDS, so no dense count of the
// vocabulary is ever stored; a history is read once per 4096 logits, from L2. Counts are sums
// of whole numbers and the bias slot a maximum, so no order of the atomics shows.
// The workgroups' best keys (value, then smaller index) meet in a second launch.

#include "hx_common.h"

namespace {

constexpr int kLrThreads = 256;
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
struct LogitElem;
template <>
struct LogitElem<float> {
  static constexpr int kVec = 4;
  typedef uint32_t raw;
  static __device__ __forceinline__ float get(raw u) { return __uint_as_float(u); }
  static __device__ __forceinline__ raw put(float f) { return __float_as_uint(f); }
};
template <typename T>
struct LogitElem {
  static constexpr int kVec = 8;
  typedef uint16_t raw;
  static __device__ __forceinline__ float get(raw u) { return hx::Elem<T>::lo(u); }
  static __device__ __forceinline__ raw put(float f) { return hx::Elem<T>::bits(f); }
};

// A key that orders by value (NaN above all, -0 like 0), then by smaller index; never 0.
__device__ __forceinline__ uint64_t key_of(float f, uint32_t v) {
  uint32_t u = __float_as_uint(f);
  const uint32_t mag = u & 0x7fffffffu;
  u = mag > 0x7f800000u ? 0xffffffffu : mag == 0 ? 0x80000000u : (u >> 31) ? ~u : u | 0x80000000u;
  return (uint64_t)u << 32 | (uint32_t)~v;
}

__device__ __forceinline__ uint64_t max_u64(uint64_t a, uint64_t b) { return a > b ? a : b; }

template <typename T, bool VEC>
__global__ __launch_bounds__(kLrThreads) void logit_rules_kernel(RuleArgs a) {
  typedef LogitElem<T> L;
  typedef typename L::raw raw;
  constexpr int kVec = VEC ? L::kVec : 1;
  constexpr int kPer = kLrSlice / kLrThreads / kVec;  // accesses a thread
  __shared__ uint32_t s_count[kLrSlice];
  __shared__ uint32_t s_bias[kLrSlice];
  __shared__ uint64_t s_key[kLrThreads / 64];
  const int tid = hx::tid_x();
  const int64_t row = hx::wg_x() / a.slices;
  const int64_t v0 = (int64_t)(hx::wg_x() % a.slices) * kLrSlice;
  const int n = a.vocab - v0 < kLrSlice ? (int)(a.vocab - v0) : kLrSlice;
  const bool hist = a.tokens != nullptr, biased = a.bias_ids != nullptr;
  for (int i = tid; i < kLrSlice; i += kLrThreads) {
    if (hist) s_count[i] = 0;
    if (biased) s_bias[i] = 0;
  }
  __syncthreads();
  if (hist) {
    const int64_t given = max(a.lengths[row], 0), len = given < a.token_cap ? given : a.token_cap;
    const int64_t prompt = a.prompt_lens != nullptr ? a.prompt_lens[row] : 0;
    const int32_t* t = a.tokens + row * a.token_stride;
    for (int64_t i = tid; i < len; i += kLrThreads) {
      const int64_t v = (int64_t)t[i] - v0;
      if (v < 0 || v >= n) continue;
      if (i >= prompt) atomicAdd(&s_count[v], 2u);  // said: twice the count
      else atomicOr(&s_count[v], 1u);               // in the prompt
    }
  }
  if (biased)
    for (int i = tid; i < a.n_bias; i += kLrThreads) {
      const int64_t v = (int64_t)a.bias_ids[row * a.bias_stride + i] - v0;
      if (v >= 0 && v < n) atomicMax(&s_bias[v], (uint32_t)i + 1u);
    }
  __syncthreads();

  const float rep = a.repetition != nullptr ? a.repetition[row] : 1.f;
  const float pres = a.presence != nullptr ? a.presence[row] : 0.f;
  const float freq = a.frequency != nullptr ? a.frequency[row] : 0.f;
  const raw* in = static_cast<const raw*>(a.logits) + row * a.row_stride + v0;
  raw* out = a.out != nullptr ? static_cast<raw*>(a.out) + row * a.out_stride + v0 : nullptr;
  uint64_t best = 0;
#pragma unroll
  for (int p = 0; p < kPer; ++p) {
    const int at = (p * kLrThreads + tid) * kVec;
    if (at >= n) continue;
    raw e[kVec];
    const bool whole = VEC && at + kVec <= n;
    if constexpr (VEC) {
      if (whole) {
        const uint4 u = *reinterpret_cast<const uint4*>(in + at);
        __builtin_memcpy(e, &u, 16);
      }
    }
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      if (!whole) {
        if (at + j >= n) continue;
        e[j] = in[at + j];
      }
      const int64_t v = v0 + at + j;
      float x = L::get(e[j]);
      if (hist) {
        const uint32_t c = s_count[at + j];
        if (c != 0) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
        if (c >> 1) x = __fsub_rn(x, __fadd_rn(__fmul_rn(freq, (float)(c >> 1)), pres));
      }
      if (biased) {
        const uint32_t i = s_bias[at + j];
        if (i != 0) x = __fadd_rn(x, a.bias_values[row * a.bias_stride + i - 1]);
      }
      e[j] = L::put(x);
      bool ok = true;
      if (a.allowed != nullptr) ok = a.allowed[row * a.allowed_stride + (v >> 5)] >> (v & 31) & 1u;
      if (!ok) e[j] = L::put(-INFINITY);
      if (ok) best = max_u64(best, key_of(L::get(e[j]), (uint32_t)v));
      if (!whole && out != nullptr) out[at + j] = e[j];
    }
    if constexpr (VEC) {
      if (whole && out != nullptr) {
        uint4 u;
        __builtin_memcpy(&u, e, 16);
        *reinterpret_cast<uint4*>(out + at) = u;
      }
    }
  }
  for (int m = 1; m < 64; m <<= 1) best = max_u64(best, __shfl_xor((unsigned long long)best, m));
  if ((tid & 63) == 0) s_key[tid >> 6] = best;
  __syncthreads();
  if (tid == 0)
    a.keys[(int64_t)hx::wg_x()] = max_u64(max_u64(s_key[0], s_key[1]), max_u64(s_key[2], s_key[3]));
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
  const int64_t vec = LogitElem<T>::kVec;
  const bool aligned = !((reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(a.out)) & 15) &&
                       a.row_stride % vec == 0 && (a.out == nullptr || a.out_stride % vec == 0);
  const dim3 grid((unsigned)(rows * a.slices));
  if (aligned) hipLaunchKernelGGL((logit_rules_kernel<T, true>), grid, dim3(kLrThreads), 0, s, a);
  else hipLaunchKernelGGL((logit_rules_kernel<T, false>), grid, dim3(kLrThreads), 0, s, a);
}

}  // namespace

extern "C" size_t hx_logit_rules_workspace_bytes(int64_t rows, int64_t vocab) {
  if (rows < 1 || vocab < 1) return 0;
  return (size_t)rows * (size_t)((vocab + kLrSlice - 1) / kLrSlice) * sizeof(uint64_t);
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
  if (!logits || !token_ids || (out && out_row_stride < vocab)) return HX_E_INVALID_ARG;
  if (tokens && (!lengths || token_cap < 0 || token_row_stride < token_cap)) return HX_E_INVALID_ARG;
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
  a.slices = (int32_t)((vocab + kLrSlice - 1) / kLrSlice);
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
  if (rows * a.slices > 0x7fffffff) return HX_E_UNSUPPORTED;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == HX_DTYPE_FP32) launch_rules<float>(a, rows, s);
  else if (dtype == HX_DTYPE_BF16) launch_rules<__bf16>(a, rows, s);
  else launch_rules<_Float16>(a, rows, s);
  hipLaunchKernelGGL(logit_rules_ids_kernel, dim3((unsigned)rows), dim3(64), 0, s, a.keys, a.slices, token_ids);
  return hx::status_from_hip(hipGetLastError());
}
