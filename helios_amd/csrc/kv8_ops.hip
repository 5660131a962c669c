// Writing and reading the 8-bit KV cache (gfx950).
//
// A head row x of a token (the key after its norm and rotation, or the value) is stored as
//   s = max(max_d |x_d| * (1 / Q), 2^-100),  c_d = round(x_d / s)  Q = 448 (e4m3) or 127 (int8)
// in fp32, 1 / Q rounded and the division by s a true one, so the codes do not depend on how a
// kernel is built. A row with an
// infinite or NaN element is stored as zeros under a NaN scale: it reads back, and is attended to,
// as NaN. Codes lie as the 16-bit pool does, [pages, page_size, kv_heads, head_dim]; scales are
// [pages, kv_heads, page_size], so that attention to one head reads consecutive ones (beside the
// codes' order a head's 4 of every 32 bytes would be read 8 times over).
//
// The norm and rotation are those of the 16-bit append (layers.py:30-40, :54-72), rounded once: to the
// queries' type, in fp32 from the projections on, or to the keys' codes and scales, in fp64 (fp32 keys
// next to a border between codes fall to either side of it: 2 in 10^6, which costs 5e-5 of a tensor's
// norm; fp64 8 % of the launch).

#include "kv8_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int64_t kMostItems = (int64_t)1 << 32;  // work-items of a launch

struct WriteArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  const float* q_norm;
  const float* k_norm;
  const float* cos;
  const float* sin;
  int64_t rope_rows;
  const int64_t* positions;
  int64_t n_rows;
  int32_t hq, hkv, head_dim;
  float eps;
  uint16_t* q_out;
  int64_t qo_row, qo_head;
  uint8_t* codes[2];   // keys, values
  float* scales[2];
  int64_t pool_rows;
  int32_t page;
  const int64_t* slots;
};

// Eight elements from 16-byte aligned memory, or one by one.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const uint16_t* p, float (&x)[8]) {
  if constexpr (VEC) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[2 * e] = hx::Elem<T>::lo(w[e]);
      x[2 * e + 1] = hx::Elem<T>::hi(w[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = hx::Elem<T>::lo((uint32_t)p[e]);
  }
}

__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}

// Over LANES neighbouring lanes, each of which gets the result: two lanes of a quad, two quads, two
// halves of 16, and further ones through the shuffle.
template <int CTRL, typename X>
__device__ __forceinline__ X other_lane(X x) {
  return __builtin_bit_cast(X, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
template <int LANES, typename X, typename F>
__device__ __forceinline__ X over_lanes(X x, F f) {
  x = f(x, other_lane<0xb1>(x));   // lane ^ 1
  x = f(x, other_lane<0x4e>(x));   // lane ^ 2
  x = f(x, other_lane<0x141>(x));  // 7 - lane
  if constexpr (LANES >= 16) x = f(x, other_lane<0x140>(x));  // 15 - lane
  if constexpr (LANES >= 32) x = f(x, __builtin_bit_cast(X, __shfl_xor(__builtin_bit_cast(int, x), 16)));
  return x;
}

// A head row to LANES lanes, 8 elements each (lanes past head_dim idle along); a workgroup takes
// kThreads / LANES of them, a token's query, key and value heads in turn. 2381 tokens of 32 + 8 + 8
// heads of 128, with norms and rotation: 18.5 us, 3.0 TB/s, 11.7 without the rotation, whose weights,
// cosines and sines are 6 times a row's own bytes, from L2, and whose sum and turn are chains across
// lanes. (Two heads to a lane, which then share the cosines, won 6 % there and lost 30 % at 64 tokens.)
// Few tokens are a launch's latency.
template <typename T, typename C, int LANES, bool ROPE, bool VEC>
__global__ __launch_bounds__(kThreads) void kv8_write_kernel(WriteArgs a) {
  const int lane = hx::tid_x() & (LANES - 1);
  const int heads = (ROPE ? a.hq : 0) + 2 * a.hkv;
  const int64_t unit = (int64_t)(uint32_t)hx::wg_x() * (kThreads / LANES) + hx::tid_x() / LANES;
  const int64_t row = (unit >> 32) == 0 ? (int64_t)((uint32_t)unit / (uint32_t)heads) : unit / heads;
  if (row >= a.n_rows) return;  // the lanes of a head row leave together
  const int h = (int)(unit - row * heads);
  const int d = 8 * lane;
  const bool mine = d < a.head_dim;
  const bool is_q = ROPE && h < a.hq;
  const int hk = h - (ROPE ? a.hq : 0);
  const int which = hk >= a.hkv ? 1 : 0;  // of codes and scales
  const int hh = is_q ? h : which ? hk - a.hkv : hk;
  int64_t slot = 0;
  if (!is_q) {
    slot = a.slots[row];
    if (slot < 0 || slot >= a.pool_rows) return;
  }
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = 0.f;
  if (mine)
    load8<T, VEC>(is_q ? a.q + row * a.q_row + hh * a.q_head + d
                       : which ? a.v + row * a.v_row + hh * a.v_head + d : a.k + row * a.k_row + hh * a.k_head + d, x);
  auto store_row = [&](uint32_t lo, uint32_t hi, bool finite, float scale) __attribute__((always_inline)) {
    if (mine) hx::st8_nt(a.codes[which] + (slot * a.hkv + hh) * a.head_dim + d, finite ? lo : 0u, finite ? hi : 0u);
    if (lane == 0) {
      const int64_t page = (slot >> 32) == 0 ? (int64_t)((uint32_t)slot / (uint32_t)a.page) : slot / a.page;
      reinterpret_cast<uint32_t*>(a.scales[which])[(page * a.hkv + hh) * a.page + (slot - page * a.page)] =
          finite ? __float_as_uint(scale) : 0x7fc00000u;
    }
  };
  if (ROPE && (is_q || !which)) {
    int64_t pos = a.positions[row];
    pos = pos < 0 ? 0 : pos >= a.rope_rows ? a.rope_rows - 1 : pos;
    const float* const norm = is_q ? a.q_norm : a.k_norm;
    const int half = a.head_dim / 16;  // lanes of half a head row
    const bool low = lane < half;
    const int turn = low ? half : -half, other = (hx::tid_x() & 63) + turn;
    float w[8], c[8], s[8];
    if (mine) {
      load8(norm + d, w);
      load8(a.cos + pos * a.head_dim + d, c);
      load8(a.sin + pos * a.head_dim + d, s);
    }
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
    ss = over_lanes<LANES>(ss, [](float p, float q) { return p + q; });
    const float r = rsqrtf(ss / (float)a.head_dim + a.eps);
    if (!is_q) {
      // A key's codes follow from its elements' ratios to the largest, which r leaves as they are: those
      // are taken in fp64, and an element next to a border between codes gets the code of its value.
      float v[8];
      if (mine) load8(norm + d + 8 * turn, v);
      double z[8];
      uint64_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float p = __shfl(x[e], other);
        z[e] = mine ? fma((double)x[e] * w[e], (double)c[e], (double)(low ? -p : p) * v[e] * (double)s[e]) : 0.;
        const uint64_t b = hx::raw_bits(z[e]) & 0x7fffffffffffffffull;
        top = b > top ? b : top;
      }
#pragma unroll
      for (int m = 1; m < LANES; m <<= 1) {
        const uint64_t b = (uint64_t)(uint32_t)__shfl_xor((int)(uint32_t)top, m) |
                           (uint64_t)(uint32_t)__shfl_xor((int)(top >> 32), m) << 32;
        top = b > top ? b : top;
      }
      const double most = (double)r * __builtin_bit_cast(double, top);
      const bool finite = top < 0x7ff0000000000000ull && (hx::raw_bits((float)most) & 0x7fffffffu) < 0x7f800000u;
      const double scale = fmax(most * (1. / C::kMost), (double)hx8::kLeastScale);
      const double by = (double)r / scale;
      uint32_t code[2];
#pragma unroll
      for (int e = 0; e < 8; e += 4)
        code[e / 4] = hx8::encode4<C>((float)(z[e] * by), (float)(z[e + 1] * by), (float)(z[e + 2] * by), (float)(z[e + 3] * by));
      store_row(code[0], code[1], finite, (float)scale);
      return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = x[e] * r * (mine ? w[e] : 0.f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float p = __shfl(x[e], other);
      s[e] = mine ? fmaf(x[e], c[e], (low ? -p : p) * s[e]) : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = s[e];
  }
  if (is_q) {
    uint16_t* const to = a.q_out + row * a.qo_row + hh * a.qo_head + d;
    if (!mine) return;
    const uint4 u = make_uint4(hx::pack2_round<T>(x[0], x[1]), hx::pack2_round<T>(x[2], x[3]),
                               hx::pack2_round<T>(x[4], x[5]), hx::pack2_round<T>(x[6], x[7]));
    if constexpr (VEC) {
      hx::st16_nt(to, u);
    } else {
      const uint32_t wd[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) to[e] = (uint16_t)(wd[e / 2] >> (16 * (e & 1)));
    }
    return;
  }
  // The largest magnitude as bits: infinities and NaN lie above every number.
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, hx::raw_bits(x[e]) & 0x7fffffffu);
  top = over_lanes<LANES>(top, [](uint32_t p, uint32_t q) { return max(p, q); });
  const bool finite = top < 0x7f800000u;
  const float scale = fmaxf(__fmul_rn(__uint_as_float(finite ? top : 0u), 1.f / C::kMost), hx8::kLeastScale);
  // x / scale, rounded once, from the rounded reciprocal, of which a row needs one (Markstein 1990):
  // with r = 1 / s rounded to nearest and y = x r, the remainder x - y s is exact and y + (x - y s) r
  // rounds to the quotient. A small scale goes up by 2^64 first, and x with it: remainders stay normal.
  const float up = scale < 0x1p-64f ? 0x1p64f : 1.f, s = scale * up, r = __fdiv_rn(1.f, s);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float n = x[e] * up, y = n * r;
    x[e] = copysignf(fmaf(fmaf(-y, s, n), r, y), n);  // (-0 stays)
  }
  uint32_t code[2];
#pragma unroll
  for (int e = 0; e < 8; e += 4) code[e / 4] = hx8::encode4<C>(x[e], x[e + 1], x[e + 2], x[e + 3]);
  store_row(code[0], code[1], finite, scale);
}

// ------------------------------------------------------------------------------ read
struct ReadArgs {
  const uint8_t* codes;
  const float* scales;
  int32_t num_pages, page, hkv, head_dim;
  const int32_t* pages;
  int64_t length;
  void* out;
};

// 16 bytes of results to a lane, from 8 codes (4 for fp32); consecutive lanes walk a head's rows, whose
// results are consecutive in memory. A thread's loads for four such pieces are in flight together, and
// one head's workgroups follow another's. 40001 tokens of 8 heads of 128 to fp16: 22 us, 5.5 TB/s (24
// with two pieces, 24 with the heads side by side, 33 with 16 codes to a lane, whose stores leave gaps).
template <typename T, typename C>
__global__ __launch_bounds__(kThreads) void kv8_read_kernel(ReadArgs a, int pieces, uint32_t wgs) {
  constexpr int kCodes = 16 / sizeof(T), kAhead = 4;
  const int h = (int)((uint32_t)hx::wg_x() / wgs);
  const uint32_t at = (uint32_t)hx::wg_x() - (uint32_t)h * wgs;
  const int64_t all = a.length * pieces;
  for (int64_t i0 = (int64_t)at * (kAhead * kThreads) + hx::tid_x(); i0 < all; i0 += (int64_t)wgs * (kAhead * kThreads)) {
    uint32_t w[kAhead][kCodes / 4];
    float s[kAhead];
    int64_t page[kAhead], in[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t i = i0 + u * kThreads < all ? i0 + u * kThreads : all - 1;
      const int64_t t = (i >> 32) == 0 ? (int64_t)((uint32_t)i / (uint32_t)pieces) : i / pieces;
      const int64_t j = (t >> 32) == 0 ? (int64_t)((uint32_t)t / (uint32_t)a.page) : t / a.page;
      page[u] = a.pages[j];
      const bool off = page[u] < 0 || page[u] >= a.num_pages;
      page[u] = off ? 0 : page[u];
      const int64_t row = t - j * a.page;
      in[u] = (row * a.hkv + h) * a.head_dim + kCodes * (i - t * pieces);
      s[u] = off ? 0.f : a.scales[(page[u] * a.hkv + h) * a.page + row];
      page[u] = off ? -1 : page[u];
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const uint8_t* const from = a.codes + (page[u] < 0 ? 0 : page[u]) * a.page * a.hkv * a.head_dim + in[u];
#pragma unroll
      for (int e = 0; e < kCodes / 4; ++e) w[u][e] = 0;
      if (page[u] < 0) continue;
      if constexpr (kCodes == 8) {
        const uint2 x = *reinterpret_cast<const uint2*>(from);
        w[u][0] = x.x;
        w[u][1] = x.y;
      } else {
        w[u][0] = *reinterpret_cast<const uint32_t*>(from);
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t i = i0 + u * kThreads;
      if (i >= all) break;
      float x[kCodes];
#pragma unroll
      for (int e = 0; e < kCodes / 4; ++e) {
        float f[4];
        hx8::decode4<C>(w[u][e], f);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[4 * e + k] = f[k] * s[u];
      }
      uint4 o;
      if constexpr (sizeof(T) == 4)
        o = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
      else
        o = make_uint4(hx::pack2_round<T>(x[0], x[1]), hx::pack2_round<T>(x[2], x[3]),
                       hx::pack2_round<T>(x[4], x[5]), hx::pack2_round<T>(x[6], x[7]));
      hx::st16_nt(static_cast<uint8_t*>(a.out) + ((int64_t)h * all + i) * 16, o);
    }
  }
}

template <typename T, typename C, int LANES, bool ROPE>
void launch_write(const WriteArgs& a, bool vec, unsigned grid, hipStream_t s) {
  if (vec) hipLaunchKernelGGL((kv8_write_kernel<T, C, LANES, ROPE, true>), dim3(grid), dim3(kThreads), 0, s, a);
  else hipLaunchKernelGGL((kv8_write_kernel<T, C, LANES, ROPE, false>), dim3(grid), dim3(kThreads), 0, s, a);
}

template <typename T, typename C, bool ROPE>
int launch_write(const WriteArgs& a, bool vec, hipStream_t s) {
  const int lanes = a.head_dim <= 64 ? 8 : a.head_dim <= 128 ? 16 : 32, per = kThreads / lanes;
  const int64_t heads = (ROPE ? a.hq : 0) + 2 * (int64_t)a.hkv;
  if (a.n_rows > kMostItems / lanes / heads - kThreads) return HX_E_UNSUPPORTED;
  const unsigned grid = (unsigned)((a.n_rows * heads + per - 1) / per);
  if (lanes == 8) launch_write<T, C, 8, ROPE>(a, vec, grid, s);
  else if (lanes == 16) launch_write<T, C, 16, ROPE>(a, vec, grid, s);
  else launch_write<T, C, 32, ROPE>(a, vec, grid, s);
  return hx::status_from_hip(hipGetLastError());
}

template <bool ROPE>
int launch_write(const WriteArgs& a, int32_t dtype, int32_t code, hipStream_t s) {
  const uintptr_t ptrs = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
                         (ROPE ? reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.q_out) : 0);
  const int64_t strides = a.k_row | a.k_head | a.v_row | a.v_head | (ROPE ? a.q_row | a.q_head | a.qo_row | a.qo_head : 0);
  const bool vec = (ptrs & 15) == 0 && (strides & 7) == 0;
  if (dtype == HX_DTYPE_BF16)
    return code == HX_CODE_E4M3 ? launch_write<__bf16, hx8::E4m3, ROPE>(a, vec, s)
                                : launch_write<__bf16, hx8::Int8, ROPE>(a, vec, s);
  return code == HX_CODE_E4M3 ? launch_write<_Float16, hx8::E4m3, ROPE>(a, vec, s)
                              : launch_write<_Float16, hx8::Int8, ROPE>(a, vec, s);
}

int check_pool(int32_t num_pages, int32_t page, int32_t hkv, int32_t head_dim, int32_t code) {
  if (code != HX_CODE_E4M3 && code != HX_CODE_INT8) return HX_E_UNSUPPORTED;
  if (num_pages < 1 || page < 1 || hkv < 1 || head_dim < 1) return HX_E_INVALID_ARG;
  return head_dim % 16 || head_dim > 256 ? HX_E_UNSUPPORTED : HX_OK;
}

bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

}  // namespace

extern "C" int hx_kv8_append(void* k_codes, void* v_codes, float* k_scales, float* v_scales, int32_t num_pages,
                             int32_t page_size, int32_t n_kv_heads, int32_t head_dim, int32_t code, const void* k_new,
                             int64_t k_row_stride, int64_t k_head_stride, const void* v_new, int64_t v_row_stride,
                             int64_t v_head_stride, const int64_t* write_slots, int64_t n_tokens, int32_t dtype,
                             void* stream) {
  const int bad = check_pool(num_pages, page_size, n_kv_heads, head_dim, code);
  if (bad != HX_OK) return bad;
  if (dtype != HX_DTYPE_BF16 && dtype != HX_DTYPE_FP16) return HX_E_UNSUPPORTED;
  if (n_tokens < 0) return HX_E_INVALID_ARG;
  if (n_tokens == 0) return HX_OK;
  if (!k_codes || !v_codes || !k_scales || !v_scales || !k_new || !v_new || !write_slots || misaligned(k_codes, 16) ||
      misaligned(v_codes, 16))
    return HX_E_INVALID_ARG;
  WriteArgs a{};
  a.k = static_cast<const uint16_t*>(k_new);
  a.v = static_cast<const uint16_t*>(v_new);
  a.k_row = k_row_stride;
  a.k_head = k_head_stride;
  a.v_row = v_row_stride;
  a.v_head = v_head_stride;
  a.n_rows = n_tokens;
  a.hkv = n_kv_heads;
  a.head_dim = head_dim;
  a.codes[0] = static_cast<uint8_t*>(k_codes);
  a.codes[1] = static_cast<uint8_t*>(v_codes);
  a.scales[0] = k_scales;
  a.scales[1] = v_scales;
  a.pool_rows = (int64_t)num_pages * page_size;
  a.page = page_size;
  a.slots = write_slots;
  return launch_write<false>(a, dtype, code, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int hx_kv8_norm_rope_append(const void* q, int64_t q_row_stride, int64_t q_head_stride, const void* k,
                                       int64_t k_row_stride, int64_t k_head_stride, const void* v, int64_t v_row_stride,
                                       int64_t v_head_stride, const float* q_norm_weight, const float* k_norm_weight,
                                       const float* cos, const float* sin, int64_t rope_rows, const int64_t* positions,
                                       int64_t n_rows, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, float eps,
                                       int32_t dtype, void* q_out, int64_t q_out_row_stride, int64_t q_out_head_stride,
                                       void* k_codes, void* v_codes, float* k_scales, float* v_scales, int32_t num_pages,
                                       int32_t page_size, int32_t code, const int64_t* write_slots, void* stream) {
  const int bad = check_pool(num_pages, page_size, n_kv_heads, head_dim, code);
  if (bad != HX_OK) return bad;
  if (dtype != HX_DTYPE_BF16 && dtype != HX_DTYPE_FP16) return HX_E_UNSUPPORTED;
  if (n_rows < 0 || n_q_heads < 1 || rope_rows < 1 || !(eps >= 0.f)) return HX_E_INVALID_ARG;
  if (n_rows == 0) return HX_OK;
  if (!q || !k || !v || !q_norm_weight || !k_norm_weight || !cos || !sin || !positions || !q_out || !k_codes ||
      !v_codes || !k_scales || !v_scales || !write_slots || misaligned(k_codes, 16) || misaligned(v_codes, 16) ||
      misaligned(q_norm_weight, 16) || misaligned(k_norm_weight, 16) || misaligned(cos, 16) || misaligned(sin, 16))
    return HX_E_INVALID_ARG;
  WriteArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.q_row = q_row_stride;
  a.q_head = q_head_stride;
  a.k_row = k_row_stride;
  a.k_head = k_head_stride;
  a.v_row = v_row_stride;
  a.v_head = v_head_stride;
  a.q_norm = q_norm_weight;
  a.k_norm = k_norm_weight;
  a.cos = cos;
  a.sin = sin;
  a.rope_rows = rope_rows;
  a.positions = positions;
  a.n_rows = n_rows;
  a.hq = n_q_heads;
  a.hkv = n_kv_heads;
  a.head_dim = head_dim;
  a.eps = eps;
  a.q_out = static_cast<uint16_t*>(q_out);
  a.qo_row = q_out_row_stride;
  a.qo_head = q_out_head_stride;
  a.codes[0] = static_cast<uint8_t*>(k_codes);
  a.codes[1] = static_cast<uint8_t*>(v_codes);
  a.scales[0] = k_scales;
  a.scales[1] = v_scales;
  a.pool_rows = (int64_t)num_pages * page_size;
  a.page = page_size;
  a.slots = write_slots;
  return launch_write<true>(a, dtype, code, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int hx_kv8_gather(const void* codes, const float* scales, int32_t num_pages, int32_t page_size,
                             int32_t n_kv_heads, int32_t head_dim, int32_t code, const int32_t* pages, int32_t n_pages,
                             int64_t length, int32_t dtype, void* out, void* stream) {
  const int bad = check_pool(num_pages, page_size, n_kv_heads, head_dim, code);
  if (bad != HX_OK) return bad;
  if (dtype != HX_DTYPE_BF16 && dtype != HX_DTYPE_FP16 && dtype != HX_DTYPE_FP32) return HX_E_UNSUPPORTED;
  if (n_pages < 0 || length < 0 || length > (int64_t)n_pages * page_size) return HX_E_INVALID_ARG;
  if (length == 0) return HX_OK;
  if (!codes || !scales || !pages || !out || misaligned(codes, 16) || misaligned(out, 16)) return HX_E_INVALID_ARG;
  ReadArgs a{static_cast<const uint8_t*>(codes), scales, num_pages, page_size, n_kv_heads, head_dim, pages, length, out};
  const int pieces = head_dim / (dtype == HX_DTYPE_FP32 ? 4 : 8);
  int64_t wgs = (length * pieces + 4 * kThreads - 1) / (4 * kThreads);
  const int64_t most = 65536 / n_kv_heads + 1;
  wgs = wgs < most ? wgs : most;
  if (wgs * n_kv_heads > kMostItems / kThreads) return HX_E_UNSUPPORTED;
  const dim3 grid((unsigned)(wgs * n_kv_heads));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, a, pieces, (uint32_t)wgs); };
  if (code == HX_CODE_E4M3) {
    if (dtype == HX_DTYPE_BF16) launch(kv8_read_kernel<__bf16, hx8::E4m3>);
    else if (dtype == HX_DTYPE_FP16) launch(kv8_read_kernel<_Float16, hx8::E4m3>);
    else launch(kv8_read_kernel<float, hx8::E4m3>);
  } else {
    if (dtype == HX_DTYPE_BF16) launch(kv8_read_kernel<__bf16, hx8::Int8>);
    else if (dtype == HX_DTYPE_FP16) launch(kv8_read_kernel<_Float16, hx8::Int8>);
    else launch(kv8_read_kernel<float, hx8::Int8>);
  }
  return hx::status_from_hip(hipGetLastError());
}
