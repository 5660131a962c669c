// The decoder block's products with 4-bit weights and group scales, for up to 64 rows (gfx950).
//
// W[n][k] = scale[g][n] * (q[n][k] - zero[g][n]) with q, zero in 0..15 and g = k / group, and
//   y = h W^T,  h = x, or RMSNorm(x) * norm_weight;
//   out = y, residual + y, or silu(y[:, :cols]) * y[:, cols:] (W then holds gate, up rows),
// in fp32 and rounded once at the end.
//
// A product of few rows is a stream of W: a quarter of the bytes of 16-bit weights. Per group
//   sum_k h_k s (q_k - z) = s (sum_k h_k (16 + q_k) - (16 + z) sum_k h_k):
// 16 + q is a bf16 (fp16) number with q in its upper mantissa bits, so a pair of weights costs
// a shift and one and-or, and the sums of h come from one more MFMA against ones. Both sums
// are fp32; the offset 16 makes the terms at most 31 / 15 times as large as they have to be.
//
// Weights are packed in the order in which the MFMA takes them: 1 KiB holds 16 rows x 128 k,
// lane l = 16 c + r of a wave reads 16 bytes, the k elements 32 s + 8 c .. + 7 of row r in its
// word s. Element j of a word sits at bits 4 (j / 2) + 16 (j % 2), where the shift above finds
// elements 2 i and 2 i + 1 at once.
//
// The norm's row factor 1 / rms multiplies y at the end; x * norm_weight is split into two
// bf16 (their sum has 16 bits), each with an MFMA of its own.
//
// A workgroup owns 16 columns of y (SwiGLU: 16 gate and the 16 up columns they multiply) and
// all rows; its waves split K and merge through LDS in wave order.

#include <type_traits>

#include "hx_common.h"

namespace {

constexpr int kI4Block = 128;  // k elements per packed block: one 16-byte load a lane

enum : int { kEpiPlain = 0, kEpiResidual = 1, kEpiSwiglu = 2 };

struct Int4Args {
  const uint16_t* x;
  int64_t x_row;
  const uint8_t* w;       // [rows of W / 16][blocks][64][16]
  const uint16_t* scale;  // [k_pad / group][w_rows_pad]
  const uint8_t* zero;
  int32_t rows, cols, k, blocks, w_pad;  // cols: of the output; w_pad: rows of W, padded to 16
  const float* norm_w;
  float eps;
  const uint16_t* res;
  int64_t res_row;
  uint16_t* out;
  int64_t out_row;
};

// Eight weights of a packed word as 16 + q in the MFMA's element type.
template <typename T>
__device__ __forceinline__ uint4 widen(uint32_t w);
template <>
__device__ __forceinline__ uint4 widen<__bf16>(uint32_t w) {
  constexpr uint32_t m = 0x00780078u, o = 0x41804180u;
  return make_uint4(((w << 3) & m) | o, ((w >> 1) & m) | o, ((w >> 5) & m) | o, ((w >> 9) & m) | o);
}
template <>
__device__ __forceinline__ uint4 widen<_Float16>(uint32_t w) {
  constexpr uint32_t m = 0x03c003c0u, o = 0x4c004c00u;
  return make_uint4(((w << 6) & m) | o, ((w << 2) & m) | o, ((w >> 2) & m) | o, ((w >> 6) & m) | o);
}

// MT: row tiles of 16. G: k elements per group (32, 64 or 128).
template <typename T, bool NORM, int EPI, int MT, int G, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void int4_gemm_kernel(Int4Args a) {
  // The normalised rows are bf16 pairs whatever the element type: x * norm_weight may leave
  // fp16's range, and 16 + q is exact in either.
  typedef typename std::conditional<NORM, __bf16, T>::type M;
  typedef hx::Elem<T> E;
  typedef hx::Elem<M> EM;
  constexpr int NV = EPI == kEpiSwiglu ? 2 : 1;
  constexpr int kSteps = kI4Block / 32, kGroups = kI4Block / G;
  __shared__ __attribute__((aligned(16))) float red[WAVES][MT * NV][256];
  __shared__ float s_ss[WAVES][MT * 16];
  const int tid = hx::tid_x(), lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = hx::wg_x() * 16;
  const int b_begin = (int)((int64_t)a.blocks * w / WAVES), b_end = (int)((int64_t)a.blocks * (w + 1) / WAVES);

  const uint8_t* wp[NV];
  int wrow[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    // A column past the last reads a row of W that is there; its sums are not stored.
    wrow[v] = min(n0 + lr, a.cols - 1) + v * a.cols;
    wp[v] = a.w + ((int64_t)(wrow[v] >> 4) * a.blocks * 64 + (wrow[v] & 15) + 16 * lg) * 16;
  }
  hx::f32x4_t acc[MT][NV];
  float ss[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    ss[t] = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) acc[t][v] = hx::f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  const typename EM::v8 ones = hx::as_v8<M>(hx::ones8<M>());

  for (int b = b_begin; b < b_end; ++b) {
    uint4 wq[NV];
    float sc[NV][kGroups], zp[NV][kGroups];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      wq[v] = hx::ld16_stream(wp[v] + (int64_t)b * 1024);
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const int64_t at = (int64_t)(b * kGroups + g) * a.w_pad + wrow[v];
        sc[v][g] = E::lo(a.scale[at]);
        zp[v][g] = 16.f + (float)a.zero[at];
      }
    }
    hx::f32x4_t ga[MT][NV], gx[MT];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int k0 = b * kI4Block + 32 * s + 8 * lg;
      const bool in = k0 < a.k;
      uint4 wf[NV];
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const uint32_t wd[4] = {wq[v].x, wq[v].y, wq[v].z, wq[v].w};
        wf[v] = widen<M>(wd[s]);
      }
      float nw[8];
      if constexpr (NORM) {
#pragma unroll
        for (int i = 0; i < 8; ++i) nw[i] = 0.f;
        if (in) {
          const float4 lo = *reinterpret_cast<const float4*>(a.norm_w + k0);
          const float4 hi = *reinterpret_cast<const float4*>(a.norm_w + k0 + 4);
          nw[0] = lo.x, nw[1] = lo.y, nw[2] = lo.z, nw[3] = lo.w;
          nw[4] = hi.x, nw[5] = hi.y, nw[6] = hi.z, nw[7] = hi.w;
        }
      }
      if (s % (G / 32) == 0) {
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          gx[t] = hx::f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int v = 0; v < NV; ++v) ga[t][v] = hx::f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
      }
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const int row = 16 * t + lr;
        uint4 xv = hx::zero4();
        if (in && row < a.rows) xv = *reinterpret_cast<const uint4*>(a.x + (int64_t)row * a.x_row + k0);
        if constexpr (NORM) {
          const uint32_t wd[4] = {xv.x, xv.y, xv.z, xv.w};
          uint32_t h[4], l[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float e0 = E::lo(wd[q]), e1 = E::hi(wd[q]);
            ss[t] = fmaf(e0, e0, ss[t]);
            ss[t] = fmaf(e1, e1, ss[t]);
            const float p0 = e0 * nw[2 * q], p1 = e1 * nw[2 * q + 1];
            h[q] = hx::pack2_round<M>(p0, p1);
            l[q] = hx::pack2_round<M>(p0 - EM::lo(h[q]), p1 - EM::hi(h[q]));
          }
          const typename EM::v8 xh = hx::as_v8<M>(make_uint4(h[0], h[1], h[2], h[3]));
          const typename EM::v8 xl = hx::as_v8<M>(make_uint4(l[0], l[1], l[2], l[3]));
          gx[t] = EM::mfma16x16x32(xh, ones, gx[t]);
          gx[t] = EM::mfma16x16x32(xl, ones, gx[t]);
#pragma unroll
          for (int v = 0; v < NV; ++v) {
            ga[t][v] = EM::mfma16x16x32(xh, hx::as_v8<M>(wf[v]), ga[t][v]);
            ga[t][v] = EM::mfma16x16x32(xl, hx::as_v8<M>(wf[v]), ga[t][v]);
          }
        } else {
          const typename EM::v8 xf = hx::as_v8<M>(xv);
          gx[t] = EM::mfma16x16x32(xf, ones, gx[t]);
#pragma unroll
          for (int v = 0; v < NV; ++v) ga[t][v] = EM::mfma16x16x32(xf, hx::as_v8<M>(wf[v]), ga[t][v]);
        }
      }
      if (s % (G / 32) == G / 32 - 1) {
        const int g = s / (G / 32);
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc[t][v][i] = fmaf(sc[v][g], fmaf(-zp[v][g], gx[t][i], ga[t][v][i]), acc[t][v][i]);
      }
    }
  }

  // Lane holds column lr of rows 4 lg .. + 3 of each tile.
#pragma unroll
  for (int t = 0; t < MT; ++t) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < 4; ++i) red[w][t * NV + v][16 * (4 * lg + i) + lr] = acc[t][v][i];
    if constexpr (NORM) {
      const float sum = hx::add_xor32(hx::add_xor16(ss[t]));
      if (lane < 16) s_ss[w][16 * t + lr] = sum;
    }
  }
  __syncthreads();
  for (int e = tid; e < MT * 256; e += 64 * WAVES) {
    const int t = e >> 8, row = e >> 4, n = n0 + (e & 15);
    if (row >= a.rows || n >= a.cols) continue;
    float y[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      y[v] = 0.f;
#pragma unroll
      for (int ww = 0; ww < WAVES; ++ww) y[v] += red[ww][t * NV + v][e & 255];
    }
    if constexpr (NORM) {
      float sum = 0.f;
#pragma unroll
      for (int ww = 0; ww < WAVES; ++ww) sum += s_ss[ww][row];
      const float r = rsqrtf(__fadd_rn(__fdiv_rn(sum, (float)a.k), a.eps));
#pragma unroll
      for (int v = 0; v < NV; ++v) y[v] *= r;
    }
    float o = y[0];
    if constexpr (EPI == kEpiSwiglu) o = hx::silu(o) * y[NV - 1];
    if constexpr (EPI == kEpiResidual) o += E::lo(a.res[(int64_t)row * a.res_row + n]);
    a.out[(int64_t)row * a.out_row + n] = E::bits(o);
  }
}

struct DequantArgs {
  const uint8_t* w;
  const uint16_t* scale;
  const uint8_t* zero;
  int32_t w_rows, k, blocks, w_pad, group;
  uint16_t* out;
  int64_t out_row;
};

// One lane per 16 packed bytes: 32 weights of a row, written as four 16-byte pieces.
template <typename T>
__global__ __launch_bounds__(256) void int4_dequant_kernel(DequantArgs a, int64_t units) {
  typedef hx::Elem<T> E;
  const int64_t u = (int64_t)hx::wg_x() * 256 + hx::tid_x();
  if (u >= units) return;
  const int lane = (int)(u & 63);
  const int64_t blk = u >> 6;
  const int b = (int)(blk % a.blocks), row = (int)(blk / a.blocks) * 16 + (lane & 15), lg = lane >> 4;
  if (row >= a.w_rows) return;
  const uint4 q = hx::ld16_stream(a.w + u * 16);
  const uint32_t wd[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int k0 = b * kI4Block + 32 * s + 8 * lg;
    if (k0 >= a.k) return;
    const int64_t at = (int64_t)(k0 / a.group) * a.w_pad + row;
    const float sc = E::lo(a.scale[at]), zp = (float)a.zero[at];
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      o[i] = hx::pack2_round<T>(sc * ((float)(wd[s] >> (4 * i) & 15u) - zp),
                                sc * ((float)(wd[s] >> (4 * i + 16) & 15u) - zp));
    *reinterpret_cast<uint4*>(a.out + (int64_t)row * a.out_row + k0) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

template <typename T, bool NORM, int EPI, int MT, int G>
void launch_one(const Int4Args& a, hipStream_t s) {
  constexpr int kWaves = MT * (EPI == kEpiSwiglu ? 2 : 1) > 4 ? 4 : 8;  // the sums fit 64 KiB of LDS
  hipLaunchKernelGGL((int4_gemm_kernel<T, NORM, EPI, MT, G, kWaves>), dim3((unsigned)((a.cols + 15) / 16)),
                     dim3(64 * kWaves), 0, s, a);
}

template <typename T, bool NORM, int EPI, int MT>
void launch_group(const Int4Args& a, int group, hipStream_t s) {
  if (group == 128) launch_one<T, NORM, EPI, MT, 128>(a, s);
  else if (group == 64) launch_one<T, NORM, EPI, MT, 64>(a, s);
  else launch_one<T, NORM, EPI, MT, 32>(a, s);
}

template <typename T, bool NORM, int EPI>
void launch_rows(const Int4Args& a, int group, hipStream_t s) {
  if (a.rows <= 16) launch_group<T, NORM, EPI, 1>(a, group, s);
  else if (a.rows <= 32) launch_group<T, NORM, EPI, 2>(a, group, s);
  else launch_group<T, NORM, EPI, 4>(a, group, s);
}

template <typename T>
void launch_epi(const Int4Args& a, int group, bool swiglu, hipStream_t s) {
  const bool norm = a.norm_w != nullptr;
  if (swiglu && norm) launch_rows<T, true, kEpiSwiglu>(a, group, s);
  else if (swiglu) launch_rows<T, false, kEpiSwiglu>(a, group, s);
  else if (a.res != nullptr && norm) launch_rows<T, true, kEpiResidual>(a, group, s);
  else if (a.res != nullptr) launch_rows<T, false, kEpiResidual>(a, group, s);
  else if (norm) launch_rows<T, true, kEpiPlain>(a, group, s);
  else launch_rows<T, false, kEpiPlain>(a, group, s);
}

bool bad_weight(const void* w, const void* scale, const void* zero, int32_t k, int32_t group) {
  return !w || !scale || !zero || (reinterpret_cast<uintptr_t>(w) & 15) || (reinterpret_cast<uintptr_t>(scale) & 1) ||
         k % group;
}

}  // namespace

extern "C" int hx_int4_gemm(const void* x, int64_t x_row_stride, int64_t rows, const void* packed, const void* scales,
                            const void* zeros, int32_t cols, int32_t k, int32_t group, int32_t dtype,
                            const float* norm_weight, float eps, const void* residual, int64_t residual_row_stride,
                            int32_t swiglu, void* out, int64_t out_row_stride, void* stream) {
  if (dtype != HX_DTYPE_BF16 && dtype != HX_DTYPE_FP16) return HX_E_UNSUPPORTED;
  if (group != 32 && group != 64 && group != 128) return HX_E_UNSUPPORTED;
  if (rows < 0 || cols < 1 || k < 1 || (norm_weight != nullptr && !(eps >= 0.f))) return HX_E_INVALID_ARG;
  if (rows > 64 || cols > (1 << 29) || k > (1 << 29)) return HX_E_UNSUPPORTED;
  if (bad_weight(packed, scales, zeros, k, group) || (swiglu && residual)) return HX_E_INVALID_ARG;
  if (rows == 0) return HX_OK;
  if (!x || !out) return HX_E_INVALID_ARG;
  if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(norm_weight)) & 15) || x_row_stride % 8 ||
      x_row_stride < k)
    return HX_E_INVALID_ARG;
  if (((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(residual)) & 1) || out_row_stride < cols ||
      (residual != nullptr && residual_row_stride < cols))
    return HX_E_INVALID_ARG;
  Int4Args a;
  a.x = static_cast<const uint16_t*>(x);
  a.x_row = x_row_stride;
  a.w = static_cast<const uint8_t*>(packed);
  a.scale = static_cast<const uint16_t*>(scales);
  a.zero = static_cast<const uint8_t*>(zeros);
  a.rows = (int32_t)rows;
  a.cols = cols;
  a.k = k;
  a.blocks = (k + kI4Block - 1) / kI4Block;
  a.w_pad = ((swiglu ? 2 * cols : cols) + 15) / 16 * 16;
  a.norm_w = norm_weight;
  a.eps = eps;
  a.res = static_cast<const uint16_t*>(residual);
  a.res_row = residual_row_stride;
  a.out = static_cast<uint16_t*>(out);
  a.out_row = out_row_stride;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == HX_DTYPE_BF16) launch_epi<__bf16>(a, group, swiglu != 0, s);
  else launch_epi<_Float16>(a, group, swiglu != 0, s);
  return hx::status_from_hip(hipGetLastError());
}

extern "C" int hx_int4_dequantize(const void* packed, const void* scales, const void* zeros, int32_t weight_rows,
                                  int32_t k, int32_t group, int32_t dtype, void* out, int64_t out_row_stride,
                                  void* stream) {
  if (dtype != HX_DTYPE_BF16 && dtype != HX_DTYPE_FP16) return HX_E_UNSUPPORTED;
  if (group != 32 && group != 64 && group != 128) return HX_E_UNSUPPORTED;
  if (weight_rows < 1 || k < 1 || weight_rows > (1 << 30) || k > (1 << 29)) return HX_E_INVALID_ARG;
  if (bad_weight(packed, scales, zeros, k, group) || !out || (reinterpret_cast<uintptr_t>(out) & 15) ||
      out_row_stride % 8 || out_row_stride < k)
    return HX_E_INVALID_ARG;
  DequantArgs a;
  a.w = static_cast<const uint8_t*>(packed);
  a.scale = static_cast<const uint16_t*>(scales);
  a.zero = static_cast<const uint8_t*>(zeros);
  a.w_rows = weight_rows;
  a.k = k;
  a.blocks = (k + kI4Block - 1) / kI4Block;
  a.w_pad = (weight_rows + 15) / 16 * 16;
  a.group = group;
  a.out = static_cast<uint16_t*>(out);
  a.out_row = out_row_stride;
  const int64_t units = (int64_t)(a.w_pad / 16) * a.blocks * 64;
  if ((units + 255) / 256 > 0x7fffffff) return HX_E_UNSUPPORTED;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)((units + 255) / 256));
  if (dtype == HX_DTYPE_BF16) hipLaunchKernelGGL(int4_dequant_kernel<__bf16>, grid, dim3(256), 0, s, a, units);
  else hipLaunchKernelGGL(int4_dequant_kernel<_Float16>, grid, dim3(256), 0, s, a, units);
  return hx::status_from_hip(hipGetLastError());
}
