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
// a rotation and one and-or, and the sums of h come from one more MFMA against ones. Both sums
// are fp32; the offset 16 makes the terms at most 31 / 15 times as large as they have to be. Where
// they are infinite (an infinite h, or one near the type's largest), the two sums cancel to a NaN:
// such a result is summed again term by term.
//
// Weights are packed in the order in which the MFMA takes them: 1 KiB holds 16 rows x 128 k,
// lane l = 16 c + r of a wave reads 16 bytes, the k elements 32 s + 8 c .. + 7 of row r in its
// word s. Element j of a word sits at bits 3 + 4 (j / 2) + 16 (j % 2), modulo 32: turned by 4 i,
// elements 2 i and 2 i + 1 lie in the upper mantissa bits of a bf16 pair.
//
// The norm's row factor 1 / rms multiplies y at the end; x * norm_weight is split into three
// bf16, which hold fp32's 24 bits. Of up to four rows they are rows 0-3, 4-7 and 8-11 of one MFMA
// operand, at no further cost; of up to eight, rows 0-7 and 8-15 of one and 0-7 of another; of
// up to sixteen, three operands. More rows are normalised by a launch of their own, which knows
// how large they can get, and scaled so that two fp16 hold 23 bits of them.
//
// A workgroup owns 16 to 64 columns of y (SwiGLU: gate and the up columns they multiply) and 16
// (8, 4) rows; its waves split K and merge through LDS in wave order.
//
// A layer of hidden 2560, 32/8 heads of 128 and ffn 9728, W from HBM, 1 / 8 / 16 rows (us): qkv
// 5.7 / 6.9 / 9.2, o 4.2 / 4.6 / 5.4, gate_up 10.3 / 12.0 / 17.2, down 6.9 / 7.6 / 9.5, in all 27 /
// 31 / 41 where the 16-bit products take 60 / 62 / 71; 17 / 64 rows 48 / 65. (Normalised rows in two
// bf16 parts, 16 bits: 27 / 29 / 38, 47 / 61.) gate_up's 26 MB are 2.5 TB/s at one row: about 4 us
// of each launch are its start, the first loads' way and the merge, as for the 16-bit products; the
// rest is the stream of W (25 MB at the copy rate: 5.4), with the address unit close behind (x, W and
// norm weights: 104 cycles a block at 8 rows; 80 with the norm weights loaded once and handed on
// through LDS take the same time), at 64 rows x's way from L2.

#include <type_traits>

#include "hx_common.h"

namespace {

constexpr int kI4Block = 128;  // k elements per packed block: one 16-byte load a lane

struct Int4Args {
  const uint16_t* x;
  const uint16_t* h;  // normalised rows (int4_norm_kernel)
  int64_t x_row;
  const uint8_t* w;       // [rows of W / 16][blocks][64][16]
  const uint32_t* steps;  // [w_pad / 16][blocks][16][128 / group]: the scale, and 16 + zero in the high half
  int32_t rows, cols, k, blocks, w_pad;  // cols: of the output; w_pad: rows of W, padded to 16
  int32_t row_tiles, col_tiles;
  const float* norm_w;
  float eps;
  const uint16_t* res;
  int64_t res_row;
  uint16_t* out;
  int64_t out_row;
};

// Constants of widen, kept in registers: v_and_or_b32 takes no literals, and one scalar operand.
template <typename T>
struct WidenBits {
  uint32_t mask, one;
  __device__ __forceinline__ WidenBits() {
    asm("s_mov_b32 %0, %1" : "=s"(mask) : "n"(__is_same(T, __bf16) ? 0x00780078 : 0x03c003c0));
    asm("v_mov_b32 %0, %1" : "=v"(one) : "n"(__is_same(T, __bf16) ? 0x41804180 : 0x4c004c00));
  }
};

// Eight weights of a packed word as 16 + q in the MFMA's element type.
template <typename T>
__device__ __forceinline__ uint4 widen(uint32_t w, const WidenBits<T>& c) {
  constexpr int kAt = __is_same(T, __bf16) ? 0 : 29;  // fp16's upper mantissa bits lie three further up
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t turned = (kAt + 4 * i) % 32 == 0 ? w : __builtin_amdgcn_alignbit(w, w, (kAt + 4 * i) % 32);
    o[i] = (turned & c.mask) | c.one;
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// Eight fp32 numbers, each as three bf16 ones that add up to it.
__device__ __forceinline__ void split8(const float (&p)[8], uint4 (&part)[3]) {
  typedef hx::Elem<__bf16> B;
  uint32_t w[3][4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float x = p[2 * q], y = p[2 * q + 1];
#pragma unroll
    for (int n = 0; n < 3; ++n) {
      w[n][q] = hx::pack2_round<__bf16>(x, y);
      x -= B::lo(w[n][q]);
      y -= B::hi(w[n][q]);
    }
  }
#pragma unroll
  for (int n = 0; n < 3; ++n) part[n] = make_uint4(w[n][0], w[n][1], w[n][2], w[n][3]);
}

// Eight elements of x times r times norm_weight.
template <typename T>
__device__ __forceinline__ void times8(uint4 u, float r, uint4 na, uint4 nb, float (&p)[8]) {
  typedef hx::Elem<T> E;
  const uint32_t wd[4] = {u.x, u.y, u.z, u.w};
  const uint32_t n[8] = {na.x, na.y, na.z, na.w, nb.x, nb.y, nb.z, nb.w};
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    p[2 * q] = E::lo(wd[q]) * r * __uint_as_float(n[2 * q]);
    p[2 * q + 1] = E::hi(wd[q]) * r * __uint_as_float(n[2 * q + 1]);
  }
}

// More rows than one tile: RMSNorm's results are below sqrt(k) `most`, the largest |norm_weight|.
// Scaled by 2^scale_of they are below 2^15 and go into two fp16, which hold 23 bits of them,
// or of small ones 2^-40 of that bound (fp16's smallest step is 2^-24).
__device__ __forceinline__ int scale_of(float most, int k) {
  const int root = (33 - __builtin_clz(k)) / 2;  // 2^root >= sqrt(k)
  return min(14 + 127 - (int)(__float_as_uint(most) >> 23) - root, 126);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

__device__ __forceinline__ float most_of(float most, uint4 u) {
  most = fmaxf(fmaxf(most, fabsf(__uint_as_float(u.x))), fabsf(__uint_as_float(u.y)));
  return fmaxf(fmaxf(most, fabsf(__uint_as_float(u.z))), fabsf(__uint_as_float(u.w)));
}
__device__ __forceinline__ float wave_most(float v) {
  v = fmaxf(v, hx::dpp<hx::kDppXor1>(v));
  v = fmaxf(v, hx::dpp<hx::kDppXor2>(v));
  v = fmaxf(v, hx::dpp<hx::kDppHalfMirror>(v));
  v = fmaxf(v, hx::dpp<hx::kDppMirror>(v));
  return hx::max_xor32(hx::max_xor16(v));
}

// RMSNorm of row r as two fp16 parts: h holds, per row tile, block of 128 k, part and step, the
// MFMA's operand [lane][8]. The first kHold x 256 pieces of a row stay in registers.
template <typename T>
__global__ __launch_bounds__(256) void int4_norm_kernel(Int4Args a, uint16_t* h) {
  constexpr int kHold = 2;
  __shared__ float s_part[4];
  __shared__ float s_most[4];
  const int row = hx::wg_x(), tid = hx::tid_x(), pieces = a.k / 8, padded = a.blocks * (kI4Block / 8);
  const uint4* x = reinterpret_cast<const uint4*>(a.x + (int64_t)row * a.x_row);
  const uint4* n = reinterpret_cast<const uint4*>(a.norm_w);
  uint4 held[kHold], nw[kHold][2];
#pragma unroll
  for (int i = 0; i < kHold; ++i) {
    const int p = tid + 256 * i;
    held[i] = nw[i][0] = nw[i][1] = hx::zero4();
    if (p >= pieces) continue;
    held[i] = x[p];
    nw[i][0] = n[2 * p];
    nw[i][1] = n[2 * p + 1];
  }
  float ss = 0.f, most = 0.f;
#pragma unroll
  for (int i = 0; i < kHold; ++i) {
    ss = hx::dot8<T>(held[i], held[i], ss);
    most = most_of(most_of(most, nw[i][0]), nw[i][1]);
  }
  for (int p = tid + 256 * kHold; p < pieces; p += 256) {
    const uint4 u = x[p];
    ss = hx::dot8<T>(u, u, ss);
    most = most_of(most_of(most, n[2 * p]), n[2 * p + 1]);
  }
  ss = hx::wave_sum_xor(ss, 1, 32);
  most = wave_most(most);
  if ((tid & 63) == 0) {
    s_part[tid >> 6] = ss;
    s_most[tid >> 6] = most;
  }
  __syncthreads();
  ss = (s_part[0] + s_part[1]) + (s_part[2] + s_part[3]);
  most = fmaxf(fmaxf(s_most[0], s_most[1]), fmaxf(s_most[2], s_most[3]));
  const float r = __builtin_amdgcn_rsqf(__fadd_rn(__fdiv_rn(ss, (float)a.k), a.eps));
  const float scale = power_of_two(scale_of(most, a.k));
  uint4* tile = reinterpret_cast<uint4*>(h) + (int64_t)(row >> 4) * a.blocks * 512 + (row & 15);
  auto put = [&](int p, uint4 u, uint4 na, uint4 nb) __attribute__((always_inline)) {
    typedef hx::Elem<_Float16> H;
    float v[8];
    times8<T>(u, r, na, nb, v);
    uint32_t high[4], low[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float v0 = v[2 * q] * scale, v1 = v[2 * q + 1] * scale;
      high[q] = hx::pack2_round<_Float16>(v0, v1);
      low[q] = hx::pack2_round<_Float16>(v0 - H::lo(high[q]), v1 - H::hi(high[q]));
    }
    uint4* to = tile + (p / 16 * 8 + p / 4 % 4) * 64 + 16 * (p % 4);
    to[0] = make_uint4(high[0], high[1], high[2], high[3]);
    to[256] = make_uint4(low[0], low[1], low[2], low[3]);
  };
#pragma unroll
  for (int i = 0; i < kHold; ++i)
    if (tid + 256 * i < padded) put(tid + 256 * i, held[i], nw[i][0], nw[i][1]);
  for (int p = tid + 256 * kHold; p < padded; p += 256)
    put(p, p < pieces ? x[p] : hx::zero4(), p < pieces ? n[2 * p] : hx::zero4(), p < pieces ? n[2 * p + 1] : hx::zero4());
}

// 16-byte buffer load at byte offset voff + soff.
__device__ __forceinline__ uint4 ld16(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff) {
  const hx::u32x4_t v =
      __builtin_bit_cast(hx::u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, (int)voff, (int)soff, 0));
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// A row's steps of a block: one load whatever the group.
__device__ __forceinline__ void load_steps(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff, uint32_t (&st)[1]) {
  st[0] = __builtin_amdgcn_raw_buffer_load_b32(r, (int)voff, (int)soff, 0);
}
__device__ __forceinline__ void load_steps(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff, uint32_t (&st)[2]) {
  const auto u = __builtin_amdgcn_raw_buffer_load_b64(r, (int)voff, (int)soff, 0);
  st[0] = u[0];
  st[1] = u[1];
}
__device__ __forceinline__ void load_steps(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff, uint32_t (&st)[4]) {
  const uint4 u = ld16(r, voff, soff);
  st[0] = u.x;
  st[1] = u.y;
  st[2] = u.z;
  st[3] = u.w;
}

// How x reaches the MFMA: as it is, up to 4, 8 or 16 rows a tile; normalised on the way, the same;
// or as int4_norm_kernel's parts.
enum : int { kRaw4, kRaw8, kRaw16, kNorm4, kNorm8, kNorm16, kParts16 };

__host__ __device__ constexpr int rows_of(int in) { return in == kNorm4 ? 4 : in == kNorm8 ? 8 : 16; }

// LDS slot of 16-byte piece p of row r: the 16 rows of a fragment read spread over the banks.
__device__ __forceinline__ int turn_piece(int r, int p) { return p ^ (r & 15); }

// Whether one of eight elements is a NaN.
template <typename T>
__device__ __forceinline__ bool has_nan(uint4 u) {
  constexpr uint32_t kInf = __is_same(T, __bf16) ? 0x7f80u : 0x7c00u;
  const uint32_t wd[4] = {u.x, u.y, u.z, u.w};
  bool nan = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) nan |= (wd[i] & 0x7fffu) > kInf || (wd[i] >> 16 & 0x7fffu) > kInf;
  return nan;
}

// sum_k x[k] W[n][k] by one lane: scale (q - zero) is exact in fp32. About a microsecond for every
// 30 elements of k, for rows that have an infinity or leave fp32; a row with a NaN costs one in all.
template <typename T, int G>
__device__ __forceinline__ float sum_of_terms(const Int4Args& a, const uint16_t* x, int n) {
  typedef hx::Elem<T> E;
  constexpr int kGroups = kI4Block / G;
  const int64_t tile = (int64_t)(n >> 4) * a.blocks;
  const uint8_t* const w = a.w + tile * 1024 + (n & 15) * 16;
  const uint32_t* const steps = a.steps + (tile * 16 + (n & 15)) * kGroups;
  float y = 0.f;
#pragma unroll 1
  for (int k0 = 0; k0 < a.k; k0 += 8) {
    const int b = k0 / kI4Block, s = k0 / 32 % 4, c = k0 / 8 % 4;
    const uint32_t step = steps[(int64_t)b * 16 * kGroups + 32 * s / G];
    const uint32_t word = *reinterpret_cast<const uint32_t*>(w + (int64_t)b * 1024 + c * 256 + 4 * s);
    const uint32_t turned = __builtin_amdgcn_alignbit(word, word, 3);
    const uint4 u = *reinterpret_cast<const uint4*>(x + k0);
    const uint32_t wd[4] = {u.x, u.y, u.z, u.w};
    const float sc = E::lo(step), zp = E::hi(step) - 16.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y = fmaf(E::lo(wd[i]), sc * ((float)(turned >> (4 * i) & 15u) - zp), y);
      y = fmaf(E::hi(wd[i]), sc * ((float)(turned >> (4 * i + 16) & 15u) - zp), y);
    }
  }
  return y;
}

// G: k elements per group (32, 64 or 128). NV: W tiles of a wave (SWIGLU: gate tiles, then the up
// tiles they multiply). D: packed blocks in flight per wave.
template <typename T, int IN, bool SWIGLU, int G, int NV, int WAVES, int D>
__global__ __launch_bounds__(64 * WAVES) void int4_gemm_kernel(Int4Args a) {
  constexpr bool kRaw = IN <= kRaw16, kNorm = IN >= kNorm4 && IN <= kNorm16, kTurn = kRaw || kNorm;
  // The parts' type, whatever the element type: 16 + q is exact in either.
  typedef typename std::conditional<kRaw, T, typename std::conditional<kNorm, __bf16, _Float16>::type>::type M;
  typedef hx::Elem<T> E;
  typedef hx::Elem<M> EM;
  typedef typename EM::v8 v8;
  constexpr int kSteps = kI4Block / 32, kGroups = kI4Block / G;
  constexpr int kTiles = SWIGLU ? NV / 2 : NV, kCols = 16 * kTiles;  // of the output
  constexpr int kRows = rows_of(IN);  // of a row tile
  constexpr int kOps = kRaw || IN == kNorm4 ? 1 : IN == kNorm16 ? 3 : 2;  // MFMA operands of a tile's rows
  // Where the parts of up to eight normalised rows lie: operand and first row.
  constexpr bool kFew = IN == kNorm4 || IN == kNorm8;
  constexpr int kAt[3][2] = {{0, 0}, {0, kRows}, {IN == kNorm8 ? 1 : 0, IN == kNorm8 ? 0 : 2 * kRows}};
  // Rows 8-15 of the second operand are one row of zeros.
  constexpr int kSecond = 4096, kZeros = kSecond + 8 * 256;
  constexpr int kTurnBytes = IN == kNorm8 ? kZeros + 256 : IN == kNorm16 ? 8192 : 4096;
  constexpr bool kSplit = IN == kNorm16;  // kept in fp32, split where the MFMA takes them
  constexpr int kLoads = IN == kParts16 ? 2 * kSteps : IN == kRaw4 || IN == kNorm4 ? 1 : IN == kRaw8 || IN == kNorm8 ? 2 : 4;
  __shared__ __attribute__((aligned(16))) float red[WAVES][NV][256];
  __shared__ __attribute__((aligned(16))) uint8_t turn[kTurn ? WAVES : 1][kTurn ? kTurnBytes : 16];
  __shared__ float s_ss[WAVES][16];
  const int tid = hx::tid_x(), lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  // Workgroups go to the XCDs in turn: the row tiles of a column tile share one, and its L2.
  const int xcd = hx::wg_x() % 8, j = hx::wg_x() / 8;
  const int rt = j % a.row_tiles, ct = j / a.row_tiles * 8 + xcd;
  if (ct >= a.col_tiles) return;
  const int n0 = ct * kCols;
  const int b_begin = (int)((int64_t)a.blocks * w / WAVES), b_end = (int)((int64_t)a.blocks * (w + 1) / WAVES);

  // Buffer loads: what varies over the lanes is one offset, what varies over the blocks a scalar
  // one. (With an address per load a third of the instructions were additions.)
  __amdgpu_buffer_rsrc_t wr[NV];
  uint32_t woff[NV], soff[NV];
  const uint32_t sbytes = (uint32_t)(a.blocks * kGroups) * a.w_pad * 4, wbytes = 2u * a.blocks * 1024;
  const __amdgpu_buffer_rsrc_t sr = hx::buffer_rsrc(a.steps, sbytes);
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    // A column past the last reads a row of W that is there; its sums are not stored.
    const int part = v / kTiles, first = min(n0 + 16 * (v % kTiles), a.cols - 1) + part * a.cols;
    const int row = min(first + lr, (part + 1) * a.cols - 1);
    wr[v] = hx::buffer_rsrc(a.w + (int64_t)(first >> 4) * a.blocks * 1024, wbytes);
    woff[v] = (uint32_t)((row >> 4) - (first >> 4)) * a.blocks * 1024 + ((row & 15) + 16 * lg) * 16;
    soff[v] = (uint32_t)((row >> 4) * a.blocks * 16 + (row & 15)) * 4 * kGroups;
  }
  // x is read in whole lines, 16 lanes to the 256 bytes of a row's block, and turned into the
  // MFMA's layout through the wave's part of LDS: lanes next to each other in that layout are
  // different rows, and a load straight into it costs an access per lane (64 cycles of the
  // address unit instead of 16: what bounded this kernel). Rows that are not there are read
  // past the buffer's end (zeros).
  const int rows = min(a.rows - rt * kRows, kRows);
  const uint16_t* xbase = kTurn ? a.x + (int64_t)rt * kRows * a.x_row : a.h + (int64_t)rt * 32 * a.blocks * kI4Block;
  const uint32_t xbytes = kTurn ? (uint32_t)((rows - 1) * a.x_row + a.k) * 2 : (uint32_t)a.blocks * 8192;
  const __amdgpu_buffer_rsrc_t xr = hx::buffer_rsrc(xbase, xbytes);
  const uint32_t nbytes = 4u * a.k;
  const __amdgpu_buffer_rsrc_t nr = hx::buffer_rsrc(kNorm ? a.norm_w : nullptr, kNorm ? nbytes : 0u);
  uint32_t xoff[kLoads];
#pragma unroll
  for (int q = 0; q < kLoads; ++q)
    xoff[q] = !kTurn ? 16u * lane + 1024u * q : 4 * q + lg < rows ? (uint32_t)((4 * q + lg) * a.x_row) * 2 + 16 * lr
                                                                  : 0x80000000u;
  // Loads complete in the order they were issued, so a block's x goes with its weights. Blocks
  // past the wave's last are loaded too, from the end of each buffer: zeros, and no traffic.
  // (With a branch around these loads every trip through the loop waited for all of them.)
  uint4 wq[D][NV], xb[D][kLoads], nb[D][kNorm ? 2 : 1];
  uint32_t st[D][NV][kGroups];
  auto load = [&](int i, int b) __attribute__((always_inline)) {
    const bool in = b < b_end;
    const uint32_t at = in ? (kTurn ? 256u : 8192u) * b : xbytes;
#pragma unroll
    for (int q = 0; q < kLoads; ++q) xb[i][q] = ld16(xr, xoff[q], at);
    if constexpr (kNorm) {
      nb[i][0] = ld16(nr, 32u * lr, in ? 512u * b : nbytes);
      nb[i][1] = ld16(nr, 32u * lr + 16, in ? 512u * b : nbytes);
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      wq[i][v] = hx::ld16_stream(wr[v], woff[v], in ? 1024u * b : wbytes);
      load_steps(sr, soff[v], in ? (uint32_t)b * 64 * kGroups : sbytes, st[i][v]);
    }
  };
#pragma unroll
  for (int i = 0; i < D; ++i) load(i, b_begin + i);

  // The first output element's residual, in flight with the weights.
  const int r_row = rt * kRows + tid / 16, r_col = n0 + tid % 16;
  uint16_t r_first = 0;
  if constexpr (!SWIGLU)
    if (a.res != nullptr && tid < kRows * 16 && r_row < a.rows && r_col < a.cols)
      r_first = a.res[(int64_t)r_row * a.res_row + r_col];

  // The norm weights that give the scale of the normalised rows' parts, in flight with the weights
  // too. (Kept in registers and looked at after the loop they cost occupancy: SwiGLU of 64 rows
  // took 1.2 us longer.)
  float most = 0.f;
  if constexpr (IN == kParts16) {
    const uint4* const n = reinterpret_cast<const uint4*>(a.norm_w);
    for (int p = tid; p < a.k / 4; p += 256 * WAVES) {
      uint4 u[4];  // past the end the last piece again
#pragma unroll
      for (int q = 0; q < 4; ++q) u[q] = n[min(p + 64 * WAVES * q, a.k / 4 - 1)];
#pragma unroll
      for (int q = 0; q < 4; ++q) most = most_of(most, u[q]);
    }
  }

  hx::f32x4_t acc[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) acc[v] = hx::f32x4_t{0.f, 0.f, 0.f, 0.f};
  float ss[kLoads];
#pragma unroll
  for (int q = 0; q < kLoads; ++q) ss[q] = 0.f;
  if constexpr (IN == kNorm8)
    if (lane < 16) reinterpret_cast<uint4*>(turn[w] + kZeros)[lane] = hx::zero4();
  const v8 ones = hx::as_v8<M>(hx::ones8<M>());
  const WidenBits<M> bits;
  auto consume = [&](int i, int b) __attribute__((always_inline)) {
    uint4 xf[kSteps][kOps];
    if constexpr (kTurn) {
#pragma unroll
      for (int q = 0; q < kLoads; ++q) {
        uint4 u = xb[i][q];
        if (G < kI4Block && b * kI4Block + 8 * lr >= a.k) u = hx::zero4();  // the next row's
        const int r = 4 * q + lg;
        uint8_t* to = turn[w] + 256 * r + 16 * turn_piece(r, lr);
        if constexpr (kNorm) {
          // x * norm_weight; 1 / rms multiplies the sums at the end.
          float p[8];
          times8<T>(u, 1.f, nb[i][0], nb[i][kNorm], p);
          ss[q] = hx::dot8<T>(u, u, ss[q]);
          if constexpr (kFew) {
            uint4 part[3];
            split8(p, part);
#pragma unroll
            for (int n = 0; n < 3; ++n) {
              const int r2 = r + kAt[n][1];
              *reinterpret_cast<uint4*>(turn[w] + kSecond * kAt[n][0] + 256 * r2 + 16 * turn_piece(r2, lr)) = part[n];
            }
          } else {  // a row's first halves of its pieces of eight, then the second ones
            float4* const to4 = reinterpret_cast<float4*>(turn[w] + 512 * r) + turn_piece(r, lr);
            to4[0] = make_float4(p[0], p[1], p[2], p[3]);
            to4[16] = make_float4(p[4], p[5], p[6], p[7]);
          }
        } else {
          *reinterpret_cast<uint4*>(to) = u;
        }
      }
      // One wave's LDS accesses complete in order: the fences hold the compiler to it. Rows that
      // are not stored here hold anything: their sums are not used, and rows do not mix.
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      if constexpr (kSplit) {
        const float4* const from = reinterpret_cast<const float4*>(turn[w] + 512 * lr) + turn_piece(lr, 4 * s + lg);
        const float4 a4 = from[0], b4 = from[16];
        const float p[8] = {a4.x, a4.y, a4.z, a4.w, b4.x, b4.y, b4.z, b4.w};
        split8(p, xf[s]);
      } else {
#pragma unroll
        for (int o = 0; o < kOps; ++o)
          xf[s][o] = kTurn ? *reinterpret_cast<const uint4*>(turn[w] + kSecond * o + 256 * (o == 0 ? lr : min(lr, 8)) +
                                                             16 * turn_piece(lr, 4 * s + lg))
                           : xb[i][(kSteps * o + s) % kLoads];
      }
    }
    if constexpr (kTurn) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      hx::f32x4_t ga[NV], gx{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < NV; ++v) ga[v] = hx::f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = g * (G / 32); s < (g + 1) * (G / 32); ++s) {
#pragma unroll
        for (int o = 0; o < kOps; ++o) gx = EM::mfma16x16x32(hx::as_v8<M>(xf[s][o]), ones, gx);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const uint32_t wd[4] = {wq[i][v].x, wq[i][v].y, wq[i][v].z, wq[i][v].w};
          const v8 wf = hx::as_v8<M>(widen<M>(wd[s], bits));
#pragma unroll
          for (int o = 0; o < kOps; ++o) ga[v] = EM::mfma16x16x32(hx::as_v8<M>(xf[s][o]), wf, ga[v]);
        }
      }
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const float sc = E::lo(st[i][v][g]), zp = E::hi(st[i][v][g]);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[v][e] = fmaf(sc, fmaf(-zp, gx[e], ga[v][e]), acc[v][e]);
      }
    }
  };
  for (int b = b_begin; b < b_end; b += D) {
#pragma unroll
    for (int i = 0; i < D; ++i) {
      if (b + i < b_end) consume(i, b + i);  // wave-uniform
      load(i, b + i + D);
    }
  }

  // Lane holds column lr of rows 4 lg .. + 3.
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int i = 0; i < 4; ++i) red[w][v][16 * (4 * lg + i) + lr] = acc[v][i];
  if constexpr (kNorm) {
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      const float sum = hx::wave_sum_xor(ss[q], 1, 8);  // over the row's 16 lanes
      if (lr == 0) s_ss[w][4 * q + lg] = sum;
    }
  }
  if constexpr (IN == kParts16) {
    most = wave_most(most);
    if (lane == 0) s_ss[w][0] = most;
  }
  __syncthreads();
  for (int e = tid; e < kTiles * kRows * 16; e += 64 * WAVES) {
    const int v0 = e / (kRows * 16), at = e % (kRows * 16);
    const int row = rt * kRows + at / 16, n = n0 + 16 * v0 + at % 16;
    constexpr int kSums = SWIGLU ? 2 : 1;
    float y[kSums];
#pragma unroll
    for (int v = 0; v < kSums; ++v) {
      y[v] = 0.f;
#pragma unroll
      for (int ww = 0; ww < WAVES; ++ww) {
        y[v] += red[ww][v0 + v * kTiles][at];
        if constexpr (kFew) y[v] += red[ww][v0 + v * kTiles][at + 16 * kRows];  // the second parts
        if constexpr (IN == kNorm4) y[v] += red[ww][v0 + v * kTiles][at + 32 * kRows];  // the third
      }
    }
    const bool there = row < a.rows && n < a.cols;
    if constexpr (kRaw) {
      bool odd = false;
#pragma unroll
      for (int v = 0; v < kSums; ++v) odd |= there && !hx::is_finite(y[v]);
      const uint64_t odds = __builtin_amdgcn_ballot_w64(odd);
      if (__builtin_expect(odds != 0, 0)) {
        // Sixteen lanes share a row of x. One with a NaN in it, which garbage may hold, stays NaN.
        const uint16_t* const x = a.x + (int64_t)row * a.x_row;
        bool nan = false;
        if ((odds >> (lane & 48) & 0xffff) != 0)
          for (int p = lr; p < a.k / 8 && !nan; p += 64)
#pragma unroll
            for (int i = 0; i < 64; i += 16)
              if (p + i < a.k / 8) nan |= has_nan<T>(reinterpret_cast<const uint4*>(x)[p + i]);
        const uint64_t nans = __builtin_amdgcn_ballot_w64(nan);
        if ((nans >> (lane & 48) & 0xffff) == 0) {
#pragma unroll
          for (int v = 0; v < kSums; ++v)
            if (odd && !hx::is_finite(y[v])) y[v] = sum_of_terms<T, G>(a, x, n + v * a.cols);
        }
      }
    }
    if (!there) continue;
    if constexpr (kNorm) {
      float sum = 0.f;
#pragma unroll
      for (int ww = 0; ww < WAVES; ++ww) sum += s_ss[ww][at / 16];
      const float r = __builtin_amdgcn_rsqf(__fadd_rn(__fdiv_rn(sum, (float)a.k), a.eps));
#pragma unroll
      for (int v = 0; v < kSums; ++v) y[v] *= r;
    }
    if constexpr (IN == kParts16) {
      float top = 0.f;
#pragma unroll
      for (int ww = 0; ww < WAVES; ++ww) top = fmaxf(top, s_ss[ww][0]);
      const float unscale = power_of_two(-scale_of(top, a.k));
#pragma unroll
      for (int v = 0; v < kSums; ++v) y[v] *= unscale;
    }
    float o = y[0];
    if constexpr (SWIGLU) o = hx::silu(o) * y[kSums - 1];
    else if (a.res != nullptr) o += E::lo(e < kRows * 16 && e == tid ? r_first : a.res[(int64_t)row * a.res_row + n]);
    a.out[(int64_t)row * a.out_row + n] = E::bits(o);
  }
}

struct DequantArgs {
  const uint8_t* w;
  const uint32_t* steps;
  int32_t w_rows, k, blocks, group;
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
    const uint32_t step = a.steps[(blk * 16 + (lane & 15)) * (kI4Block / a.group) + 32 * s / a.group];
    const float sc = E::lo(step), zp = E::hi(step) - 16.f;
    const uint32_t turned = __builtin_amdgcn_alignbit(wd[s], wd[s], 3);
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      o[i] = hx::pack2_round<T>(sc * ((float)(turned >> (4 * i) & 15u) - zp),
                                sc * ((float)(turned >> (4 * i + 16) & 15u) - zp));
    *reinterpret_cast<uint4*>(a.out + (int64_t)row * a.out_row + k0) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

template <typename T, int IN, bool SWIGLU, int G, int NV>
int launch_tiles(Int4Args a, hipStream_t s) {
  constexpr int kCols = SWIGLU ? 8 * NV : 16 * NV, kRows = rows_of(IN);
  a.row_tiles = (a.rows + kRows - 1) / kRows;
  a.col_tiles = (a.cols + kCols - 1) / kCols;
  // Waves that split K, and blocks in flight. bf16, 1 / 8 / 16 rows, W from HBM (us): 9728 + 9728
  // columns of 2560 with SwiGLU, 4 waves and 1 block 10.3 / 12.1 / 17.1, 2 blocks 10.3 / 12.4 /
  // 17.4, 8 waves 10.2 / 13.3 / 25.4 (their LDS leaves one workgroup to a CU at 16 rows); 2560
  // columns of 9728, 8 waves and 2 blocks 6.6 / 7.4 / 9.4, 3 blocks 6.3 / 7.5 / 9.8, 4 waves
  // 9.1 / 10.0 / 11.0. Three W tiles and more are enough in flight at one block: 64 rows of the
  // columns of 9728, three tiles, 11.9, 2 blocks 12.7; 6144 columns of 2560, normalised, four tiles,
  // 17 / 64 rows, 8 waves and 1 block 11.6 / 16.2, 4 waves 13.2 / 16.5, 4 waves and 2 blocks 11.8 /
  // 16.0 (SwiGLU's 9728 20.2 / 29.0, 2 blocks 21.9 / 31.9).
  constexpr int kWaves = SWIGLU ? 4 : 8, kDepth = SWIGLU || NV >= 3 ? 1 : 2;
  const auto fn = int4_gemm_kernel<T, IN, SWIGLU, G, NV, kWaves, kDepth>;
  hipLaunchKernelGGL(fn, dim3((unsigned)((a.col_tiles + 7) / 8 * 8 * a.row_tiles)), dim3(64 * kWaves), 0, s, a);
  return hx::status_from_hip(hipGetLastError());
}

// W tiles of a workgroup. Two where x costs more than a load (6144 columns of 2560, normalised,
// 1 / 8 / 16 rows: 5.5 / 6.8 / 9.0 us, one tile 5.9 / 7.6 / 14.1), one where it does not (2560
// columns of 9728: 6.6 / 7.4 / 9.4, two tiles 8.2 / 9.2 / 11.0). Past one row tile, x's way from
// L2 bounds the kernel and more tiles share it: four of normalised rows, whose parts are twice
// the bytes (17 / 64 rows, 6144 columns 11.6 / 16.2, two tiles 14.0 / 18.9, eight 14.8 / 15.6; 9728
// columns and SwiGLU 20.0 / 29.0, two 24.0 / 36.6, eight 25.5 / 36.3), otherwise the fewest of two,
// three and four that make at most one workgroup a CU (2560 columns of 9728, 17 / 48 rows two 10.1 /
// 10.7, four 13.0 / 13.6; 64 rows two 17.1, three 11.9, four 13.5).
template <typename T, int IN, bool SWIGLU, int NV = SWIGLU || IN >= kNorm4 ? 2 : 1>
int launch_group(const Int4Args& a, int group, hipStream_t s) {
  if (group == 128) return launch_tiles<T, IN, SWIGLU, 128, NV>(a, s);
  if (group == 64) return launch_tiles<T, IN, SWIGLU, 64, NV>(a, s);
  return launch_tiles<T, IN, SWIGLU, 32, NV>(a, s);
}

// Rows that each workgroup normalises on their way in; more of them are normalised once, in a
// launch of about 3 us (6144 columns of 2560: 16 rows 9.0 us, 17 rows 11.6, 64 rows 16.2; normalised
// by every workgroup 17 rows 16.6, 64 rows 24.7).
constexpr int kFusedNormRows = 16;

template <typename T, bool SWIGLU>
int launch_in(const Int4Args& a, int group, hipStream_t s) {
  constexpr int kRawPair = SWIGLU ? 16 : 32;  // columns of two W tiles
  if (a.norm_w == nullptr) {
    if (a.rows <= 4) return launch_group<T, kRaw4, SWIGLU>(a, group, s);
    if (a.rows <= 8) return launch_group<T, kRaw8, SWIGLU>(a, group, s);
    if (a.rows <= 16) return launch_group<T, kRaw16, SWIGLU>(a, group, s);
    const int tiles = (a.rows + 15) / 16;
    if (tiles * (int64_t)((a.cols + kRawPair - 1) / kRawPair) <= 256) return launch_group<T, kRaw16, SWIGLU, 2>(a, group, s);
    if constexpr (!SWIGLU)
      if (tiles * (int64_t)((a.cols + 47) / 48) <= 256) return launch_group<T, kRaw16, SWIGLU, 3>(a, group, s);
    return launch_group<T, kRaw16, SWIGLU, 4>(a, group, s);
  }
  if (a.rows <= 4) return launch_group<T, kNorm4, SWIGLU>(a, group, s);
  if (a.rows <= 8) return launch_group<T, kNorm8, SWIGLU>(a, group, s);
  if (a.rows <= kFusedNormRows) return launch_group<T, kNorm16, SWIGLU>(a, group, s);
  hipLaunchKernelGGL(int4_norm_kernel<T>, dim3((unsigned)a.rows), dim3(256), 0, s, a, const_cast<uint16_t*>(a.h));
  return launch_group<T, kParts16, SWIGLU, 4>(a, group, s);
}

bool bad_weight(const void* w, const void* steps, int32_t k, int32_t group) {
  return !w || !steps || ((reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(steps)) & 15) || k % group;
}

}  // namespace

extern "C" size_t hx_int4_workspace_bytes(int64_t rows, int32_t k, int32_t norm) {
  const int64_t blocks = ((int64_t)k + kI4Block - 1) / kI4Block;
  if (!norm || rows <= kFusedNormRows || k < 1) return 0;
  return (size_t)((rows + 15) / 16 * 32) * (size_t)blocks * kI4Block * 2;
}

extern "C" int hx_int4_gemm(const void* x, int64_t x_row_stride, int64_t rows, const void* packed, const void* steps,
                            int32_t cols, int32_t k, int32_t group, int32_t dtype,
                            const float* norm_weight, float eps, const void* residual, int64_t residual_row_stride,
                            int32_t swiglu, void* out, int64_t out_row_stride, void* workspace,
                            size_t workspace_bytes, void* stream) {
  if (dtype != HX_DTYPE_BF16 && dtype != HX_DTYPE_FP16) return HX_E_UNSUPPORTED;
  if (group != 32 && group != 64 && group != 128) return HX_E_UNSUPPORTED;
  if (rows < 0 || cols < 1 || k < 1 || (norm_weight != nullptr && !(eps >= 0.f))) return HX_E_INVALID_ARG;
  // 32-bit buffer offsets within a row tile of x, a column tile of W and the steps.
  if (rows > 64 || cols > (1 << 26) || k > (1 << 20) || x_row_stride > (1 << 26) ||
      ((int64_t)k / group + 4) * (2 * (int64_t)cols + 16) * 4 > 0x7fffffff)
    return HX_E_UNSUPPORTED;
  if (bad_weight(packed, steps, k, group) || (swiglu && residual)) return HX_E_INVALID_ARG;
  if (rows == 0) return HX_OK;
  if (!x || !out) return HX_E_INVALID_ARG;
  if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(norm_weight)) & 15) || x_row_stride % 8 ||
      x_row_stride < k)
    return HX_E_INVALID_ARG;
  if (((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(residual)) & 1) || out_row_stride < cols ||
      (residual != nullptr && residual_row_stride < cols))
    return HX_E_INVALID_ARG;
  const size_t need = hx_int4_workspace_bytes(rows, k, norm_weight != nullptr);
  if (need && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < need))
    return HX_E_WORKSPACE;
  Int4Args a;
  a.x = static_cast<const uint16_t*>(x);
  a.h = static_cast<const uint16_t*>(workspace);
  a.x_row = x_row_stride;
  a.w = static_cast<const uint8_t*>(packed);
  a.steps = static_cast<const uint32_t*>(steps);
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
  if (dtype == HX_DTYPE_BF16)
    return swiglu ? launch_in<__bf16, true>(a, group, s) : launch_in<__bf16, false>(a, group, s);
  return swiglu ? launch_in<_Float16, true>(a, group, s) : launch_in<_Float16, false>(a, group, s);
}

extern "C" int hx_int4_dequantize(const void* packed, const void* steps, int32_t weight_rows, int32_t k, int32_t group,
                                  int32_t dtype, void* out, int64_t out_row_stride,
                                  void* stream) {
  if (dtype != HX_DTYPE_BF16 && dtype != HX_DTYPE_FP16) return HX_E_UNSUPPORTED;
  if (group != 32 && group != 64 && group != 128) return HX_E_UNSUPPORTED;
  if (weight_rows < 1 || k < 1 || weight_rows > (1 << 30) || k > (1 << 29)) return HX_E_INVALID_ARG;
  if (bad_weight(packed, steps, k, group) || !out || (reinterpret_cast<uintptr_t>(out) & 15) ||
      out_row_stride % 8 || out_row_stride < k)
    return HX_E_INVALID_ARG;
  DequantArgs a;
  a.w = static_cast<const uint8_t*>(packed);
  a.steps = static_cast<const uint32_t*>(steps);
  a.w_rows = weight_rows;
  a.k = k;
  a.blocks = (k + kI4Block - 1) / kI4Block;
  a.group = group;
  a.out = static_cast<uint16_t*>(out);
  a.out_row = out_row_stride;
  const int64_t units = ((int64_t)weight_rows + 15) / 16 * a.blocks * 64;
  if (units > 0xffffff00ll) return HX_E_UNSUPPORTED;  // work-items of a launch: 32 bits
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)((units + 255) / 256));
  if (dtype == HX_DTYPE_BF16) hipLaunchKernelGGL(int4_dequant_kernel<__bf16>, grid, dim3(256), 0, s, a, units);
  else hipLaunchKernelGGL(int4_dequant_kernel<_Float16>, grid, dim3(256), 0, s, a, units);
  return hx::status_from_hip(hipGetLastError());
}
