// Attention over selected blocks of the paged KV cache (gfx950): the key bounds of each block,
// the selection by them, and the attention that reads the selected blocks only.
//
// A block is `block` consecutive tokens of a page (a power of two from 16 that divides the
// page). Per block and KV head
//   lower[d] = min_j k_j[d],  upper[d] = max_j k_j[d]           (block_bounds_kernel)
// bound the scores of its keys: q . k_j <= sum_d max(q[d] lower[d], q[d] upper[d]). Summed over
// the G query heads that share the KV head the bound is linear in two vectors,
//   s = sum_d (sum_g min(q_g[d], 0)) lower[d] + (sum_g max(q_g[d], 0)) upper[d]
// (an infinite bound whose vector is 0 there left out: no query takes it),
// and the blocks with the largest s, with the first `sink` and the last `recent` ones, are the
// row's selection for that KV head (block_scores_kernel, select_blocks_kernel). The attention is
// the softmax over the keys of those blocks alone (sparse_attn_kernel).

#include "hx_common.h"

namespace {

// Work-items of a launch: a 32-bit number.
constexpr int64_t kMostItems = 0xffffffff;

// HIP's min and max go through double for some mixes of 64-bit types.
template <typename I>
__device__ __forceinline__ I least_of(I a, I b) { return b < a ? b : a; }
template <typename I>
__device__ __forceinline__ I most_of(I a, I b) { return a < b ? b : a; }

// ------------------------------------------------------------------------- key bounds
//
// The bounds of every block that a tick's new tokens touched, from all of its keys so far and
// never from its former bounds: a dropped draft or a reused page leaves no trace in them, and
// the order of ticks none either. At most `block` keys are read for a sequence's first block.
// A workgroup takes one block and 32 16-byte pieces of the key rows, eight tokens at a time.
//
// 8 heads of 128, blocks of 64: the last blocks of 64 sequences (4.8 MB) 5.8 us, three chunks of
// 7145 tokens in all (15 MB) 7.2: the launch and three loads that wait for one another, not HBM.

constexpr int kBdThreads = 256;
constexpr int kBdPieces = 32, kBdTokens = kBdThreads / kBdPieces;

typedef short s16x2_t __attribute__((ext_vector_type(2)));

struct BoundsArgs {
  const uint16_t* k;
  uint16_t* bounds;  // [num_pages][page / block][heads][2][head_dim]
  int32_t num_pages, page, block, pieces, pieces_head;  // 16-byte pieces of a token row, of a head
  const int32_t* table;
  int64_t table_stride;
  int32_t table_width;
  const int32_t* cu_q;
  const int32_t* used;
  int32_t groups, chunks;  // workgroups along a sequence's blocks and along the pieces
  uint16_t inf;            // bits of the type's infinity
};

// bf16 / fp16 bits in the order of their values as signed integers, and back (an involution).
__device__ __forceinline__ s16x2_t ordered(s16x2_t x) { return x ^ ((x >> 15) & (short)0x7fff); }

__global__ __launch_bounds__(kBdThreads) void block_bounds_kernel(BoundsArgs a) {
  __shared__ s16x2_t s_low[kBdTokens][kBdPieces][4], s_high[kBdTokens][kBdPieces][4], s_mag[kBdTokens][kBdPieces][4];
  const int tid = hx::tid_x(), at = tid % kBdPieces, tl = tid / kBdPieces;
  int wg = hx::wg_x();
  const int piece = wg % a.chunks * kBdPieces + at;
  wg /= a.chunks;
  const int g = wg % a.groups, b = wg / a.groups;
  const int len = a.used[b], fresh = min(a.cu_q[b + 1] - a.cu_q[b], len);
  if (fresh <= 0) return;
  const int per_page = a.page / a.block, last = (len - 1) / a.block;
  for (int j = (len - fresh) / a.block + g; j <= last; j += a.groups) {
    if (j / per_page >= a.table_width) return;
    const int page = a.table[(int64_t)b * a.table_stride + j / per_page];
    if (page < 0 || page >= a.num_pages) continue;  // uniform over the workgroup
    const int64_t block0 = (int64_t)page * per_page + j % per_page;
    const int keys = min(a.block, len - j * a.block);
    s16x2_t low[4], high[4], mag[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      low[q] = s16x2_t{0x7fff, 0x7fff};
      high[q] = s16x2_t{(short)0x8000, (short)0x8000};
      mag[q] = s16x2_t{0, 0};
    }
    if (piece < a.pieces) {
      const uint4* p = reinterpret_cast<const uint4*>(a.k) + block0 * a.block * a.pieces + piece;
#pragma unroll 8
      for (int i = tl; i < keys; i += kBdTokens) {
        const uint4 u = p[(int64_t)i * a.pieces];
        const uint32_t wd[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const s16x2_t x = __builtin_bit_cast(s16x2_t, wd[q]), o = ordered(x);
          low[q] = __builtin_elementwise_min(low[q], o);
          high[q] = __builtin_elementwise_max(high[q], o);
          mag[q] = __builtin_elementwise_max(mag[q], (s16x2_t)(x & (short)0x7fff));
        }
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      s_low[tl][at][q] = low[q];
      s_high[tl][at][q] = high[q];
      s_mag[tl][at][q] = mag[q];
    }
    __syncthreads();
    if (tl == 0 && piece < a.pieces) {
      uint32_t lo[4], hi[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
#pragma unroll
        for (int t = 1; t < kBdTokens; ++t) {
          low[q] = __builtin_elementwise_min(low[q], s_low[t][at][q]);
          high[q] = __builtin_elementwise_max(high[q], s_high[t][at][q]);
          mag[q] = __builtin_elementwise_max(mag[q], s_mag[t][at][q]);
        }
        s16x2_t l = ordered(low[q]), h = ordered(high[q]);
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if ((uint16_t)mag[q][e] > a.inf) l[e] = h[e] = 0x7fff;  // a NaN key: both bounds NaN
        lo[q] = __builtin_bit_cast(uint32_t, l);
        hi[q] = __builtin_bit_cast(uint32_t, h);
      }
      const int64_t row = block0 * (a.pieces / a.pieces_head) + piece / a.pieces_head;
      uint4* out = reinterpret_cast<uint4*>(a.bounds) + row * 2 * a.pieces_head + piece % a.pieces_head;
      out[0] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      out[a.pieces_head] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    }
    __syncthreads();
  }
}

// -------------------------------------------------------------------------- selection
//
// block_scores_kernel reads the bounds once, HBM-bound: LANES lanes hold a query row's sums for
// one KV head, eight dims each, and take kScPer blocks, all in flight at once. The sums are
// 64-bit: the blocks at the border of a selection lie close together, and a sum in another order
// would choose others. Their keys (64-bit integers in the scores' order) go to the workspace.
// select_blocks_kernel holds a row's keys in registers and finds the r-th largest free one by
// counting keys in bins.
//
// 8 heads of 128: 64 rows of 256-640 blocks (113 MB of bounds) 31 us (3.6 TB/s; the loads alone,
// in the same order, 24.5: what is left is 64-bit arithmetic that they do not hide) and 5.7 us
// for the selection; one row of 2047 blocks 6.2 and 6.2 us, latency both. One workgroup a row and
// head for scores and selection: 71 and 137 us.

constexpr int kScThreads = 256;
constexpr int kScPer = 4;
constexpr int kSelMaxBlocks = 16384;  // keys in the registers of one workgroup
constexpr int kSelBins = 1024, kSelPasses = 7;  // 10 bits of the range a pass

struct SelectArgs {
  const uint16_t* q;
  int64_t q_row, q_head, q_rows;
  const int64_t* rows;     // query row of each selection (null: itself)
  const int32_t* row_seq;  // its sequence (null: itself)
  const int32_t* keys;
  int32_t n_heads, group, head_dim;
  const uint16_t* bounds;
  int32_t num_pages, page, block;
  const int32_t* table;
  int64_t table_stride;
  int32_t batch, table_width;
  int32_t budget, sink, recent;
  uint32_t page_magic;             // 2^32 / blocks of a page, rounded up
  int32_t chunks, stretch, most;  // workgroups along a row's blocks, blocks of one; blocks the table covers
  uint64_t* order;       // [n][n_heads][most]
  int32_t* out;
};

// Keys of blocks that are taken in any case, and of those on a page outside the pool; every
// other block's is above both.
constexpr uint64_t kKeyTaken = 0, kKeyLast = 1;

__device__ __forceinline__ uint64_t ordered_key(double s) {
  const uint64_t u = hx::raw_bits(s + 0.0);  // -0 like 0
  if ((u & 0x7fffffffffffffffull) > 0x7ff0000000000000ull) return 0xfff0000000000000ull;  // NaN like +inf
  return (u >> 63) ? ~u : u | 0x8000000000000000ull;
}

// Blocks that row i sees: 0 where its row or sequence is not there.
__device__ __forceinline__ int selected_from(const SelectArgs& a, int64_t i, int64_t& row, int64_t& seq) {
  row = a.rows != nullptr ? a.rows[i] : i;
  seq = a.row_seq != nullptr ? a.row_seq[i] : i;
  if (seq < 0 || seq >= a.batch || row < 0 || row >= a.q_rows) return 0;
  const int64_t n = least_of<int64_t>(max(a.keys[i], 0), (int64_t)a.table_width * a.page);
  return (int)((n + a.block - 1) / a.block);
}

// Sum over LANES lanes next to each other, in all of them (pairings as in hx::dpp).
template <int CTRL>
__device__ __forceinline__ double add_dpp(double v) {
  typedef int i2 __attribute__((ext_vector_type(2)));
  i2 u = __builtin_bit_cast(i2, v);
  u.x = __builtin_amdgcn_update_dpp(0, u.x, CTRL, 0xF, 0xF, false);
  u.y = __builtin_amdgcn_update_dpp(0, u.y, CTRL, 0xF, 0xF, false);
  return v + __builtin_bit_cast(double, u);
}
template <int LANES>
__device__ __forceinline__ double lanes_sum(double v) {
  v = add_dpp<hx::kDppHalfMirror>(add_dpp<hx::kDppXor2>(add_dpp<hx::kDppXor1>(v)));
  if constexpr (LANES >= 16) v = add_dpp<hx::kDppMirror>(v);
  if constexpr (LANES >= 32) v += __shfl_xor(v, 16);
  return v;
}

// Bits of the type's infinity.
template <typename T>
__device__ __forceinline__ constexpr uint32_t inf_bits() { return __is_same(T, __bf16) ? 0x7f80u : 0x7c00u; }

// A workgroup takes a stretch of a row's blocks for one KV head, kGroups x kScPer at a time.
template <typename T, int LANES>
__global__ __launch_bounds__(kScThreads) void block_scores_kernel(SelectArgs a) {
  typedef hx::Elem<T> E;
  constexpr int kGroups = kScThreads / LANES, kPass = kGroups * kScPer;
  __shared__ double2 s_q[256];
  const int tid = hx::tid_x(), li = tid % LANES, g = tid / LANES;
  const int begin = hx::wg_x() % a.chunks * a.stretch;
  const int64_t ih = hx::wg_x() / a.chunks, i = ih / a.n_heads;
  const int h = (int)(ih % a.n_heads);
  int64_t row, seq;
  const int count = selected_from(a, i, row, seq);
  if (count <= a.budget || begin >= count) return;
  const int end = min(begin + a.stretch, count);
  const int32_t* table = a.table + seq * a.table_stride;
  const int per_page = a.page / a.block, d = 8 * li;
  const bool dims = d < a.head_dim;
  const uint32_t block_elems = (uint32_t)a.n_heads * 2 * a.head_dim;
  const uint16_t* const bounds = a.bounds + h * 2 * a.head_dim + d;
  uint4 low[kScPer], high[kScPer];
  uint32_t bad = 0;
  auto page_of = [&](int at, int& in_page) __attribute__((always_inline)) {
    const uint32_t j = min(at, count - 1);
    const uint32_t k = per_page == 1 ? j : (uint32_t)((uint64_t)j * a.page_magic >> 32);  // j / per_page
    in_page = j - k * per_page;
    return table[k];
  };
  auto load = [&](int j0) __attribute__((always_inline)) {
    int page[kScPer], in_page[kScPer];
#pragma unroll
    for (int p = 0; p < kScPer; ++p) page[p] = page_of(j0 + g + p * kGroups, in_page[p]);
    bad = 0;
#pragma unroll
    for (int p = 0; p < kScPer; ++p) {
      const bool off = page[p] < 0 || page[p] >= a.num_pages;
      bad |= (uint32_t)off << p;
      low[p] = high[p] = hx::zero4();
      if (off || !dims) continue;
      const uint16_t* at = bounds + ((int64_t)page[p] * per_page + in_page[p]) * block_elems;
      low[p] = hx::ld16_stream(at);
      high[p] = hx::ld16_stream(at + a.head_dim);
    }
  };
  load(begin);
  // Sums over the group of min(q, 0) and max(q, 0), by the sign bit: a NaN counts in one of them.
  for (int e = tid; e < a.head_dim; e += kScThreads) {
    const uint16_t* q = a.q + row * a.q_row + (int64_t)h * a.group * a.q_head + e;
    double neg = 0.0, pos = 0.0;
    for (int k = 0; k < a.group; ++k) {
      const uint32_t bits = __float_as_uint(E::lo(q[k * a.q_head])), minus = (uint32_t)((int32_t)bits >> 31);
      neg += (double)__uint_as_float(bits & minus);
      pos += (double)__uint_as_float(bits & ~minus);
    }
    s_q[e] = make_double2(neg, pos);
  }
  __syncthreads();
  double neg[8], pos[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const double2 v = s_q[dims ? d + e : 0];
    neg[e] = dims ? v.x : 0.0;
    pos[e] = dims ? v.y : 0.0;
  }
  uint64_t* const order = a.order + ih * a.most;
  auto key_at = [&](int j, bool off, double s) __attribute__((always_inline)) {
    return j < a.sink || j >= count - a.recent ? kKeyTaken : off ? kKeyLast : ordered_key(s);
  };
  uint32_t most = 0;  // of the upper halves of the sums' magnitudes
  for (int j0 = begin;;) {
    double s[kScPer];
#pragma unroll
    for (int p = 0; p < kScPer; ++p) {
      const uint32_t lw[4] = {low[p].x, low[p].y, low[p].z, low[p].w};
      const uint32_t hw[4] = {high[p].x, high[p].y, high[p].z, high[p].w};
      s[p] = 0.0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[p] = fma((double)(e % 2 ? E::hi(lw[e / 2]) : E::lo(lw[e / 2])), neg[e], s[p]);
        s[p] = fma((double)(e % 2 ? E::hi(hw[e / 2]) : E::lo(hw[e / 2])), pos[e], s[p]);
      }
    }
    const uint32_t was_bad = bad;
    const int j1 = j0 + kPass;
    if (j1 < end) load(j1);
#pragma unroll
    for (int p = 0; p < kScPer; ++p) {
      s[p] = lanes_sum<LANES>(s[p]);
      most = max(most, (uint32_t)(hx::raw_bits(s[p]) >> 32) & 0x7fffffffu);
      const int j = j0 + g + p * kGroups;
      if (li == 0 && j < end) order[j] = key_at(j, was_bad >> p & 1, s[p]);
    }
    if (j1 >= end) break;
    j0 = j1;
  }
  // Of a wave with an infinite or NaN sum, all again: 0 * inf is a NaN in the two products of a
  // dim, but not in max(q lower, q upper) unless a query is 0 itself. An infinite bound with a
  // weight of 0 and no such query is left out.
  if (__builtin_amdgcn_ballot_w64(most >= 0x7ff00000u) == 0) return;
  uint32_t zero = 0;  // dims in which a query is 0
  if (dims)
    for (int k = 0; k < a.group; ++k)
      for (int e = 0; e < 8; ++e)
        zero |= (a.q[row * a.q_row + (int64_t)(h * a.group + k) * a.q_head + d + e] & 0x7fffu) == 0 ? 1u << e : 0u;
  for (int j = begin + g; j - g < end; j += kGroups) {  // as many rounds for every group of lanes
    int in_page;
    const int page = page_of(j, in_page);
    const bool off = page < 0 || page >= a.num_pages;
    double s = 0.0;
    if (!off && dims) {
      const uint16_t* at = bounds + ((int64_t)page * per_page + in_page) * block_elems;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t lo = at[e], hi = at[a.head_dim + e], keep = zero >> e & 1;
        const bool no_lo = !keep && (lo & 0x7fffu) == inf_bits<T>() && hx::raw_bits(neg[e]) << 1 == 0;
        const bool no_hi = !keep && (hi & 0x7fffu) == inf_bits<T>() && hx::raw_bits(pos[e]) << 1 == 0;
        s = fma((double)E::lo(no_lo ? 0 : lo), neg[e], s);
        s = fma((double)E::lo(no_hi ? 0 : hi), pos[e], s);
      }
    }
    s = lanes_sum<LANES>(s);
    if (li == 0 && j < end) order[j] = key_at(j, off, s);
  }
}

// The largest of a wave's values, in all lanes.
template <int CTRL>
__device__ __forceinline__ uint64_t max_dpp(uint64_t v) {
  const uint32_t x = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, 0xF, 0xF, false);
  const uint32_t y = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, 0xF, 0xF, false);
  return most_of<uint64_t>(v, (uint64_t)y << 32 | x);
}
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
  v = max_dpp<hx::kDppHalfMirror>(max_dpp<hx::kDppXor2>(max_dpp<hx::kDppXor1>(v)));
  v = max_dpp<hx::kDppMirror>(v);  // of each row of 16 lanes
  uint64_t best = 0;
#pragma unroll
  for (int r = 0; r < 64; r += 16)
    best = most_of<uint64_t>(best, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), r) << 32 |
                                       (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, r));
  return best;
}

// Sum of the lanes' values up to and with each lane's own.
__device__ __forceinline__ int wave_prefix(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // the row before's last, into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // lane 31's, into rows 2 and 3
  return v;
}

// Wave w holds blocks 64 PER w .. + 64 PER - 1, block 64 PER w + 64 t + lane in key[t].
template <int WAVES, int PER>
__global__ __launch_bounds__(64 * WAVES) void select_blocks_kernel(SelectArgs a) {
  __shared__ uint64_t s_ends[2][WAVES];
  __shared__ __attribute__((aligned(16))) int s_bins[kSelBins];
  __shared__ int s_above[WAVES], s_ties[WAVES], s_taken[WAVES];
  __shared__ uint64_t s_few[64];
  __shared__ int s_listed;
  const int tid = hx::tid_x(), lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t ih = hx::wg_x();
  int32_t* out = a.out + ih * a.budget;
  int64_t row, seq;
  const int count = selected_from(a, ih / a.n_heads, row, seq);
  if (count <= a.budget) {
    for (int j = tid; j < a.budget; j += 64 * WAVES) out[j] = j < count ? j : -1;
    return;
  }
  const int first = 64 * PER * w + lane;
  uint64_t key[PER], hi = 0, lo = ~0ull;
#pragma unroll
  for (int t = 0; t < PER; ++t) {
    key[t] = kKeyTaken;
    if (first + 64 * t < count) key[t] = a.order[ih * a.most + first + 64 * t];
  }
#pragma unroll
  for (int t = 0; t < PER; ++t) {
    hi = most_of(hi, key[t]);
    if (key[t] != kKeyTaken) lo = least_of(lo, key[t]);
  }
  hi = wave_max(hi);
  lo = ~wave_max(~lo);
  if constexpr (WAVES > 1) {
    if (lane == 0) {
      s_ends[0][w] = hi;
      s_ends[1][w] = lo;
    }
    __syncthreads();
#pragma unroll
    for (int ww = 0; ww < WAVES; ++ww) {
      hi = most_of(hi, s_ends[0][ww]);
      lo = least_of(lo, s_ends[1][ww]);
    }
  }
  // The need-th largest free key: counts of the keys between lo and hi in up to 1024 equal bins,
  // then of those in the bin it lies in, until that bin is wanted whole, is a single key or holds
  // no more than a wave does. One or two passes of keys that spread out, at most seven.
  const int need = a.budget - a.sink - a.recent;
  uint64_t least = ~0ull;  // above every key
  for (int want = need, pass = 0; want > 0 && pass < kSelPasses; ++pass) {
    const int bits = lo == hi ? 0 : 64 - __builtin_clzll(hi - lo), shift = bits > 10 ? bits - 10 : 0;
    for (int e = tid; e < kSelBins / 4; e += 64 * WAVES) reinterpret_cast<uint4*>(s_bins)[e] = hx::zero4();
    if (tid == 0) s_listed = 0;
    __syncthreads();
#pragma unroll
    for (int t = 0; t < PER; ++t)
      if (key[t] >= lo && key[t] <= hi) atomicAdd(&s_bins[(key[t] - lo) >> shift], 1);
    __syncthreads();
    int in[16], sum = 0;  // every wave reads them all: bins 16 lane .. + 15
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int4 u = reinterpret_cast<const int4*>(s_bins)[4 * lane + e / 4];
      in[e] = u.x, in[e + 1] = u.y, in[e + 2] = u.z, in[e + 3] = u.w;
      sum += (u.x + u.y) + (u.z + u.w);
    }
    const int upto = wave_prefix(sum), all = __builtin_amdgcn_readlane(upto, 63);
    // Keys in the lane's bins and above, and above them alone.
    int from = all - upto + sum, above = all - upto, bin = 0, count_of = 0;
    const int owner = __builtin_ctzll(__builtin_amdgcn_ballot_w64(from >= want && above < want));
    bool found = false;
#pragma unroll
    for (int e = 15; e >= 0; --e) {
      const bool here = !found && above + in[e] >= want;
      bin = here ? 16 * lane + e : bin;
      count_of = here ? in[e] : count_of;
      found |= here;
      above += found ? 0 : in[e];
    }
    bin = __builtin_amdgcn_readlane(bin, owner);
    count_of = __builtin_amdgcn_readlane(count_of, owner);
    want -= __builtin_amdgcn_readlane(above, owner);
    lo += (uint64_t)bin << shift;
    if (shift == 0 || count_of == want) {
      least = lo;
      break;
    }
    hi = lo + least_of<uint64_t>(hi - lo, (1ull << shift) - 1);  // lo + 2^shift may pass 2^64
    __syncthreads();
    if (count_of > 64) continue;
    // Few enough to compare each with each: a lane's key is the one wanted if fewer than want
    // lie above it and it is not above want of them; every wave finds it.
#pragma unroll
    for (int t = 0; t < PER; ++t)
      if (key[t] >= lo && key[t] <= hi) s_few[atomicAdd(&s_listed, 1)] = key[t];
    __syncthreads();
    const uint64_t mine = lane < count_of ? s_few[lane] : 0;
    int greater = 0, equal = 0;
    for (int o = 0; o < count_of; ++o) {
      greater += s_few[o] > mine ? 1 : 0;
      equal += s_few[o] == mine ? 1 : 0;
    }
    const uint64_t is = __builtin_amdgcn_ballot_w64(lane < count_of && greater < want && greater + equal >= want);
    least = s_few[__builtin_ctzll(is)];
    break;
  }
  // Keys above the threshold, and of those equal to it the first ones, make up the rest.
  int above = 0, tied = 0, taken = 0;
#pragma unroll
  for (int t = 0; t < PER; ++t) {
    above += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key[t] > least));
    tied += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key[t] == least));
    taken += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key[t] == kKeyTaken && first + 64 * t < count));
  }
  int ties = need - above, at = 0;
  if constexpr (WAVES > 1) {
    if (lane == 0) {
      s_above[w] = above;
      s_ties[w] = tied;
      s_taken[w] = above + taken;
    }
    __syncthreads();
    ties = need;
#pragma unroll
    for (int ww = 0; ww < WAVES; ++ww) ties -= s_above[ww];
    for (int ww = 0; ww < w; ++ww) {
      const int had = min(max(ties, 0), s_ties[ww]);
      at += s_taken[ww] + had;
      ties -= s_ties[ww];
    }
  }
  const uint64_t before = (1ull << lane) - 1ull;
#pragma unroll
  for (int t = 0; t < PER; ++t) {
    const int j = first + 64 * t;
    const bool there = j < count;
    const bool tie = there && key[t] == least;
    const uint64_t equal = __builtin_amdgcn_ballot_w64(tie);
    const bool take = there && (key[t] == kKeyTaken || key[t] > least ||
                                (tie && __builtin_popcountll(equal & before) < ties));
    ties -= __builtin_popcountll(equal);  // at 0 or below no later tie is taken
    const uint64_t goes = __builtin_amdgcn_ballot_w64(take);
    const int to = at + __builtin_popcountll(goes & before);
    if (take && to < a.budget) out[to] = j;
    at += __builtin_popcountll(goes);
  }
}

template <typename T, int LANES>
void launch_scores(SelectArgs a, int64_t n, hipStream_t s) {
  constexpr int kPass = kScThreads / LANES * kScPer;
  const int64_t passes = (a.most + kPass - 1) / kPass;
  // Several passes a workgroup, one in flight while the last is summed, where that leaves
  // workgroups enough.
  int64_t loops = n * a.n_heads * passes / 2048;
  loops = loops < 1 ? 1 : loops > 8 ? 8 : loops;
  a.stretch = (int32_t)(loops * kPass);
  a.chunks = (int32_t)((passes + loops - 1) / loops);
  hipLaunchKernelGGL((block_scores_kernel<T, LANES>), dim3((unsigned)(n * a.n_heads * a.chunks)), dim3(kScThreads), 0,
                     s, a);
}

template <typename T>
void launch_select(const SelectArgs& a, int64_t n, hipStream_t s) {
  if (a.most > a.budget) {
    if (a.head_dim <= 64) launch_scores<T, 8>(a, n, s);
    else if (a.head_dim <= 128) launch_scores<T, 16>(a, n, s);
    else launch_scores<T, 32>(a, n, s);
  }
  const dim3 grid((unsigned)(n * a.n_heads));
  // Few keys a thread, few waves to a barrier. One row / 64 rows, 8 heads, us: 900 blocks 5.2 /
  // 6.3, 8 waves 5.6 / 8.2, 2 waves 5.9 / 7.2; 2000 blocks 6.2 / 8.4, 16 waves 8.1 / 12.2, 4 waves
  // 8.7 / 10.3; 4000 blocks 7.1 / 14.1, 16 waves 8.0 / 19.3, 4 waves 8.2 / 13.6; 12000 blocks of 4
  // rows 13.5, 8 waves 17.2.
  if (a.most <= 1024) hipLaunchKernelGGL((select_blocks_kernel<4, 4>), grid, dim3(256), 0, s, a);
  else if (a.most <= 2048) hipLaunchKernelGGL((select_blocks_kernel<8, 4>), grid, dim3(512), 0, s, a);
  else if (a.most <= 4096) hipLaunchKernelGGL((select_blocks_kernel<8, 8>), grid, dim3(512), 0, s, a);
  else hipLaunchKernelGGL((select_blocks_kernel<16, 16>), grid, dim3(1024), 0, s, a);
}

// -------------------------------------------------------------------------- attention
//
// One query row and KV head to a workgroup and split: the G query heads (8 at a time) share
// each K / V read, which HBM bounds. The list's blocks are cut into units of 16 tokens; a wave
// takes two units (32 keys) at a time through its own part of LDS, the next two in flight in
// registers meanwhile, so the waves never wait for one another. Rows past a sequence's keys
// are read past the end of the unit's buffer resource and come back as zeros: what a page
// holds behind its last key never reaches the sums.
//
// S^T = K Q^T has the query heads as its columns, twice: of each key's weight p, columns 0-7
// carry its rounding to the element type into P V and columns 8-15 that of the remainder, so one
// MFMA sums both. S^T's registers are the P operand as they are. Two fp16 hold 23 bits of p, less
// than exp2's error; bf16 takes a third part, in columns 8-15 of a second MFMA, and holds all 24.
// (Two bf16 parts showed where values cancel: two keys with weights 2^-13 apart came out up to 6 %
// off. The third takes 0.15 us of one row's 9.1, and nothing of 64 rows' 181.)
// Weights are scaled by a power of two: bf16's by 2^-24, so that values up to the type's largest
// cannot leave fp32 in the sums over a list's keys, fp16's by 2^14, so that small ones keep
// their bits (unscaled, those below 2^-25 were lost: 940 of e^-18 are 1.4e-5 of a sum).
//
// 32/8 heads of 128, blocks of 64: 64 rows of 4096 keys (1.07 GB) 177 us, 6.1 TB/s, what this
// card reads at most; one row of 2048 keys (8.4 MB) 7.1 us and 3.2 for the join of its 16 splits,
// the launches' and dependent loads' latency.

constexpr int kSpWaves = 4;
constexpr int kSpHeads = 8;       // query heads of a workgroup
constexpr int kSpMaxUnits = 64;   // 16-token units of a split
constexpr float kSpLog2e = 1.44269504088896340736f;

struct SparseArgs {
  const uint16_t* q;
  int64_t q_row, q_head, q_rows;
  const int64_t* rows;
  const int32_t* row_seq;
  const int32_t* keys;
  const uint16_t* k;
  const uint16_t* v;
  int32_t num_pages, page, block;
  const int32_t* blocks;  // [n][n_heads][budget]
  int32_t budget;
  const int32_t* table;
  int64_t table_stride;
  int32_t batch, table_width;
  int32_t n_heads, group, head_dim, head_blocks;
  float scale_log2;
  uint16_t* out;
  int64_t out_row, out_head;
  float* part_o;  // [n][query heads][splits][head_dim]
  float* part_ml; // [n][query heads][splits][2]
  int32_t splits, units;  // units of a split, even
};

// LDS slot of 16-byte piece p of tile row r: a fragment read (16 rows, one piece each) and a
// transposing read (4 rows, two pieces each) then spread over the banks.
template <int DP>
__device__ __forceinline__ int sp_piece(int r, int p) {
  return DP == 64 ? p ^ ((r >> 1) & 7) : p ^ (r & 15);
}

// By which the weights are scaled.
template <typename T>
__device__ __forceinline__ constexpr float weight_scale() { return __is_same(T, __bf16) ? 0x1p-24f : 0x1p14f; }

template <typename T, int DP>
__global__ __launch_bounds__(64 * kSpWaves) void sparse_attn_kernel(SparseArgs a) {
  typedef hx::Elem<T> E;
  typedef typename E::v8 v8;
  constexpr int kRowBytes = 2 * DP, kPieces = DP / 8, kSteps = DP / 32, kDims = DP / 16;
  constexpr int kPerLoad = 64 / kPieces, kLoads = 16 / kPerLoad;  // tokens a load, loads a unit
  constexpr int kTile = 32 * kRowBytes;
  constexpr int kStage = 2 * kTile;
  __shared__ __attribute__((aligned(16))) uint8_t smem[kSpWaves * kStage];
  __shared__ int64_t s_row[kSpMaxUnits];
  __shared__ int s_cnt[kSpMaxUnits];
  __shared__ float s_m[kSpWaves][kSpHeads], s_l[kSpWaves][kSpHeads];
  const int tid = hx::tid_x(), lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  int wg = hx::wg_x();
  const int split = wg % a.splits;
  wg /= a.splits;
  const int hb = wg % a.head_blocks;
  wg /= a.head_blocks;
  const int h = wg % a.n_heads;
  const int64_t i = wg / a.n_heads;
  const int64_t row = a.rows != nullptr ? a.rows[i] : i;
  const int64_t seq = a.row_seq != nullptr ? a.row_seq[i] : i;
  if (row < 0 || row >= a.q_rows) return;  // no such query, and no such output row
  int n = (int)least_of<int64_t>(max(a.keys[i], 0), (int64_t)a.table_width * a.page);
  if (seq < 0 || seq >= a.batch) n = 0;
  const int per_page = a.page / a.block, per_block = a.block / 16;
  const int64_t row_elems = (int64_t)a.n_heads * a.head_dim;

  if (tid < a.units) {
    const int u = split * a.units + tid, e = u / per_block;
    int64_t at = 0;
    int cnt = 0;
    if (e < a.budget) {
      // A block that starts below n has a first token that fits 32 bits, as n does.
      const int j = a.blocks[((int64_t)i * a.n_heads + h) * a.budget + e], in = u % per_block * 16;
      if (n > 0 && j >= 0 && j <= (n - 1) / a.block && j * a.block < n - in) {
        const int page = a.table[seq * a.table_stride + j / per_page];
        if (page >= 0 && page < a.num_pages) {
          at = (int64_t)page * a.page + j % per_page * a.block + in;
          cnt = min(16, n - in - j * a.block);
        }
      }
    }
    s_row[tid] = at;
    s_cnt[tid] = cnt;
  }

  const int heads = min(kSpHeads, a.group - hb * kSpHeads);
  const int head0 = h * a.group + hb * kSpHeads;
  v8 qf[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    uint4 u = hx::zero4();
    const int d = 32 * s + 8 * lg;
    if ((lr & 7) < heads && d < a.head_dim)
      u = *reinterpret_cast<const uint4*>(a.q + row * a.q_row + (int64_t)(head0 + (lr & 7)) * a.q_head + d);
    qf[s] = hx::as_v8<T>(u);
  }
  __syncthreads();

  // Lane l of a load takes piece l % kPieces of token l / kPieces; a piece past the head's
  // dims is read past the buffer's end (zeros).
  const uint32_t row_bytes = (uint32_t)row_elems * 2;
  const int piece = lane % kPieces, ltok = lane / kPieces;
  const uint32_t voff = 8 * piece < a.head_dim ? ltok * row_bytes + 16 * piece : 0x7ffffff0u;
  uint4 kb[2][kLoads], vb[2][kLoads];
  auto load = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int64_t at = s_row[2 * tile + u];
      const int cnt = __builtin_amdgcn_readfirstlane(s_cnt[2 * tile + u]);
      const int64_t pool_row = (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at) |
                               (int64_t)__builtin_amdgcn_readfirstlane((int)(at >> 32)) << 32;
      const int64_t base = pool_row * row_elems + (int64_t)h * a.head_dim;
      const uint32_t bytes = cnt > 0 ? (uint32_t)(cnt - 1) * row_bytes + 2 * a.head_dim : 0u;
      const __amdgpu_buffer_rsrc_t kr = hx::buffer_rsrc(a.k + base, bytes), vr = hx::buffer_rsrc(a.v + base, bytes);
#pragma unroll
      for (int q = 0; q < kLoads; ++q) {
        // A piece past the head's dims stays past the buffer's end: 0x7ffffff0 + 2^29 at most.
        kb[u][q] = hx::ld16_stream(kr, voff + q * kPerLoad * row_bytes, 0);
        vb[u][q] = hx::ld16_stream(vr, voff + q * kPerLoad * row_bytes, 0);
      }
    }
  };

  uint8_t* const kt = smem + w * kStage;
  uint8_t* const vt = kt + kTile;
  float m_run = -INFINITY, l_run = 0.f;
  hx::f32x4_t o[kDims];
#pragma unroll
  for (int d = 0; d < kDims; ++d) o[d] = hx::f32x4_t{0.f, 0.f, 0.f, 0.f};

  const int tiles = a.units / 2;
  auto live = [&](int tile) __attribute__((always_inline)) {
    return __builtin_amdgcn_readfirstlane(s_cnt[2 * tile] | s_cnt[2 * tile + 1]) != 0;
  };
  // The wave's next tile with a key in it.
  auto next = [&](int tile) __attribute__((always_inline)) {
    while (tile < tiles && !live(tile)) tile += kSpWaves;
    return tile;
  };
  int tile = next(w);
  if (tile < tiles) load(tile);
  while (tile < tiles) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int q = 0; q < kLoads; ++q) {
        const int r = 16 * u + q * kPerLoad + ltok;
        const int to = r * kRowBytes + 16 * sp_piece<DP>(r, piece);
        *reinterpret_cast<uint4*>(kt + to) = kb[u][q];
        *reinterpret_cast<uint4*>(vt + to) = vb[u][q];
      }
    // Lanes read what other lanes of the wave stored: a wave's LDS accesses complete in order,
    // the fences hold the compiler to it.
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    int cnt[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) cnt[u] = __builtin_amdgcn_readfirstlane(s_cnt[2 * tile + u]);
    tile = next(tile + kSpWaves);
    if (tile < tiles) load(tile);

    hx::f32x4_t sc[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      sc[u] = hx::f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int r = 16 * u + lr;
        const uint4 kf = *reinterpret_cast<const uint4*>(kt + r * kRowBytes + 16 * sp_piece<DP>(r, 4 * s + lg));
        sc[u] = E::mfma16x16x32(hx::as_v8<T>(kf), qf[s], sc[u]);
      }
    }
    float mx = m_run;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sc[u][e] = 4 * lg + e < cnt[u] ? sc[u][e] * a.scale_log2 : -INFINITY;
        mx = fmaxf(mx, sc[u][e]);
      }
    mx = hx::max_xor32(hx::max_xor16(mx));
    const float alpha = mx == -INFINITY ? 1.f : hx::fast_exp2(m_run - mx);
    const float neg = mx == -INFINITY ? 0.f : -mx;
    m_run = mx;
    l_run *= alpha;
#pragma unroll
    for (int d = 0; d < kDims; ++d) o[d] *= alpha;
    uint32_t pw[4], pl[4];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const float p0 = hx::fast_exp2(sc[u][e] + neg) * weight_scale<T>();
        const float p1 = hx::fast_exp2(sc[u][e + 1] + neg) * weight_scale<T>();
        l_run += p0;
        l_run += p1;
        const uint32_t top = hx::pack2_round<T>(p0, p1);
        const float r0 = p0 - E::lo(top), r1 = p1 - E::hi(top);
        const uint32_t rest = hx::pack2_round<T>(r0, r1);
        pw[2 * u + e / 2] = lr < 8 ? top : rest;
        pl[2 * u + e / 2] = lr < 8 ? 0u : hx::pack2_round<T>(r0 - E::lo(rest), r1 - E::hi(rest));
      }
    const v8 pf = hx::as_v8<T>(make_uint4(pw[0], pw[1], pw[2], pw[3]));
    const v8 pf2 = hx::as_v8<T>(make_uint4(pl[0], pl[1], pl[2], pl[3]));
#pragma unroll
    for (int d = 0; d < kDims; ++d) {
      uint2 f[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int r = 16 * u + 4 * lg + (lr >> 2);
        f[u] = hx::ld8_lds_tr16(vt + r * kRowBytes + 16 * sp_piece<DP>(r, 2 * d + ((lr & 3) >> 1)) + 8 * (lr & 1));
      }
      const v8 vf = hx::as_v8<T>(make_uint4(f[0].x, f[0].y, f[1].x, f[1].y));
      o[d] = E::mfma16x16x32(vf, pf, o[d]);
      if constexpr (__is_same(T, __bf16)) o[d] = E::mfma16x16x32(vf, pf2, o[d]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }

  // Lane: dims 16 d + 4 lg .. + 3 of head lr % 8; the parts of P summed.
  l_run = hx::add_xor32(hx::add_xor16(l_run));
  float all = 0.f;
#pragma unroll
  for (int d = 0; d < kDims; ++d)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[d][e] += hx::dpp<0x128>(o[d][e]);  // the lane 8 apart in its row of 16
      all += o[d][e];
    }
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(!hx::is_finite(all)) != 0, 0)) {
    // An infinite or NaN sum. The parts of P made NaN of an infinite V too (0 * inf): what the
    // wave's keys have in each dim is looked up again, and is the dim's result at any weight.
    uint32_t has = 0;  // +inf, -inf, NaN: a bit for each of the piece's dims
    for (int t = next(w); t < tiles; t = next(t + kSpWaves)) {
      load(t);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int q = 0; q < kLoads; ++q) {
          const uint32_t wd[4] = {vb[u][q].x, vb[u][q].y, vb[u][q].z, vb[u][q].w};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t x = wd[e / 2] >> (16 * (e % 2)) & 0xffffu, mag = x & 0x7fffu;
            const uint32_t at = mag > inf_bits<T>() ? 16 : x >> 15 ? 8 : 0;
            has |= mag >= inf_bits<T>() ? 1u << (at + e) : 0u;
          }
        }
    }
    for (int m = kPieces; m < 64; m <<= 1) has |= __shfl_xor(has, m);
#pragma unroll
    for (int d = 0; d < kDims; ++d) {
      const uint32_t of = __shfl(has, 2 * d + (lg >> 1)) >> (4 * (lg & 1));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool up = of >> e & 1, down = of >> (8 + e) & 1, nan = of >> (16 + e) & 1;
        if (up || down || nan)
          o[d][e] = __uint_as_float(nan || (up && down) ? 0x7fc00000u : up ? 0x7f800000u : 0xff800000u);
      }
    }
  }
  __syncthreads();  // every wave is done with its stage
  float (*const s_o)[kSpHeads][DP] = reinterpret_cast<float (*)[kSpHeads][DP]>(smem);
  if (lr < kSpHeads) {
#pragma unroll
    for (int d = 0; d < kDims; ++d)
      *reinterpret_cast<float4*>(&s_o[w][lr][16 * d + 4 * lg]) = make_float4(o[d][0], o[d][1], o[d][2], o[d][3]);
    if (lg == 0) {
      s_m[w][lr] = m_run;
      s_l[w][lr] = l_run;
    }
  }
  __syncthreads();
  const int half = a.head_dim / 2;  // head_dim is a multiple of 8
  for (int e = tid; e < heads * half; e += 64 * kSpWaves) {
    const int hd = e / half, d = 2 * (e % half);
    float m = s_m[0][hd];
#pragma unroll
    for (int ww = 1; ww < kSpWaves; ++ww) m = fmaxf(m, s_m[ww][hd]);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int ww = 0; ww < kSpWaves; ++ww) {
      const float f = hx::fast_exp2(s_m[ww][hd] - ref);
      l = fmaf(f, s_l[ww][hd], l);
      x = fmaf(f, s_o[ww][hd][d], x);
      y = fmaf(f, s_o[ww][hd][d + 1], y);
    }
    if (__builtin_expect(!hx::is_finite(x + y), 0)) {  // an infinite part counts at any weight, 0 too
      x = y = 0.f;
      for (int ww = 0; ww < kSpWaves; ++ww) {
        const float f = hx::fast_exp2(s_m[ww][hd] - ref);
        x = hx::add_weighed<true>(f, s_o[ww][hd][d], x);
        y = hx::add_weighed<true>(f, s_o[ww][hd][d + 1], y);
      }
    }
    const int64_t head = head0 + hd;
    if (a.splits == 1) {
      const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
      *reinterpret_cast<uint32_t*>(a.out + row * a.out_row + head * a.out_head + d) = hx::pack2_round<T>(x * inv, y * inv);
    } else {
      const int64_t p = (i * a.n_heads * a.group + head) * a.splits + split;
      *reinterpret_cast<float2*>(a.part_o + p * a.head_dim + d) = make_float2(x, y);
      if (d == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * p) = make_float2(m, l);
    }
  }
}

// The splits of a row and query head, in order; one wave each, with the first kCbAtOnce splits'
// sums on their way before the maxima are known (loaded one after another: 7.5 us for 3.4).
constexpr int kCbAtOnce = 16;

template <typename T>
__global__ __launch_bounds__(64) void sparse_combine_kernel(SparseArgs a) {
  const int lane = hx::tid_x();
  const int64_t t = hx::wg_x();
  const int n_q = a.n_heads * a.group, i = hx::wg_x() / n_q, head = hx::wg_x() % n_q;
  const int64_t row = a.rows != nullptr ? a.rows[i] : i;
  if (row < 0 || row >= a.q_rows) return;
  const float2* const ml = reinterpret_cast<const float2*>(a.part_ml) + t * a.splits;
  const float* const sums = a.part_o + t * a.splits * a.head_dim;
  for (int d0 = 0; d0 < a.head_dim; d0 += 128) {
    const int d = d0 + 2 * lane, from = d < a.head_dim ? d : 0;
    float2 o[kCbAtOnce];
    auto load = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < kCbAtOnce; ++k) {
        const int at = s0 + k < a.splits ? s0 + k : a.splits - 1;
        o[k] = *reinterpret_cast<const float2*>(sums + (int64_t)at * a.head_dim + from);
      }
    };
    load(0);
    float m = -INFINITY;
    for (int s = lane; s < a.splits; s += 64) m = fmaxf(m, ml[s].x);
    m = fmaxf(m, hx::dpp<hx::kDppXor1>(m));
    m = fmaxf(m, hx::dpp<hx::kDppXor2>(m));
    m = fmaxf(m, hx::dpp<hx::kDppHalfMirror>(m));
    m = fmaxf(m, hx::dpp<hx::kDppMirror>(m));
    m = hx::max_xor32(hx::max_xor16(m));
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f, x = 0.f, y = 0.f;
    for (int s0 = 0; s0 < a.splits; s0 += 64) {
      const float2 mine = s0 + lane < a.splits ? ml[s0 + lane] : make_float2(-INFINITY, 0.f);
      const float f = hx::fast_exp2(mine.x - ref);
      l = fmaf(f, mine.y, l);
      for (int k0 = 0; k0 < 64 && s0 + k0 < a.splits; k0 += kCbAtOnce) {
#pragma unroll
        for (int k = 0; k < kCbAtOnce; ++k) {
          const float fk = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(f), k0 + k));
          if (s0 + k0 + k < a.splits) {
            x = fmaf(fk, o[k].x, x);
            y = fmaf(fk, o[k].y, y);
          }
        }
        if (s0 + k0 + kCbAtOnce < a.splits) load(s0 + k0 + kCbAtOnce);
      }
    }
    l += hx::dpp<hx::kDppXor1>(l);
    l += hx::dpp<hx::kDppXor2>(l);
    l += hx::dpp<hx::kDppHalfMirror>(l);
    l += hx::dpp<hx::kDppMirror>(l);
    l = hx::add_xor32(hx::add_xor16(l));
    if (__builtin_expect(!hx::is_finite(x + y), 0)) {
      // An infinite part counts at any weight, 0 too. (In the loop above this took 0.3 us of 3.)
      x = y = 0.f;
      for (int at = 0; at < a.splits; ++at) {
        const float2 part = *reinterpret_cast<const float2*>(sums + (int64_t)at * a.head_dim + from);
        const float f = hx::fast_exp2(ml[at].x - ref);
        x = hx::add_weighed<true>(f, part.x, x);
        y = hx::add_weighed<true>(f, part.y, y);
      }
    }
    const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
    if (d < a.head_dim)
      *reinterpret_cast<uint32_t*>(a.out + row * a.out_row + head * a.out_head + d) = hx::pack2_round<T>(x * inv, y * inv);
  }
}

struct Split {
  int32_t units, splits;
};

// Splits of a row's list: about four workgroups a CU where the rows and heads alone give fewer,
// of at least 128 and at most 1024 keys.
Split sparse_split(int64_t n, int32_t n_heads, int32_t head_blocks, int32_t budget, int32_t block) {
  const int64_t row_heads = n * n_heads * head_blocks, total = (int64_t)budget * (block / 16);
  const int64_t want = (1024 + row_heads - 1) / row_heads;
  int64_t units = ((total + want - 1) / want + 7) / 8 * 8;
  units = units < 8 ? 8 : units > kSpMaxUnits ? kSpMaxUnits : units;
  return {(int32_t)units, (int32_t)((total + units - 1) / units)};
}

template <typename T, int DP>
void launch_sparse(const SparseArgs& a, int64_t n, hipStream_t s) {
  const dim3 grid((unsigned)(n * a.n_heads * a.head_blocks * a.splits));
  hipLaunchKernelGGL((sparse_attn_kernel<T, DP>), grid, dim3(64 * kSpWaves), 0, s, a);
}

template <typename T>
void launch_sparse_dims(const SparseArgs& a, int64_t n, hipStream_t s) {
  if (a.head_dim <= 64) launch_sparse<T, 64>(a, n, s);
  else if (a.head_dim <= 128) launch_sparse<T, 128>(a, n, s);
  else launch_sparse<T, 256>(a, n, s);
  if (a.splits > 1) {
    hipLaunchKernelGGL(sparse_combine_kernel<T>, dim3((unsigned)(n * a.n_heads * a.group)), dim3(64), 0, s, a);
  }
}

bool power_of_two(int32_t x) { return x > 0 && (x & (x - 1)) == 0; }

int check_layout(int32_t num_pages, int32_t page, int32_t block, int32_t n_heads, int32_t head_dim, int32_t dtype) {
  if (dtype != HX_DTYPE_BF16 && dtype != HX_DTYPE_FP16) return HX_E_UNSUPPORTED;
  if (num_pages < 1 || page < 1 || n_heads < 1 || head_dim < 1) return HX_E_INVALID_ARG;
  if (head_dim % 8 || head_dim > 256 || !power_of_two(block) || block < 16 || block > 1024 || page % block)
    return HX_E_UNSUPPORTED;
  if ((int64_t)n_heads * head_dim > (1 << 24)) return HX_E_UNSUPPORTED;  // a unit within a buffer resource
  return HX_OK;
}

}  // namespace

extern "C" int hx_kv_block_bounds(const void* k_pool, void* bounds, int32_t num_pages, int32_t page_size,
                                  int32_t block_size, int32_t n_kv_heads, int32_t head_dim, int32_t dtype,
                                  const int32_t* block_table, int64_t block_table_stride, int32_t block_table_width,
                                  const int32_t* cu_seq_q, const int32_t* seqused_k, int32_t batch, int32_t max_q,
                                  void* stream) {
  const int bad = check_layout(num_pages, page_size, block_size, n_kv_heads, head_dim, dtype);
  if (bad != HX_OK) return bad;
  if (batch < 0 || max_q < 0 || block_table_width < 1 || block_table_stride < block_table_width)
    return HX_E_INVALID_ARG;
  if (batch == 0 || max_q == 0) return HX_OK;
  if (!k_pool || !bounds || !block_table || !cu_seq_q || !seqused_k ||
      ((reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(bounds)) & 15))
    return HX_E_INVALID_ARG;
  BoundsArgs a;
  a.k = static_cast<const uint16_t*>(k_pool);
  a.bounds = static_cast<uint16_t*>(bounds);
  a.num_pages = num_pages;
  a.page = page_size;
  a.block = block_size;
  a.pieces = n_kv_heads * head_dim / 8;
  a.pieces_head = head_dim / 8;
  a.table = block_table;
  a.table_stride = block_table_stride;
  a.table_width = block_table_width;
  a.cu_q = cu_seq_q;
  a.used = seqused_k;
  a.groups = (max_q - 1) / block_size + 2;
  a.chunks = (a.pieces + kBdPieces - 1) / kBdPieces;
  a.inf = dtype == HX_DTYPE_BF16 ? 0x7f80 : 0x7c00;
  const int64_t wgs = (int64_t)batch * a.groups * a.chunks;
  if (wgs > kMostItems / kBdThreads) return HX_E_UNSUPPORTED;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(block_bounds_kernel, dim3((unsigned)wgs), dim3(kBdThreads), 0, s, a);
  return hx::status_from_hip(hipGetLastError());
}

extern "C" size_t hx_select_blocks_workspace_bytes(int64_t n, int32_t n_kv_heads, int64_t blocks) {
  return n < 1 || n_kv_heads < 1 || blocks < 1 ? 0 : (size_t)n * n_kv_heads * (size_t)blocks * sizeof(uint64_t);
}

extern "C" int hx_select_blocks(const void* q, int64_t q_row_stride, int64_t q_head_stride, int64_t q_rows,
                                const int64_t* rows, const int32_t* row_seq, const int32_t* key_counts, int64_t n,
                                int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int32_t dtype,
                                const void* bounds, int32_t num_pages, int32_t page_size, int32_t block_size,
                                const int32_t* block_table, int64_t block_table_stride, int32_t batch,
                                int32_t block_table_width, int32_t budget, int32_t sink, int32_t recent,
                                int32_t* blocks, void* workspace, size_t workspace_bytes, void* stream) {
  const int bad = check_layout(num_pages, page_size, block_size, n_kv_heads, head_dim, dtype);
  if (bad != HX_OK) return bad;
  if (n < 0 || q_rows < 0 || n_q_heads < 1 || n_q_heads % n_kv_heads || batch < 0 || block_table_width < 1 ||
      block_table_stride < block_table_width || budget < 1 || sink < 0 || recent < 1 ||
      (int64_t)sink + recent > budget)
    return HX_E_INVALID_ARG;
  const int64_t most = (int64_t)block_table_width * (page_size / block_size);
  if (most > kSelMaxBlocks || page_size / block_size > (1 << 16) || n > 0x7fffffff / n_kv_heads / (most + 1) ||
      n > kMostItems / 1024 / n_kv_heads)
    return HX_E_UNSUPPORTED;
  if (n == 0) return HX_OK;
  if (!q || !key_counts || !bounds || !block_table || !blocks ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(bounds)) & 15) || q_row_stride % 8 ||
      q_head_stride % 8 || (rows == nullptr && n > q_rows) ||
      (row_seq == nullptr && n > batch))
    return HX_E_INVALID_ARG;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 7) ||
      workspace_bytes < hx_select_blocks_workspace_bytes(n, n_kv_heads, most))
    return HX_E_WORKSPACE;
  SelectArgs a;
  a.q = static_cast<const uint16_t*>(q);
  a.q_row = q_row_stride;
  a.q_head = q_head_stride;
  a.q_rows = q_rows;
  a.rows = rows;
  a.row_seq = row_seq;
  a.keys = key_counts;
  a.n_heads = n_kv_heads;
  a.group = n_q_heads / n_kv_heads;
  a.head_dim = head_dim;
  a.bounds = static_cast<const uint16_t*>(bounds);
  a.num_pages = num_pages;
  a.page = page_size;
  a.block = block_size;
  a.table = block_table;
  a.table_stride = block_table_stride;
  a.batch = batch;
  a.table_width = block_table_width;
  a.budget = budget;
  a.sink = sink;
  a.recent = recent;
  a.most = (int32_t)most;
  // j * magic >> 32 = j / per_page while j * per_page < 2^32: j is below 16384.
  const uint32_t per_page = (uint32_t)(page_size / block_size);
  a.page_magic = per_page > 1 ? (uint32_t)(((1ull << 32) + per_page - 1) / per_page) : 0;
  a.order = static_cast<uint64_t*>(workspace);
  a.out = blocks;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == HX_DTYPE_BF16) launch_select<__bf16>(a, n, s);
  else launch_select<_Float16>(a, n, s);
  return hx::status_from_hip(hipGetLastError());
}

extern "C" size_t hx_block_sparse_workspace_bytes(int64_t n, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                                                  int32_t budget, int32_t block_size) {
  if (n < 1 || n_kv_heads < 1 || n_q_heads < 1 || n_q_heads % n_kv_heads || head_dim < 1 || budget < 1 ||
      block_size < 16)
    return 0;
  const int32_t head_blocks = (n_q_heads / n_kv_heads + kSpHeads - 1) / kSpHeads;
  const Split sp = sparse_split(n, n_kv_heads, head_blocks, budget, block_size);
  return sp.splits == 1 ? 0 : (size_t)n * n_q_heads * sp.splits * (head_dim + 2) * sizeof(float);
}

extern "C" int hx_block_sparse_attn(const void* q, int64_t q_row_stride, int64_t q_head_stride, int64_t q_rows,
                                    const int64_t* rows, const int32_t* row_seq, const int32_t* key_counts, int64_t n,
                                    const void* k_pool, const void* v_pool, int32_t num_pages, int32_t page_size,
                                    int32_t block_size, const int32_t* blocks, int32_t budget,
                                    const int32_t* block_table, int64_t block_table_stride, int32_t batch,
                                    int32_t block_table_width, int32_t n_q_heads, int32_t n_kv_heads,
                                    int32_t head_dim, float scale, int32_t dtype, void* out, int64_t out_row_stride,
                                    int64_t out_head_stride, void* workspace, size_t workspace_bytes, void* stream) {
  const int bad = check_layout(num_pages, page_size, block_size, n_kv_heads, head_dim, dtype);
  if (bad != HX_OK) return bad;
  if (n < 0 || q_rows < 0 || n_q_heads < 1 || n_q_heads % n_kv_heads || batch < 0 || block_table_width < 1 ||
      block_table_stride < block_table_width || budget < 1 || budget > (1 << 24))
    return HX_E_INVALID_ARG;
  if (n == 0) return HX_OK;
  if (!q || !key_counts || !k_pool || !v_pool || !blocks || !block_table || !out || (rows == nullptr && n > q_rows) ||
      (row_seq == nullptr && n > batch))
    return HX_E_INVALID_ARG;
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool)) &
       15) ||
      q_row_stride % 8 || q_head_stride % 8 || (reinterpret_cast<uintptr_t>(out) & 3) || out_row_stride % 2 ||
      out_head_stride % 2)
    return HX_E_INVALID_ARG;
  SparseArgs a;
  a.q = static_cast<const uint16_t*>(q);
  a.q_row = q_row_stride;
  a.q_head = q_head_stride;
  a.q_rows = q_rows;
  a.rows = rows;
  a.row_seq = row_seq;
  a.keys = key_counts;
  a.k = static_cast<const uint16_t*>(k_pool);
  a.v = static_cast<const uint16_t*>(v_pool);
  a.num_pages = num_pages;
  a.page = page_size;
  a.block = block_size;
  a.blocks = blocks;
  a.budget = budget;
  a.table = block_table;
  a.table_stride = block_table_stride;
  a.batch = batch;
  a.table_width = block_table_width;
  a.n_heads = n_kv_heads;
  a.group = n_q_heads / n_kv_heads;
  a.head_dim = head_dim;
  a.head_blocks = (a.group + kSpHeads - 1) / kSpHeads;
  a.scale_log2 = scale * kSpLog2e;
  a.out = static_cast<uint16_t*>(out);
  a.out_row = out_row_stride;
  a.out_head = out_head_stride;
  const Split sp = sparse_split(n, n_kv_heads, a.head_blocks, budget, block_size);
  a.splits = sp.splits;
  a.units = sp.units;
  a.part_o = a.part_ml = nullptr;
  if (a.splits > 1) {
    const size_t parts = (size_t)n * n_q_heads * a.splits;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) ||
        workspace_bytes < parts * (head_dim + 2) * sizeof(float))
      return HX_E_WORKSPACE;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + parts * head_dim;
  }
  if ((double)n * n_q_heads * a.splits > kMostItems / (64 * kSpWaves)) return HX_E_UNSUPPORTED;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == HX_DTYPE_BF16) launch_sparse_dims<__bf16>(a, n, s);
  else launch_sparse_dims<_Float16>(a, n, s);
  return hx::status_from_hip(hipGetLastError());
}
