// Varlen GQA attention over the paged 8-bit KV cache (gfx950).
//
// With key codes c, value codes v, scales s_k and s_v per token and KV head:
//   u_j = log2(e) scale (q . c_j) s_kj + log2 s_vj,   w_j = 2^(u_j - M),   M = max_j u_j
//   out = sum_j w_j v_j / sum_j (w_j / s_vj)
// The value's scale rides on the softmax's exponent: the weights that meet the codes have their
// maximum at 1 whatever the scales of the values are, and fit fp16 together with the codes, which
// fp16 holds exactly. q goes into the products as fp16 too, each row and head after a power of two of
// its own that puts its largest element at 2^14: exact down to 2^-28 of that element (smaller ones
// within 2^-39 of it). Sums are fp32.
//
// Two kernels over a plan's work lists, in one launch where a tick has both, and one that joins splits:
//   few_kernel    sequences whose (row, query head) pairs of a KV head fit one MFMA's 16 columns
//                 (decode rows, a few drafted ones), split over their keys. Bound by HBM: 64
//                 decoders with 8 KV heads of 128, 306 MB, take 61 us with the join, 5.0 TB/s
//                 (the loads alone 50 to 55); one of 32768 keys 22, 4.1 TB/s in the launch.
//   chunk_kernel  the others: blocks of rows over 64-key tiles, split over their tiles where the
//                 blocks alone leave CUs without work. Bound by MFMA, the reads of its operands from
//                 LDS and the softmax, which overlap only in part: 4096 rows that see 4096 keys and
//                 their own, 32 heads of 128, take 603 us, 685 TFLOP/s, the matrix units busy for 43 %
//                 of the time. (The 16-bit cache's kernel takes 350: a prompt is faster from there.)

#include "kv8_common.h"

#include <math.h>

namespace {

constexpr int64_t kMostItems = (int64_t)1 << 32;  // work-items of a launch
constexpr float kLog2e = 1.44269504088896340736f;

constexpr int kFewUnits = 16;     // (row, head) pairs of a few_kernel item
constexpr int kFewThreads = 256;  // 4 waves, each on its own 32-key tiles
constexpr int kFewTile = 32;
// Work of few_kernel's rows is dealt in equal parts of the tick's tiles, whatever the sequences are:
// a part ends in the middle of one and goes on in the next. A sequence counts kFewStart tiles more
// than it has, for what its start costs (loads that wait for one another, the waves' merge).
constexpr int kFewWGs = 768;      // workgroups, about: 3 a CU, all at once
constexpr int kFewStart = 8;
constexpr int kFewLeast = 24;     // of a part, at least: tiles and starts
constexpr int kFewMost = 256;     // and at most
constexpr int kChunkUnits = 128;  // (row, head) pairs of a chunk block
constexpr int kChunkTile = 64;
// Workgroups below which row blocks are split, and into about as many. (512 would be on the CUs at
// once, but partial results cost too: decoders beside chunks whose blocks are 344 workgroups take 107 us
// split for 384, 110 for 512, 113 as they are, 115 for 768.)
constexpr int kChunkWGs = 384;
constexpr int kChunkLeast = 4;    // tiles of a split, at least
constexpr int kShortJoin = 4;     // splits that a part of a wave joins; a workgroup does more
constexpr int kPlanThreads = 1024;

// Plan header words.
enum { H_PARTS = 0, H_CHUNK = 1, H_JOIN = 2, H_ERR = 3, H_STAMP = 4, H_SHORT = 12, H_STAMP2 = 13, H_WORDS = 16 };

__host__ __device__ inline int ceil_div(int a, int b) { return (a + b - 1) / b; }
inline int64_t ceil_div64(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

// What a plan is built for; its runs must agree, which is checked on the device.
struct Shape {
  int32_t batch, total_q, max_q, max_k, hq, hkv, head_dim, page;
  int32_t left, right, width;
};

struct Sizes {
  int32_t group;
  int32_t few_heads, head_blocks;  // query heads of a few item, and items over a group's heads
  int32_t few_rows;                // rows of a sequence that few_kernel takes
  int32_t few_cap;                 // most tiles of a part
  int32_t chunk_rows;              // rows of a chunk block
};


inline Sizes sizes_of(const Shape& s) {
  Sizes z;
  z.group = s.hq / s.hkv;
  z.few_heads = z.group < kFewUnits ? z.group : kFewUnits;
  z.head_blocks = ceil_div(z.group, kFewUnits);
  z.few_rows = z.group <= kFewUnits ? kFewUnits / z.group : 1;
  const int pages = 62 * (s.page / kFewTile);  // a wave holds a part's page ids of a sequence, one a lane
  z.few_cap = pages < kFewMost ? pages : kFewMost;
  z.chunk_rows = kChunkUnits / z.group;
  return z;
}

struct Layout {
  size_t seq, part, few, chunk, join, ml, o, total;
  int64_t most_parts, most_few, most_chunk, most_join, slots;
};

inline Layout layout_of(const Shape& s) {
  const Sizes z = sizes_of(s);
  Layout l;
  const int64_t few_rows = s.max_q < z.few_rows ? s.max_q : z.few_rows;
  l.most_parts = ceil_div64(kFewWGs, (int64_t)s.hkv * z.head_blocks) +
                 ceil_div64((int64_t)s.batch * (s.max_k / kFewTile + 2 + kFewStart), z.few_cap) + 1;
  l.most_few = l.most_parts + s.batch;  // a part's end cuts one item in two
  l.slots = l.most_few * few_rows;
  l.most_join = (int64_t)s.batch * few_rows;
  l.most_chunk = 0;
  if (s.max_q > z.few_rows) {
    const int64_t rows = s.max_q < z.chunk_rows ? s.max_q : z.chunk_rows;
    const int64_t unsplit = ceil_div64(kChunkWGs, s.hkv);  // splits exist below this many blocks
    int64_t blocks = (int64_t)s.batch * ceil_div64(s.max_q, z.chunk_rows);
    const int64_t by_rows = s.total_q / z.chunk_rows + s.batch;
    blocks = blocks < by_rows ? blocks : by_rows;
    l.most_chunk = blocks + unsplit + 1;
    l.slots += (2 * unsplit + 1) * rows;
    l.most_join += unsplit * rows;
  }
  size_t off = align256(H_WORDS * sizeof(int32_t));
  l.seq = off;    off = align256(off + (size_t)s.batch * sizeof(int4));
  l.part = off;   off = align256(off + (size_t)(l.most_parts + 1) * 3 * sizeof(int4));
  l.few = off;    off = align256(off + (size_t)l.most_few * 2 * sizeof(int4));
  l.chunk = off;  off = align256(off + (size_t)l.most_chunk * 2 * sizeof(int4));
  l.join = off;   off = align256(off + (size_t)l.most_join * sizeof(int4));
  l.ml = off;     off = align256(off + (size_t)l.slots * s.hq * sizeof(float2));
  l.o = off;      off = align256(off + (size_t)l.slots * s.hq * s.head_dim * sizeof(float));
  l.total = off;
  return l;
}

// -------------------------------------------------------------------------------- plan
//
// Work lists, two int4 an entry:
//   few:   {sequence, first key, key end, slot or -1} {first query row, rows, keys, -}, in the
//          sequences' order
//   part:  {its first entry of few} and that entry; it goes on to the next part's
//   chunk: {sequence, first row, first tile, tile end} {first query row, rows, keys, slot or -1}
//   join:  {output row, first slot, slots from one split to the next, splits}; those of up to
//          kShortJoin splits from the list's end backwards
// A slot holds the partial result of one query row, all heads.
struct PlanArgs {
  const int32_t* cu_q;
  const int32_t* used;
  int32_t* hdr;
  int4* seq;
  int4* part;
  int4* few;
  int4* chunk;
  int4* join;
  int64_t most_parts, most_few, most_chunk, most_join, slots;
  Shape s;
  Sizes z;
};

// Keys [lo, hi) that rows [row0, row0 + rows) of a sequence with n rows and L keys see.
__device__ __forceinline__ void keys_of(const Shape& s, int n, int L, int row0, int rows, int* lo, int* hi) {
  const int64_t first = (int64_t)L - n + row0;
  int64_t a = s.left >= 0 ? first - s.left : 0, b = s.right >= 0 ? first + rows + s.right : L;
  a = a < 0 ? 0 : a;
  b = b > L ? L : b;
  *lo = (int)(a < L ? a : L);
  *hi = (int)(b > *lo ? b : *lo);
}

// Exclusive prefix sum over the workgroup of three values; their totals.
__device__ int3 plan_scan(int3 v, int3* total, int3 (*waves)) {
  const int lane = hx::tid_x() & 63, w = hx::tid_x() >> 6;
  int3 x = v;
  for (int m = 1; m < 64; m <<= 1) {
    const int a = __shfl_up(x.x, m), b = __shfl_up(x.y, m), c = __shfl_up(x.z, m);
    if (lane >= m) {
      x.x += a;
      x.y += b;
      x.z += c;
    }
  }
  __syncthreads();
  if (lane == 63) waves[w] = x;
  __syncthreads();
  int3 before = make_int3(0, 0, 0), all = make_int3(0, 0, 0);
  for (int i = 0; i < kPlanThreads / 64; ++i) {
    if (i < w) {
      before.x += waves[i].x;
      before.y += waves[i].y;
      before.z += waves[i].z;
    }
    all.x += waves[i].x;
    all.y += waves[i].y;
    all.z += waves[i].z;
  }
  *total = all;
  return make_int3(before.x + x.x - v.x, before.y + x.y - v.y, before.z + x.z - v.z);
}

// Which of the prefix sums p[0 .. n] (n of them and the total) holds i: the last at or below it.
__device__ __forceinline__ int plan_find(const int* p, int n, int i) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int block_tiles(const PlanArgs& a, int n, int L, int row0, int* first) {
  int lo, hi;
  keys_of(a.s, n, L, row0, n - row0 < a.z.chunk_rows ? n - row0 : a.z.chunk_rows, &lo, &hi);
  *first = lo / kChunkTile;
  return hi > lo ? ceil_div(hi, kChunkTile) - *first : 0;
}

// 32-key tiles of a sequence of few rows, and the first.
__device__ __forceinline__ int few_tiles(const PlanArgs& a, int n, int L, int* lo, int* hi) {
  keys_of(a.s, n, L, 0, n, lo, hi);
  return *hi > *lo ? ceil_div(*hi, kFewTile) - *lo / kFewTile : 0;
}

__global__ __launch_bounds__(kPlanThreads) void kv8_plan_kernel(PlanArgs a) {
  __shared__ int3 s_waves[kPlanThreads / 64];
  __shared__ int s_items[kPlanThreads], s_slots[kPlanThreads], s_blocks[kPlanThreads], s_cost[kPlanThreads];
  __shared__ unsigned long long s_few, s_tiles;
  __shared__ int s_err, s_nblocks, s_join, s_short;
  const int tid = hx::tid_x(), batch = a.s.batch;
  if (tid == 0) {
    s_few = s_tiles = 0;
    s_err = s_nblocks = s_join = s_short = 0;
  }
  __syncthreads();
  const int64_t room = (int64_t)a.s.width * a.s.page;
  // Every sequence's rows and keys, checked, and the tick's tiles.
  for (int b0 = 0; b0 < batch; b0 += kPlanThreads) {
    const int b = b0 + tid;
    int n = 0, L = 0, blocks = 0;
    if (b < batch) {
      const int q0 = a.cu_q[b], q1 = a.cu_q[b + 1];
      int err = 0;
      L = a.used[b];
      if (q0 < 0 || q1 < q0 || q1 > a.s.total_q) {
        err |= HX_WERR_BAD_CU_SEQ;
      } else {
        n = q1 - q0;
        if (n > a.s.max_q) {
          n = a.s.max_q;
          err |= HX_WERR_CLAMPED_LEN;
        }
      }
      const int64_t most = a.s.max_k < room ? a.s.max_k : room;
      if (L < 0 || L > most) {
        L = L < 0 ? 0 : (int)most;
        err |= HX_WERR_CLAMPED_LEN;
      }
      if (err) atomicOr(&s_err, err);
      a.seq[b] = make_int4(q0, n, L, 0);
      if (n > 0 && n <= a.z.few_rows) {
        int lo, hi;
        atomicAdd(&s_few, (unsigned long long)(few_tiles(a, n, L, &lo, &hi) + kFewStart));
      } else if (n > 0) {
        blocks = ceil_div(n, a.z.chunk_rows);
      }
    }
    int3 total;
    const int3 at = plan_scan(make_int3(blocks, 0, 0), &total, s_waves);
    __syncthreads();
    s_blocks[tid] = at.x;
    if (tid == 0) s_nblocks += total.x;
    __syncthreads();
    unsigned long long tiles = 0;
    for (int i = tid; i < total.x; i += kPlanThreads) {
      const int j = plan_find(s_blocks, kPlanThreads, i);
      const int4 si = a.seq[b0 + j];
      int first;
      tiles += (unsigned long long)block_tiles(a, si.y, si.z, (i - s_blocks[j]) * a.z.chunk_rows, &first);
    }
    if (tiles) atomicAdd(&s_tiles, tiles);
    __syncthreads();
  }
  // Parts of the few rows' tiles; blocks of chunk rows are split only when they are fewer than
  // kChunkWGs.
  const int64_t few_wgs = kFewWGs / (a.s.hkv * a.z.head_blocks) > 0 ? kFewWGs / (a.s.hkv * a.z.head_blocks) : 1;
  const int64_t even = ((int64_t)s_few + few_wgs - 1) / few_wgs;
  const int share = (int)(even > a.z.few_cap ? a.z.few_cap : even < kFewLeast ? kFewLeast : even);
  const int parts = (int)(((int64_t)s_few + share - 1) / share);
  int chunk_split = 1 << 30;
  if ((int64_t)s_nblocks * a.s.hkv < kChunkWGs) {
    const int64_t t = ((int64_t)s_tiles * a.s.hkv + kChunkWGs - 1) / kChunkWGs;
    chunk_split = (int)(t < kChunkLeast ? kChunkLeast : t);
  }
  int few_base = 0, cost_base = 0, chunk_base = 0, slot_base = 0;
  // Rows to join, from `of` on; their order in the list is of no account.
  auto add_joins = [&](int4 of, int rows) {
    const bool is_short = of.w <= kShortJoin;
    const int at = atomicAdd(is_short ? &s_short : &s_join, rows);
    for (int r = 0; r < rows; ++r) {
      const int64_t to = is_short ? a.most_join - 1 - (at + r) : at + r;
      if (to >= 0 && to < a.most_join) a.join[to] = make_int4(of.x + r, of.y + r, of.z, of.w);
    }
  };
  for (int b0 = 0; b0 < batch; b0 += kPlanThreads) {
    const int b = b0 + tid;
    int4 si = make_int4(0, 0, 0, 0);
    int cost = 0, tiles = 0, blocks = 0, rows = 0;
    if (b < batch) {
      si = a.seq[b];
      if (si.y > 0 && si.y <= a.z.few_rows) {
        int lo, hi;
        tiles = few_tiles(a, si.y, si.z, &lo, &hi);
        cost = tiles + kFewStart;
        rows = si.y;
      } else if (si.y > 0) {
        blocks = ceil_div(si.y, a.z.chunk_rows);
      }
    }
    int3 sum;
    const int3 place = plan_scan(make_int3(cost, blocks, 0), &sum, s_waves);
    // Tile x of the sequence lies at its place, and kFewStart, and x: its first and last part.
    const int from = cost_base + place.x, first_part = (tiles ? from + kFewStart : from + cost - 1) / share;
    const int splits = rows ? (from + cost - 1) / share - first_part + 1 : 0;
    const int joined = splits > 1 ? rows : 0;
    int3 total;
    const int3 at = plan_scan(make_int3(splits, joined * splits, 0), &total, s_waves);
    __syncthreads();
    s_items[tid] = at.x;
    s_slots[tid] = at.y;
    s_blocks[tid] = place.y;
    s_cost[tid] = from;
    __syncthreads();
    if (joined) add_joins(make_int4(si.x, slot_base + at.y, rows, splits), joined);
    for (int i = tid; i < total.x; i += kPlanThreads) {
      const int j = plan_find(s_items, kPlanThreads, i);
      const int4 of = a.seq[b0 + j];
      int lo, hi;
      const int n = few_tiles(a, of.y, of.z, &lo, &hi), sp = i - s_items[j], start = s_cost[j];
      const int first = (n ? start + kFewStart : start + kFewStart - 1) / share, last = (start + kFewStart + n - 1) / share;
      const int part = first + sp, t0 = lo / kFewTile, base = start + kFewStart;
      int begin = part * share - base, end = begin + share;
      begin = t0 + (begin > 0 ? begin : 0);
      end = t0 + (end < n ? end : n);
      const int64_t entry = (int64_t)few_base + i;
      const int4 e0 = make_int4(b0 + j, begin * kFewTile > lo ? begin * kFewTile : lo, end * kFewTile < hi ? end * kFewTile : hi,
                                last > first ? slot_base + s_slots[j] + sp * of.y : -1);
      const int4 e1 = make_int4(of.x, of.y, of.z, 0);
      if (entry < a.most_few) {
        a.few[2 * entry] = e0;
        a.few[2 * entry + 1] = e1;
      }
      // The first entry of its part, and of parts that have none.
      for (int q = sp ? part : start ? (start - 1) / share + 1 : 0; q <= part; ++q)
        if (q < a.most_parts) {
          a.part[3 * q] = make_int4((int)entry, 0, 0, 0);
          a.part[3 * q + 1] = e0;
          a.part[3 * q + 2] = e1;
        }
    }
    cost_base += sum.x;
    const int3 total2 = make_int3(sum.y, 0, 0);
    few_base += total.x;
    slot_base += total.y;
    // Chunk blocks, a round of the threads at a time: their items, slots and joined rows follow
    // those of the blocks before them. Later blocks of a sequence first: they see more keys.
    for (int i0 = 0; i0 < total2.x; i0 += kPlanThreads) {
      const int i = i0 + tid;
      int n = 0, tiles = 0, first = 0, row0 = 0, rows_here = 0, j = 0;
      int4 of = make_int4(0, 0, 0, 0);
      if (i < total2.x) {
        j = plan_find(s_blocks, kPlanThreads, i);
        of = a.seq[b0 + j];
        row0 = (ceil_div(of.y, a.z.chunk_rows) - 1 - (i - s_blocks[j])) * a.z.chunk_rows;
        rows_here = of.y - row0 < a.z.chunk_rows ? of.y - row0 : a.z.chunk_rows;
        tiles = block_tiles(a, of.y, of.z, row0, &first);
        n = tiles > 0 ? ceil_div(tiles, chunk_split) : 1;
      }
      const int joins = n > 1 ? rows_here : 0;
      int3 all;
      const int3 to = plan_scan(make_int3(n, joins * n, 0), &all, s_waves);
      const int share = n > 0 ? ceil_div(tiles, n) : 0;
      for (int sp = 0; sp < n; ++sp) {
        const int64_t entry = (int64_t)chunk_base + to.x + sp;
        if (entry >= a.most_chunk) break;
        const int from = first + (sp * share < tiles ? sp * share : tiles);
        const int end = from + share < first + tiles ? from + share : first + tiles;
        a.chunk[2 * entry] = make_int4(b0 + j, row0, from, end);
        a.chunk[2 * entry + 1] = make_int4(of.x, of.y, of.z, n > 1 ? slot_base + to.y + sp * rows_here : -1);
      }
      if (joins) add_joins(make_int4(of.x + row0, slot_base + to.y, rows_here, n), joins);
      chunk_base += all.x;
      slot_base += all.y;
    }
    __syncthreads();
  }
  if (tid == 0) {
    int err = s_err;
    // By the bounds that the workspace was sized with none of these can happen.
    if (parts > a.most_parts || few_base > a.most_few || chunk_base > a.most_chunk ||
        (int64_t)s_join + s_short > a.most_join || slot_base > a.slots) err |= HX_WERR_GRID;
    const int most = (int)(parts < a.most_parts ? parts : a.most_parts);
    a.hdr[H_PARTS] = most;
    a.part[3 * most] = make_int4(few_base < a.most_few ? few_base : (int)a.most_few, 0, 0, 0);
    a.hdr[H_CHUNK] = chunk_base < a.most_chunk ? chunk_base : (int)a.most_chunk;
    a.hdr[H_JOIN] = s_join < a.most_join ? s_join : (int)a.most_join;
    a.hdr[H_SHORT] = s_short < a.most_join ? s_short : (int)a.most_join;
    a.hdr[H_ERR] = err;
    const int32_t stamp[8] = {a.s.batch, a.s.total_q, a.s.max_q, a.s.max_k, a.s.hq, a.s.hkv, a.s.head_dim, a.s.page};
    for (int i = 0; i < 8; ++i) a.hdr[H_STAMP + i] = stamp[i];
    a.hdr[H_STAMP2] = a.s.left;
    a.hdr[H_STAMP2 + 1] = a.s.right;
    a.hdr[H_STAMP2 + 2] = a.s.width;
  }
}

// --------------------------------------------------------------------------------- run
struct RunArgs {
  const uint16_t* q;
  int64_t q_row, q_head;
  const uint8_t* k;
  const uint8_t* v;
  const float* k_scale;
  const float* v_scale;
  int32_t num_pages;
  const int32_t* table;
  int64_t table_stride;
  float scale_log2;
  uint16_t* out;
  int64_t out_row, out_head;
  int32_t* hdr;
  const int4* part;
  const int4* few;
  const int4* chunk;
  const int4* join;
  float2* part_ml;
  float* part_o;
  int64_t slots, most_join;
  Shape s;
  Sizes z;
};

// The plan's counts, if it was built for this shape.
__device__ __forceinline__ bool plan_ok(const RunArgs& a, int4* counts) {
  const int4 h0 = *reinterpret_cast<const int4*>(a.hdr), h1 = *reinterpret_cast<const int4*>(a.hdr + H_STAMP),
             h2 = *reinterpret_cast<const int4*>(a.hdr + H_STAMP + 4), h3 = *reinterpret_cast<const int4*>(a.hdr + H_SHORT);
  *counts = h0;
  const bool ok = h1.x == a.s.batch && h1.y == a.s.total_q && h1.z == a.s.max_q && h1.w == a.s.max_k && h2.x == a.s.hq &&
                  h2.y == a.s.hkv && h2.z == a.s.head_dim && h2.w == a.s.page && h3.y == a.s.left && h3.z == a.s.right &&
                  h3.w == a.s.width;
  if (!ok && hx::wg_x() == 0 && hx::tid_x() == 0) atomicOr(&a.hdr[H_ERR], HX_WERR_PLAN_MISMATCH);
  return ok;
}

__device__ __forceinline__ int4 uniform4(const int4* p) {
  const int4 v = *p;
  return make_int4(__builtin_amdgcn_readfirstlane(v.x), __builtin_amdgcn_readfirstlane(v.y),
                   __builtin_amdgcn_readfirstlane(v.z), __builtin_amdgcn_readfirstlane(v.w));
}

// The power of two that takes magnitudes up to `top` (bits) to [2^14, 2^15), and its inverse.
// Below 2^-107 magnitudes stay smaller than that: what they lose is nothing to a score.
__device__ __forceinline__ float fit_up(uint32_t top) { return __uint_as_float((268u - max(top >> 23, 20u)) << 23); }
__device__ __forceinline__ float fit_down(uint32_t top) { return __uint_as_float((max(top >> 23, 20u) - 14u) << 23); }

// The largest finite magnitude among packed elements, as their type's bits (a step further than
// `top`), and those bits as fp32's. (An infinite or NaN element passes through any power of two.)
template <typename T>
__device__ __forceinline__ uint32_t largest(uint4 u, uint32_t top) {
  constexpr uint32_t kInf = __is_same(T, __bf16) ? 0x7f80u : 0x7c00u;
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t lo = w[e] & 0x7fffu, hi = w[e] >> 16 & 0x7fffu;
    top = max(top, lo < kInf ? lo : 0u);
    top = max(top, hi < kInf ? hi : 0u);
  }
  return top;
}
template <typename T>
__device__ __forceinline__ uint32_t magnitude(uint32_t top) { return __float_as_uint(hx::Elem<T>::lo(top)); }

// A value's scale as the softmax takes it. (Sums of weights over scales fit fp32 for 2^17 keys of scales
// above 2^-96; values below those, 1e-26, may come out as 0. Weights times scales below 2^-126 of the
// row's largest are 0.) A NaN makes the weight NaN through its logarithm, and has an inverse that
// leaves the weight 0 of a row that does not see the key alone.
struct ValueScale {
  float log, inverse;
};
__device__ __forceinline__ ValueScale value_scale(float s) {
  const bool nan = (hx::raw_bits(s) & 0x7fffffffu) > 0x7f800000u;
  const float at_least = nan ? 1.f : fmaxf(s, hx8::kLeastScale);
  return {nan ? __uint_as_float(0x7fc00000u) : __builtin_amdgcn_logf(at_least), __builtin_amdgcn_rcpf(at_least)};
}

// Key positions `at + more`, which may lie far past the last key.
__device__ __forceinline__ int beyond(int at, int more) {
  const int64_t x = (int64_t)at + more;
  return x < 0x7fffffff ? (int)x : 0x7fffffff;
}

template <typename T>
__device__ __forceinline__ void widen8(uint4 u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = hx::Elem<T>::lo(w[e]);
    x[2 * e + 1] = hx::Elem<T>::hi(w[e]);
  }
}

__device__ __forceinline__ uint4 pack8(const float (&x)[8], float by) {
  return make_uint4(hx::pack2_round<_Float16>(x[0] * by, x[1] * by), hx::pack2_round<_Float16>(x[2] * by, x[3] * by),
                    hx::pack2_round<_Float16>(x[4] * by, x[5] * by), hx::pack2_round<_Float16>(x[6] * by, x[7] * by));
}

template <typename C>
__device__ __forceinline__ hx::f16x8_t codes8(uint2 w) {
  const uint2 a = hx8::to_f16<C>(w.x), b = hx8::to_f16<C>(w.y);
  return hx::as_v8<_Float16>(make_uint4(a.x, a.y, b.x, b.y));
}

__device__ __forceinline__ uint2 ld8_lds_tr8(const void* p) {
  typedef int v2i __attribute__((ext_vector_type(2)));
  const v2i r = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i*)(p));
  return __builtin_bit_cast(uint2, r);
}

// The score that a softmax's weights are relative to: SHIFT below the largest, so that weights fill
// fp16 and their remainders stay normal. It moves when a score exceeds that largest one by more than
// LAZY; SHIFT + LAZY <= 15, all in log2. Past 2^22 fp32's steps are of their size, and its rounding
// could take a weight past fp16: there it is the largest score itself, and moves with each larger one.
constexpr float kStepsFit = 0x1p22f;
__device__ __forceinline__ float reference_of(float most, float shift) {
  return fabsf(most) < kStepsFit ? most - shift : most;
}
__device__ __forceinline__ float moves_past(float ref, float by) { return fabsf(ref) < kStepsFit ? ref + by : ref; }

constexpr float kFewShift = 14.f, kFewLazy = 1.f;

template <int DP>
struct FewLds {
  union {
    // The waves' codes. Rows of an odd number of 16-byte pieces: 16 rows' pieces of one dim block
    // cover all banks once.
    struct {
      __attribute__((aligned(16))) uint8_t k[4][kFewTile * (DP + 16)];
      __attribute__((aligned(16))) uint8_t v[4][kFewTile * (DP + 16)];
    };
    __attribute__((aligned(16))) float o[4][kFewUnits][DP];    // their results
  };
  __attribute__((aligned(16))) float scale[4][3][kFewTile];    // of a tile: keys' scales, log2 and inverse of values'
  float m[4][kFewUnits], l[4][kFewUnits];
};

struct FewItem {
  int seq, k0, k1, slot;  // keys [k0, k1)
  int q0, n, L;
  int h, head0, heads;    // KV head, first query head and how many
};

// One item and KV head (and block of 16 query heads) to a workgroup. The units, (row, head) pairs,
// are the columns of S^T = K Q^T. A wave walks every fourth 32-key tile on its own through its part
// of LDS, the next one's codes in flight in registers. Row r of the MFMA's operand for block u is key
// 8 (r / 4) + 4 u + r % 4, so that a lane's 8 scores belong to 8 consecutive keys; value codes are
// read transposed. TWICE: up to 8 units, whose
// second set of columns carries the weights' remainders; more take a second MFMA: 22 bits.
template <typename T, typename C, int DP, bool TWICE>
__device__ __forceinline__ void few_item(const RunArgs& a, FewLds<DP>& lds, const FewItem& it) {
  typedef hx::f16x8_t v8;
  typedef hx::Elem<_Float16> E;
  constexpr int kLoads = DP / 64, kSteps = DP / 32, kDims = DP / 16, kPieces = DP / 16, kVLoads = DP / 32;
  const int tid = hx::tid_x(), lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int D = a.s.head_dim, page = a.s.page, k0 = it.k0, k1 = it.k1, heads = it.heads, units = it.n * heads;
  const uint32_t row_bytes = (uint32_t)a.s.hkv * (uint32_t)D;
  uint8_t *const kt = lds.k[w], *const vt = lds.v[w];
  const int unit = TWICE ? lr & 7 : lr;
  const bool live = unit < units;
  const int urow = live ? unit / heads : 0, uhead = it.head0 + (live ? unit - urow * heads : 0);

  const int t0 = k0 / kFewTile, t1 = k1 > k0 ? (k1 + kFewTile - 1) / kFewTile : t0;
  // Page ids of the item's keys: lane j holds that of page pg0 + j.
  const int pg0 = t0 * kFewTile / page;
  int ids = -1;
  if (t1 > t0 && pg0 + lane <= (k1 - 1) / page) ids = a.table[(int64_t)it.seq * a.table_stride + pg0 + lane];

  v8 qf[kSteps];
  float qc;  // of this lane's unit: log2(e) scale, and what undoes q's power of two
  {
    uint4 raw[kSteps];
    const uint16_t* const qp = a.q + (int64_t)(it.q0 + urow) * a.q_row + (int64_t)uhead * a.q_head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = 64 * (s >> 1) + 16 * lg + 8 * (s & 1);
      raw[s] = live && d < D ? *reinterpret_cast<const uint4*>(qp + d) : hx::zero4();
    }
    uint32_t top = 0;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) top = largest<T>(raw[s], top);
    top = max(top, (uint32_t)__shfl_xor((int)top, 16));
    top = max(top, (uint32_t)__shfl_xor((int)top, 32));
    top = magnitude<T>(top);
    const float up = fit_up(top);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      float x[8];
      widen8<T>(raw[s], x);
      qf[s] = hx::as_v8<_Float16>(pack8(x, up));
    }
    qc = a.scale_log2 * fit_down(top);
  }
  // Keys this lane's unit sees of the item's. (Columns without a unit have q = 0 and go nowhere.)
  int klo = k0, khi = k1 - 1;
  {
    const int at = it.L - it.n + urow;
    if (a.s.left >= 0) klo = max(klo, at > a.s.left ? at - a.s.left : 0);
    if (a.s.right >= 0) khi = min(khi, beyond(at, a.s.right));
  }

  // Lane l of a load takes piece l % kPieces of row l / kPieces: whole rows, side by side. Past
  // head_dim its offset is one that no tile reaches.
  constexpr int kRows = 64 / kPieces;  // rows of a load
  const uint32_t off = 16 * (lane % kPieces) < D ? (uint32_t)(lane / kPieces) * row_bytes + 16u * (lane % kPieces) : 0x7ffffff0u;
  const int to = lane / kPieces * (DP + 16) + 16 * (lane % kPieces);
  uint4 kb[kVLoads], vb[kVLoads];
  float sreg;  // lanes 0-31: the keys' scales, 32-63: the values'
  int next_cnt = 0;
  bool bad = false;
  auto load = [&](int t) __attribute__((always_inline)) {
    const int key0 = t * kFewTile, j = key0 / page;
    int id = __builtin_amdgcn_readlane(ids, j - pg0);
    const bool none = (unsigned)id >= (unsigned)a.num_pages;
    bad |= none;
    id = none ? 0 : id;
    const int cnt = none ? 0 : min(kFewTile, k1 - key0);
    next_cnt = cnt;
    const int64_t in = key0 - j * page;
    const int64_t base = (((int64_t)id * page + in) * a.s.hkv + it.h) * D;
    const uint32_t bytes = cnt > 0 ? (uint32_t)(cnt - 1) * row_bytes + (uint32_t)D : 0u;
    const __amdgpu_buffer_rsrc_t kr = hx::buffer_rsrc(a.k + base, bytes), vr = hx::buffer_rsrc(a.v + base, bytes);
#pragma unroll
    for (int q = 0; q < kVLoads; ++q) kb[q] = hx::ld16_stream(kr, off, q * kRows * row_bytes);
    const float* const sp = lane < 32 ? a.k_scale : a.v_scale;
    sreg = sp[((int64_t)id * a.s.hkv + it.h) * page + in + (lane & 31)];
#pragma unroll
    for (int q = 0; q < kVLoads; ++q) vb[q] = hx::ld16_stream(vr, off, q * kRows * row_bytes);
  };

  float ref = -INFINITY, l_run = 0.f;  // the weights' reference, and their sum
  hx::f32x4_t o[kDims];
#pragma unroll
  for (int d = 0; d < kDims; ++d) o[d] = hx::f32x4_t{0.f, 0.f, 0.f, 0.f};

  int t = t0 + w;
  if (t < t1) load(t);
  while (t < t1) {
    const int key0 = t * kFewTile, cnt = next_cnt;
    t += 4;
#pragma unroll
    for (int q = 0; q < kVLoads; ++q) {
      *reinterpret_cast<uint4*>(kt + to + q * kRows * (DP + 16)) = kb[q];
      *reinterpret_cast<uint4*>(vt + to + q * kRows * (DP + 16)) = vb[q];
    }
    // A lane's key or value scale to where its 16 columns' lanes find 8 in a row.
    {
      const ValueScale v = value_scale(sreg);
      lds.scale[w][lane < 32 ? 0 : 1][lane & 31] = lane < 32 ? sreg : v.log;
      if (lane >= 32) lds.scale[w][2][lane & 31] = v.inverse;
    }
    // Lanes read what others of the wave stored: a wave's LDS accesses complete in order, the
    // fences hold the compiler to it.
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (t < t1) load(t);
    hx::f32x4_t sc[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      sc[u] = hx::f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < kLoads; ++q) {
        const uint4 kw = *reinterpret_cast<const uint4*>(kt + (8 * (lr >> 2) + 4 * u + (lr & 3)) * (DP + 16) + 64 * q + 16 * lg);
        sc[u] = E::mfma16x16x32(codes8<C>(make_uint2(kw.x, kw.y)), qf[2 * q], sc[u]);
        sc[u] = E::mfma16x16x32(codes8<C>(make_uint2(kw.z, kw.w)), qf[2 * q + 1], sc[u]);
      }
    }
    float u[8], inv[8];
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      const float4 ks = *reinterpret_cast<const float4*>(&lds.scale[w][0][8 * lg + e]);
      const float4 lv = *reinterpret_cast<const float4*>(&lds.scale[w][1][8 * lg + e]);
      const float4 iv = *reinterpret_cast<const float4*>(&lds.scale[w][2][8 * lg + e]);
      u[e] = fmaf(sc[e / 4][0], ks.x * qc, lv.x);
      u[e + 1] = fmaf(sc[e / 4][1], ks.y * qc, lv.y);
      u[e + 2] = fmaf(sc[e / 4][2], ks.z * qc, lv.z);
      u[e + 3] = fmaf(sc[e / 4][3], ks.w * qc, lv.w);
      inv[e] = iv.x;
      inv[e + 1] = iv.y;
      inv[e + 2] = iv.z;
      inv[e + 3] = iv.w;
    }
    const int from = key0 + 8 * lg, last = min(khi, key0 + cnt - 1);
    if (__any(from < klo || from + 7 > last)) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool seen = from + e >= klo && from + e <= last;
        u[e] = seen ? u[e] : -INFINITY;
      }
    }
    float mx = fmaxf(u[0], u[1]);
#pragma unroll
    for (int e = 2; e < 8; ++e) mx = fmaxf(mx, u[e]);
    mx = hx::max_xor32(hx::max_xor16(mx));
    const bool move = mx > moves_past(ref, kFewShift + kFewLazy);
    if (__any(move)) {
      const float to = move ? reference_of(mx, kFewShift) : ref;
      const float alpha = move ? hx::fast_exp2(ref - to) : 1.f;
      ref = to;
      l_run *= alpha;
#pragma unroll
      for (int d = 0; d < kDims; ++d) o[d] *= alpha;
    }
    const float neg = ref == -INFINITY ? 0.f : -ref;
    uint32_t pw[4], pr[4];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float p0 = hx::fast_exp2(u[e] + neg), p1 = hx::fast_exp2(u[e + 1] + neg);
      l_run = fmaf(p0, inv[e], l_run);
      l_run = fmaf(p1, inv[e + 1], l_run);
      pw[e / 2] = hx::pack2_round<_Float16>(p0, p1);
      pr[e / 2] = hx::pack2_round<_Float16>(p0 - E::lo(pw[e / 2]), p1 - E::hi(pw[e / 2]));
      if (TWICE) pw[e / 2] = lr >= 8 ? pr[e / 2] : pw[e / 2];
    }
    const v8 pf = hx::as_v8<_Float16>(make_uint4(pw[0], pw[1], pw[2], pw[3]));
    const v8 pf2 = hx::as_v8<_Float16>(make_uint4(pr[0], pr[1], pr[2], pr[3]));
    const uint8_t* const vp = vt + (8 * lg + (lr >> 1)) * (DP + 16) + 8 * (lr & 1);
#pragma unroll
    for (int d0 = 0; d0 < kDims; d0 += 4) {
      uint2 vw[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) vw[e] = ld8_lds_tr8(vp + 16 * (d0 + e));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const v8 vv = codes8<C>(vw[e]);
        o[d0 + e] = E::mfma16x16x32(vv, pf, o[d0 + e]);
        if (!TWICE) o[d0 + e] = E::mfma16x16x32(vv, pf2, o[d0 + e]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  if (bad && lane == 0) atomicOr(&a.hdr[H_ERR], HX_WERR_BAD_PAGE);

  // Lane: dims 16 d + 4 lg .. + 3 of its unit; remainders' columns added.
  l_run = hx::add_xor32(hx::add_xor16(l_run));
  if (TWICE) {
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[d][e] += hx::dpp<0x128>(o[d][e]);  // the lane 8 apart in its row of 16
  }
  __syncthreads();  // every wave is done with its stage
  if (lr < units) {
#pragma unroll
    for (int d = 0; d < kDims; ++d)
      *reinterpret_cast<float4*>(&lds.o[w][lr][16 * d + 4 * lg]) = make_float4(o[d][0], o[d][1], o[d][2], o[d][3]);
    if (lg == 0) {
      lds.m[w][lr] = ref;
      lds.l[w][lr] = l_run;
    }
  }
  __syncthreads();
  const int half = D / 2;
  for (int e = tid; e < units * half; e += kFewThreads) {
    const int un = e / half, d = 2 * (e % half);
    float m = lds.m[0][un];
#pragma unroll
    for (int ww = 1; ww < 4; ++ww) m = fmaxf(m, lds.m[ww][un]);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int ww = 0; ww < 4; ++ww) {
      const float f = hx::fast_exp2(lds.m[ww][un] - ref);
      l = fmaf(f, lds.l[ww][un], l);
      x = fmaf(f, lds.o[ww][un][d], x);
      y = fmaf(f, lds.o[ww][un][d + 1], y);
    }
    const int row = un / heads, head = it.head0 + un - row * heads;
    if (it.slot < 0) {
      const float r = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
      *reinterpret_cast<uint32_t*>(a.out + (int64_t)(it.q0 + row) * a.out_row + (int64_t)head * a.out_head + d) =
          hx::pack2_round<T>(x * r, y * r);
    } else if ((int64_t)it.slot + row < a.slots) {
      const int64_t p = ((int64_t)it.slot + row) * a.s.hq + head;
      *reinterpret_cast<float2*>(a.part_o + p * D + d) = make_float2(x, y);
      if (d == 0) a.part_ml[p] = make_float2(m, l);
    }
  }
  __syncthreads();  // the next item's stages take the place of the results
}

template <typename T, typename C, int DP>
__device__ __forceinline__ void few_items(const RunArgs& a, FewLds<DP>& lds, const int4& counts, int wg, int n_wg) {
  // All parts of one head, then of the next: a head's rows are every eighth 128 bytes of memory, say,
  // and what one head's reads bring along of its neighbours' is there when theirs come. (Heads side
  // by side: 3.9 to 5.4 TB/s of loads alone; this way 5.8 to 6.4.)
  const int64_t work = (int64_t)counts.x * a.s.hkv * a.z.head_blocks;
  for (int64_t i = wg; i < work; i += n_wg) {
    const int sub = (int)((uint32_t)i / (uint32_t)counts.x), part = (int)((uint32_t)i - (uint32_t)sub * (uint32_t)counts.x);
    const int hb = sub / a.s.hkv, h = sub - hb * a.s.hkv;
    int4 e0 = uniform4(a.part + 3 * part + 1), e1 = uniform4(a.part + 3 * part + 2);
    const int first = __builtin_amdgcn_readfirstlane(a.part[3 * part].x), end = __builtin_amdgcn_readfirstlane(a.part[3 * part + 3].x);
    for (int item = first; item < end; ++item) {
      if (item > first) {
        e0 = uniform4(a.few + 2 * (int64_t)item);
        e1 = uniform4(a.few + 2 * (int64_t)item + 1);
      }
      const FewItem it{e0.x, e0.y, e0.z, e0.w, e1.x, e1.y, e1.z, h, h * a.z.group + hb * kFewUnits,
                       min(a.z.few_heads, a.z.group - hb * kFewUnits)};
      if (it.n * it.heads <= 8) few_item<T, C, DP, true>(a, lds, it);
      else few_item<T, C, DP, false>(a, lds, it);
    }
  }
}

template <typename T, typename C, int DP>
__global__ __launch_bounds__(kFewThreads, DP == 256 ? 2 : DP == 128 ? 3 : 4) void kv8_few_kernel(RunArgs a, int n_wg) {
  __shared__ FewLds<DP> lds;
  int4 counts;
  if (plan_ok(a, &counts)) few_items<T, C, DP>(a, lds, counts, hx::wg_x(), n_wg);
}

// ------------------------------------------------------------------------------- chunks
constexpr int chunk_threads(int dp) { return dp == 256 ? 512 : 256; }
constexpr float kChunkShift = 7.f, kChunkLazy = 8.f;

// Rows of fp16 with 16 and 32 bytes more, so that neighbouring rows begin in other banks. Conflicts are
// left: 51M cycles of the 357M that the CUs are busy on the prompt, by which accesses is not known.
constexpr int chunk_k_row(int dp) { return 2 * dp + 16; }
constexpr int chunk_v_row(int dp) { return 2 * dp + 32; }

template <int DP>
struct ChunkLds {
  __attribute__((aligned(16))) uint8_t k[2][kChunkTile * chunk_k_row(DP)], v[2][kChunkTile * chunk_v_row(DP)];
  __attribute__((aligned(16))) float k_scale[2][kChunkTile], v_log[2][kChunkTile], v_inverse[2][kChunkTile];
};

// One item and KV head to a workgroup: wave w owns units 16 RB w .. + 16 RB - 1, (row, head) pairs
// with the group's heads fastest. 64-key tiles of K and V go from HBM through registers, where the
// workgroup widens their codes to fp16 once for all waves, into two LDS buffers in turn: a tile's
// loads are in flight for a whole tile, and one barrier a tile suffices.
// Up to 128 dims a workgroup is 4 waves, and the two on a CU are out of step: one's products run
// under the other's softmax. 8 waves with 256 units halve the staging but wait in step: 1 % faster
// on a long prompt, 11 % slower on a tick of chunks, whose blocks and splits are then twice as large
// (both with weights of one fp16).
// (A power of two for all units of a block would ride on the keys' scales, 2 % of the prompt's time,
// and lose rows that are 2^28 smaller than their neighbours.)
// The weights go into P V as two fp16, 22 bits, as those of few rows do: one alone (11 bits) turns the
// rounding of one bf16 output in ten, and takes 499 us on the prompt for 603.
template <typename T, typename C, int DP>
__device__ __forceinline__ void chunk_items(const RunArgs& a, ChunkLds<DP>& lds, const int4& counts, int wg, int n_wg) {
  typedef hx::f16x8_t v8;
  typedef hx::Elem<_Float16> E;
  constexpr int RB = DP == 256 ? 1 : 2, kSteps = DP / 32, kDims = DP / 16, kPieces = DP / 16;
  constexpr int kThreads = chunk_threads(DP), kWaves = kThreads / 64;
  constexpr int kAhead = 2;  // operands of V read before the softmax, and ahead of their products
  constexpr int kMine = 8 * DP / kThreads;  // 16-byte pieces of codes that a thread moves
  constexpr int kKRow = chunk_k_row(DP), kVRow = chunk_v_row(DP);
  const int tid = hx::tid_x(), lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int D = a.s.head_dim, page = a.s.page, G = a.z.group;
  const int64_t work = (int64_t)counts.y * a.s.hkv;
  const uint32_t row_bytes = (uint32_t)a.s.hkv * (uint32_t)D;

  for (int64_t i = wg; i < work; i += n_wg) {
    const int item = (int)((uint32_t)i / (uint32_t)a.s.hkv), h = (int)((uint32_t)i % (uint32_t)a.s.hkv);
    const int4 it = uniform4(a.chunk + 2 * (int64_t)item), si = uniform4(a.chunk + 2 * (int64_t)item + 1);
    const int row0 = it.y, t_begin = it.z, t_end = it.w, n = si.y, L = si.z;
    const int rows = min(a.z.chunk_rows, n - row0), units = rows * G;

    // Q^T as the MFMA's B operand, and the keys each of this lane's units sees.
    v8 qf[RB][kSteps];
    float qc[RB];  // of this lane's units: log2(e) scale, and what undoes q's power of two
    int klo[RB], khi[RB], urow[RB], uhead[RB];
    bool live[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int u = 16 * (RB * w + rb) + lr;
      live[rb] = u < units;
      urow[rb] = live[rb] ? u / G : 0;
      uhead[rb] = h * G + (live[rb] ? u - urow[rb] * G : 0);
      const int at = L - n + row0 + urow[rb];
      klo[rb] = a.s.left >= 0 && at > a.s.left ? at - a.s.left : 0;
      khi[rb] = a.s.right >= 0 ? min(L - 1, beyond(at, a.s.right)) : L - 1;
    }
    uint4 raw[RB][kSteps];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const uint16_t* const qp = a.q + (int64_t)(si.x + row0 + urow[rb]) * a.q_row + (int64_t)uhead[rb] * a.q_head;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int d = 32 * s + 8 * lg;
        raw[rb][s] = live[rb] && d < D ? *reinterpret_cast<const uint4*>(qp + d) : hx::zero4();
      }
    }
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      uint32_t top = 0;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) top = largest<T>(raw[rb][s], top);
      top = max(top, (uint32_t)__shfl_xor((int)top, 16));
      top = max(top, (uint32_t)__shfl_xor((int)top, 32));
      top = magnitude<T>(top);
      const float up = fit_up(top);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        float x[8];
        widen8<T>(raw[rb][s], x);
        qf[rb][s] = hx::as_v8<_Float16>(pack8(x, up));
      }
      qc[rb] = a.scale_log2 * fit_down(top);
    }
    // Keys that any unit of the wave sees, and those that all of them do.
    int any_lo = 0x7fffffff, any_hi = -1, all_lo = 0, all_hi = 0x7fffffff;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      any_lo = live[rb] ? min(any_lo, klo[rb]) : any_lo;
      any_hi = live[rb] ? max(any_hi, khi[rb]) : any_hi;
      all_lo = live[rb] ? max(all_lo, klo[rb]) : all_lo;
      all_hi = live[rb] ? min(all_hi, khi[rb]) : all_hi;
    }
    for (int m = 1; m < 16; m <<= 1) {
      any_lo = min(any_lo, __shfl_xor(any_lo, m));
      any_hi = max(any_hi, __shfl_xor(any_hi, m));
      all_lo = max(all_lo, __shfl_xor(all_lo, m));
      all_hi = min(all_hi, __shfl_xor(all_hi, m));
    }
    any_lo = __builtin_amdgcn_readfirstlane(any_lo);
    any_hi = __builtin_amdgcn_readfirstlane(any_hi);
    all_lo = __builtin_amdgcn_readfirstlane(all_lo);
    all_hi = __builtin_amdgcn_readfirstlane(all_hi);

    // Page ids, 64 at a time: lane j holds that of page pg0 + j.
    const int last_pg = t_end > t_begin ? (min(L, t_end * kChunkTile) - 1) / page : -1;
    int pg0 = t_begin * kChunkTile / page, ids = -1;
    auto fetch = [&]() {
      ids = pg0 + lane <= last_pg ? a.table[(int64_t)it.x * a.table_stride + pg0 + lane] : -1;
    };
    fetch();
    bool bad = false;
    uint4 reg[kMine];
    float sreg = 0.f;
    int cnt_next = 0;
    auto load = [&](int t) __attribute__((always_inline)) {
      const int key0 = t * kChunkTile, j = key0 / page;
      if (j - pg0 >= 64) {
        pg0 = j;
        fetch();
      }
      int id = __builtin_amdgcn_readlane(ids, j - pg0);
      const bool off = (unsigned)id >= (unsigned)a.num_pages;
      bad |= off;
      id = off ? 0 : id;
      cnt_next = off ? 0 : min(kChunkTile, L - key0);
      const int64_t in = key0 - j * page;
      const int64_t base = (((int64_t)id * page + in) * a.s.hkv + h) * D;
      const uint32_t bytes = cnt_next > 0 ? (uint32_t)(cnt_next - 1) * row_bytes + (uint32_t)D : 0u;
      const __amdgpu_buffer_rsrc_t kr = hx::buffer_rsrc(a.k + base, bytes), vr = hx::buffer_rsrc(a.v + base, bytes);
#pragma unroll
      for (int e = 0; e < kMine; ++e) {
        // The first half of the pieces are K's.
        const bool of_v = 2 * e >= kMine;
        const int p = tid + (of_v ? e - kMine / 2 : e) * kThreads;
        const int r = p / kPieces, c = p % kPieces;
        reg[e] = hx::ld16_buf(of_v ? vr : kr, 16 * c < D ? (uint32_t)r * row_bytes + 16u * c : 0x7ffffff0u);
      }
      if (w < 2) sreg = (w ? a.v_scale : a.k_scale)[((int64_t)id * a.s.hkv + h) * page + in + lane];
    };
    // Into buffer b: codes as fp16, scales as the softmax takes them.
    auto store = [&](int b, int cnt) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < kMine; ++e) {
        const bool of_v = 2 * e >= kMine;
        const int p = tid + (of_v ? e - kMine / 2 : e) * kThreads;
        const int r = p / kPieces, c = p % kPieces;
        const uint2 x0 = hx8::to_f16<C>(reg[e].x), x1 = hx8::to_f16<C>(reg[e].y), x2 = hx8::to_f16<C>(reg[e].z),
                    x3 = hx8::to_f16<C>(reg[e].w);
        uint8_t* const to = (of_v ? lds.v[b] + r * kVRow : lds.k[b] + r * kKRow) + 32 * c;
        *reinterpret_cast<uint4*>(to) = make_uint4(x0.x, x0.y, x1.x, x1.y);
        *reinterpret_cast<uint4*>(to + 16) = make_uint4(x2.x, x2.y, x3.x, x3.y);
      }
      if (w == 0) {
        lds.k_scale[b][lane] = lane < cnt ? sreg : 0.f;
      } else if (w == 1) {
        const ValueScale v = value_scale(lane < cnt ? sreg : 1.f);
        lds.v_log[b][lane] = v.log;
        lds.v_inverse[b][lane] = v.inverse;
      }
    };

    hx::f32x4_t o[kDims][RB];
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) o[d][rb] = hx::f32x4_t{0.f, 0.f, 0.f, 0.f};
    float ref[RB], l_run[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      ref[rb] = -INFINITY;
      l_run[rb] = 0.f;
    }

    int cnt = 0;
    if (t_begin < t_end) {
      load(t_begin);
      cnt = cnt_next;
      store(t_begin & 1, cnt);
      if (t_begin + 1 < t_end) load(t_begin + 1);
    }
    for (int t = t_begin; t < t_end; ++t) {
      const int b = t & 1, key0 = t * kChunkTile, here = cnt;
      __syncthreads();  // tile t is stored, and every wave is done with tile t - 1
      if (t + 1 < t_end) {
        cnt = cnt_next;
        store(b ^ 1, cnt);
        if (t + 2 < t_end) load(t + 2);
      }
      if (key0 > any_hi || key0 + kChunkTile - 1 < any_lo) continue;

      const uint8_t* const kp = lds.k[b] + lr * kKRow + 16 * lg;
      const uint8_t* const vp = lds.v[b] + (4 * lg + (lr >> 2)) * kVRow + 16 * ((lr >> 1) & 1) + 8 * (lr & 1);
      hx::f32x4_t sc[4][RB];
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) sc[kb][rb] = hx::f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
          const v8 kf = hx::as_v8<_Float16>(*reinterpret_cast<const uint4*>(kp + 16 * kb * kKRow + 64 * s));
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) sc[kb][rb] = E::mfma16x16x32(kf, qf[rb][s], sc[kb][rb]);
        }
      // V^T operands, read transposed: keys 32 ks + 4 lg + 0..3 and 16 further of dim 16 d + lr.
      auto read_v = [&](int ks, int d) __attribute__((always_inline)) {
        const uint2 lo = hx::ld8_lds_tr16(vp + 32 * ks * kVRow + 32 * d);
        const uint2 hi = hx::ld8_lds_tr16(vp + (32 * ks + 16) * kVRow + 32 * d);
        return hx::as_v8<_Float16>(make_uint4(lo.x, lo.y, hi.x, hi.y));
      };
      v8 vf[kAhead];
#pragma unroll
      for (int d = 0; d < kAhead; ++d) vf[d] = read_v(0, d);
      // Lane: keys 16 kb + 4 lg + e of its units.
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) {
        const float4 ks = *reinterpret_cast<const float4*>(&lds.k_scale[b][16 * kb + 4 * lg]);
        const float4 lv = *reinterpret_cast<const float4*>(&lds.v_log[b][16 * kb + 4 * lg]);
        const float k4[4] = {ks.x, ks.y, ks.z, ks.w}, l4[4] = {lv.x, lv.y, lv.z, lv.w};
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[kb][rb][e] = fmaf(sc[kb][rb][e], k4[e] * qc[rb], l4[e]);
      }
      const bool whole = here == kChunkTile && key0 >= all_lo && key0 + kChunkTile - 1 <= all_hi;
      float mx[RB];
      bool move[RB];
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        if (!whole) {
          const int from = key0 + 4 * lg, lo = klo[rb] - from, hi = min(khi[rb], key0 + here - 1) - from;
#pragma unroll
          for (int kb = 0; kb < 4; ++kb)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint64_t hidden =
                  __builtin_amdgcn_ballot_w64(16 * kb + e < lo) | __builtin_amdgcn_ballot_w64(16 * kb + e > hi);
              sc[kb][rb][e] = hx::lane_sel(hidden, -INFINITY, sc[kb][rb][e]);
            }
        }
        float m = fmaxf(fmaxf(sc[0][rb][0], sc[0][rb][1]), fmaxf(sc[0][rb][2], sc[0][rb][3]));
#pragma unroll
        for (int kb = 1; kb < 4; ++kb)
          m = fmaxf(m, fmaxf(fmaxf(sc[kb][rb][0], sc[kb][rb][1]), fmaxf(sc[kb][rb][2], sc[kb][rb][3])));
        mx[rb] = hx::max_xor32(hx::max_xor16(m));
        move[rb] = mx[rb] > moves_past(ref[rb], kChunkShift + kChunkLazy);
      }
      bool moved = move[0];
#pragma unroll
      for (int rb = 1; rb < RB; ++rb) moved = moved || move[rb];
      if (__any(moved)) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          const float to = move[rb] ? reference_of(mx[rb], kChunkShift) : ref[rb];
          const float alpha = move[rb] ? hx::fast_exp2(ref[rb] - to) : 1.f;
          ref[rb] = to;
          l_run[rb] *= alpha;
#pragma unroll
          for (int d = 0; d < kDims; ++d) o[d][rb] *= alpha;
        }
      }
      v8 pf[2][RB], pf2[2][RB];
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const float neg = ref[rb] == -INFINITY ? 0.f : -ref[rb];
        float sum = 0.f;
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
          const float4 iv = *reinterpret_cast<const float4*>(&lds.v_inverse[b][16 * kb + 4 * lg]);
          const float i4[4] = {iv.x, iv.y, iv.z, iv.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            sc[kb][rb][e] = hx::fast_exp2(sc[kb][rb][e] + neg);
            // A key that is hidden has the weight 0 under any scale, a NaN too.
            sum = fmaf(sc[kb][rb][e], i4[e], sum);
          }
        }
        l_run[rb] += sum;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          const hx::f32x4_t &x = sc[2 * ks][rb], &y = sc[2 * ks + 1][rb];
          const uint32_t p[4] = {hx::pack2_round<_Float16>(x[0], x[1]), hx::pack2_round<_Float16>(x[2], x[3]),
                                 hx::pack2_round<_Float16>(y[0], y[1]), hx::pack2_round<_Float16>(y[2], y[3])};
          pf[ks][rb] = hx::as_v8<_Float16>(make_uint4(p[0], p[1], p[2], p[3]));
          pf2[ks][rb] = hx::as_v8<_Float16>(
              make_uint4(hx::pack2_round<_Float16>(x[0] - E::lo(p[0]), x[1] - E::hi(p[0])),
                         hx::pack2_round<_Float16>(x[2] - E::lo(p[1]), x[3] - E::hi(p[1])),
                         hx::pack2_round<_Float16>(y[0] - E::lo(p[2]), y[1] - E::hi(p[2])),
                         hx::pack2_round<_Float16>(y[2] - E::lo(p[3]), y[3] - E::hi(p[3]))));
        }
      }
      // O^T += V^T P^T
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int d = 0; d < kDims; ++d) {
          const int i = ks * kDims + d, next = i + kAhead;
          const v8 vv = vf[i % kAhead];
          if (next < 2 * kDims) vf[i % kAhead] = read_v(next / kDims, next % kDims);
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) {
            o[d][rb] = E::mfma16x16x32(vv, pf[ks][rb], o[d][rb]);
            o[d][rb] = E::mfma16x16x32(vv, pf2[ks][rb], o[d][rb]);
          }
        }
    }
    if (bad && tid == 0) atomicOr(&a.hdr[H_ERR], HX_WERR_BAD_PAGE);

#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const float l = hx::add_xor32(hx::add_xor16(l_run[rb]));
      if (!live[rb]) continue;
      if (si.w < 0) {
        const float r = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
        uint16_t* const to = a.out + (int64_t)(si.x + row0 + urow[rb]) * a.out_row + (int64_t)uhead[rb] * a.out_head;
#pragma unroll
        for (int d = 0; d < kDims; ++d)
          if (16 * d < D) {
            uint32_t* const p = reinterpret_cast<uint32_t*>(to + 16 * d + 4 * lg);
            p[0] = hx::pack2_round<T>(o[d][rb][0] * r, o[d][rb][1] * r);
            p[1] = hx::pack2_round<T>(o[d][rb][2] * r, o[d][rb][3] * r);
          }
      } else if ((int64_t)si.w + urow[rb] < a.slots) {
        const int64_t p = ((int64_t)si.w + urow[rb]) * a.s.hq + uhead[rb];
#pragma unroll
        for (int d = 0; d < kDims; ++d)
          if (16 * d < D)
            *reinterpret_cast<float4*>(a.part_o + p * D + 16 * d + 4 * lg) = make_float4(o[d][rb][0], o[d][rb][1], o[d][rb][2], o[d][rb][3]);
        if (lg == 0) a.part_ml[p] = make_float2(ref[rb], l);
      }
    }
    __syncthreads();  // every wave is done with the last tile before the next item's first is stored
  }
}

template <typename T, typename C, int DP>
__global__ __launch_bounds__(chunk_threads(DP), 2) void kv8_chunk_kernel(RunArgs a, int n_wg) {
  __shared__ ChunkLds<DP> lds;
  int4 counts;
  if (plan_ok(a, &counts)) chunk_items<T, C, DP>(a, lds, counts, hx::wg_x(), n_wg);
}

// A tick of both: its few rows' reads go beside the chunks' products, up to 128 dims (where both take
// 4 waves). 32 decoders and two chunks: 107 us, 116 in two launches, of 31 and 84.
template <typename T, typename C, int DP>
__global__ __launch_bounds__(kFewThreads, 2) void kv8_both_kernel(RunArgs a, int n_chunk, int n_few) {
  static_assert(chunk_threads(DP) == kFewThreads);
  __shared__ union Lds {
    FewLds<DP> few;
    ChunkLds<DP> chunk;
    __device__ Lds() {}
  } lds;
  int4 counts;
  if (!plan_ok(a, &counts)) return;
  const int wg = hx::wg_x();
  if (wg < n_chunk) chunk_items<T, C, DP>(a, lds.chunk, counts, wg, n_chunk);
  else few_items<T, C, DP>(a, lds.few, counts, wg - n_chunk, n_few);
}

// -------------------------------------------------------------------------------- join
// The splits of an output row and query head. Many: a workgroup's thread takes four dims of every
// n-th split, in order, then the groups of threads are summed in order. Few: a part of a wave with
// four dims a lane takes them in order, four loads at once.
constexpr int kJoinThreads = 256;

template <typename T>
__global__ __launch_bounds__(kJoinThreads) void kv8_join_kernel(RunArgs a, int n_wg) {
  __shared__ float s_max[4];
  __shared__ float4 s_o[kJoinThreads];
  __shared__ float s_l[kJoinThreads];
  int4 counts;
  if (!plan_ok(a, &counts)) return;
  const int tid = hx::tid_x(), D = a.s.head_dim, quads = D / 4, groups = kJoinThreads / quads;
  const int g = tid / quads, d = 4 * (tid % quads);
  const int64_t work = (int64_t)counts.z * a.s.hq;
  for (int64_t i = hx::wg_x(); i < work; i += n_wg) {
    const int rec = (int)((uint32_t)i / (uint32_t)a.s.hq), head = (int)((uint32_t)i % (uint32_t)a.s.hq);
    const int4 r = uniform4(a.join + rec);
    const int splits = r.w;
    if (r.x < 0 || r.x >= a.s.total_q || r.y < 0 || splits < 1 || (int64_t)r.y + (int64_t)(splits - 1) * r.z >= a.slots) continue;
    float m = -INFINITY;
    for (int s = tid; s < splits; s += kJoinThreads) m = fmaxf(m, a.part_ml[((int64_t)r.y + (int64_t)s * r.z) * a.s.hq + head].x);
    for (int k = 1; k < 64; k <<= 1) m = fmaxf(m, __shfl_xor(m, k));
    if ((tid & 63) == 0) s_max[tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (g < groups) {
      for (int s = g; s < splits; s += groups) {
        const int64_t p = ((int64_t)r.y + (int64_t)s * r.z) * a.s.hq + head;
        const float2 ml = a.part_ml[p];
        const float4 o = *reinterpret_cast<const float4*>(a.part_o + p * D + d);
        const float f = hx::fast_exp2(ml.x - ref);
        l = fmaf(f, ml.y, l);
        x.x = fmaf(f, o.x, x.x);
        x.y = fmaf(f, o.y, x.y);
        x.z = fmaf(f, o.z, x.z);
        x.w = fmaf(f, o.w, x.w);
      }
    }
    s_o[tid] = x;
    s_l[tid] = l;
    __syncthreads();
    if (tid < quads) {
      for (int k = 1; k < groups; ++k) {
        const float4 o = s_o[tid + k * quads];
        l += s_l[tid + k * quads];
        x.x += o.x;
        x.y += o.y;
        x.z += o.z;
        x.w += o.w;
      }
      const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
      uint32_t* const to = reinterpret_cast<uint32_t*>(a.out + (int64_t)r.x * a.out_row + (int64_t)head * a.out_head + d);
      to[0] = hx::pack2_round<T>(x.x * inv, x.y * inv);
      to[1] = hx::pack2_round<T>(x.z * inv, x.w * inv);
    }
    __syncthreads();
  }
  const int lane = tid & 63, each = 64 / quads, mine = lane / quads, d4 = 4 * (lane % quads);
  if (mine >= each) return;
  const int64_t short_work = (int64_t)a.hdr[H_SHORT] * a.s.hq, step = (int64_t)n_wg * (kJoinThreads / 64) * each;
  for (int64_t i = ((int64_t)hx::wg_x() * (kJoinThreads / 64) + (tid >> 6)) * each + mine; i < short_work; i += step) {
    const int rec = (int)((uint32_t)i / (uint32_t)a.s.hq), head = (int)((uint32_t)i % (uint32_t)a.s.hq);
    const int4 r = a.join[a.most_join - 1 - rec];
    const int splits = r.w;
    if (r.x < 0 || r.x >= a.s.total_q || r.y < 0 || splits < 1 || (int64_t)r.y + (int64_t)(splits - 1) * r.z >= a.slots) continue;
    float m = -INFINITY, l = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0; s0 < splits; s0 += 4) {
      float2 ml[4];
      float4 o[4];
      float top = m;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t p = ((int64_t)r.y + (int64_t)min(s0 + e, splits - 1) * r.z) * a.s.hq + head;
        ml[e] = a.part_ml[p];
        o[e] = *reinterpret_cast<const float4*>(a.part_o + p * D + d4);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, ml[e].x);
      const float ref = top == -INFINITY ? 0.f : top, before = hx::fast_exp2(m - ref);
      l *= before;
      x.x *= before;
      x.y *= before;
      x.z *= before;
      x.w *= before;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (s0 + e >= splits) break;
        const float f = hx::fast_exp2(ml[e].x - ref);
        l = fmaf(f, ml[e].y, l);
        x.x = fmaf(f, o[e].x, x.x);
        x.y = fmaf(f, o[e].y, x.y);
        x.z = fmaf(f, o[e].z, x.z);
        x.w = fmaf(f, o[e].w, x.w);
      }
      m = top;
    }
    const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
    uint32_t* const to = reinterpret_cast<uint32_t*>(a.out + (int64_t)r.x * a.out_row + (int64_t)head * a.out_head + d4);
    to[0] = hx::pack2_round<T>(x.x * inv, x.y * inv);
    to[1] = hx::pack2_round<T>(x.z * inv, x.w * inv);
  }
}

// -------------------------------------------------------------------------------- host
int check_shape(const Shape& s) {
  if (s.batch < 0 || s.total_q < 0 || s.max_q < 0 || s.max_k < 0 || s.hq < 1 || s.hkv < 1 || s.hq % s.hkv || s.width < 1 ||
      s.head_dim < 1 || s.page < 1)
    return HX_E_INVALID_ARG;
  if (s.head_dim % 16 || s.head_dim > 256 || s.page % 64 || s.hq / s.hkv > 128 || s.max_k > 0x7fffff00 - s.page ||
      (int64_t)s.hkv * s.head_dim > (1 << 22) || s.hkv > 1024)
    return HX_E_UNSUPPORTED;  // a tile must fit a buffer resource, item indexes 32 bits
  // The plan counts the few rows' tiles and starts, and a part's past their end, in 32 bits.
  if ((int64_t)s.batch * (s.max_k / kFewTile + 2 + kFewStart) > 0x7fffffff - 2 * kFewMost) return HX_E_UNSUPPORTED;
  return HX_OK;
}

struct Run {
  RunArgs a;
  Layout l;
  hipStream_t s;
};

template <typename T, typename C, int DP>
void launch_run(const Run& r, bool few, bool chunk) {
  const RunArgs& a = r.a;
  const int64_t most_few = r.l.most_parts * a.s.hkv * a.z.head_blocks, most_chunk = r.l.most_chunk * a.s.hkv;
  const int n_few = (int)(most_few < 65536 ? most_few : 65536), n_chunk = (int)(most_chunk < 8192 ? most_chunk : 8192);
  if constexpr (chunk_threads(DP) == kFewThreads) {
    if (few && chunk) {
      hipLaunchKernelGGL((kv8_both_kernel<T, C, DP>), dim3(n_chunk + n_few), dim3(kFewThreads), 0, r.s, a, n_chunk, n_few);
      return;
    }
  }
  if (few) hipLaunchKernelGGL((kv8_few_kernel<T, C, DP>), dim3(n_few), dim3(kFewThreads), 0, r.s, a, n_few);
  if (chunk) hipLaunchKernelGGL((kv8_chunk_kernel<T, C, DP>), dim3(n_chunk), dim3(chunk_threads(DP)), 0, r.s, a, n_chunk);
}

template <typename T, typename C>
void launch_run(const Run& r, bool few, bool chunk) {
  if (r.a.s.head_dim <= 64) launch_run<T, C, 64>(r, few, chunk);
  else if (r.a.s.head_dim <= 128) launch_run<T, C, 128>(r, few, chunk);
  else launch_run<T, C, 256>(r, few, chunk);
}

template <typename T>
int launch_run(const Run& r, int32_t code, bool few, bool chunk) {
  if (code == HX_CODE_E4M3) launch_run<T, hx8::E4m3>(r, few, chunk);
  else launch_run<T, hx8::Int8>(r, few, chunk);
  // Sequences may be cut wherever a part ends; blocks of chunk rows past the least of a split.
  if (few || (chunk && r.a.s.max_k > kChunkLeast * kChunkTile - kChunkTile)) {
    const int64_t most = r.l.most_join * r.a.s.hq;
    const int n = (int)(most < 4096 ? most : 4096);
    hipLaunchKernelGGL(kv8_join_kernel<T>, dim3(n), dim3(kJoinThreads), 0, r.s, r.a, n);
  }
  return hx::status_from_hip(hipGetLastError());
}

bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

}  // namespace

extern "C" size_t hx_kv8_attn_workspace_bytes(int32_t batch, int32_t total_q, int32_t max_q, int32_t max_k,
                                              int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int32_t page_size) {
  const Shape s{batch, total_q, max_q, max_k, n_q_heads, n_kv_heads, head_dim, page_size, -1, -1, 1};
  return check_shape(s) == HX_OK ? layout_of(s).total : 0;
}

extern "C" size_t hx_kv8_attn_error_word_offset(void) { return H_ERR * sizeof(int32_t); }

extern "C" int hx_kv8_attn_plan(const int32_t* cu_seq_q, const int32_t* seqused_k, int32_t batch, int32_t total_q,
                                int32_t max_q, int32_t max_k, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                                int32_t page_size, int32_t block_table_width, int32_t window_left, int32_t window_right,
                                void* workspace, size_t workspace_bytes, void* stream) {
  const Shape s{batch,     total_q,     max_q,        max_k,            n_q_heads, n_kv_heads, head_dim,
                page_size, window_left, window_right, block_table_width};
  const int bad = check_shape(s);
  if (bad != HX_OK) return bad;
  if (batch == 0 || total_q == 0 || max_q == 0) return HX_OK;
  if (!cu_seq_q || !seqused_k) return HX_E_INVALID_ARG;
  const Layout l = layout_of(s);
  if (!workspace || misaligned(workspace, 256) || workspace_bytes < l.total) return HX_E_WORKSPACE;
  if (l.slots > 0x7fffffff || l.most_chunk > 0x7fffffff / n_kv_heads || l.most_parts > 0x7ffffff / n_q_heads) return HX_E_UNSUPPORTED;
  uint8_t* const base = static_cast<uint8_t*>(workspace);
  PlanArgs a;
  a.cu_q = cu_seq_q;
  a.used = seqused_k;
  a.hdr = reinterpret_cast<int32_t*>(base);
  a.seq = reinterpret_cast<int4*>(base + l.seq);
  a.part = reinterpret_cast<int4*>(base + l.part);
  a.few = reinterpret_cast<int4*>(base + l.few);
  a.chunk = reinterpret_cast<int4*>(base + l.chunk);
  a.join = reinterpret_cast<int4*>(base + l.join);
  a.most_parts = l.most_parts;
  a.most_few = l.most_few;
  a.most_chunk = l.most_chunk;
  a.most_join = l.most_join;
  a.slots = l.slots;
  a.s = s;
  a.z = sizes_of(s);
  hipLaunchKernelGGL(kv8_plan_kernel, dim3(1), dim3(kPlanThreads), 0, reinterpret_cast<hipStream_t>(stream), a);
  return hx::status_from_hip(hipGetLastError());
}

extern "C" int hx_kv8_attn_run(const void* q, int64_t q_row_stride, int64_t q_head_stride, const void* k_codes,
                               const void* v_codes, const float* k_scales, const float* v_scales, int32_t num_pages,
                               int32_t page_size, int32_t code, const int32_t* block_table, int64_t block_table_stride,
                               int32_t block_table_width, int32_t batch, int32_t total_q, int32_t max_q, int32_t max_k,
                               int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, float scale, int32_t window_left,
                               int32_t window_right, int32_t dtype, void* out, int64_t out_row_stride,
                               int64_t out_head_stride, int32_t kinds, void* workspace, size_t workspace_bytes, void* stream) {
  const Shape s{batch,     total_q,     max_q,        max_k,            n_q_heads, n_kv_heads, head_dim,
                page_size, window_left, window_right, block_table_width};
  const int bad = check_shape(s);
  if (bad != HX_OK) return bad;
  if ((dtype != HX_DTYPE_BF16 && dtype != HX_DTYPE_FP16) || (code != HX_CODE_E4M3 && code != HX_CODE_INT8)) return HX_E_UNSUPPORTED;
  if (num_pages < 1 || block_table_stride < block_table_width || !(scale > 0.f) || !isfinite(scale)) return HX_E_INVALID_ARG;
  if (batch == 0 || total_q == 0 || max_q == 0) return HX_OK;
  if (!q || !k_codes || !v_codes || !k_scales || !v_scales || !block_table || !out || misaligned(q, 16) ||
      misaligned(k_codes, 16) || misaligned(v_codes, 16) || misaligned(k_scales, 16) || misaligned(v_scales, 16) ||
      q_row_stride % 8 || q_head_stride % 8 || misaligned(out, 4) || out_row_stride % 2 || out_head_stride % 2)
    return HX_E_INVALID_ARG;
  Run r;
  r.l = layout_of(s);
  r.s = reinterpret_cast<hipStream_t>(stream);
  if (!workspace || misaligned(workspace, 256) || workspace_bytes < r.l.total) return HX_E_WORKSPACE;
  uint8_t* const base = static_cast<uint8_t*>(workspace);
  RunArgs& a = r.a;
  a.q = static_cast<const uint16_t*>(q);
  a.q_row = q_row_stride;
  a.q_head = q_head_stride;
  a.k = static_cast<const uint8_t*>(k_codes);
  a.v = static_cast<const uint8_t*>(v_codes);
  a.k_scale = k_scales;
  a.v_scale = v_scales;
  a.num_pages = num_pages;
  a.table = block_table;
  a.table_stride = block_table_stride;
  a.scale_log2 = scale * kLog2e;
  a.out = static_cast<uint16_t*>(out);
  a.out_row = out_row_stride;
  a.out_head = out_head_stride;
  a.hdr = reinterpret_cast<int32_t*>(base);
  a.part = reinterpret_cast<const int4*>(base + r.l.part);
  a.few = reinterpret_cast<const int4*>(base + r.l.few);
  a.chunk = reinterpret_cast<const int4*>(base + r.l.chunk);
  a.join = reinterpret_cast<const int4*>(base + r.l.join);
  a.part_ml = reinterpret_cast<float2*>(base + r.l.ml);
  a.part_o = reinterpret_cast<float*>(base + r.l.o);
  a.slots = r.l.slots;
  a.most_join = r.l.most_join;
  a.s = s;
  a.z = sizes_of(s);
  const bool chunk = max_q > a.z.few_rows && (kinds & HX_KV8_CHUNK_ROWS), few = (kinds & HX_KV8_FEW_ROWS) != 0;
  return dtype == HX_DTYPE_BF16 ? launch_run<__bf16>(r, code, few, chunk) : launch_run<_Float16>(r, code, few, chunk);
}
