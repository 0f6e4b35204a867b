// Attention over the 8-bit cache: decoding rows, and chunks of a few new rows a request, in one kernel.
//
// For the query q at position p over the keys j that it sees (codes kc_j, vc_j with scales ks_j, vs_j):
//     s_j = scale ks_j (q . kc_j)  (a cap, a distance bias: as in the other attention kernels),   out = sum_j e^(s_j - m) vs_j vc_j / sum_j e^(s_j - m)
// so the codes go through the tensor cores as they are and the scales meet the scores and the weights.  It cannot do without the codes'
// bytes, read once: 2 (width + 4) per key and key/value head.  What bounds it now is the latency of dependent instructions, three warps a
// scheduler, and the joins at the ends of pieces (neither memory nor a pipe is full), so few instructions are spent on a code:
//   * scores: mma.sync on signed bytes, keys as they lie in memory.  A query's numbers become whole numbers times a power of two of its
//     own, cut into signed bytes, so the products are exact: four bytes for bfloat16 rows and five for 32-bit rows, which hold a number
//     to 2^-30 and 2^-38 of the query's LARGEST one.  So a channel keeps all its bits (8 and 24) down to 2^-22 and 2^-14 of the largest,
//     and a large channel that no key has anything in costs the others nothing (three bytes left 2^-22: a channel 2^-10 of the largest kept 12 bits);
//   * values: mma.sync on bfloat16, which holds a code exactly, with the weights times vs_j cut into two bfloat16 parts for bfloat16 rows
//     (an error of 2^-17: one part costs 2^-9 of the result's size against 64 bits, as much as the rounding of the result itself) and
//     into three for 32-bit rows.
//
// Both products are taken with the operands swapped, keys and values as the 16-row operand and the queries as the 8 columns:
// S^T = K Q^T, O^T = V^T P^T.  The query heads that share a key/value head, and a chunk's rows, are the columns, so up to 8 of them cost
// what one does (16 take a second set of columns; more were slower everywhere).  The order of the contraction, and that of the output's
// rows, is free: a lane's share of the values is 16-byte pieces of its four keys.  They come through shared memory, a ring of stages for
// every warp alone, which it fills with 16-byte asynchronous copies and reads without two lanes on one bank (q8_place): what is on its
// way holds no registers, so three or four blocks fit on an SM, and a block asks for the first tiles of its next piece before it finishes
// the one in hand.
//
// The tiles of 16 keys of all (row, head) pairs, and for every pair a few more for what it costs beside them, are one row that is cut
// evenly over the blocks: every block works out its part from the positions on the device.  A cut that would leave a short end of a
// pair is moved to the pair's end: a pair that lies in several blocks is merged by the last one to finish it.
//
// Measured on one B200, in a graph (copies run at 6.45 TB/s): 64 rows of 120 to 1,400 keys under 16 heads of 128 52.1 us, 4.0 TB/s; 5 rows
// of 7,000 to 30,011 keys, 16 heads over 4, 29.4 us, 3.1 TB/s (over a bfloat16 cache 59 and 71 us); one row of 1,100 keys, 16 heads,
// 10.0 us, of which 2 go by before the first keys are asked for, 1.5 until they are there and 4 in the join, the ticket and the merge
// (where the kernel stores the current token, which takes a fence and a barrier before a piece's first keys are asked for, 56.1, 30.7 and 11.0); in 32 bits 16 rows of
// 300 to 2,000 keys, 8 heads of 32, 13.6 us; chunks of 2 to 7 rows of twelve requests, 25 heads of 64, 17.4 us.
// A tile of a head takes some 475 warp instructions, 128 of them to make bfloat16 numbers of the values' codes; the schedulers are
// busy 46 % of the time, with three warps each.
#pragma once
#include "cache_q8.cuh"
#include "mma_sync.cuh"
#include <atomic>
#include <math.h>
#include <type_traits>

namespace cbis {

constexpr int Q8_WARPS = 4, Q8_THREADS = Q8_WARPS * 32, Q8_MAX_ITEMS = 4096;
constexpr int Q8_MOST_SMEM = 227 * 1024;      // what a block may have: the launcher's plans and the kernels' limits go by it
constexpr int Q8_PAIR = 6;      // what a pair costs beside its keys, in tiles
constexpr float LOG2E = 1.4426950408889634f;

struct Q8Args {
  const void* q;
  void* out;
  int8_t *kc, *vc;
  float *ks, *vs;
  const int *block_table, *row_seq, *positions, *slot_mapping, *cu_rows, *seg_start;
  float* part;
  unsigned* counters;
  const float *sinks, *slopes, *rates;
  int n_rows, ld, out_ld, k_off, v_off, max_blocks, num_pages, n_seqs, seg0, n_items, tiles_per_seg, n_head, n_kv_head, heads_per, head_blocks, rows_per;
  int stages, join_cols, page_rows, hd, ps, ps_shift, window, keep, temp_every;      // ps_shift: log2 of the page size, -1 where that is no whole number
  int heads_inv;                  // ceil(2^16 / heads_per)
  float scale, cap, temp_coef, grid_inv;
};

// Rows of one item: a decoding row, or some consecutive rows of a request's chunk.
struct Q8Item {
  int row0, n_rows, seq, pos0;
};
constexpr int Q8_MAX_POSITION = 1 << 30;      // a block table covers fewer tokens; later positions are all the same, and sums with them hold in 32 bits
__device__ __forceinline__ Q8Item q8_item(const Q8Args& a, int i) {
  Q8Item it;
  if (a.cu_rows == nullptr) {
    it.row0 = i;
    it.n_rows = 1;
    it.seq = a.row_seq[i];
    it.pos0 = min(a.positions[i], Q8_MAX_POSITION);
    if (it.seq >= a.n_seqs || it.pos0 < 0) it.seq = -1;
  } else {
    const int s = a.seg0 + i / a.tiles_per_seg, skip = (i % a.tiles_per_seg) * a.rows_per, r0 = a.cu_rows[s], r1 = min(a.cu_rows[s + 1], a.n_rows);
    const int start = min(a.seg_start[s], Q8_MAX_POSITION);
    const bool ok = r0 >= 0 && r0 < r1 && start >= 0;
    it.seq = s;
    it.row0 = ok ? r0 + skip : 0;
    it.n_rows = ok ? min(r1 - r0 - skip, a.rows_per) : 0;
    it.pos0 = ok ? start + skip : 0;
  }
  return it;
}

// The tiles of 16 keys that an item's rows see, numbered from 0: the nk tiles that hold kept first keys, then those of the window.
struct Q8Span {
  int nk, skipped, tiles;      // the tile numbered n is tile n of the request for n < nk, else n + skipped
};
template <bool EXT>
__device__ __forceinline__ Q8Span q8_span(const Q8Args& a, const Q8Item& it) {
  Q8Span s = {0, 0, 0};
  if (it.seq < 0 || it.n_rows <= 0) return s;
  const int last = it.pos0 + it.n_rows - 1, first_tile = first_seen(it.pos0, a.window) >> 4;
  s.nk = EXT ? min((kept_end(last, a.window, a.keep) + 15) >> 4, first_tile) : 0;
  s.skipped = first_tile - s.nk;
  const int held = (min(last, a.max_blocks * a.ps - 1) >> 4) + 1;      // behind the table's end a row sees the kept keys still
  s.tiles = max(held - s.skipped, min(s.nk, held));
  return s;
}

// The two bytes of `w` that hold signed codes (byte 0 and byte 2; the others are anything) as two bfloat16: 128 + the low seven bits,
// less 128 or 256 as the sign bit says.  `base`: 0x43004300 from a register, or each of the two would be two instructions.
__device__ __forceinline__ unsigned q8_pair(unsigned w, unsigned base) {
  unsigned low, off;
  asm("lop3.b32 %0, %1, 0x007f007f, %2, 0xea;" : "=r"(low) : "r"(w), "r"(base));      // (w & mask) | base
  asm("lop3.b32 %0, %1, 0x00800080, %2, 0xea;" : "=r"(off) : "r"(w), "r"(base));
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&low), *reinterpret_cast<const __nv_bfloat162*>(&off));
  return *reinterpret_cast<const unsigned*>(&r);
}
__device__ __forceinline__ void mma_16832_s8(int (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16832_s8_first(int (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {      // c = the product
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ unsigned transposed(unsigned v) {      // an 8 x 8 tile of 16-bit numbers, a row to four lanes
  unsigned r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float load_float(const float* p) {      // what another block may have written
  float r;
  asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(r) : "l"(p) : "memory");
  return r;
}
// Asynchronous copies to shared memory; of 16 bytes, or of none and zeros instead.
__device__ __forceinline__ void copy16(unsigned to, const void* from, bool ok) {
  const int n = ok ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(n) : "memory");
}
__device__ __forceinline__ void copy16(unsigned to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ void copy4(unsigned to, const void* from) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ void copies_close() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Where byte `byte` of the row of key `row` (0..15) lies in a tile of rows of HDP bytes: the 16-byte pieces of a 128-byte line are
// exchanged by the row's number, so that the same piece of eight keys (ldmatrix), and the pieces that eight lanes read of keys 2t,
// lie on different banks.
template <int HDP>
__device__ __forceinline__ int q8_place(int row, int byte) {
  const int at = row * HDP + byte;
  if constexpr (HDP == 128) return at ^ ((row & 7) << 4);
  if constexpr (HDP == 64) return at ^ ((((row >> 1) & 3) | ((row & 2) << 1)) << 4);
  if constexpr (HDP == 32) return at ^ ((row >> 2 & 1) * 48);
  return at ^ (((row & 4) | ((row >> 1) & 1) | ((row & 1) << 1)) << 4);
}
template <int WORDS>
__device__ __forceinline__ void read_words(unsigned* r, unsigned at) {
  if constexpr (WORDS == 1) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r[0]) : "r"(at) : "memory");
  else if constexpr (WORDS == 2) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(at) : "memory");
  else asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ float read_float(unsigned at) {
  float r;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(r) : "r"(at) : "memory");
  return r;
}
// floor(x / d) for x >= 0 and a quotient below 2^20, from the reciprocal inv of d (good to 2^-22, so the product is off by less than one): a
// division takes some 200 cycles, and a block of few tiles forms five before it asks for its first key.
__device__ __forceinline__ int quotient(long long x, long long d, float inv) {
  int q = (int)((float)x * inv);
  const long long r = x - (long long)q * d;
  if (r < 0) --q;
  if (r >= d) ++q;
  return q;
}
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// The bytes 32 x .. 32 x + 31 of 16 keys as the A fragment of a product on signed bytes, from a lane's share of the addresses.
__device__ __forceinline__ void read_keys(unsigned (&r)[4], unsigned at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
// What q8_place adds to a lane's first place, as an exchange of address bits and a distance: 32 bytes x further in a row, for key 2t + 1
// instead of 2t, and for step i of a copy (32 pieces of 16 bytes a step).
template <int HDP>
struct Q8Place {
  static __device__ __forceinline__ unsigned key(unsigned at, int x) { return (at ^ ((x & 3) * 32)) + (x >> 2) * 128; }
  static __device__ __forceinline__ unsigned odd(unsigned at) {
    return HDP == 256 ? (at ^ 32) + 256 : (HDP == 128 ? (at ^ 16) + 128 : at ^ (HDP == 64 ? 64 : 32));
  }
  static __device__ __forceinline__ unsigned copy(unsigned at, int i) {
    return (HDP == 256 ? at ^ ((i & 1 ? 16 : 0) | (i & 2 ? 64 : 0)) : (HDP == 128 ? at ^ (i & 1 ? 64 : 0) : at)) + i * 512;
  }
};

// HDP: the width rounded up to 32, 64, 128 or 256; NT: columns of queries / 8; PARTS: bfloat16 parts of a weight (2: bfloat16 rows, 3:
// 32-bit rows); EXT: kept first keys, a cap, a distance bias, a query temperature; FAST: the width is HDP and pages are a multiple of 16 keys.
__host__ __device__ constexpr int q8_digits(int parts) { return parts + 2; }      // signed bytes of a query's number
template <int HDP, int NT, int PARTS>
struct Q8Shape {
  static constexpr int TPW = HDP >= 256 ? 1 : (HDP == 128 ? (NT == 1 ? 2 : 1) : 128 / HDP);        // tiles a warp takes through one update of its maxima and sums: a stage of its ring
  static constexpr int UNIT = Q8_WARPS * TPW;                   // tiles that the warps take in a round
  static constexpr int NQ = 8 * NT;
  static constexpr int LDS = HDP + 8;                           // floats of a query's sums in shared memory
  static constexpr int LDQ = HDP >= 128 ? HDP + 16 : HDP;       // bytes of a query's row in shared memory: no two lanes of a load on one bank
  static constexpr int TILE = 32 * HDP + 128;                   // bytes of 16 keys: codes of keys, of values, their scales
  static constexpr int STAGE = TPW * TILE;
  static constexpr int BLOCKS = NT == 1 && HDP < 256 ? (PARTS == 2 && HDP < 128 ? 4 : 3) : 2;      // per SM, as far as registers go
};
// Shared memory of a block (in this order): the warps' rings; sums of jq columns from four warps, maxima of 8; the queries' bytes; the
// columns' powers of two, merged maxima and sums; a few integers; the items.
struct Q8Smem {
  int ring, join, stats, queries, columns, ints, items, bytes;
};
__host__ __device__ inline Q8Smem q8_smem(int stage, int lds, int ldq, int stages, int live, int jq, int n_items, int digits) {
  Q8Smem s;
  s.ring = 0;
  s.join = Q8_WARPS * stages * stage;
  s.stats = s.join + (Q8_WARPS * jq * lds * 4 > 2048 ? Q8_WARPS * jq * lds * 4 : 2048);      // (2 KB: the groups' sums of a merge)
  s.queries = s.stats + Q8_WARPS * 8 * 2 * 4;
  s.columns = s.queries + digits * live * ldq;
  s.ints = s.columns + 3 * 16 * 4;
  s.items = s.ints + 32;
  s.bytes = s.items + (4 * n_items + 1) * 4;
  return s;
}

template <int HDP, int NT, int PARTS, bool EXT, bool FAST>
__global__ void __launch_bounds__(Q8_THREADS, Q8Shape<HDP, NT, PARTS>::BLOCKS)
attention_q8_kernel(const __grid_constant__ Q8Args a) {
  using Shape = Q8Shape<HDP, NT, PARTS>;
  using TT = typename std::conditional<PARTS == 2, __nv_bfloat16, float>::type;
  constexpr int TPW = Shape::TPW, UNIT = Shape::UNIT, NQ = Shape::NQ, LDS = Shape::LDS, LDQ = Shape::LDQ, KS = HDP / 16;
  constexpr int STEPS = HDP / 32, VW = HDP / 32, PW = VW < 4 ? VW : 4;      // steps of the scores' product; words of a value that a lane takes, of one load
  constexpr int DIGITS = q8_digits(PARTS);
  constexpr bool Q_IN_REGS = NT * HDP <= 128;
  extern __shared__ __align__(128) char smem[];
  const int cols = a.rows_per * a.heads_per;            // live columns at most
  const Q8Smem at = q8_smem(Shape::STAGE, LDS, LDQ, a.stages, cols, a.join_cols, a.n_items, DIGITS);
  float* sm_acc = reinterpret_cast<float*>(smem + at.join);          // [warp][join_cols][LDS]
  float* sm_m = reinterpret_cast<float*>(smem + at.stats);           // [warp][8]
  float* sm_l = sm_m + Q8_WARPS * 8;                                 // [warp][8]
  int8_t* sm_q = reinterpret_cast<int8_t*>(smem + at.queries);       // [DIGITS][cols][LDQ] the queries' bytes, the highest first
  float* sm_f = reinterpret_cast<float*>(smem + at.columns);         // [16] a query's power of two, [16] maximum and [16] sum of merged pieces
  float* sm_w = sm_f + 16;
  int* sm_i = reinterpret_cast<int*>(smem + at.ints);                // [8]
  int* before = reinterpret_cast<int*>(smem + at.items);             // [n_items + 1] tiles of the items before this one
  int* item_row = before + a.n_items + 1;                            // [n_items] first row; request or rows; first position
  int* item_seq = item_row + a.n_items;
  int* item_pos = item_seq + a.n_items;
  const int hd = FAST ? HDP : a.hd;
  unsigned base;
  asm volatile("mov.b32 %0, 0x43004300;" : "=r"(base));
  pdl_trigger();
  // the arguments' lines, and what does not depend on the kernels before, while those end
  asm volatile("" ::"l"(a.q), "l"(a.block_table), "l"(a.part), "r"(a.n_rows), "r"(a.n_kv_head), "r"(a.hd), "f"(a.scale));
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;

  // the items' tiles, summed up
  int total = 0;
  for (int i0 = 0; i0 < a.n_items; i0 += Q8_THREADS) {
    const int i = i0 + tid;
    int n = 0;
    if (i < a.n_items) {
      const Q8Item it = q8_item(a, i);
      if (it.n_rows > 0) n = Q8_PAIR + q8_span<EXT>(a, it).tiles;      // a row without keys has its zeros written too
      item_row[i] = it.row0;
      item_seq[i] = a.cu_rows ? it.n_rows : it.seq;
      item_pos[i] = it.pos0;
    }
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (lane == 31) sm_i[warp] = sum;
    __syncthreads();
    int sofar = total;
#pragma unroll
    for (int w = 0; w < Q8_WARPS; ++w) {
      if (w < warp) sofar += sm_i[w];
      total += sm_i[w];
    }
    if (i < a.n_items) before[i] = sofar + sum - n;
    __syncthreads();
  }
  if (tid == 0) before[a.n_items] = total;
  __syncthreads();
  const int n_hg = a.n_kv_head * a.head_blocks, group = a.n_head / a.n_kv_head;
  if (total == 0) return;
  // At least a round of the warps to a block (16 heads of 1,100 keys: 10.0 us with one, 12.5 with two, 15 with three); cuts are moved by
  // up to three rounds (a merge takes about as long), by less where a block has much to do, for all wait for the one that got more.
  const long long all = (long long)total * n_hg, per = max((long long)((float)all * a.grid_inv) + 1, (long long)(UNIT > Q8_PAIR + 1 ? UNIT : Q8_PAIR + 2));      // (grid_inv is a little too large)
  const float total_inv = reciprocal((float)total), per_inv = reciprocal((float)per);
  const int slack = (int)min(per <= 6 * UNIT ? per - 1 : max(per / 16, (long long)Q8_PAIR), max(3LL * UNIT, (long long)Q8_PAIR));
  // the item in which tile `rem` of a head lies: the last one that begins at or before it
  auto item_at = [&](int rem) {
    int lo = 0, hi = a.n_items - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (before[mid] <= rem) lo = mid; else hi = mid - 1;
    }
    return lo;
  };
  auto cut = [&](long long x) {      // a block's end, moved to that of an item that is near
    if (x >= all) return all;
    const int rem = (int)(x - (long long)quotient(x, total, total_inv) * total), i = item_at(rem), d = rem - before[i], e = before[i + 1] - rem;
    return d <= slack ? x - d : (e <= slack ? x + e : x);
  };
  long long w_at = cut(blockIdx.x * per);
  const long long w_end = cut((blockIdx.x + 1) * per);
  if (w_at >= w_end) return;

  auto inverse = [&](int n_h) { return n_h == a.heads_per ? a.heads_inv : (65536 + n_h - 1) / n_h; };
  // A block's part of one item's keys under the heads that share a key/value head: from tile `from` to end_tile.
  struct Piece {
    Q8Item it;
    Q8Span span;
    int hg, hk, h0, n_h, item, from, end_tile;
    bool begins, ends;      // whether the item does with it
    const int* bt;
    const int8_t *k_lane, *v_lane;      // FAST: the lane's piece of the head's first row, and its scale
    const float* s_lane;
  };
  int at_hg = quotient(w_at, total, total_inv), at_item = item_at((int)(w_at - (long long)at_hg * total)), at_tile = (int)(w_at - (long long)at_hg * total) - before[at_item];
  auto find_piece = [&](Piece& p) {
    const int lo = at_item, slots = before[lo + 1] - before[lo], to = (int)min((long long)slots, at_tile + (w_end - w_at));
    p.hg = at_hg;
    p.item = lo;
    p.begins = at_tile == 0;
    p.ends = to == slots;
    p.from = p.begins ? 0 : at_tile - Q8_PAIR;
    p.end_tile = to - Q8_PAIR;
    w_at += to - at_tile;
    at_tile = to;
    if (p.ends) {
      at_tile = 0;
      do {
        if (++at_item == a.n_items) {
          at_item = 0;
          ++at_hg;
        }
      } while (w_at < w_end && before[at_item + 1] == before[at_item]);
    }
    p.it.row0 = item_row[lo];
    p.it.pos0 = item_pos[lo];
    p.it.n_rows = a.cu_rows ? item_seq[lo] : 1;
    p.it.seq = a.cu_rows ? a.seg0 + lo / a.tiles_per_seg : item_seq[lo];
    p.span = q8_span<EXT>(a, p.it);
    p.hk = a.head_blocks == 1 ? p.hg : p.hg / a.head_blocks;
    const int hb = p.hg - p.hk * a.head_blocks;
    p.h0 = p.hk * group + hb * a.heads_per;
    p.n_h = min(a.heads_per, group - hb * a.heads_per);
    p.bt = a.block_table + (size_t)max(p.it.seq, 0) * a.max_blocks;
    // the query that the warp converts first, on its way while the pages are looked up
    if (lane * 128 < hd * (int)sizeof(TT) && warp < p.it.n_rows * p.n_h) {
      const int row = inverse(p.n_h) * warp >> 16;
      asm volatile("prefetch.global.L1 [%0];" ::"l"(static_cast<const TT*>(a.q) + (size_t)(p.it.row0 + row) * a.ld + (p.h0 + warp - row * p.n_h) * hd + lane * (128 / (int)sizeof(TT))));
    }
    if constexpr (FAST) {
      const long long first = (long long)p.hk * a.ps;
      p.k_lane = a.kc + first * HDP + lane * 16;
      p.v_lane = a.vc + first * HDP + lane * 16;
      p.s_lane = (lane < 16 ? a.ks : a.vs) + first + (lane & 15);
    }
    // the current token's key and value are stored by the block that reads them
    if (a.k_off >= 0 && p.ends && p.it.seq >= 0) {
      const int slot = a.slot_mapping[p.it.row0];
      if (slot >= 0 && slot < a.num_pages * a.ps && warp < 2) {
        const TT* src = static_cast<const TT*>(a.q) + (size_t)p.it.row0 * a.ld + (warp ? a.v_off : a.k_off) + p.hk * hd;
        float x[HDP / 32];
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < HDP / 32; ++i) {
          x[i] = i * 32 + lane < hd ? to_f32(src[i * 32 + lane]) : 0.f;
          top = max(top, q8_bits(x[i]));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float s = q8_scale(top), inv = q8_inverse(s);
        const size_t row = ((size_t)(slot / a.ps) * a.n_kv_head + p.hk) * a.ps + slot % a.ps;
        int8_t* dst = (warp ? a.vc : a.kc) + row * hd;
#pragma unroll
        for (int i = 0; i < HDP / 32; ++i)
          if (i * 32 + lane < hd) dst[i * 32 + lane] = (int8_t)q8_code(x[i], s, inv);
        if (lane == 0) (warp ? a.vs : a.ks)[row] = s;
      }
      __threadfence();
      __syncthreads();
    }
  };

  // The warp's ring: `fill` is the stage to be filled next, `use` the one to be read next (as shared addresses).
  const unsigned ring = (unsigned)__cvta_generic_to_shared(smem) + warp * a.stages * Shape::STAGE, ring_end = ring + a.stages * Shape::STAGE;
  unsigned fill = ring, use = ring;
  const unsigned k_place = q8_place<HDP>((lane & 7) + (lane & 8), lane >> 4 << 4), v_place = q8_place<HDP>(2 * t, g * 4 * VW) + 16 * HDP;
  const unsigned c_place = q8_place<HDP>(lane / (HDP / 16), lane % (HDP / 16) * 16);
  auto real_tile = [&](const Piece& p, int n) { return !EXT || n >= p.span.nk ? n + p.span.skipped : n; };
  int ahead[TPW];                          // FAST: the pages of the tiles to be asked for next, as the table names them
  auto find_pages = [&](const Piece& p, int tile) {
#pragma unroll
    for (int u = 0; u < TPW; ++u) {
      const int j0 = real_tile(p, min(tile + u, p.end_tile - 1)) << 4;
      ahead[u] = p.bt[a.ps_shift >= 0 ? j0 >> a.ps_shift : j0 / a.ps];
    }
  };
  // Asks for the warp's tiles from `tile` on, as far as they lie in the piece.  A key whose page the cache does not have gets scale -1, which
  // no row has: it is hidden.  (Every address that is worked out lies in the cache, whether it is used or not.)
  auto ask = [&](const Piece& p, int tile) {
#pragma unroll
    for (int u = 0; u < TPW; ++u) {
      if (tile + u < p.end_tile) {
        const unsigned to = fill + u * Shape::TILE;
        const int j0 = real_tile(p, tile + u) << 4;
        if constexpr (FAST) {
          const bool ok = (unsigned)ahead[u] < (unsigned)a.num_pages;
          const int in_page = a.ps_shift >= 0 ? j0 & (a.ps - 1) : j0 % a.ps;
          const int row = ok ? ahead[u] * a.page_rows + in_page : 0;      // rows of codes from the head's first one on: fewer than 2^31 in all
          const int8_t *kp = p.k_lane + (long long)row * HDP, *vp = p.v_lane + (long long)row * HDP;
#pragma unroll
          for (int i = 0; i < HDP / 32; ++i) {
            copy16(Q8Place<HDP>::copy(to + c_place, i), kp + i * 512);
            copy16(Q8Place<HDP>::copy(to + c_place, i) + 16 * HDP, vp + i * 512);
          }
          const unsigned s_to = to + 32 * HDP + lane * 4;
          if (ok) copy4(s_to, p.s_lane + row);
          else asm volatile("st.shared.f32 [%0], %1;" ::"r"(s_to), "f"(-1.f) : "memory");
        } else {
#pragma unroll
          for (int i = 0; i < HDP / 32; ++i) {
            const int row = (lane + 32 * i) / (HDP / 16), byte = (lane + 32 * i) % (HDP / 16) * 16, j = j0 + row;
            const int jt = min(j, a.max_blocks * a.ps - 1), page = p.bt[jt / a.ps];
            const bool ok = j == jt && page >= 0 && page < a.num_pages;
            const long long base = (ok ? (long long)page * a.page_rows + j % a.ps : 0) + p.hk * a.ps;
            const int place = q8_place<HDP>(row, byte);
            copy16(to + place, a.kc + base * hd + (byte < hd ? byte : 0), ok && byte < hd);
            copy16(to + 16 * HDP + place, a.vc + base * hd + (byte < hd ? byte : 0), ok && byte < hd);
            if (byte == 0) {
              const unsigned s_to = to + 32 * HDP + row * 4;
              if (ok) {
                copy4(s_to, a.ks + base);
                copy4(s_to + 64, a.vs + base);
              } else {
                asm volatile("st.shared.f32 [%0], %1;\n\tst.shared.f32 [%0 + 64], %1;" ::"r"(s_to), "f"(-1.f) : "memory");
              }
            }
          }
        }
      }
    }
    copies_close();
    fill = fill + Shape::STAGE == ring_end ? ring : fill + Shape::STAGE;
  };
  auto ask_first = [&](const Piece& p) {      // all stages but one
    const int tile = p.from + warp * TPW;
    if (FAST && tile < p.end_tile) find_pages(p, tile);
    for (int s = 0; s < a.stages - 1; ++s) {
      ask(p, tile + s * UNIT);
      if (FAST && tile + (s + 1) * UNIT < p.end_tile) find_pages(p, tile + (s + 1) * UNIT);
    }
  };

  int owed = 0;                            // 1: a ticket of the first piece, 2: of the last
  unsigned ticket0 = 0, ticket1 = 0;       // of one thread
  Piece cur;
  find_piece(cur);
  ask_first(cur);
  while (true) {
    const int live = cur.it.n_rows * cur.n_h, n_h = cur.n_h;
    const int n_h_inv = inverse(n_h);
    auto row_in = [&](int m) { return m * n_h_inv >> 16; };      // m / n_h, exact for m and n_h up to 16
    // queries as signed bytes, a warp to a query
    for (int m = warp; m < live; m += Q8_WARPS) {
      float x[HDP / 32];
      unsigned top = 0;
      const TT* src = static_cast<const TT*>(a.q) + (size_t)(cur.it.row0 + row_in(m)) * a.ld + (cur.h0 + m - row_in(m) * n_h) * hd;
#pragma unroll
      for (int i = 0; i < HDP / 32; ++i) {
        x[i] = i * 32 + lane < hd ? to_f32(src[i * 32 + lane]) : 0.f;
        top = max(top, q8_bits(x[i]));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      const int up = min(275 - (int)(top >> 23), 253);      // 2^(up - 127) brings the largest into [2^21, 2^22)
      const float f = __uint_as_float((unsigned)up << 23);
#pragma unroll
      for (int i = 0; i < HDP / 32; ++i) {
        // the whole part, and what it leaves (exact, a half at most) as more bytes behind the point
        const float y = x[i] * f;
        int v = top < 0x7f800000u ? __float2int_rn(y) : 0, rest = top < 0x7f800000u ? __float2int_rn((y - (float)v) * (float)(1 << 8 * (DIGITS - 3))) : 0;
        int8_t* dst = sm_q + m * LDQ + (lane >> 2 & 3) * (HDP / 4) + i * 8 + (lane >> 4) * 4 + (lane & 3);      // number d = 32 i + 16 h + 4 t + byte: what lane t needs lies together
#pragma unroll
        for (int digit = DIGITS - 1; digit > 0; --digit) {
          if (digit == 2) v += rest;
          int& from = digit > 2 ? rest : v;
          const int low = (int)(int8_t)from;
          dst[digit * cols * LDQ] = (int8_t)low;
          from = (from - low) >> 8;
        }
        dst[0] = (int8_t)v;
      }
      if (lane == 0) sm_f[m] = top < 0x7f800000u ? __uint_as_float((unsigned)(254 - up) << 23) : __uint_as_float(0x7fc00000u);
    }
    __syncthreads();
    // ... as B fragments: column g of each n-tile (a dead column repeats a live one)
    constexpr int QW = 2 * STEPS < 4 ? 2 * STEPS : 4;      // words of a load
    const unsigned q_at = (unsigned)__cvta_generic_to_shared(sm_q) + t * (HDP / 4);
    auto q_words = [&](int digit, int nt, int x, unsigned* w) { read_words<QW>(w, q_at + (digit * cols + min(nt * 8 + g, live - 1)) * LDQ + x * 8); };
    unsigned qf[Q_IN_REGS ? DIGITS : 1][Q_IN_REGS ? NT : 1][Q_IN_REGS ? 2 * STEPS : 1];
    if constexpr (Q_IN_REGS) {
#pragma unroll
      for (int digit = 0; digit < DIGITS; ++digit)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < STEPS; x += QW / 2) q_words(digit, nt, x, &qf[digit][nt][2 * x]);
    }
    // this lane's columns 2t and 2t + 1 of each n-tile: position, first key seen, factor of the score
    int qp[NT][2], qs[NT][2], qk[NT][2];
    float qx[NT][2], qslope[NT][2];
    const float* qrate[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int m = min(nt * 8 + 2 * t + e, live - 1);
        const float back = sm_f[m] * a.scale;
        qp[nt][e] = cur.it.pos0 + row_in(m);
        qs[nt][e] = first_seen(qp[nt][e], a.window);
        qx[nt][e] = back * LOG2E;
        if constexpr (EXT) {
          const int h = cur.h0 + m - row_in(m) * n_h;
          qk[nt][e] = kept_end(qp[nt][e], a.window, a.keep);
          qx[nt][e] = back;
          if (a.temp_every > 0) qx[nt][e] *= 1.0f + a.temp_coef * logf((float)((qp[nt][e] + 1) / a.temp_every + 1));
          qslope[nt][e] = a.slopes ? a.slopes[h] : 0.f;
          qrate[nt][e] = a.rates ? a.rates + h : nullptr;
        }
      }
    const int whole_from = first_seen(cur.it.pos0 + cur.it.n_rows - 1, a.window), whole_to = cur.it.pos0;      // keys that every row sees

    float o[NT][KS][4], m_run[NT][2], l_run[NT][2], ref[NT][2];      // ref: the running maximum, 0 while there is none
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < KS; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
      m_run[nt][0] = m_run[nt][1] = -INFINITY;
      l_run[nt][0] = l_run[nt][1] = ref[nt][0] = ref[nt][1] = 0.f;
    }

    for (int tile = cur.from + warp * TPW; tile < cur.end_tile; tile += UNIT) {
      // the oldest stage has arrived, and every lane is done with the one before it, which is filled again
      if (a.stages == 2) copies_wait<0>();
      else copies_wait<1>();
      __syncwarp();
      {
        const int next = tile + (a.stages - 1) * UNIT;
        ask(cur, next);
        if (FAST && next + UNIT < cur.end_tile) find_pages(cur, next + UNIT);
      }
      const unsigned stage = use;
      use = use + Shape::STAGE == ring_end ? ring : use + Shape::STAGE;
      float s[TPW][NT][4], vx[TPW][2];
      bool whole = true;       // every row sees every key of the warp's tiles
      bool hidden = false;
#pragma unroll
      for (int u = 0; u < TPW; ++u) {
        if (tile + u >= cur.end_tile) {
          whole = false;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) s[u][nt][0] = s[u][nt][1] = s[u][nt][2] = s[u][nt][3] = -INFINITY;
          continue;
        }
        const unsigned st = stage + u * Shape::TILE, sc = st + 32 * HDP + g * 4;
        const int j0 = real_tile(cur, tile + u) << 4;
        unsigned kw[STEPS][4];
#pragma unroll
        for (int x = 0; x < STEPS; ++x) read_keys(kw[x], Q8Place<HDP>::key(st + k_place, x));
        const float kx[2] = {read_float(sc), read_float(sc + 32)};
        vx[u][0] = read_float(sc + 64);
        vx[u][1] = read_float(sc + 96);
        whole = whole && j0 >= whole_from && j0 + 15 <= whole_to;
        hidden = hidden || fminf(kx[0], kx[1]) < 0.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          int qk_sum[DIGITS][4];
#pragma unroll
          for (int x0 = 0; x0 < STEPS; x0 += QW / 2) {
#pragma unroll
            for (int digit = 0; digit < DIGITS; ++digit) {
              unsigned q[QW];
              if constexpr (Q_IN_REGS) {
#pragma unroll
                for (int w = 0; w < QW; ++w) q[w] = qf[digit][nt][2 * x0 + w];
              } else {
                q_words(digit, nt, x0, q);
              }
#pragma unroll
              for (int w = 0; w < QW; w += 2) {
                const int x = x0 + w / 2;
                if (x == 0) mma_16832_s8_first(qk_sum[digit], kw[x], q[w], q[w + 1]);
                else mma_16832_s8(qk_sum[digit], kw[x], q[w], q[w + 1]);
              }
            }
          }
          // scores in the base-2 domain
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int c = e & 1;
            // two bytes' sums together hold in 32 bits (256 * 127 * 128 * 257 < 2^31)
            const float low = (float)(qk_sum[DIGITS - 2][e] * 256 + qk_sum[DIGITS - 1][e]), high = (float)(qk_sum[DIGITS - 4][e] * 256 + qk_sum[DIGITS - 3][e]);
            float v = DIGITS == 4 ? fmaf(low, 0x1p-8f, high * 256.f) : fmaf((float)qk_sum[0][e], 65536.f, fmaf(low, 0x1p-16f, high));
            v *= kx[e >> 1] * qx[nt][c];
            if constexpr (EXT) {
              v = capped_score(v, a.cap);
              if (a.slopes) v -= distance_bias(qslope[nt][c], qrate[nt][c], (float)max(qp[nt][c] - (j0 + g + 8 * (e >> 1)), 0));
              v *= LOG2E;
            }
            s[u][nt][e] = v;
          }
        }
      }
      whole = whole && !__any_sync(0xffffffffu, hidden);
      if (!whole) {             // -inf where the query does not see the key
#pragma unroll
        for (int u = 0; u < TPW; ++u) {
          if (tile + u >= cur.end_tile) continue;
          const int j0 = real_tile(cur, tile + u) << 4;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int j = j0 + g + 8 * i;
            const bool there = !(read_float(stage + u * Shape::TILE + 32 * HDP + (g + 8 * i) * 4) < 0.f);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                const bool ok = there && j <= qp[nt][c] && (j >= qs[nt][c] || (EXT && j < qk[nt][c]));
                s[u][nt][2 * i + c] = ok ? s[u][nt][2 * i + c] : -INFINITY;
              }
          }
        }
      }
      float mx[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mx[nt][0] = mx[nt][1] = -INFINITY;
#pragma unroll
        for (int u = 0; u < TPW; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx[nt][e & 1] = fmaxf(mx[nt][e & 1], s[u][nt][e]);
      }
      bool moved = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) mx[nt][c] = fmaxf(mx[nt][c], __shfl_xor_sync(0xffffffffu, mx[nt][c], x));
          moved |= mx[nt][c] > m_run[nt][c];
        }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float corr[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float m_new = fmaxf(m_run[nt][c], mx[nt][c]);
            ref[nt][c] = m_new == -INFINITY ? 0.f : m_new;
            corr[c] = ex2(m_run[nt][c] - ref[nt][c]);
            m_run[nt][c] = m_new;
            l_run[nt][c] *= corr[c];
          }
#pragma unroll
          for (int j = 0; j < KS; ++j) {
            o[nt][j][0] *= corr[0];
            o[nt][j][1] *= corr[1];
            o[nt][j][2] *= corr[0];
            o[nt][j][3] *= corr[1];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < TPW; ++u) {
        if (tile + u >= cur.end_tile) continue;
        unsigned pf[PARTS][NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            p[e] = ex2(s[u][nt][e] - ref[nt][e & 1]);
            l_run[nt][e & 1] += p[e];
            p[e] = whole || s[u][nt][e] != -INFINITY ? p[e] * vx[u][e >> 1] : 0.f;      // a hidden key's scale may be anything
          }
          {
            unsigned a0[PARTS], a1[PARTS];
            cut_parts(p[0], p[1], a0);
            cut_parts(p[2], p[3], a1);
#pragma unroll
            for (int i = 0; i < PARTS; ++i) {
              pf[i][nt][0] = transposed(a0[i]);
              pf[i][nt][1] = transposed(a1[i]);
            }
          }
        }
        const unsigned v_at = stage + u * Shape::TILE + v_place;
#pragma unroll
        for (int w0 = 0; w0 < VW; w0 += PW) {
          unsigned vw[4][PW];
#pragma unroll
          for (int i = 0; i < 4; ++i) read_words<PW>(vw[i], (i & 1 ? Q8Place<HDP>::odd(v_at ^ (w0 * 4)) : v_at ^ (w0 * 4)) + (i >> 1) * 8 * HDP);
#pragma unroll
          for (int j = 0; j < 2 * PW; ++j) {
            const int w = j >> 1;
            const unsigned lo = j & 1 ? 0x0602 : 0x0400, hi = j & 1 ? 0x0703 : 0x0501;
            const unsigned A[4] = {q8_pair(__byte_perm(vw[0][w], vw[1][w], lo), base), q8_pair(__byte_perm(vw[0][w], vw[1][w], hi), base),
                                   q8_pair(__byte_perm(vw[2][w], vw[3][w], lo), base), q8_pair(__byte_perm(vw[2][w], vw[3][w], hi), base)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float (&sum)[4] = o[nt][2 * w0 + j];
              if constexpr (PARTS == 3) {      // the tensor cores cut their sums instead of rounding them: 32-bit rows add the tiles' own sums
                float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int p = PARTS - 1; p >= 0; --p) mma_16816(part, A, pf[p][nt][0], pf[p][nt][1]);
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] += part[e];
              } else {
#pragma unroll
                for (int p = PARTS - 1; p >= 0; --p) mma_16816(sum, A, pf[p][nt][0], pf[p][nt][1]);
              }
            }
          }
        }
      }
    }
    // what was asked for behind the piece's end is nothing; the next piece's first tiles are on their way while this one is finished
    copies_wait<0>();
    __syncwarp();
    fill = use = ring;
    const bool more = w_at < w_end;
    const Piece done = cur;
    if (more) {
      find_piece(cur);
      ask_first(cur);
    }

    // the warps' results joined, a few columns at a time
    const bool alone = done.begins && done.ends;
    float* mine = a.part + (size_t)(2 * blockIdx.x + done.begins) * NQ * (HDP + 4);      // a column: HDP sums, the maximum, the denominator
    // entry i of a query's row in shared memory is [pair of dims j][lane g][2]: the dim
    auto dim_of = [&](int i) { return ((i >> 1) & 7) * (HDP / 8) + (i >> 4) * 2 + (i & 1); };
    const int jq = a.join_cols;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      for (int q0 = 0; q0 < 8 && nt * 8 + q0 < live; q0 += jq) {
        if (nt + q0 > 0) __syncthreads();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int q = 2 * t + c;
          if (q0 == 0) {
            float l = l_run[nt][c];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
            if (g == 0) {
              sm_m[warp * 8 + q] = m_run[nt][c];
              sm_l[warp * 8 + q] = l;
            }
          }
          if (nt * 8 + q < live && q >= q0 && q < q0 + jq) {
            float* dst = sm_acc + (size_t)(warp * jq + q - q0) * LDS + g * 2;
#pragma unroll
            for (int j = 0; j < KS; ++j) *reinterpret_cast<float2*>(dst + j * 16) = make_float2(o[nt][j][c], o[nt][j][2 + c]);
          }
        }
        __syncthreads();
        for (int x = tid; x < min(live - nt * 8 - q0, jq) * HDP; x += Q8_THREADS) {
          const int mq = q0 + x / HDP, i = x % HDP, m = nt * 8 + mq, d = dim_of(i);
          float mw[Q8_WARPS], M = -INFINITY, l = 0.f, v = 0.f;
#pragma unroll
          for (int w = 0; w < Q8_WARPS; ++w) {
            mw[w] = sm_m[w * 8 + mq];
            M = fmaxf(M, mw[w]);
          }
#pragma unroll
          for (int w = 0; w < Q8_WARPS; ++w) {
            const float f = mw[w] == -INFINITY && M != -INFINITY ? 0.f : ex2(mw[w] - (M == -INFINITY ? 0.f : M));
            v = fmaf(f, sm_acc[(size_t)(w * jq + mq - q0) * LDS + i], v);
            l = fmaf(f, sm_l[w * 8 + mq], l);
          }
          if (alone) {
            const int h = done.h0 + m - row_in(m) * n_h;
            float keep1 = 1.f;
            if (a.sinks) {
              const float sk = a.sinks[h] * LOG2E, mm = fmaxf(M, sk), r = mm == -INFINITY ? 0.f : mm;      // (a head without a sink has -inf)
              keep1 = ex2(M - r);
              l = fmaf(l, keep1, ex2(sk - r));
            }
            if (d < hd) from_f32(static_cast<TT*>(a.out)[(size_t)(done.it.row0 + row_in(m)) * a.out_ld + h * hd + d], l == 0.f ? 0.f : v * keep1 / l);
          } else {
            float* p = mine + m * (HDP + 4);
            p[i] = v;
            if (i == 0) {
              p[HDP] = M;
              p[HDP + 1] = l;
            }
          }
        }
      }
    }
    // A piece of an item that others have a part of: a ticket is drawn now and looked at when the block is done with its last piece, so
    // that nothing waits for it.  (Such are a block's first piece and its last; the barrier puts the block's stores before the fence.)
    if (!alone) {
      __syncthreads();
      owed |= more ? 1 : 2;
      if (tid == Q8_THREADS - 32) {
        sm_i[more ? 4 : 6] = done.item;
        sm_i[more ? 5 : 7] = done.hg;
        __threadfence();
        const unsigned drawn = atomicAdd(a.counters + (size_t)done.item * n_hg + done.hg, 1u);
        if (more) ticket0 = drawn; else ticket1 = drawn;
      }
    }
    if (!more) break;
    __syncthreads();      // the next piece's queries and sums go where this one's were
  }
  if (!owed) return;

  // The last one to finish a piece of an item merges them.  The cuts left inside the item: the piece behind cut c is block c's, the first
  // piece that of the block before.
  auto pieces_of = [&](int item, int hg, int& b_first) {
    const long long begin = (long long)hg * total + before[item], end = begin + before[item + 1] - before[item];
    b_first = quotient(begin + slack, per, per_inv);
    return quotient(end - slack - 1, per, per_inv) - b_first + 1;
  };
  if (tid == Q8_THREADS - 32) {
    bool last[2] = {false, false};
#pragma unroll
    for (int w = 0; w < 2; ++w)
      if (owed >> w & 1) {
        int b_first;
        last[w] = (w ? ticket1 : ticket0) == (unsigned)(pieces_of(sm_i[4 + 2 * w], sm_i[5 + 2 * w], b_first) - 1);
        sm_i[w] = last[w];
      }
    __threadfence();
#pragma unroll
    for (int w = 0; w < 2; ++w)
      if (last[w]) a.counters[(size_t)sm_i[4 + 2 * w] * n_hg + sm_i[5 + 2 * w]] = 0;
  }
  __syncthreads();
#pragma unroll 1
  for (int w = 0; w < 2; ++w) {
    if (!(owed >> w & 1) || !sm_i[w]) continue;
    const int item = sm_i[4 + 2 * w], hg = sm_i[5 + 2 * w], hk = a.head_blocks == 1 ? hg : hg / a.head_blocks, hb = hg - hk * a.head_blocks, h0 = hk * group + hb * a.heads_per;
    const int n_h = min(a.heads_per, group - hb * a.heads_per), live = (a.cu_rows ? item_seq[item] : 1) * n_h, row0 = item_row[item];
    const int n_h_inv = inverse(n_h);
    auto row_in = [&](int m) { return m * n_h_inv >> 16; };
    auto dim_of = [&](int i) { return ((i >> 1) & 7) * (HDP / 8) + (i >> 4) * 2 + (i & 1); };
    int b_first;
    const int n_pieces = pieces_of(item, hg, b_first);
    auto piece = [&](int b) { return a.part + (size_t)(2 * (b_first + b) + (b == 0)) * NQ * (HDP + 4); };
    // four entries of a column to a thread, eight pieces in flight; with few columns the pieces go to several groups of threads
    const int quads = live * (HDP / 4), groups = n_pieces <= 8 || 2 * quads > Q8_THREADS ? 1 : (4 * quads > Q8_THREADS ? 2 : 4), shift = groups >> 1;      // (log2 of 1, 2, 4)
    auto part_of = [&](int x) { return groups == 1 ? x >= quads : (x >= quads) + (x >= 2 * quads) + (groups > 2 ? (x >= 3 * quads) + (x >= 4 * quads) : 0); };
    float pm[8];
    float4 pv[8];
    auto fetch = [&](int b0, int to, int m, int i) {
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        const float* p = piece(min(b0 + b, to - 1)) + m * (HDP + 4);
        pm[b] = load_float(p + HDP);
        asm volatile("ld.global.cg.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(pv[b].x), "=f"(pv[b].y), "=f"(pv[b].z), "=f"(pv[b].w) : "l"(p + i) : "memory");
      }
    };
    {      // the first of them beside the maxima and denominators
      const int part = part_of(tid), q = tid - part * quads;
      if (part < groups) fetch(n_pieces * part >> shift, n_pieces * (part + 1) >> shift, q / (HDP / 4), q % (HDP / 4) * 4);
    }
    // every column's maximum and denominator over the pieces
    for (int m = warp; m < live; m += Q8_WARPS) {
      float M = -INFINITY, l = 0.f;
      for (int b = lane; b < n_pieces; b += 32) {
        const float* p = piece(b) + m * (HDP + 4) + HDP;
        const float pm = load_float(p), pl = load_float(p + 1), top = fmaxf(M, pm), r = top == -INFINITY ? 0.f : top;
        l = fmaf(l, ex2(M - r), pl * ex2(pm - r));
        M = top;
      }
      const float sk = a.sinks ? a.sinks[h0 + m - row_in(m) * n_h] * LOG2E : -INFINITY, mm = fmaxf(warp_max(M), sk), r = mm == -INFINITY ? 0.f : mm;
      l = warp_sum(l * ex2(M - r)) + (a.sinks ? ex2(sk - r) : 0.f);
      if (lane == 0) {
        sm_w[m] = r;
        sm_w[16 + m] = l;
      }
    }
    __syncthreads();
    for (int x0 = 0; x0 < quads * groups; x0 += Q8_THREADS) {
      const int x = x0 + tid, part = part_of(x), q = x - part * quads, m = q / (HDP / 4), i = q % (HDP / 4) * 4;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      if (part < groups) {
        const float r = sm_w[m];
        const int from = n_pieces * part >> shift, to = n_pieces * (part + 1) >> shift;
        for (int b0 = from; b0 < to; b0 += 8) {
          if (x0 > 0 || b0 > from) fetch(b0, to, m, i);
#pragma unroll
          for (int b = 0; b < 8; ++b)
            if (b0 + b < to) {
              const float f = ex2(pm[b] - r);
              v[0] = fmaf(f, pv[b].x, v[0]);
              v[1] = fmaf(f, pv[b].y, v[1]);
              v[2] = fmaf(f, pv[b].z, v[2]);
              v[3] = fmaf(f, pv[b].w, v[3]);
            }
        }
      }
      if (groups > 1) {       // one round of threads then: the groups' sums are added in their order
        float4* sum = reinterpret_cast<float4*>(sm_acc);
        if (part > 0 && part < groups) sum[x - quads] = make_float4(v[0], v[1], v[2], v[3]);
        __syncthreads();
        if (part > 0) continue;
        for (int k = 0; k < groups - 1; ++k) {
          const float4 o4 = sum[k * quads + q];
          v[0] += o4.x;
          v[1] += o4.y;
          v[2] += o4.z;
          v[3] += o4.w;
        }
      }
      if (part < groups) {
        const float l = sm_w[16 + m];
        const int h = h0 + m - row_in(m) * n_h;
        TT* out = static_cast<TT*>(a.out) + (size_t)(row0 + row_in(m)) * a.out_ld + h * hd;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (dim_of(i + e) < hd) from_f32(out[dim_of(i + e)], l == 0.f ? 0.f : v[e] / l);
      }
    }
    __syncthreads();      // (the second item's sums go where this one's were)
  }
}

// How a launch is laid out.
struct Q8Plan {
  int hdp, nt, heads_per, head_blocks, rows_per, tiles_per_seg, stages, join_cols, smem;
  long long items, blocks, floats, counters;
};

template <int HDP, int NT, int PARTS, bool EXT, bool FAST>
int q8_launch(const Q8Args& a, const Q8Plan& p, cudaStream_t st) {
  auto kern = attention_q8_kernel<HDP, NT, PARTS, EXT, FAST>;
  // the kernel's limit on shared memory is set once a device (a call takes the host some 10 us)
  static std::atomic<unsigned long long> set{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev < 0 || dev >= 64 || !(set.load(std::memory_order_acquire) >> dev & 1)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Q8_MOST_SMEM);
    if (e != cudaSuccess) return (int)e;
    if (dev >= 0 && dev < 64) set.fetch_or(1ull << dev, std::memory_order_release);
  }
  return (int)launch_pdl(kern, dim3((unsigned)p.blocks), dim3(Q8_THREADS), p.smem, st, a);
}
template <int HDP, int NT, int PARTS>
int q8_launch2(const Q8Args& a, const Q8Plan& p, bool ext, cudaStream_t st) {
  if (a.ps % 16 == 0 && a.hd == HDP) return ext ? q8_launch<HDP, NT, PARTS, true, true>(a, p, st) : q8_launch<HDP, NT, PARTS, false, true>(a, p, st);
  return ext ? q8_launch<HDP, NT, PARTS, true, false>(a, p, st) : q8_launch<HDP, NT, PARTS, false, false>(a, p, st);
}
// The kernels of one padded width are compiled in a file of their own (attention_q8_w*.cu).
template <int HDP>
int q8_run(const Q8Args& a, const Q8Plan& p, bool ext, int f32, cudaStream_t st) {
  if (f32) {
    if (p.nt == 1) return q8_launch2<HDP, 1, 3>(a, p, ext, st);
    if constexpr (HDP < 256)
      if (p.nt == 2) return q8_launch2<HDP, 2, 3>(a, p, ext, st);
    return CBIS_ERR_BAD_SIZE;
  }
  return p.nt == 1 ? q8_launch2<HDP, 1, 2>(a, p, ext, st) : q8_launch2<HDP, 2, 2>(a, p, ext, st);
}

}  // namespace cbis
