// Attention over the 8-bit cache: decoding rows, and chunks of a few new rows a request, in one kernel.
//
// For the query q at position p over the keys j that it sees (codes kc_j, vc_j with scales ks_j, vs_j):
//     s_j = scale ks_j (q . kc_j)  (a cap, a distance bias: as in the other attention kernels),   out = sum_j e^(s_j - m) vs_j vc_j / sum_j e^(s_j - m)
// so the codes go through the tensor cores as they are and the scales meet the scores and the weights.  What bounds it is the codes'
// bytes, read once: 2 (width + 4) per key and key/value head; close behind come the instructions, so few are spent on a code:
//   * scores: mma.sync on signed bytes, keys as they lie in memory.  A query's numbers become whole numbers below 2^22 times a power of
//     two of its own, cut into three signed bytes each, so the products are exact and a number is off by 2^-23 of the query's
//     largest at most, for bfloat16 and for 32-bit rows alike;
//   * values: mma.sync on bfloat16, which holds a code exactly, with the weights times vs_j rounded to bfloat16 (half a step, 2^-8, as the
//     other attention kernels round theirs), or in three bfloat16 parts for 32-bit rows.
//
// Both products are taken with the operands swapped, keys and values as the 16-row operand and the queries as the 8 columns:
// S^T = K Q^T, O^T = V^T P^T.  The query heads that share a key/value head, and a chunk's rows, are the columns, so up to 8 of them cost
// what one does.  A lane loads 16-byte pieces of its two keys (K) and of its four keys (V); the order of the contraction, and that of
// the output's rows, is free, so the pieces are fragments as they come, without shared memory.
//
// The keys of all (row, head) pairs are one row of units (64 or 128 keys), which is cut evenly over the blocks: every block works out
// its part from the positions on the device.  A pair that lies in several blocks is merged by the last one to finish it.
#pragma once
#include "cache_q8.cuh"
#include "mma_sync.cuh"
#include <math.h>
#include <type_traits>

namespace cbis {

constexpr int Q8_WARPS = 4, Q8_THREADS = Q8_WARPS * 32, Q8_MAX_ITEMS = 4096;
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
  int hd, ps, ps_shift, window, keep, temp_every;      // ps_shift: log2 of the page size, -1 where that is no whole number
  float scale, cap, temp_coef;
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
  s.tiles = max(((min(last, a.max_blocks * a.ps - 1) >> 4) + 1) - s.skipped, 0);
  return s;
}

// The two bytes of `w` that hold signed codes (byte 0 and byte 2; the others are anything) as two bfloat16: 128 + the low seven bits,
// less 128 or 256 as the sign bit says.
__device__ __forceinline__ unsigned q8_pair(unsigned w) {
  const unsigned low = (w & 0x007f007fu) | 0x43004300u, off = (w & 0x00800080u) | 0x43004300u;
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&low), *reinterpret_cast<const __nv_bfloat162*>(&off));
  return *reinterpret_cast<const unsigned*>(&r);
}
__device__ __forceinline__ void mma_16832_s8(int (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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

__device__ __forceinline__ float load_float(const float* p) {
  float r;
  asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(r) : "l"(p) : "memory");
  return r;
}
template <int HDP>
struct Q8Lane {                       // what a lane loads of a key: PIECES pieces of WORDS words; of a value: VWORDS words in a row
  static constexpr int WORDS = HDP >= 64 ? 4 : 2, PIECES = HDP / (16 * WORDS), VWORDS = HDP / 32;
};
template <int WORDS>
__device__ __forceinline__ void load_words(unsigned* r, const int8_t* p) {
  if constexpr (WORDS == 1) {
    asm volatile("ld.global.cg.u32 %0, [%1];" : "=r"(r[0]) : "l"(p) : "memory");
  } else if constexpr (WORDS == 2) {
    asm volatile("ld.global.cg.v2.u32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "l"(p) : "memory");
  } else {
    asm volatile("ld.global.cg.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "l"(p) : "memory");
  }
}

// HDP: the width rounded up to 32, 64, 128 or 256; NT: columns of queries / 8; PARTS: bfloat16 parts of a weight (1: bfloat16 rows, 3:
// 32-bit rows); EXT: kept first keys, a cap, a distance bias, a query temperature; FAST: the width is HDP and pages are a multiple of 16 keys.
template <int HDP, int NT, int PARTS>
struct Q8Shape {
  static constexpr int TPW = HDP * NT <= 32 ? 4 : (HDP * NT <= 128 ? 2 : 1);      // tiles a warp takes through one update of its maxima and sums
  static constexpr int UNIT = Q8_WARPS * TPW;                                     // tiles of a unit
  static constexpr int NQ = 8 * NT;
  static constexpr int LDS = HDP + 8;                                             // floats of a query's sums in shared memory
  static constexpr int LDQ = HDP >= 128 ? HDP + 64 : HDP;                         // bytes of a query's row in shared memory: no two lanes of a load on one bank
  static constexpr int BLOCKS = NT == 1 && HDP < 256 ? 3 : 2;                     // per SM
  static constexpr int FLOATS = Q8_WARPS * NQ * (LDS + 2) + 3 * NQ + 8;
  static size_t smem(int n_items) { return (size_t)FLOATS * 4 + 3 * NQ * LDQ + (size_t)(n_items + 1) * 4; }
};

template <int HDP, int NT, int PARTS, bool EXT, bool FAST>
__global__ void __launch_bounds__(Q8_THREADS, Q8Shape<HDP, NT, PARTS>::BLOCKS)
attention_q8_kernel(const __grid_constant__ Q8Args a) {
  using Shape = Q8Shape<HDP, NT, PARTS>;
  using Lane = Q8Lane<HDP>;
  using TT = typename std::conditional<PARTS == 1, __nv_bfloat16, float>::type;
  constexpr int TPW = Shape::TPW, UNIT = Shape::UNIT, NQ = Shape::NQ, LDS = Shape::LDS, LDQ = Shape::LDQ, KS = HDP / 16;
  constexpr int W = Lane::WORDS, PIECES = Lane::PIECES, VW = Lane::VWORDS;
  constexpr bool Q_IN_REGS = NT * HDP <= 128;
  extern __shared__ __align__(16) float sm[];
  float* sm_acc = sm;                                   // [warp][NQ][LDS]
  float* sm_m = sm_acc + Q8_WARPS * NQ * LDS;           // [warp][NQ]
  float* sm_l = sm_m + Q8_WARPS * NQ;                   // [warp][NQ]
  float* sm_w = sm_l + Q8_WARPS * NQ;                   // [NQ] maximum, [NQ] sum of the merged pieces
  float* sm_f = sm_w + 2 * NQ;                          // [NQ] a query's power of two
  int* sm_i = reinterpret_cast<int*>(sm_f + NQ);        // [8]
  int8_t* sm_q = reinterpret_cast<int8_t*>(sm + Shape::FLOATS);      // [3][NQ][LDQ] the queries' bytes, the highest first
  int* before = reinterpret_cast<int*>(sm_q + 3 * NQ * LDQ);         // [n_items + 1] units of the items before this one
  const int hd = FAST ? HDP : a.hd;
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;

  // the items' units, summed up
  int total = 0;
  for (int i0 = 0; i0 < a.n_items; i0 += Q8_THREADS) {
    const int i = i0 + tid;
    int n = 0;
    if (i < a.n_items) {
      const Q8Item it = q8_item(a, i);
      if (it.n_rows > 0) n = max((q8_span<EXT>(a, it).tiles + UNIT - 1) / UNIT, 1);      // a row without keys has its zeros written too
    }
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (lane == 31) sm_i[warp] = sum;
    __syncthreads();
    int at = total;
#pragma unroll
    for (int w = 0; w < Q8_WARPS; ++w) {
      if (w < warp) at += sm_i[w];
      total += sm_i[w];
    }
    if (i < a.n_items) before[i] = at + sum - n;
    __syncthreads();
  }
  if (tid == 0) before[a.n_items] = total;
  __syncthreads();
  const int n_hg = a.n_kv_head * a.head_blocks;
  const long long all = (long long)total * n_hg, per = (all + gridDim.x - 1) / gridDim.x;
  const long long w_end = min(all, (blockIdx.x + 1) * per);

  for (long long w_at = blockIdx.x * per; w_at < w_end;) {
    const int hg = (int)(w_at / total), rem = (int)(w_at % total);
    int lo = 0, hi = a.n_items - 1;                    // the last item that begins at or before rem
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (before[mid] <= rem) lo = mid; else hi = mid - 1;
    }
    const int item = lo, units = before[item + 1] - before[item], u0 = rem - before[item];
    const int u1 = (int)min((long long)units, u0 + (w_end - w_at));
    const Q8Item it = q8_item(a, item);
    const Q8Span span = q8_span<EXT>(a, it);
    const int hk = hg / a.head_blocks, hb = hg % a.head_blocks, group = a.n_head / a.n_kv_head;
    const int h0 = hk * group + hb * a.heads_per, n_h = min(a.heads_per, group - hb * a.heads_per), live = it.n_rows * n_h;
    const int* bt = a.block_table + (size_t)max(it.seq, 0) * a.max_blocks;
    const int last = it.pos0 + it.n_rows - 1;
    const int end_tile = min(u1 * UNIT, span.tiles);

    // the current token's key and value are stored by the block that reads them
    if (a.k_off >= 0 && u1 == units && it.seq >= 0) {
      const int slot = a.slot_mapping[it.row0];
      if (slot >= 0 && slot < a.num_pages * a.ps && warp < 2) {
        const TT* src = static_cast<const TT*>(a.q) + (size_t)it.row0 * a.ld + (warp ? a.v_off : a.k_off) + hk * hd;
        float x[HDP / 32];
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < HDP / 32; ++i) {
          x[i] = i * 32 + lane < hd ? to_f32(src[i * 32 + lane]) : 0.f;
          top = max(top, q8_bits(x[i]));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float s = q8_scale(top), inv = 1.f / s;
        const size_t row = ((size_t)(slot / a.ps) * a.n_kv_head + hk) * a.ps + slot % a.ps;
        int8_t* dst = (warp ? a.vc : a.kc) + row * hd;
#pragma unroll
        for (int i = 0; i < HDP / 32; ++i)
          if (i * 32 + lane < hd) dst[i * 32 + lane] = (int8_t)q8_code(x[i], s, inv);
        if (lane == 0) (warp ? a.vs : a.ks)[row] = s;
      }
      __syncthreads();
    }

    // queries as three signed bytes a number, a warp to a query
    for (int m = warp; m < NQ; m += Q8_WARPS) {
      float x[HDP / 32];
      unsigned top = 0;
      const TT* src = static_cast<const TT*>(a.q) + (size_t)(it.row0 + m / n_h) * a.ld + (h0 + m % n_h) * hd;
#pragma unroll
      for (int i = 0; i < HDP / 32; ++i) {
        x[i] = m < live && i * 32 + lane < hd ? to_f32(src[i * 32 + lane]) : 0.f;
        top = max(top, q8_bits(x[i]));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      const int up = min(275 - (int)(top >> 23), 253);      // 2^(up - 127) brings the largest into [2^21, 2^22)
      const float f = __uint_as_float((unsigned)up << 23);
#pragma unroll
      for (int i = 0; i < HDP / 32; ++i) {
        const int v = top < 0x7f800000u ? __float2int_rn(x[i] * f) : 0;
        const int lo = (int)(int8_t)v, v1 = (v - lo) >> 8, mid = (int)(int8_t)v1;
        int8_t* dst = sm_q + m * LDQ + i * 32 + lane;
        dst[0] = (int8_t)((v1 - mid) >> 8);
        dst[NQ * LDQ] = (int8_t)mid;
        dst[2 * NQ * LDQ] = (int8_t)lo;
      }
      if (lane == 0) sm_f[m] = top < 0x7f800000u ? __uint_as_float((unsigned)(254 - up) << 23) : __uint_as_float(0x7fc00000u);
    }
    __syncthreads();
    // ... as B fragments: column g of each n-tile; the contraction's order is that of the keys' pieces
    auto q_words = [&](int digit, int nt, int c, unsigned (&w)[W]) {
      const int8_t* p = sm_q + (digit * NQ + nt * 8 + g) * LDQ + (c * 16 + t * 4) * W;
      if constexpr (W == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
      } else {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x; w[1] = v.y;
      }
    };
    unsigned qf[Q_IN_REGS ? 3 : 1][Q_IN_REGS ? NT : 1][Q_IN_REGS ? PIECES : 1][W];
    if constexpr (Q_IN_REGS) {
#pragma unroll
      for (int digit = 0; digit < 3; ++digit)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < PIECES; ++c) q_words(digit, nt, c, qf[digit][nt][c]);
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
        const float back = sm_f[nt * 8 + 2 * t + e] * a.scale;
        qp[nt][e] = it.pos0 + max(m, 0) / n_h;
        qs[nt][e] = first_seen(qp[nt][e], a.window);
        qx[nt][e] = back * LOG2E;
        if constexpr (EXT) {
          const int h = h0 + max(m, 0) % n_h;
          qk[nt][e] = kept_end(qp[nt][e], a.window, a.keep);
          qx[nt][e] = back;
          if (a.temp_every > 0) qx[nt][e] *= 1.0f + a.temp_coef * logf((float)((qp[nt][e] + 1) / a.temp_every + 1));
          qslope[nt][e] = a.slopes ? a.slopes[h] : 0.f;
          qrate[nt][e] = a.rates ? a.rates + h : nullptr;
        }
      }
    const int whole_from = first_seen(last, a.window), whole_to = it.pos0;      // keys that every row sees

    float o[NT][KS][4], m_run[NT][2], l_run[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < KS; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
      m_run[nt][0] = m_run[nt][1] = -INFINITY;
      l_run[nt][0] = l_run[nt][1] = 0.f;
    }

    unsigned kw[TPW][2][PIECES * W], vw[TPW][4][VW];
    float ksc[TPW][2], vsc[TPW][2];
    long long base[TPW];                     // FAST: the row of codes that a loaded tile begins with
    int ahead[TPW];                          // FAST: the pages of the tiles to be loaded next, as the table names them
    unsigned held = 0;                       // two bits a tile: this lane's keys g and g + 8 lie in a page of the cache
    auto real_tile = [&](int n) { return n < span.nk ? n : n + span.skipped; };
    auto find_pages = [&](int tile) {
#pragma unroll
      for (int u = 0; u < TPW; ++u) {
        const int j0 = real_tile(min(tile + u, end_tile - 1)) << 4;
        ahead[u] = bt[a.ps_shift >= 0 ? j0 >> a.ps_shift : j0 / a.ps];
      }
    };
    // The row of codes of the key at j.  Where the table names no page of the cache that is the head's first row of page 0, and `ok` is
    // false: every address that is worked out here lies in the cache, whether it is used or not.
    auto row_of = [&](int j, bool& ok) -> long long {
      const int at = min(j, a.max_blocks * a.ps - 1), page = bt[at / a.ps];
      ok = j == at && page >= 0 && page < a.num_pages;
      return ok ? ((long long)page * a.n_kv_head + hk) * a.ps + j % a.ps : (long long)hk * a.ps;
    };
    auto load_keys = [&](int tile) {
      held = 0;
#pragma unroll
      for (int u = 0; u < TPW; ++u) {
        if (tile + u >= end_tile) continue;
        const int j0 = real_tile(tile + u) << 4;
        if constexpr (FAST) {
          const bool ok = ahead[u] >= 0 && ahead[u] < a.num_pages;
          const int in_page = a.ps_shift >= 0 ? j0 & (a.ps - 1) : j0 % a.ps;
          base[u] = ok ? ((long long)ahead[u] * a.n_kv_head + hk) * a.ps + in_page : (long long)hk * a.ps;
          held |= ok ? 3u << (2 * u) : 0u;
          const int8_t* p = a.kc + base[u] * HDP + (g * HDP + t * 4 * W);
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int c = 0; c < PIECES; ++c) load_words<W>(&kw[u][i][c * W], p + i * 8 * HDP + c * 16 * W);
          const float *ps = a.ks + base[u] + g, *vs = a.vs + base[u] + g;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            ksc[u][i] = load_float(ps + 8 * i);
            vsc[u][i] = load_float(vs + 8 * i);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            bool ok;
            const long long row = row_of(j0 + g + 8 * i, ok);
            if (ok) held |= 1u << (2 * u + i);
            const int8_t* p = a.kc + row * hd;
#pragma unroll
            for (int c = 0; c < PIECES; ++c) {
              const int d0 = c * 16 * W + t * 4 * W;
              load_words<W>(&kw[u][i][c * W], p + (d0 < hd ? d0 : 0));
              if (d0 >= hd) {
#pragma unroll
                for (int w = 0; w < W; ++w) kw[u][i][c * W + w] = 0;
              }
            }
            ksc[u][i] = load_float(a.ks + row);
            vsc[u][i] = load_float(a.vs + row);
          }
        }
      }
    };
    auto load_values = [&](int tile) {      // after load_keys(tile), before the next load_keys
#pragma unroll
      for (int u = 0; u < TPW; ++u) {
        if (tile + u >= end_tile) continue;
        constexpr int PW = VW < 4 ? VW : 4;      // words of a load
        if constexpr (FAST) {
          const int8_t* p = a.vc + base[u] * HDP + (2 * t * HDP + g * 4 * VW);
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int w0 = 0; w0 < VW; w0 += PW) load_words<PW>(&vw[u][i][w0], p + ((i & 1) + 8 * (i >> 1)) * HDP + 4 * w0);
        } else {
          const int j0 = real_tile(tile + u) << 4;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            bool ok;
            const int8_t* p = a.vc + row_of(j0 + 2 * t + (i & 1) + 8 * (i >> 1), ok) * hd;
#pragma unroll
            for (int w0 = 0; w0 < VW; w0 += PW) {
              const int d0 = (g * VW + w0) * 4;
              load_words<PW>(&vw[u][i][w0], p + (d0 < hd ? d0 : 0));
              if (d0 >= hd) {
#pragma unroll
                for (int w = 0; w < PW; ++w) vw[u][i][w0 + w] = 0;
              }
            }
          }
        }
      }
    };
    // tiles behind the last are not loaded: their products are masked, but have to be of something
#pragma unroll
    for (int u = 0; u < TPW; ++u) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ksc[u][i] = vsc[u][i] = 0.f;
#pragma unroll
        for (int w = 0; w < PIECES * W; ++w) kw[u][i][w] = 0;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int w = 0; w < VW; ++w) vw[u][i][w] = 0;
    }

    int tile = u0 * UNIT + warp * TPW;
    if (tile < end_tile) {
      if constexpr (FAST) find_pages(tile);
      load_keys(tile);
      load_values(tile);
      if constexpr (FAST) find_pages(tile + UNIT);
    }
    // A round: the scores are taken from the keys, the keys of the next round are asked for, the maxima, sums and products with the
    // values follow, and the next values are asked for: a warp has loads on their way all the time.
    for (; tile < end_tile; tile += UNIT) {
      float s[TPW][NT][4];
#pragma unroll
      for (int u = 0; u < TPW; ++u) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          int sh[4] = {0, 0, 0, 0}, sd[4] = {0, 0, 0, 0}, sl[4] = {0, 0, 0, 0};
#pragma unroll
          for (int c = 0; c < PIECES; ++c) {
            unsigned q0[W], q1[W], q2[W];
            if constexpr (Q_IN_REGS) {
#pragma unroll
              for (int w = 0; w < W; ++w) {
                q0[w] = qf[0][nt][c][w];
                q1[w] = qf[1][nt][c][w];
                q2[w] = qf[2][nt][c][w];
              }
            } else {
              q_words(0, nt, c, q0);
              q_words(1, nt, c, q1);
              q_words(2, nt, c, q2);
            }
#pragma unroll
            for (int w = 0; w < W; w += 2) {
              const unsigned A[4] = {kw[u][0][c * W + w], kw[u][1][c * W + w], kw[u][0][c * W + w + 1], kw[u][1][c * W + w + 1]};
              mma_16832_s8(sh, A, q0[w], q0[w + 1]);
              mma_16832_s8(sd, A, q1[w], q1[w + 1]);
              mma_16832_s8(sl, A, q2[w], q2[w + 1]);
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) s[u][nt][e] = fmaf((float)sh[e], 65536.f, (float)(sd[e] * 256 + sl[e]));
        }
      }
      float kx[TPW][2], vx[TPW][2];
      const unsigned in_page = held;
#pragma unroll
      for (int u = 0; u < TPW; ++u)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          kx[u][i] = ksc[u][i];
          vx[u][i] = vsc[u][i];
        }
      if (tile + UNIT < end_tile) {
        load_keys(tile + UNIT);
        if constexpr (FAST) find_pages(tile + 2 * UNIT);
      }
      // scores in the base-2 domain; -inf where the query does not see the key
      bool whole = true;       // every row sees every key of the warp's tiles
      float mx[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mx[nt][0] = mx[nt][1] = -INFINITY;
#pragma unroll
      for (int u = 0; u < TPW; ++u) {
        const int j0 = real_tile(tile + u) << 4;
        whole = whole && tile + u < end_tile && j0 >= whole_from && j0 + 15 <= whole_to;
        if constexpr (FAST) whole = whole && ((in_page >> (2 * u)) & 3u) == 3u;      // the same in all lanes
        else whole = whole && __all_sync(0xffffffffu, ((in_page >> (2 * u)) & 3u) == 3u);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = e >> 1, c = e & 1;
            float v = s[u][nt][e] * (kx[u][i] * qx[nt][c]);
            if constexpr (EXT) {
              v = capped_score(v, a.cap);
              if (a.slopes) v -= distance_bias(qslope[nt][c], qrate[nt][c], (float)max(qp[nt][c] - (j0 + g + 8 * i), 0));
              v *= LOG2E;
            }
            s[u][nt][e] = v;
          }
      }
      if (!whole) {
#pragma unroll
        for (int u = 0; u < TPW; ++u) {
          const int j0 = real_tile(tile + u) << 4;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int i = e >> 1, c = e & 1, j = j0 + g + 8 * i;
              const bool ok = tile + u < end_tile && j <= qp[nt][c] && (j >= qs[nt][c] || (EXT && j < qk[nt][c])) && ((in_page >> (2 * u + i)) & 1u);
              s[u][nt][e] = ok ? s[u][nt][e] : -INFINITY;
            }
        }
      }
#pragma unroll
      for (int u = 0; u < TPW; ++u)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx[nt][e & 1] = fmaxf(mx[nt][e & 1], s[u][nt][e]);
      bool moved = false;
      float corr[NT][2], ref[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) mx[nt][c] = fmaxf(mx[nt][c], __shfl_xor_sync(0xffffffffu, mx[nt][c], x));
          const float m_new = fmaxf(m_run[nt][c], mx[nt][c]);
          moved |= m_new != m_run[nt][c];
          ref[nt][c] = m_new == -INFINITY ? 0.f : m_new;
          corr[nt][c] = ex2(m_run[nt][c] - ref[nt][c]);
          m_run[nt][c] = m_new;
        }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          l_run[nt][0] *= corr[nt][0];
          l_run[nt][1] *= corr[nt][1];
#pragma unroll
          for (int j = 0; j < KS; ++j) {
            o[nt][j][0] *= corr[nt][0];
            o[nt][j][1] *= corr[nt][1];
            o[nt][j][2] *= corr[nt][0];
            o[nt][j][3] *= corr[nt][1];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < TPW; ++u) {
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
          if constexpr (PARTS == 1) {
            pf[0][nt][0] = transposed(pack_bf16(p[0], p[1]));
            pf[0][nt][1] = transposed(pack_bf16(p[2], p[3]));
          } else {
            unsigned a0[3], a1[3];
            cut3(p[0], p[1], a0);
            cut3(p[2], p[3], a1);
#pragma unroll
            for (int i = 0; i < PARTS; ++i) {
              pf[i][nt][0] = transposed(a0[i]);
              pf[i][nt][1] = transposed(a1[i]);
            }
          }
        }
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          const int w = j >> 1;
          const unsigned lo = j & 1 ? 0x0602 : 0x0400, hi = j & 1 ? 0x0703 : 0x0501;
          const unsigned A[4] = {q8_pair(__byte_perm(vw[u][0][w], vw[u][1][w], lo)), q8_pair(__byte_perm(vw[u][0][w], vw[u][1][w], hi)),
                                 q8_pair(__byte_perm(vw[u][2][w], vw[u][3][w], lo)), q8_pair(__byte_perm(vw[u][2][w], vw[u][3][w], hi))};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int p = PARTS - 1; p >= 0; --p) mma_16816(o[nt][j], A, pf[p][nt][0], pf[p][nt][1]);
        }
      }
      if (tile + UNIT < end_tile) load_values(tile + UNIT);
    }

    // the warps' results joined
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float l = l_run[nt][c];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
        const int m = nt * 8 + 2 * t + c;
        if (g == 0) {
          sm_m[warp * NQ + m] = m_run[nt][c];
          sm_l[warp * NQ + m] = l;
        }
        if (m < live) {
          float* dst = sm_acc + (size_t)(warp * NQ + m) * LDS + g * 2;      // [pair of dims j][lane g][2]
#pragma unroll
          for (int j = 0; j < KS; ++j) *reinterpret_cast<float2*>(dst + j * 16) = make_float2(o[nt][j][c], o[nt][j][2 + c]);
        }
      }
    __syncthreads();
    const bool alone = u0 == 0 && u1 == units;
    const long long item_at = (long long)hg * total + before[item];
    const int b_first = (int)(item_at / per), b_last = (int)((item_at + units - 1) / per);
    float* mine = a.part + (size_t)(2 * blockIdx.x + (u0 == 0)) * NQ * (HDP + 2);
    for (int x = tid; x < live * HDP; x += Q8_THREADS) {
      const int m = x / HDP, i = x % HDP, d = ((i >> 1) & 7) * (HDP / 8) + (i >> 4) * 2 + (i & 1);
      float mw[Q8_WARPS], M = -INFINITY, l = 0.f, v = 0.f;
#pragma unroll
      for (int w = 0; w < Q8_WARPS; ++w) {
        mw[w] = sm_m[w * NQ + m];
        M = fmaxf(M, mw[w]);
      }
#pragma unroll
      for (int w = 0; w < Q8_WARPS; ++w) {
        const float f = mw[w] == -INFINITY && M != -INFINITY ? 0.f : ex2(mw[w] - (M == -INFINITY ? 0.f : M));
        v = fmaf(f, sm_acc[(size_t)(w * NQ + m) * LDS + i], v);
        l = fmaf(f, sm_l[w * NQ + m], l);
      }
      if (alone) {
        const int h = h0 + m % n_h;
        float keep1 = 1.f;
        if (a.sinks) {
          const float sk = a.sinks[h] * LOG2E, mm = fmaxf(M, sk);
          keep1 = ex2(M - mm);
          l = fmaf(l, keep1, ex2(sk - mm));
        }
        if (d < hd) from_f32(static_cast<TT*>(a.out)[(size_t)(it.row0 + m / n_h) * a.out_ld + h * hd + d], l == 0.f ? 0.f : v * keep1 / l);
      } else {
        float* p = mine + m * (HDP + 2);
        p[2 + i] = v;
        if (i == 0) {
          p[0] = M;
          p[1] = l;
        }
      }
    }
    if (!alone) {
      __threadfence();
      __syncthreads();
      unsigned* counter = a.counters + (size_t)item * n_hg + hg;
      if (tid == 0) sm_i[0] = atomicAdd(counter, 1u) == (unsigned)(b_last - b_first);
      __syncthreads();
      if (sm_i[0]) {
        __threadfence();
        const int n_pieces = b_last - b_first + 1;
        auto piece = [&](int b) { return a.part + (size_t)(2 * (b_first + b) + (b == 0)) * NQ * (HDP + 2); };
        // every query's maximum and sum over the pieces first
        for (int m = warp; m < live; m += Q8_WARPS) {
          float M = -INFINITY, l = 0.f;
          for (int b = lane; b < n_pieces; b += 32) M = fmaxf(M, load_float(piece(b) + m * (HDP + 2)));
          M = warp_max(M);
          const float sk = a.sinks ? a.sinks[h0 + m % n_h] * LOG2E : -INFINITY, mm = fmaxf(M, sk), r = mm == -INFINITY ? 0.f : mm;
          for (int b = lane; b < n_pieces; b += 32) l = fmaf(ex2(load_float(piece(b) + m * (HDP + 2)) - r), load_float(piece(b) + m * (HDP + 2) + 1), l);
          l = warp_sum(l) + (a.sinks ? ex2(sk - r) : 0.f);
          if (lane == 0) {
            sm_w[m] = r;
            sm_w[NQ + m] = l;
          }
        }
        __syncthreads();
        for (int x = tid; x < live * HDP; x += Q8_THREADS) {
          const int m = x / HDP, i = x % HDP, d = ((i >> 1) & 7) * (HDP / 8) + (i >> 4) * 2 + (i & 1);
          const float r = sm_w[m], l = sm_w[NQ + m];
          float v = 0.f;
          for (int b0 = 0; b0 < n_pieces; b0 += 8) {      // eight in flight
            float pm[8], pv[8];
#pragma unroll
            for (int b = 0; b < 8; ++b) {
              const float* p = piece(min(b0 + b, n_pieces - 1)) + m * (HDP + 2);
              pm[b] = load_float(p);
              pv[b] = load_float(p + 2 + i);
            }
#pragma unroll
            for (int b = 0; b < 8; ++b) v = b0 + b < n_pieces ? fmaf(ex2(pm[b] - r), pv[b], v) : v;
          }
          const int h = h0 + m % n_h;
          if (d < hd) from_f32(static_cast<TT*>(a.out)[(size_t)(it.row0 + m / n_h) * a.out_ld + h * hd + d], l == 0.f ? 0.f : v / l);
        }
        if (tid == 0) *counter = 0;
      }
    }
    __syncthreads();
    w_at += u1 - u0;
  }
}

// How a launch is laid out.
struct Q8Plan {
  int hdp, nt, heads_per, head_blocks, rows_per, tiles_per_seg;
  long long items, blocks, floats, counters;
};

template <int HDP, int NT, int PARTS, bool EXT, bool FAST>
int q8_launch(const Q8Args& a, const Q8Plan& p, cudaStream_t st) {
  auto kern = attention_q8_kernel<HDP, NT, PARTS, EXT, FAST>;
  const size_t smem = Q8Shape<HDP, NT, PARTS>::smem(a.n_items);
  const cudaError_t e = allow_smem(kern, smem);
  if (e != cudaSuccess) return (int)e;
  return (int)launch_pdl(kern, dim3((unsigned)p.blocks), dim3(Q8_THREADS), smem, st, a);
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
  if (p.nt == 1) return q8_launch2<HDP, 1, 1>(a, p, ext, st);
  if (p.nt == 2) return q8_launch2<HDP, 2, 1>(a, p, ext, st);
  if constexpr (HDP < 256)
    if (p.nt == 4) return q8_launch2<HDP, 4, 1>(a, p, ext, st);
  return CBIS_ERR_BAD_SIZE;
}


}  // namespace cbis
