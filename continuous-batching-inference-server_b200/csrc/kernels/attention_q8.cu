// Launcher of the attention over the 8-bit cache (attention_q8.cuh).
#include "attention_q8.cuh"
#include <string.h>

namespace cbis {
extern template int q8_run<32>(const Q8Args&, const Q8Plan&, bool, int, cudaStream_t);
extern template int q8_run<64>(const Q8Args&, const Q8Plan&, bool, int, cudaStream_t);
extern template int q8_run<128>(const Q8Args&, const Q8Plan&, bool, int, cudaStream_t);
extern template int q8_run<256>(const Q8Args&, const Q8Plan&, bool, int, cudaStream_t);
}  // namespace cbis

using namespace cbis;

namespace {

int padded_width(int hd) { return hd <= 32 ? 32 : (hd <= 64 ? 64 : (hd <= 128 ? 128 : 256)); }

// Columns of queries / 8: as many as the query heads and rows that share keys fill, up to what the accumulators' registers allow.
int columns8(int hdp, int f32, long long queries) {
  return queries <= 8 || (hdp == 256 && f32) ? 1 : 2;
}
int blocks_per_sm(int hdp, int nt, int f32) { return nt == 1 && hdp < 256 ? (f32 || hdp == 128 ? 3 : 4) : 2; }      // as Q8Shape::BLOCKS

// rows_of_seg 0: decoding, `n` rows; else `n` requests of at most so many rows.
Q8Plan q8_plan(int n, int rows_of_seg, int n_head, int n_kv_head, int hd, int f32, int max_context) {
  Q8Plan p = {};
  const int group = n_head / n_kv_head;
  p.hdp = padded_width(hd);
  p.nt = columns8(p.hdp, f32, (long long)group * (rows_of_seg ? rows_of_seg : 1));
  p.heads_per = group < 8 * p.nt ? group : 8 * p.nt;
  p.head_blocks = (group + p.heads_per - 1) / p.heads_per;
  const long long rows = rows_of_seg ? rows_of_seg : 1, fit = 8 * p.nt / p.heads_per;
  p.rows_per = (int)(rows < fit ? rows : fit);
  p.tiles_per_seg = (int)((rows + p.rows_per - 1) / p.rows_per);
  p.items = (long long)n * p.tiles_per_seg;
  if (p.items > Q8_MAX_ITEMS) return p;
  // as many blocks on an SM as registers allow, if need be with two stages a warp instead of three, and with fewer columns joined at a time
  const int tpw = p.hdp >= 256 ? 1 : (p.hdp == 128 ? (p.nt == 1 ? 2 : 1) : 128 / p.hdp);
  const int stage = tpw * (32 * p.hdp + 128), ldq = p.hdp >= 128 ? p.hdp + 16 : p.hdp, cols = p.rows_per * p.heads_per;
  for (int fit_blocks = blocks_per_sm(p.hdp, p.nt, f32);; --fit_blocks) {
    bool fits = false;
    for (int least = cols < 2 || p.nt > 1 ? 8 : 2, x = 0; x < 4 && !fits; ++x) {
      p.stages = x < 2 ? 3 : 2;
      p.join_cols = x % 2 == 0 ? 8 : least;
      if (p.join_cols > cols) p.join_cols = cols;
      p.smem = q8_smem(stage, p.hdp + 8, ldq, p.stages, cols, p.join_cols, (int)p.items, q8_digits(f32 ? 3 : 2)).bytes;
      fits = p.smem <= Q8_MOST_SMEM && fit_blocks * (p.smem + 1024) <= 228 * 1024;      // (1 KB a block is the system's)
    }
    if (fits) {
      p.blocks = 148LL * fit_blocks;
      break;
    }
    if (fit_blocks == 1) {      // (not with Q8_MAX_ITEMS as it is)
      p.items = Q8_MAX_ITEMS + 1;
      return p;
    }
  }
  const long long pairs = p.items * n_kv_head * p.head_blocks, most = pairs * (max_context / (64 * tpw) + 2);      // no more blocks than there can be pieces
  if (most < p.blocks) p.blocks = most;
  p.floats = p.blocks * 2 * 8 * p.nt * (p.hdp + 4);
  p.counters = pairs;
  return p;
}

}  // namespace

// Scratch of a launch over `n` decoding rows (rows_of_seg 0) or `n` requests of at most rows_of_seg rows: floats for partial results
// and counters (zero before the first launch; every launch leaves them zero).  Returns a status.
CBIS_EXPORT int cbis_attention_q8_scratch(int n, int rows_of_seg, int n_head, int n_kv_head, int hd, int dtype, int max_context,
                                          long long* floats, long long* counters) {
  *floats = *counters = 0;
  if (n <= 0) return CBIS_OK;
  if (n_kv_head <= 0 || n_head <= 0 || n_head % n_kv_head || hd <= 0 || hd > 256 || rows_of_seg < 0 || max_context < 0) return CBIS_ERR_BAD_SIZE;
  const Q8Plan p = q8_plan(n, rows_of_seg, n_head, n_kv_head, hd, dtype == CBIS_F32, max_context);
  *floats = p.floats;
  *counters = p.counters;
  return p.items > Q8_MAX_ITEMS ? CBIS_ERR_TOO_LARGE : CBIS_OK;
}

// rows_of_seg 0: n decoding rows (row_seq, positions; with k_off >= 0 the current token's key and value are taken from q's rows, quantised
// and stored at slot_mapping[row]); else the n requests from seg0 on, whose rows are cu_rows[s] .. cu_rows[s + 1] - 1 at positions from
// seg_start[s] on.  A row whose request is no row of the block table, or that sees no key, gets zeros.
// The call is one record of 8-byte fields.
struct Q8Call {
  long long q, ld, k_off, v_off, kc, ks, vc, vs, block_table, max_blocks, n_seqs, num_pages, row_seq, positions, slot_mapping, cu_rows, seg_start,
      seg0, n, rows_of_seg, n_rows, out, out_ld, part, part_floats, counters, n_counters, n_head, n_kv_head, hd, ps, window, max_context, dtype,
      stream, sinks, slopes, rates, temp_every, keep;
  double scale, temp_coef, cap;
};
CBIS_EXPORT int cbis_attention_q8(const void* call) {
  Q8Call x;
  memcpy(&x, call, sizeof x);
  const int n = q8_int(x.n), rows_of_seg = q8_int(x.rows_of_seg), dtype = (int)x.dtype, hd = q8_int(x.hd), ps = q8_int(x.ps), n_head = q8_int(x.n_head),
            n_kv_head = q8_int(x.n_kv_head), max_blocks = q8_int(x.max_blocks), num_pages = q8_int(x.num_pages), n_seqs = q8_int(x.n_seqs),
            max_context = q8_int(x.max_context), keep = q8_int(x.keep), window = q8_int(x.window), n_rows = q8_int(x.n_rows), seg0 = q8_int(x.seg0),
            ld = (int)x.ld;
  float* part = (float*)x.part;
  if (n <= 0) return CBIS_OK;
  if (dtype != CBIS_F32 && dtype != CBIS_BF16) return CBIS_ERR_BAD_DTYPE;
  if (hd <= 0 || hd > 256 || hd % 16 || ps <= 0 || n_kv_head <= 0 || n_head <= 0 || n_head % n_kv_head || max_blocks <= 0 || keep < 0 ||
      num_pages <= 0 || rows_of_seg < 0 || rows_of_seg > Q8_MAX_POSITION || max_context < 0 || n_rows < 0 || (rows_of_seg && (seg0 < 0 || seg0 + n > n_seqs)) || (!rows_of_seg && n > n_rows))
    return CBIS_ERR_BAD_SIZE;
  if (x.ld > 0x7fffffffLL || x.out_ld > 0x7fffffffLL) return CBIS_ERR_TOO_LARGE;
  if ((long long)max_blocks * ps >= Q8_MAX_POSITION || (long long)num_pages * ps * n_kv_head > 0x7fffffffLL) return CBIS_ERR_TOO_LARGE;
  if (window < -Q8_MAX_POSITION) return CBIS_ERR_BAD_SIZE;
  const int f32 = dtype == CBIS_F32, align = f32 ? 4 : 8;
  if (ld % align || ((x.q | x.kc | x.vc) & 15)) return CBIS_ERR_ALIGNMENT;
  const Q8Plan p = q8_plan(n, rows_of_seg, n_head, n_kv_head, hd, f32, max_context);
  if (p.items > Q8_MAX_ITEMS || p.items * ((long long)max_blocks * ps / 16 + 8) > 0x7fffffffLL) return CBIS_ERR_TOO_LARGE;      // the tiles are counted in 32 bits
  if ((uintptr_t)part & 15) return CBIS_ERR_ALIGNMENT;
  if (x.part_floats < p.floats || x.n_counters < p.counters || (x.k_off >= 0 && !x.slot_mapping)) return CBIS_ERR_BAD_SIZE;
  Q8Args a = {};
  a.q = (const void*)x.q; a.out = (void*)x.out; a.kc = (int8_t*)x.kc; a.vc = (int8_t*)x.vc; a.ks = (float*)x.ks; a.vs = (float*)x.vs;
  a.block_table = (const int*)x.block_table; a.row_seq = (const int*)x.row_seq; a.positions = (const int*)x.positions;
  a.slot_mapping = (const int*)x.slot_mapping;
  a.cu_rows = rows_of_seg ? (const int*)x.cu_rows : nullptr; a.seg_start = (const int*)x.seg_start; a.part = part; a.counters = (unsigned*)x.counters;
  a.sinks = (const float*)x.sinks; a.slopes = (const float*)x.slopes; a.rates = (const float*)x.rates;
  a.n_rows = n_rows; a.ld = ld; a.out_ld = (int)x.out_ld; a.k_off = q8_int(x.k_off); a.v_off = q8_int(x.v_off); a.max_blocks = max_blocks; a.num_pages = num_pages; a.n_seqs = n_seqs;
  a.seg0 = seg0; a.n_items = (int)p.items; a.tiles_per_seg = p.tiles_per_seg; a.n_head = n_head; a.n_kv_head = n_kv_head;
  a.heads_per = p.heads_per; a.heads_inv = (65536 + p.heads_per - 1) / p.heads_per; a.head_blocks = p.head_blocks; a.rows_per = p.rows_per;
  a.stages = p.stages; a.join_cols = p.join_cols; a.page_rows = n_kv_head * ps; a.hd = hd; a.ps = ps; a.ps_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (ps == 1 << i) a.ps_shift = i;
  a.window = window; a.keep = keep; a.temp_every = q8_int(x.temp_every); a.scale = (float)x.scale; a.cap = (float)x.cap;
  a.temp_coef = (float)x.temp_coef;
  a.grid_inv = p.blocks ? 1.000001f / (float)p.blocks : 0.f;
  const bool ext = a.cap > 0.f || (keep > 0 && window != 0) || a.slopes || a.temp_every > 0;
  cudaStream_t st = (cudaStream_t)x.stream;
  switch (p.hdp) {
    case 32: return q8_run<32>(a, p, ext, f32, st);
    case 64: return q8_run<64>(a, p, ext, f32, st);
    case 128: return q8_run<128>(a, p, ext, f32, st);
    default: return q8_run<256>(a, p, ext, f32, st);
  }
}
