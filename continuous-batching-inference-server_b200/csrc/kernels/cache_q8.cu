// The 8-bit cache: a step's keys and values written as codes and scales, and codes and scales read back as values.
// Codes of one layer: [num_pages][heads][page_size][width], one byte each; scales: [num_pages][heads][page_size], 32-bit.
//
// Both are bound by their bytes once there are some megabytes of them, and by the launch below that.
#include "cache_q8.cuh"

namespace cbis {

// Rows with 16-byte loads: `lpr` lanes (a power of two) to a row, each with IT pieces of 16 bytes of it.  A row's largest magnitude
// is found with shuffles inside its lanes while the numbers stay in registers, so the row is read once.
template <typename TT, int IT>
__global__ void __launch_bounds__(128)
kv_write_q8_kernel(const TT* qkv, int ld, int k_off, int v_off, int8_t* kc, float* ks, int8_t* vc, float* vs, const int* slot_mapping,
                   int n_slots, long long n_rows, int heads, int hd, int hd_v, int ps, int lpr, int both) {
  constexpr int E = 16 / sizeof(TT);
  pdl_trigger();
  pdl_wait();
  const int sub = threadIdx.x % lpr;
  const long long unit = (long long)blockIdx.x * (128 / lpr) + threadIdx.x / lpr;      // token, key or value, head
  const int per_token = heads << both;
  const bool in_range = unit < n_rows;
  const int token = in_range ? (int)(unit / per_token) : 0;
  const int place = in_range ? (int)(unit % per_token) : 0;
  const int which = place / heads, h = place % heads, width = which ? hd_v : hd;
  const int slot = in_range ? slot_mapping[token] : -1;
  const bool live = slot >= 0 && slot < n_slots;
  const TT* src = qkv + (size_t)token * ld + (which ? v_off : k_off) + (size_t)h * width;
  float x[IT][E];
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int at = (i * lpr + sub) * E;
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (live && at < width) raw = *reinterpret_cast<const uint4*>(src + at);
    const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (E == 8) {
        x[i][2 * e] = __uint_as_float(w[e] << 16);
        x[i][2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
      } else {
        x[i][e] = __uint_as_float(w[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) top = max(top, q8_bits(x[i][e]));
  }
  for (int o = lpr / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (!live) return;
  const float scale = q8_scale(top), inv = 1.f / scale;
  const size_t row = ((size_t)(slot / ps) * heads + h) * ps + slot % ps;
  int8_t* dst = (which ? vc : kc) + row * width;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int at = (i * lpr + sub) * E;
    if (at >= width) continue;
    unsigned out[E / 4];
#pragma unroll
    for (int e = 0; e < E / 4; ++e) {
      out[e] = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b) out[e] |= (unsigned)(q8_code(x[i][4 * e + b], scale, inv) & 0xff) << (8 * b);
    }
    if constexpr (E == 8) *reinterpret_cast<uint2*>(dst + at) = make_uint2(out[0], out[1]);
    else *reinterpret_cast<unsigned*>(dst + at) = out[0];
  }
  if (sub == 0) (which ? vs : ks)[row] = scale;
}

// Any width and alignment: a warp to a row, which is read twice.
template <typename TT>
__global__ void __launch_bounds__(128)
kv_write_q8_any_kernel(const TT* qkv, int ld, int k_off, int v_off, int8_t* kc, float* ks, int8_t* vc, float* vs, const int* slot_mapping,
                       int n_slots, long long n_rows, int heads, int hd, int hd_v, int ps, int both) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (unit >= n_rows) return;
  const int per_token = heads << both, token = (int)(unit / per_token), place = (int)(unit % per_token);
  const int which = place / heads, h = place % heads, width = which ? hd_v : hd;
  const int slot = slot_mapping[token];
  if (slot < 0 || slot >= n_slots) return;
  const TT* src = qkv + (size_t)token * ld + (which ? v_off : k_off) + (size_t)h * width;
  unsigned top = 0;
  for (int i = lane; i < width; i += 32) top = max(top, q8_bits(to_f32(src[i])));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float scale = q8_scale(top), inv = 1.f / scale;
  const size_t row = ((size_t)(slot / ps) * heads + h) * ps + slot % ps;
  int8_t* dst = (which ? vc : kc) + row * width;
  for (int i = lane; i < width; i += 32) dst[i] = (int8_t)q8_code(to_f32(src[i]), scale, inv);
  if (lane == 0) (which ? vs : ks)[row] = scale;
}

// grid (pages of a request that may be read, requests): a block takes one page of one request, keys and values of all heads.  N
// codes (N output bytes = 16) to a thread and step, so that a warp's stores fill whole lines.
template <typename TT, int N>
__global__ void __launch_bounds__(256)
kv_read_q8_kernel(const int8_t* kc, const float* ks, const int8_t* vc, const float* vs, TT* ko, TT* vo, const int* block_table, int max_blocks,
                  int num_pages, const int* seg_start, const int* seg_ctx, int heads, int hd, int hd_v, int ps, int window, int keep,
                  int kept_blocks, int whole) {
  pdl_trigger();
  pdl_wait();
  const int s = blockIdx.y, ctx = min(seg_ctx[s], max_blocks * ps);
  if (ctx <= 0) return;
  int first = first_seen(min(max(seg_start[s], 0), ctx - 1), window), kept = kept_end(ctx - 1, window, keep);
  if (whole) {
    first -= first % ps;
    kept = (kept + ps - 1) / ps * ps;
  }
  // the pages of the kept first tokens come first, then those from `first` on (a page that both name is taken by the second)
  const int block = (int)blockIdx.x < kept_blocks ? (int)blockIdx.x : first / ps + (int)blockIdx.x - kept_blocks;
  if ((int)blockIdx.x < kept_blocks && (block * ps >= kept || block >= first / ps)) return;
  if (block * ps >= ctx) return;
  const int page = block_table[(size_t)s * max_blocks + block];
  if (page < 0 || page >= num_pages) return;
  for (int which = 0; which < 2; ++which) {
    if (which && vc == nullptr) break;
    const int width = which ? hd_v : hd, per = width / N, units = heads * ps * per;
    const size_t row0 = (size_t)page * heads * ps;
    const int8_t* src = (which ? vc : kc) + row0 * width;
    const float* scales = (which ? vs : ks) + row0;
    TT* dst = (which ? vo : ko) + row0 * width;
#pragma unroll 4
    for (int u = threadIdx.x; u < units; u += 256) {
      const int row = u / per, j = block * ps + row % ps;
      if (j >= ctx || (j < first && j >= kept)) continue;
      const float scale = scales[row];
      if constexpr (N == 1) {
        from_f32(dst[u], (float)src[u] * scale);
      } else if constexpr (N == 4) {
        const char4 c = *reinterpret_cast<const char4*>(src + (size_t)u * 4);
        *reinterpret_cast<float4*>(dst + (size_t)u * 4) = make_float4(c.x * scale, c.y * scale, c.z * scale, c.w * scale);
      } else {
        const uint2 c = *reinterpret_cast<const uint2*>(src + (size_t)u * 8);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)(int8_t)((e < 4 ? c.x : c.y) >> (8 * (e & 3))) * scale;
        store8(dst + (size_t)u * 8, v);
      }
    }
  }
}

}  // namespace cbis

using namespace cbis;

// hd_v 0: the keys' width.  vc null: one array stands for keys and values and takes the rows at k_off.  n_slots: num_pages * ps; rows
// whose slot is none of these are not written.
CBIS_EXPORT int cbis_kv_write_q8(const void* qkv, int ld, int k_off, int v_off, void* kc, void* ks, void* vc, void* vs,
                                 const int* slot_mapping, int n_slots, int T, int heads, int hd, int hd_v, int ps, int dtype,
                                 void* stream) {
  if (T <= 0) return CBIS_OK;
  if (hd_v <= 0) hd_v = hd;
  if (heads <= 0 || hd <= 0 || ps <= 0 || n_slots < 0) return CBIS_ERR_BAD_SIZE;
  if (dtype != CBIS_F32 && dtype != CBIS_BF16) return CBIS_ERR_BAD_DTYPE;
  const int both = vc != nullptr, E = dtype == CBIS_F32 ? 4 : 8, widest = both && hd_v > hd ? hd_v : hd;
  const long long n_rows = (long long)T * (heads << both);
  cudaStream_t st = (cudaStream_t)stream;
  const bool vec = hd % E == 0 && (!both || hd_v % E == 0) && ld % E == 0 && k_off % E == 0 && (!both || v_off % E == 0) &&
                   widest <= 32 * 4 * E && !(((uintptr_t)qkv | (uintptr_t)kc | (uintptr_t)vc) & 15);
  int lpr = 1;
  while (lpr < 32 && lpr * E < widest) lpr *= 2;
  const int its = (widest + lpr * E - 1) / (lpr * E);
  const long long blocks = vec ? (n_rows + 128 / lpr - 1) / (128 / lpr) : (n_rows + 3) / 4;
  if (blocks > 0x7fffffffLL) return CBIS_ERR_TOO_LARGE;
#define CBIS_WRITE(TT, IT)                                                                                                        \
  return (int)launch_pdl(kv_write_q8_kernel<TT, IT>, dim3((unsigned)blocks), dim3(128), 0, st, (const TT*)qkv, ld, k_off, v_off,  \
                         (int8_t*)kc, (float*)ks, (int8_t*)vc, (float*)vs, slot_mapping, n_slots, n_rows, heads, hd, hd_v, ps, lpr, both)
#define CBIS_WRITE_ANY(TT)                                                                                                        \
  return (int)launch_pdl(kv_write_q8_any_kernel<TT>, dim3((unsigned)blocks), dim3(128), 0, st, (const TT*)qkv, ld, k_off, v_off,  \
                         (int8_t*)kc, (float*)ks, (int8_t*)vc, (float*)vs, slot_mapping, n_slots, n_rows, heads, hd, hd_v, ps, both)
  if (dtype == CBIS_F32) {
    if (!vec) CBIS_WRITE_ANY(float);
    if (its == 1) CBIS_WRITE(float, 1);
    if (its == 2) CBIS_WRITE(float, 2);
    CBIS_WRITE(float, 4);
  }
  if (!vec) CBIS_WRITE_ANY(__nv_bfloat16);
  if (its == 1) CBIS_WRITE(__nv_bfloat16, 1);
  if (its == 2) CBIS_WRITE(__nv_bfloat16, 2);
  CBIS_WRITE(__nv_bfloat16, 4);
#undef CBIS_WRITE
#undef CBIS_WRITE_ANY
}

// Values of the first n_seg requests' tokens go to the pages of the same numbers in ko and vo (vc and vo null: one array).  Of request s
// the tokens that its queries at seg_start[s] .. seg_ctx[s] - 1 see: those from first_seen(seg_start[s]) on, at most max_tokens of
// them, and the kept first ones.  whole: the rest of these tokens' pages too, up to seg_ctx[s] (a kernel that brings pages in whole
// multiplies what it masks by zero, which only numbers survive).
CBIS_EXPORT int cbis_kv_read_q8(const void* kc, const void* ks, const void* vc, const void* vs, void* ko, void* vo, const int* block_table,
                                int max_blocks, int num_pages, const int* seg_start, const int* seg_ctx, int n_seg, int max_tokens,
                                int heads, int hd, int hd_v, int ps, int window, int keep, int whole, int dtype, void* stream) {
  if (n_seg <= 0 || max_tokens <= 0) return CBIS_OK;
  if (hd_v <= 0) hd_v = hd;
  if (heads <= 0 || hd <= 0 || ps <= 0 || max_blocks <= 0 || keep < 0 || n_seg > 65535) return CBIS_ERR_BAD_SIZE;
  if ((long long)max_blocks * ps > 0x7fffffffLL || (long long)heads * ps * (hd > hd_v ? hd : hd_v) > 0x7fffffffLL) return CBIS_ERR_TOO_LARGE;
  if (dtype != CBIS_F32 && dtype != CBIS_BF16) return CBIS_ERR_BAD_DTYPE;
  const int kept_blocks = window != 0 ? (keep + ps - 1) / ps : 0;
  long long blocks = (long long)(max_tokens - 1) / ps + 2;
  if (blocks > max_blocks) blocks = max_blocks;
  blocks += kept_blocks < max_blocks ? kept_blocks : max_blocks;
  const int kb = kept_blocks < max_blocks ? kept_blocks : max_blocks;
  const int N = dtype == CBIS_F32 ? 4 : 8;
  const bool vec = hd % N == 0 && (!vc || hd_v % N == 0) &&
                   !(((uintptr_t)kc | (uintptr_t)vc | (uintptr_t)ko | (uintptr_t)vo) & 15);
  cudaStream_t st = (cudaStream_t)stream;
  const dim3 grid((unsigned)blocks, n_seg);
#define CBIS_READ(TT, NN)                                                                                                              \
  return (int)launch_pdl(kv_read_q8_kernel<TT, NN>, grid, dim3(256), 0, st, (const int8_t*)kc, (const float*)ks, (const int8_t*)vc,    \
                         (const float*)vs, (TT*)ko, (TT*)vo, block_table, max_blocks, num_pages, seg_start, seg_ctx, heads, hd, hd_v, \
                         ps, window, keep, kb, whole)
  if (dtype == CBIS_F32) {
    if (vec) CBIS_READ(float, 4);
    CBIS_READ(float, 1);
  }
  if (vec) CBIS_READ(__nv_bfloat16, 8);
  CBIS_READ(__nv_bfloat16, 1);
#undef CBIS_READ
}
