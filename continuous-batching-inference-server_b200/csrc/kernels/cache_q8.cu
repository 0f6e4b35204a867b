// The 8-bit cache: a step's keys and values written as codes and scales, and codes and scales read back as values.
// Codes of one layer: [num_pages][heads][page_size][width], one byte each; scales: [num_pages][heads][page_size], 32-bit.
//
// Both are bound by their bytes once there are some megabytes of them, and by the launch below that.  One B200, in a graph: 8 tokens of 16
// heads of 128 written in 1.6 us, 2,048 in 9.9 (25.4 MB read and written); 23 requests of 90 to 1,100 tokens, 25 heads of 64, read back in
// 29.4 us (134.9 MB, 4.6 TB/s), 32,767 tokens of 8 heads of 32 to 32 bits in 14.8 (86 MB, some of it from L2).
#include "cache_q8.cuh"
#include "packed.cuh"
#include <string.h>

namespace cbis {

// Rows with 16-byte loads: `lpr` lanes (a power of two) to a row, each with IT pieces of 16 bytes of it.  A row's largest magnitude
// is found with shuffles inside its lanes while the numbers stay in registers, so the row is read once.
// (More rows to a thread gained nothing: 2,048 tokens of 16 heads of 128 were 11.2 us with one, 11.4 with two and 12.0 with four.)
template <typename TT, int IT>
__global__ void __launch_bounds__(128)
kv_write_q8_kernel(const TT* qkv, int ld, int k_off, int v_off, int8_t* kc, float* ks, int8_t* vc, float* vs, const int* slot_mapping,
                   int n_slots, unsigned n_rows, int heads, int hd, int hd_v, int ps, int ps_shift, int lpr_shift, int token_shift, int both) {
  constexpr int E = 16 / sizeof(TT);
  pdl_trigger();
  const int lpr = 1 << lpr_shift, sub = threadIdx.x & (lpr - 1);
  const unsigned unit = (blockIdx.x << (7 - lpr_shift)) + (threadIdx.x >> lpr_shift), per_token = heads << both;      // token, key or value, head
  const bool in_range = unit < n_rows;
  const unsigned token = in_range ? (token_shift >= 0 ? unit >> token_shift : unit / per_token) : 0, place = in_range ? unit - token * per_token : 0;
  const bool which = place >= (unsigned)heads;
  const int h = which ? place - heads : place, width = which ? hd_v : hd;
  const TT* src = qkv + (size_t)token * ld + (which ? v_off : k_off) + h * width;
  pdl_wait();
  const int slot = in_range ? slot_mapping[token] : -1;
  const bool live = slot >= 0 && slot < n_slots;
  uint4 raw[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) {      // beside the slot, not after it
    const int at = (i * lpr + sub) * E;
    raw[i] = in_range && at < width ? *reinterpret_cast<const uint4*>(src + at) : make_uint4(0, 0, 0, 0);
  }
  unsigned top = 0;      // bfloat16: the upper and the lower half of every word at once
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const unsigned w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) top = E == 8 ? __vmaxu2(top, w[e] & 0x7fff7fffu) : max(top, w[e] & 0x7fffffffu);
  }
  for (int o = lpr / 2; o > 0; o >>= 1) {
    const unsigned other = __shfl_xor_sync(0xffffffffu, top, o);
    top = E == 8 ? __vmaxu2(top, other) : max(top, other);
  }
  if (!live) return;
  if (E == 8) top = max(top & 0xffff0000u, top << 16);
  const float scale = q8_scale(top), inv = q8_inverse(scale);
  const int page = ps_shift >= 0 ? slot >> ps_shift : slot / ps;
  const size_t row = ((size_t)page * heads + h) * ps + (slot - page * ps);
  int8_t* dst = (which ? vc : kc) + row * width;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int at = (i * lpr + sub) * E;
    if (at >= width) continue;
    const unsigned w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
    float x[E];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (E == 8) {
        x[2 * e] = __uint_as_float(w[e] << 16);
        x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
      } else {
        x[e] = __uint_as_float(w[e]);
      }
    }
    if constexpr (E == 8) *reinterpret_cast<uint2*>(dst + at) = make_uint2(q8_codes4(x, scale, inv), q8_codes4(x + 4, scale, inv));
    else *reinterpret_cast<unsigned*>(dst + at) = q8_codes4(x, scale, inv);
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
  const float scale = q8_scale(top), inv = q8_inverse(scale);
  const size_t row = ((size_t)(slot / ps) * heads + h) * ps + slot % ps;
  int8_t* dst = (which ? vc : kc) + row * width;
  for (int i = lane; i < width; i += 32) dst[i] = (int8_t)q8_code(to_f32(src[i]), scale, inv);
  if (lane == 0) (which ? vs : ks)[row] = scale;
}

// Four codes as numbers: with the sign bit turned round a code is u = code + 128, and 0x4b0000uu is 2^23 + u.
__device__ __forceinline__ void q8_numbers(unsigned w, float* v) {
  w ^= 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; i += 2)
    unpack2(add2(pack2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7650 | i)), __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7651 | i))),
                 pack2(-8388736.f, -8388736.f)), v[i], v[i + 1]);
}

// grid (pages of a request that may be read, requests, parts of a page): a block takes a part of the rows (head, token) of one page of
// one request, of the keys and of the values.  A thread takes N codes (16 output bytes) of a row at a time, `lpr` threads (a power of
// two) side by side a row, and asks for four rows before it uses one.
template <typename TT, int N>
__global__ void __launch_bounds__(256)
kv_read_q8_kernel(const int8_t* kc, const float* ks, const int8_t* vc, const float* vs, TT* ko, TT* vo, const int* block_table, int max_blocks,
                  int num_pages, const int* seg_start, const int* seg_ctx, int heads, int hd, int hd_v, int ps, int window, int keep,
                  int kept_blocks, int whole, int as_codes, int lpr_shift) {
  pdl_wait();      // no early start for the kernel behind: those that read pages ask for the first of them before they wait
  const int s = blockIdx.y, ctx = min(seg_ctx[s], max_blocks * ps);
  if (ctx <= 0) return;
  int first = first_seen(min(max(seg_start[s], 0), ctx - 1), window), kept = kept_end(ctx - 1, window, keep);
  if (whole) {
    first -= first % ps;
    kept = (kept + ps - 1) / ps * ps;
  }
  // the pages of the kept first tokens come first, then those from `first` on (a page that both name is taken by the second)
  const int block = (int)blockIdx.x < kept_blocks ? (int)blockIdx.x : first / ps + (int)blockIdx.x - kept_blocks, j0 = block * ps;
  if ((int)blockIdx.x < kept_blocks && (j0 >= kept || block >= first / ps)) return;
  if (j0 >= ctx) return;
  const int page = block_table[(size_t)s * max_blocks + block];
  if (page < 0 || page >= num_pages) return;
  const int hi = min(ps, ctx - j0), lo = j0 < kept ? 0 : max(first - j0, 0), n = hi - lo;
  const float inv_n = 1.f / n;
  const size_t row0 = (size_t)page * heads * ps;
  const int lpr = 1 << lpr_shift, sub = threadIdx.x & (lpr - 1), rows = heads * n, step = (256 >> lpr_shift) * gridDim.z;
  for (int which = 0; which < 2; ++which) {
    if (which && vc == nullptr) break;
    const int width = which ? hd_v : hd;
    const int8_t* src = (which ? vc : kc) + row0 * width;
    const float* scales = (which ? vs : ks) + row0;
    TT* dst = (which ? vo : ko) + row0 * width;
    if (N > 1 && n == ps && (first <= j0 || kept >= j0 + ps) && width == N << lpr_shift) {
      // a whole page of rows of a power of two of pieces: one run of codes, four pieces of it on their way to a thread
      const int units = rows << lpr_shift;
      for (int u0 = blockIdx.z * 1024 + threadIdx.x; u0 < units; u0 += gridDim.z * 1024) {
        float scale[4];
        uint2 raw[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int u = min(u0 + k * 256, units - 1);
          scale[k] = as_codes ? 1.f : scales[u >> lpr_shift];
          if constexpr (N == 8) raw[k] = reinterpret_cast<const uint2*>(src)[u];
          else raw[k].x = reinterpret_cast<const unsigned*>(src)[u];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (u0 + k * 256 >= units) break;
          float v[8];
          q8_numbers(raw[k].x, v);
          if constexpr (N == 8) q8_numbers(raw[k].y, v + 4);
          const unsigned long long s2 = pack2(scale[k], scale[k]);
#pragma unroll
          for (int e = 0; e < N; e += 2) unpack2(mul2(pack2(v[e], v[e + 1]), s2), v[e], v[e + 1]);
          TT* p = dst + (size_t)(u0 + k * 256) * N;
          if constexpr (N == 8) store8(p, v);
          else *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        }
      }
      continue;
    }
    for (int r0 = blockIdx.z * (256 >> lpr_shift) + (threadIdx.x >> lpr_shift); r0 < rows; r0 += 4 * step) {
      int at[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int r = r0 + k * step, h = (int)((r + 0.5f) * inv_n), slot = lo + r - h * n, j = j0 + slot;      // r / n: exact below 2^22
        at[k] = r < rows && (j >= first || j < kept) ? h * ps + slot : -1;
      }
      for (int c = sub * N; c < width; c += lpr * N) {
        float scale[4];
        uint2 raw[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (at[k] < 0) continue;
          const int8_t* p = src + (size_t)at[k] * width + c;
          scale[k] = as_codes ? 1.f : scales[at[k]];
          if constexpr (N == 8) raw[k] = *reinterpret_cast<const uint2*>(p);
          else if constexpr (N == 4) raw[k].x = *reinterpret_cast<const unsigned*>(p);
          else raw[k].x = (unsigned)(int)*p;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (at[k] < 0) continue;
          TT* p = dst + (size_t)at[k] * width + c;
          float v[8];
          if constexpr (N == 1) {
            from_f32(*p, (float)(int)raw[k].x * scale[k]);
          } else {
            q8_numbers(raw[k].x, v);
            if constexpr (N == 8) q8_numbers(raw[k].y, v + 4);
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] *= scale[k];
            if constexpr (N == 8) store8(p, v);
            else *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
          }
        }
      }
    }
  }
  // The kernel behind starts when the last block ends, and if it is a decode kernel it reads these pages before it waits: they have to be
  // visible by then.  Only whole pages of values are for such a kernel, and the fence is not free (23 requests, 25 heads of 64: 29.9 us
  // without, 33.0 with; 32,767 tokens to 32 bits 15.2 and 19.4); the one over codes waits first.
  if (whole && !as_codes) __threadfence();
}

}  // namespace cbis

using namespace cbis;

// hd_v 0: the keys' width.  vc null: one array stands for keys and values and takes the rows at k_off.  n_slots: num_pages * ps; rows
// whose slot is none of these are not written.
// The call is one record of 8-byte fields, as below.
struct KvWriteCall {
  long long qkv, ld, k_off, v_off, kc, ks, vc, vs, slot_mapping, n_slots, T, heads, hd, hd_v, ps, dtype, stream;
};
CBIS_EXPORT int cbis_kv_write_q8(const void* call) {
  KvWriteCall x;
  memcpy(&x, call, sizeof x);
  const void* qkv = (const void*)x.qkv;
  void *kc = (void*)x.kc, *ks = (void*)x.ks, *vc = (void*)x.vc, *vs = (void*)x.vs, *stream = (void*)x.stream;
  const int* slot_mapping = (const int*)x.slot_mapping;
  int hd_v = (int)x.hd_v;
  const int ld = (int)x.ld, k_off = q8_int(x.k_off), v_off = q8_int(x.v_off), T = q8_int(x.T), heads = q8_int(x.heads), hd = q8_int(x.hd),
            ps = q8_int(x.ps), dtype = (int)x.dtype;
  if (x.n_slots > 0x7fffffffLL || x.ld > 0x7fffffffLL) return CBIS_ERR_TOO_LARGE;
  const int n_slots = (int)x.n_slots;
  if (T <= 0) return CBIS_OK;
  if (hd_v <= 0) hd_v = hd;
  if (heads <= 0 || hd <= 0 || ps <= 0 || n_slots < 0) return CBIS_ERR_BAD_SIZE;
  if (dtype != CBIS_F32 && dtype != CBIS_BF16) return CBIS_ERR_BAD_DTYPE;
  const int both = vc != nullptr, E = dtype == CBIS_F32 ? 4 : 8, widest = both && hd_v > hd ? hd_v : hd;
  const long long n_rows = (long long)T * (heads << both);
  cudaStream_t st = (cudaStream_t)stream;
  const bool vec = hd % E == 0 && (!both || hd_v % E == 0) && ld % E == 0 && k_off % E == 0 && (!both || v_off % E == 0) &&
                   widest <= 32 * 4 * E && !(((uintptr_t)qkv | (uintptr_t)kc | (uintptr_t)vc) & 15);
  int lpr = 1, shift = 0;
  while (lpr < 32 && lpr * E < widest) lpr *= 2, ++shift;
  const int its = (widest + lpr * E - 1) / (lpr * E);
  const long long blocks = vec ? (n_rows + 128 / lpr - 1) / (128 / lpr) : (n_rows + 3) / 4;
  if (n_rows > 0x7fffffffLL || blocks > 0x7fffffffLL) return CBIS_ERR_TOO_LARGE;
  int token_shift = -1, ps_shift = -1;
  for (int i = 0; i < 31; ++i) {
    if (heads << both == 1 << i) token_shift = i;
    if (ps == 1 << i) ps_shift = i;
  }
#define CBIS_WRITE(TT, IT)                                                                                                        \
  return (int)launch_pdl(kv_write_q8_kernel<TT, IT>, dim3((unsigned)blocks), dim3(128), 0, st, (const TT*)qkv, ld, k_off, v_off,  \
                         (int8_t*)kc, (float*)ks, (int8_t*)vc, (float*)vs, slot_mapping, n_slots, (unsigned)n_rows, heads, hd,    \
                         hd_v, ps, ps_shift, shift, token_shift, both)
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
// multiplies what it masks by zero, which only numbers survive).  as_codes: the codes as they are, without their scales.
struct KvReadCall {
  long long kc, ks, vc, vs, ko, vo, block_table, max_blocks, num_pages, seg_start, seg_ctx, n_seg, max_tokens, heads, hd, hd_v, ps, window, keep,
      flags, stream;      // whole | dtype << 1 | as_codes << 2
};
CBIS_EXPORT int cbis_kv_read_q8(const void* call) {
  KvReadCall x;
  memcpy(&x, call, sizeof x);
  const void *kc = (const void*)x.kc, *ks = (const void*)x.ks, *vc = (const void*)x.vc, *vs = (const void*)x.vs;
  void *ko = (void*)x.ko, *vo = (void*)x.vo, *stream = (void*)x.stream;
  const int *block_table = (const int*)x.block_table, *seg_start = (const int*)x.seg_start, *seg_ctx = (const int*)x.seg_ctx;
  int hd_v = (int)x.hd_v;
  const int max_blocks = q8_int(x.max_blocks), num_pages = q8_int(x.num_pages), n_seg = q8_int(x.n_seg), max_tokens = q8_int(x.max_tokens), heads = (int)x.heads,
            hd = (int)x.hd, ps = (int)x.ps, window = q8_int(x.window), keep = q8_int(x.keep), whole = (int)x.flags & 1, dtype = (int)x.flags >> 1 & 1, as_codes = (int)x.flags >> 2;
  if (n_seg <= 0 || max_tokens <= 0) return CBIS_OK;
  if (hd_v <= 0) hd_v = hd;
  if (heads <= 0 || hd <= 0 || ps <= 0 || max_blocks <= 0 || keep < 0 || n_seg > 65535) return CBIS_ERR_BAD_SIZE;
  if (window < -(1 << 30)) return CBIS_ERR_BAD_SIZE;
  if ((long long)max_blocks * ps >= 1 << 30 || (long long)heads * ps * (hd > hd_v ? hd : hd_v) > 0x7fffffffLL) return CBIS_ERR_TOO_LARGE;
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
  int shift = 0;
  const int widest = vc && hd_v > hd ? hd_v : hd;
  while (shift < 5 && (vec ? N : 1) << shift < widest) ++shift;
  // parts of a page: eight rows to a thread if there are blocks enough (23 requests of 90 to 1,100 tokens, 25 heads of 64: 8 % slower with
  // four), fewer rows for a few pages
  const long long rows = (long long)heads * ps, per_block = 256 >> shift, pages = blocks * n_seg;
  long long parts = (rows + 8 * per_block - 1) / (8 * per_block), finest = (rows + per_block - 1) / per_block;
  if (pages * parts < 4 * 148) parts = (4 * 148 + pages - 1) / pages;
  if (parts > finest) parts = finest;
  if (parts > 65535) parts = 65535;
  if (rows > 1 << 22) return CBIS_ERR_TOO_LARGE;
  const dim3 grid((unsigned)blocks, n_seg, (unsigned)parts);
#define CBIS_READ(TT, NN)                                                                                                              \
  return (int)launch_pdl(kv_read_q8_kernel<TT, NN>, grid, dim3(256), 0, st, (const int8_t*)kc, (const float*)ks, (const int8_t*)vc,    \
                         (const float*)vs, (TT*)ko, (TT*)vo, block_table, max_blocks, num_pages, seg_start, seg_ctx, heads, hd, hd_v, \
                         ps, window, keep, kb, whole, as_codes, shift)
  if (dtype == CBIS_F32) {
    if (vec) CBIS_READ(float, 4);
    CBIS_READ(float, 1);
  }
  if (vec) CBIS_READ(__nv_bfloat16, 8);
  CBIS_READ(__nv_bfloat16, 1);
#undef CBIS_READ
}
