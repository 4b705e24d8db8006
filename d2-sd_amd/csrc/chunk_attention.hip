// gfx950 kernels of the attention of each request's newest tokens over its
// paged KV cache, which already holds them:
//
//   o_i = sum_j softmax_j(s q_i . k_j) v_j,   pos_i - window <= j <= pos_i,
//   pos_i = cache length - new tokens + i,    lse_i = log sum_j exp(s q_i . k_j),
//   o_i *= sigmoid(lse_i - sink)              (with sinks)
//
// for a chunk of a prompt, a single token, or a batch of both, over a cache in
// bf16, fp8 (one scale per kv head) or the block formats mxfp8 and mxfp4.
//
//   chunk_attn_kernel   one workgroup per work item: packed rows of one
//                       (request, kv head) against a chunk of their visible
//                       keys, with a running maximum and sum (one pass over the
//                       cache), state in registers
//   chunk_merge_kernel  joins the partial states of rows whose keys were split
//
// Rows are packed (token, query head of the kv head) pairs, row = token * g + j,
// so that a key is read once for all query heads that share it.  S^T = K Q^T
// and O^T += V^T P^T: a lane holds scores and output of one row, so the softmax
// stays in a lane and its one (tile items) or three (token items) partners, and
// P^T goes back as an operand without leaving the registers.  Codes are expanded
// to bf16 by the converters that apply a block's scale as they go; that is exact,
// so quantised caches cost no accuracy beyond their own.
//
// Two kinds of item, by packed rows:
//  * tile items (more than 32 rows): v_mfma_f32_32x32x16_bf16; each wave owns 32
//    rows, the workgroup stages tiles of 64 keys into LDS (bf16 straight, codes
//    through registers; two buffers, one barrier a tile).  Bound by MFMA and the
//    softmax's vector instructions, which the lock-step of the waves lets overlap
//    only in part: 2 x 2048 tokens at 16384 keys, 32 heads of 128, take 0.93 to
//    0.98 ms, 1.05 PFLOP/s, where a large library product reaches 1.36; a tile is
//    2048 cycles of MFMA (of both waves of a SIMD) in 3700.
//  * token items (up to 32 rows: decoding): v_mfma_f32_16x16x32_bf16; all waves
//    share the rows, and wave w of W takes every W-th tile of 32 keys.  Keys go
//    from the cache straight to the MFMA operand: the sum over head dims may run
//    in any order, so lane l takes a quarter of key l % 16's dims (through LDS
//    instead: 168 -> 233 us on 32 x 8..32k mxfp4).  Values pass through the
//    wave's own LDS to be read transposed.  No barrier until the waves' states
//    are joined.  Bound by HBM: 32 requests of 8..32k tokens read
//    6.2 TB/s in bf16, 5.7 in mxfp8, 5.2 in mxfp4 (1 KB of a page at a time).
//
// Plans whose requests share their first keys (shared_attn_kernel, shared_merge_kernel)
// compute those once for the rows of a whole group, at the rate of matrix products:
// bytes of the shared keys fall by the group's size, and decoding 96 requests behind
// 32K keys becomes the work of a prompt's chunk.  Three kinds of item:
//  * shared keys: 32 rows a wave (256 or 128 an item), the loop of shared_tile.h;
//  * keys of a request's own, up to 32 rows: a wave each, without a partner or a
//    barrier, so that a workgroup holds as many requests and heads as waves (token
//    items, one a workgroup, spent most of their time on their start and joins: 64
//    requests behind 16K bf16 keys took 65 us, now 43);
//  * a request's own rows beyond 32: tile items.
// A plan of so few rows that no tile fills takes the kernels above over all of its
// parts.  Partial states over shared keys lie as the registers hold them; 20 MB of
// partial states otherwise cost as many lines a store as rows.  Measured, one token
// a request, heads of 128: 4 requests behind 2K bf16 keys 12 us, most of it two
// launches; 32 behind 8K in mxfp8 26; 64 behind 16K in bf16 43.  96 behind 32K in
// mxfp8 with 64 query heads 158: their products take 79 at a library's rate and
// their own keys, 0.32 GB, 65 beside them, but the two share power and memory.  Six
// chunks of 100..700 tokens behind 8K in mxfp4 257, products 185.
//
// Keys outside an item's visible range are never read: their addresses are
// clamped to the range, so what lies behind a cache's end (or before its
// window) may hold anything.  What lies inside and is not finite reaches the rows
// that see it alone ("values that are not finite" below).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "d2sd_internal.h"
#include "kernel_common.h"
#include "plan.h"

namespace d2sd {

namespace {

typedef __attribute__((address_space(3))) char lds_char;

// Bytes of one cache row (one token's head) and the formats' properties.
template <int D, int FMT>
struct Format {
  static constexpr bool MX = FMT == CACHE_MXFP8 || FMT == CACHE_MXFP4;
  static constexpr int ROW = FMT == CACHE_BF16 ? 2 * D : FMT == CACHE_MXFP4 ? D / 2 : D;
};

__device__ __forceinline__ float xor32(float x, int hh) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(hh ? r[0] : r[1]);
}

// 8 codes (two words of fp8, one of fp4) as bf16
template <int FMT>
__device__ __forceinline__ bf16x8 expand(unsigned w0, unsigned w1, float sc) {
  u32x4 u;
  if constexpr (FMT == CACHE_MXFP4) {
    u[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w0, sc, 0));
    u[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w0, sc, 1));
    u[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w0, sc, 2));
    u[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w0, sc, 3));
  } else {
    u[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, sc, false));
    u[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, sc, true));
    u[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, sc, false));
    u[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, sc, true));
  }
  return __builtin_bit_cast(bf16x8, u);
}

__device__ __forceinline__ float block_scale(unsigned byte) {
  return __uint_as_float(byte == 255u ? 0x7FC00000u : byte == 0u ? 0x00400000u : byte << 23);
}

// What an item's rows see: query i of the request sits at pos0 + i.
struct Span {
  int pos0;       // position of the request's query 0 (negative: it has no key yet; items of shared keys: unused)
  int lo, hi;     // keys [lo, hi) are visible to some row of the item
  int all_lo, all_hi;  // keys [all_lo, all_hi) are visible to every row
};

__device__ __forceinline__ Span item_span(const ChunkParams& p, const ChunkItem& w, int t0, int t1) {
  Span s;
  const int len = min(p.kv_len[w.req], (w.page_end - w.page_begin) << p.log2_page);
  s.pos0 = len - w.nq;
  const int first = s.pos0 + t0, last = s.pos0 + t1;
  s.hi = max(last + 1, 0);
  s.lo = p.window_left >= 0 ? max(first - p.window_left, 0) : 0;
  s.all_hi = first + 1;
  s.all_lo = p.window_left >= 0 ? max(last - p.window_left, 0) : 0;
  return s;
}

// ---- shared keys ----
// Plans whose requests share their first keys (SHARED) have three parts of work:
// the rows of a whole group of requests over the keys that they share
// (PART_SHARED: keys [0, bound) of the group's first request), each request's rows
// over its keys from `bound` on (PART_OWN), and requests that share nothing.  Rows
// of a group lie one after the other, so that an item's rows are packed as ever;
// but they sit at positions of their own.
__device__ __forceinline__ int shared_pos(const ChunkParams& p, const ChunkItem& w, int row) {
  const int4 t = ((const int4*)p.tokens)[w.q0 + (w.row0 + row) / p.group];  // request, tokens to its end, tokens its pages hold
  return min(p.kv_len[t.x], t.z) - t.y;
}

__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) x = min(x, __shfl_xor(x, m));
  return __builtin_amdgcn_readfirstlane(x);
}

// The span of packed rows row_a .. row_b of the item.  edges: all_lo and all_hi are
// wanted too.  (Without a window an item of shared keys takes lo and hi as they are
// planned, so that its first keys wait for no length.)
template <bool SHARED>
__device__ __forceinline__ Span rows_span(const ChunkParams& p, const ChunkItem& w, int row_a, int row_b, bool edges = true) {
  if constexpr (!SHARED) return item_span(p, w, (w.row0 + row_a) / p.group, (w.row0 + row_b) / p.group);
  if (w.part != PART_SHARED) {
    Span s = item_span(p, w, (w.row0 + row_a) / p.group, (w.row0 + row_b) / p.group);
    s.lo = max(s.lo, w.bound);
    s.all_lo = max(s.all_lo, w.bound);
    return s;
  }
  Span s{0, 0, w.bound, w.bound, 0};
  if (!edges && p.window_left < 0) return s;
  int first = 0x7FFFFFFF, past = 0x7FFFFFFF;  // lowest position; 0 - highest
  for (int row = row_a + (threadIdx.x & 63); row <= row_b; row += 64) {
    const int pos = shared_pos(p, w, row);
    first = min(first, pos);
    past = min(past, -pos);
  }
  first = wave_min(first);
  const int last = -wave_min(past);
  s.all_lo = 0, s.all_hi = min(w.bound, first + 1);
  if (p.window_left >= 0) {
    s.hi = min(w.bound, max(last + 1, 0));
    s.lo = max(first - p.window_left, 0);
    s.all_lo = max(last - p.window_left, 0);
  }
  return s;
}

// Keys [0, this) are visible to every row of the item, which is one of shared keys
// without a window.  (Arguments and item are read again: nothing need be kept for here
// over the tile loop.)
__device__ __forceinline__ int seen_by_all_rows() {
  auto at = (const __attribute__((address_space(4))) char*)__builtin_amdgcn_kernarg_segment_ptr();
  __asm__ volatile("" : "+s"(at));
  const ChunkParams& p = *(const ChunkParams*)at;
  const ChunkItem w = p.items[blockIdx.x];
  return rows_span<true>(p, w, 0, w.nrows - 1).all_hi;
}

// Keys that a row at `pos` sees: first and last of the item's.
template <bool SHARED>
__device__ __forceinline__ int row_first(const ChunkParams& p, const ChunkItem& w, int pos) {
  const int lo = p.window_left >= 0 ? max(pos - p.window_left, 0) : 0;
  if constexpr (SHARED) return w.part == PART_SHARED ? lo : max(lo, w.bound);
  return lo;
}
template <bool SHARED>
__device__ __forceinline__ int row_last(const ChunkItem& w, int pos) {
  if constexpr (SHARED) return w.part == PART_SHARED ? min(pos, w.bound - 1) : pos;
  return pos;
}
template <bool SHARED>
__device__ __forceinline__ int row_pos(const ChunkParams& p, const ChunkItem& w, int pos0, int row) {
  if constexpr (SHARED)
    if (w.part == PART_SHARED) return shared_pos(p, w, row);
  return pos0 + (w.row0 + row) / p.group;
}
// Whether the item's state is one of several of its rows.
template <bool SHARED>
__device__ __forceinline__ bool is_partial(const ChunkItem& w) {
  return w.nchunks > 1 || (SHARED && w.part != PART_ALONE);
}

// Partial states of a wave's 32 rows over shared keys are stored as the registers
// hold them (lane hh * 32 + row has dims 32 mt + 8 q + 4 hh .. + 3 of its row), 1 KB
// a store: by rows a store would touch 32 lines.  Blocks of 32 rows follow each
// other, then chunks.
template <int D>
__device__ __forceinline__ long long image_at(long long row0, int d4, int row) {
  return row0 * D + (((d4 >> 1) * 64 + (d4 & 1) * 32 + row) << 2);  // row0: the block's first
}
template <int D>
__device__ __forceinline__ void store_image(const ChunkParams& p, const ChunkItem& w, const f32x16 (&o)[D / 32], float inv,
                                            float lse2, int wrow, int l32, int hh) {
  if (wrow + l32 >= w.nrows) return;
  const long long row0 = w.slot + (long long)w.chunk * ((w.nrows + 31) & ~31) + wrow;
#pragma unroll
  for (int mt = 0; mt < D / 32; ++mt)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *(f32x4*)(p.part_o + image_at<D>(row0, 8 * mt + 2 * q + hh, l32)) =
          (f32x4){o[mt][4 * q] * inv, o[mt][4 * q + 1] * inv, o[mt][4 * q + 2] * inv, o[mt][4 * q + 3] * inv};
  if (hh == 0) p.part_lse[row0 + l32] = lse2;
}

// Online softmax of 16 * N scores of this lane's row: the running maximum m (raw
// score units) may trail the true one by kRescaleSlack before the state is
// rescaled; then probabilities into s and their sum into l (32 bits, before
// they are rounded to bf16 for the second product, whose operands are bf16).
template <int N, int MT>
__device__ __forceinline__ void softmax_step(f32x16 (&s)[N], f32x16 (&o)[MT], float& m, float& l, float c,
                                             float slack, int hh) {
  float m4[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};
#pragma unroll
  for (int i = 4; i < 16 * N; ++i) m4[i & 3] = fmaxf(m4[i & 3], s[i >> 4][i & 15]);
  float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
  mx = fmaxf(mx, xor32(mx, hh));
  if (__any(mx > m + slack)) {
    const float mn = fmaxf(m, mx);
    const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mn) * c);
    l *= a;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) o[mt] *= a;
    m = mn;
  }
  const float mc = m == -INFINITY ? 0.f : m * c;
  float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 16 * N; ++i) {
    const float e = __builtin_amdgcn_exp2f(fmaf(s[i >> 4][i & 15], c, -mc));
    ls[i & 3] += e;
    s[i >> 4][i & 15] = e;
  }
  l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
}

// Probabilities 8j .. 8j + 7 as the B operand of keys 16j .. 16j + 15
__device__ __forceinline__ bf16x8 p_operand(const f32x16& s, int j) {
  u32x4 u;
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = pack_bf16x2(s[8 * j + 2 * i], s[8 * j + 2 * i + 1]);
  return __builtin_bit_cast(bf16x8, u);
}

// Hides the scores of keys that the row (visible keys [lo, hi]) does not see:
// register r of a 32-key block at kb is key kb + 8 (r / 4) + 4 hh + r % 4.
__device__ __forceinline__ void hide(f32x16& s, int kb, int lo, int hi, int hh) {
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int key = kb + 8 * (r >> 2) + 4 * hh + (r & 3);
    s[r] = key >= lo && key <= hi ? s[r] : -INFINITY;
  }
}

// This lane's byte offsets of V^T operands (head dims 32mt.., keys 0..15) in a
// chunk-swizzled tile of D-wide bf16 rows: lane k of a 16-lane group names key
// 4 hh + k / 4 (+ 8 for the second read) and 4 head dims.
template <int D>
struct ValueRead {
  unsigned off0[D / 32], off1[D / 32];
  __device__ __forceinline__ explicit ValueRead(int lane) {
    const int hh = lane >> 5, k16 = lane & 15, row = 4 * hh + (k16 >> 2);
    const int dsub = 16 * ((lane >> 4) & 1) + 4 * (k16 & 3);
#pragma unroll
    for (int mt = 0; mt < D / 32; ++mt) {
      const int d = 32 * mt + dsub;
      off0[mt] = (row * D + 8 * ((d >> 3) ^ chunk_swizzle<D>(row)) + (d & 7)) * 2;
      off1[mt] = ((row + 8) * D + 8 * ((d >> 3) ^ chunk_swizzle<D>(row + 8)) + (d & 7)) * 2;
    }
  }
  // keys 16j .. 16j + 15 of the tile at `at`
  __device__ __forceinline__ bf16x8 operator()(const lds_char* at, int mt, int j) const {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + off0[mt] + j * 16 * D * 2));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + off1[mt] + j * 16 * D * 2));
    const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
    return __builtin_bit_cast(bf16x8, (u32x4){a[0], a[1], b[0], b[1]});
  }
};

// Bits of an operand's words that belong to element e of the lanes that are `on`.
__device__ __forceinline__ u32x4 one_element(int e, bool on) {
  const unsigned bits = on ? 0xFFFFu << 16 * (e & 1) : 0u;
  u32x4 x;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = i == e >> 1 ? bits : 0u;
  return x;
}

// Byte offset of a cache row / its block scales (head 0) in page `page`: strides
// below 2^32, one 32 x 32 -> 64-bit multiply each.
__device__ __forceinline__ unsigned long long row_offset(const ChunkParams& p, unsigned page, unsigned slot) {
  return (unsigned long long)page * p.stride_page + slot * p.stride_tok;
}
__device__ __forceinline__ unsigned long long scale_offset(const ChunkParams& p, unsigned page, unsigned slot) {
  return (unsigned long long)page * p.scale_stride_page + slot * p.scale_stride_tok;
}

template <int D>
__device__ __forceinline__ lds_char* lds_piece(lds_char* tile, int row, int chunk) {
  return tile + row * D * 2 + 16 * (chunk ^ chunk_swizzle<D>(row));
}

// A lane that expands N chunks of a row (part `col` of it) writes them in the
// order i ^ turn, so that 8 lanes beside each other write 8 different 16-byte
// columns of the 128 bytes that LDS takes at a time.  (In order they meet in 4 or
// 2 of them: half of the LDS cycles of quantised batches were conflicts.)
template <int D, int N>
__device__ __forceinline__ unsigned write_turn(int row, int col) {
  if constexpr (D == 64) return row & (N - 1);
  if constexpr (N == 2) return col >> 2 & 1;
  return (col >> 1 & 1) | (row & 1) << 1;
}
// chunk i of d becomes chunk i ^ turn
template <int N, int WORDS>
__device__ __forceinline__ void turn_chunks(unsigned (&d)[N * WORDS], unsigned turn) {
#pragma unroll
  for (int bit = 1; bit < N; bit *= 2) {
    const bool swap = turn & bit;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i & bit) continue;
#pragma unroll
      for (int e = 0; e < WORDS; ++e) {
        const unsigned a = d[i * WORDS + e], b = d[(i | bit) * WORDS + e];
        d[i * WORDS + e] = swap ? b : a;
        d[(i | bit) * WORDS + e] = swap ? a : b;
      }
    }
  }
}

// Output of one row's state: normalised O and LSE to the output, or a partial.
struct RowOut {
  int token, head;
  __device__ __forceinline__ RowOut(const ChunkParams& p, const ChunkItem& w, int row) {
    const int r = w.row0 + row;
    token = w.q0 + r / p.group;
    head = w.kvh * p.group + r % p.group;
  }
};

// (A row without a key has output 0 whatever its sink: -inf less -inf is no number.)
__device__ __forceinline__ float sink_factor(const ChunkParams& p, int head, float lse2) {
  if (!p.sinks || lse2 == -INFINITY) return 1.f;
  return 1.f / (1.f + __builtin_amdgcn_exp2f((p.sinks[head] - lse2 * kLn2) * kLog2e));
}

// ---- values that are not finite ----
// A hidden key has probability 0, but 0 times an infinite or NaN value is NaN: the
// second product would carry it into the rows of its tile that do not see the key.
// Where a row does not see all of a wave's keys and a sum came out not finite, the
// wave takes its keys again, and those that some row does not see one at a time, each
// for the rows that see it.  The check, one instruction an output once an item, is all
// that other items pay (24 requests with a chunk of 1000 in mxfp4 55.2 -> 55.7 us, 4 x
// 1024 tokens of 64 heads of 64 with a window 27.8 -> 28.3); items that meet one take
// about three times as long (2 x 2048 at 16384 keys, a NaN in each request's newest
// token: bf16 1.1 -> 3.3 ms).
// Tile items: a wave's 32 rows over their part of the item's chunk of keys, straight
// from the cache, values through 32 rows of its own LDS.  o, m, l: from the start.
template <int D, int FMT, bool SHARED>
__device__ __forceinline__ void tile_rows_by_key(lds_char* lds, f32x16 (&o)[D / 32], float& m, float& l) {
  constexpr int MT = D / 32, KS = D / 16;
  constexpr bool MX = Format<D, FMT>::MX;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, l32 = lane & 31, hh = lane >> 5;
  // (arguments and item are read again: nothing need be kept for here over the tile loop)
  auto at = (const __attribute__((address_space(4))) char*)__builtin_amdgcn_kernarg_segment_ptr();
  __asm__ volatile("" : "+s"(at));
  const ChunkParams& p = *(const ChunkParams*)at;
  const ChunkItem w = p.items[blockIdx.x];
  const Span all = rows_span<SHARED>(p, w, 0, w.nrows - 1, false);
  const Span own = rows_span<SHARED>(p, w, 32 * wv, min(32 * wv + 31, w.nrows - 1));
  if (own.lo == own.all_lo && own.hi == own.all_hi) return;
  const int ntiles = max(all.hi - all.lo + 63, 0) >> 6;
  const int from = max(all.lo + 64 * (int)((long long)ntiles * w.chunk / w.nchunks), own.lo);
  const int to = min(all.lo + 64 * (int)((long long)ntiles * (w.chunk + 1) / w.nchunks), own.hi);
  lds_char* vt = lds + wv * 32 * D * 2;
  const int row = min(32 * wv + l32, w.nrows - 1), pos = row_pos<SHARED>(p, w, all.pos0, row),
            hi = min(row_last<SHARED>(w, pos), to - 1);
  const RowOut qat(p, w, row);
  const bf16_t* qp = (const bf16_t*)p.q + (long long)qat.token * p.q_stride_n + (long long)qat.head * p.q_stride_h + 8 * hh;
  const int row_lo = row_first<SHARED>(p, w, pos);
  float c = p.sm_scale * kLog2e;
  if constexpr (FMT == CACHE_FP8) c *= ((const float*)p.ks.scale)[w.kvh];
  const float slack = c > 0.f ? kRescaleSlack / c : 0.f;
  const unsigned last_page = (unsigned)p.num_pages - 1u;
  const int pmask = (1 << p.log2_page) - 1;
  // 8 elements of a key's row from `d` on
  auto piece = [&](const CacheSide& s, int key, int d) -> bf16x8 {
    const unsigned page = min((unsigned)p.page_table[w.page_begin + (key >> p.log2_page)], last_page), slot = key & pmask;
    const char* row = (const char*)s.codes + w.kvh * p.stride_head + row_offset(p, page, slot);
    if constexpr (FMT == CACHE_BF16) return *(const bf16x8*)(row + 2 * d);
    float f = 1.f;
    if constexpr (MX) f = block_scale(((const uint8_t*)s.scale + w.kvh * p.scale_stride_head)[scale_offset(p, page, slot) + d / 32]);
    if constexpr (FMT == CACHE_MXFP4) return expand<FMT>(*(const unsigned*)(row + d / 2), 0u, f);
    const u32x2 x = *(const u32x2*)(row + (FMT == CACHE_MXFP4 ? 0 : d));
    return expand<FMT>(x[0], x[1], f);
  };
  const ValueRead<D> vread(lane);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) o[mt] = f32x16{};
  m = -INFINITY, l = 0.f;
  for (int kb = from; kb < to; kb += 32) {
    f32x16 s[1];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      s[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(piece(p.ks, min(kb + l32, to - 1), 16 * ks + 8 * hh), *(const bf16x8*)(qp + 16 * ks),
                                                     ks ? s[0] : f32x16{}, 0, 0, 0);
    hide(s[0], kb, row_lo, hi, hh);
    softmax_step<1, MT>(s, o, m, l, c, slack, hh);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 1
    for (int i = lane; i < 32 * (D / 8); i += 64)
      *(__attribute__((address_space(3))) bf16x8*)lds_piece<D>(vt, i / (D / 8), i % (D / 8)) =
          piece(p.vs, min(kb + i / (D / 8), to - 1), 8 * (i % (D / 8)));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (kb >= own.all_lo && kb + 32 <= min(own.all_hi, to)) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          o[mt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vread(vt, mt, j), p_operand(s[0], j), o[mt], 0, 0, 0);
      continue;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const u32x4 pb = __builtin_bit_cast(u32x4, p_operand(s[0], j));
#pragma unroll 1
      for (int k = 0; k < 16; ++k) {
        const u32x4 keep = one_element(4 * (k >> 3) + (k & 3), hh == (k >> 2 & 1));
        const int key = kb + 16 * j + k;
        const bool sees = key >= row_lo && key <= hi;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const f32x16 x = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, vread(vt, mt, j)) & keep),
              __builtin_bit_cast(bf16x8, pb & keep), f32x16{}, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < 16; ++i) o[mt][i] = sees ? o[mt][i] + x[i] : o[mt][i];
        }
      }
    }
  }
}

// ---- tile items ----
template <int D, int FMT, int W, bool SHARED>
__device__ __forceinline__ void tile_item(const ChunkParams& p, const ChunkItem& w, lds_char* lds) {
  constexpr int MT = D / 32, KS = D / 16, ROW = Format<D, FMT>::ROW, TB = 64 * D * 2;
  constexpr bool MX = Format<D, FMT>::MX;
  const int tid = threadIdx.x, wv = tid >> 6, lane = tid & 63, l32 = lane & 31, hh = lane >> 5;

  const Span all = rows_span<SHARED>(p, w, 0, w.nrows - 1, false);
  // tiles of 64 keys from the first visible one on
  const int ntiles = max(all.hi - all.lo + 63, 0) >> 6;
  const int tb = (int)((long long)ntiles * w.chunk / w.nchunks);
  const int te = (int)((long long)ntiles * (w.chunk + 1) / w.nchunks);

  // this wave's rows
  const int wrow = 32 * wv, row = min(wrow + l32, w.nrows - 1);
  const bool wave_on = wrow < w.nrows;
  const int pos = row_pos<SHARED>(p, w, all.pos0, row);
  const int row_lo = row_first<SHARED>(p, w, pos), row_hi = row_last<SHARED>(w, pos);
  const Span own = rows_span<SHARED>(p, w, min(wrow, w.nrows - 1), min(wrow + 31, w.nrows - 1));
  const RowOut at(p, w, row);
  bf16x8 qf[KS];
  {
    const bf16_t* qp = (const bf16_t*)p.q + (long long)at.token * p.q_stride_n + (long long)at.head * p.q_stride_h + 8 * hh;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *(const bf16x8*)(qp + 16 * ks);
  }
  float c = p.sm_scale * kLog2e, vscale = 1.f;
  if constexpr (FMT == CACHE_FP8) {
    c *= ((const float*)p.ks.scale)[w.kvh];
    vscale = ((const float*)p.vs.scale)[w.kvh];
  }
  const float slack = c > 0.f ? kRescaleSlack / c : 0.f;

  // staging of a tile's keys (then values) into chunk-swizzled bf16 rows
  // (a page id is clamped where it is used: clamped where it is loaded, the
  // wait for it would be a wait for all the tile's loads before it)
  auto page_of = [&](int key) -> unsigned { return (unsigned)p.page_table[w.page_begin + (key >> p.log2_page)]; };
  const unsigned last_page = (unsigned)p.num_pages - 1u;
  auto key_of = [&](int tile, int row_) -> int { return min(all.lo + 64 * tile + row_, all.hi - 1); };
  const int pmask = (1 << p.log2_page) - 1;
  // bf16: a wave copies 64 / W rows straight into LDS, 1 KB (1024 / ROW rows) at a time
  constexpr int RPC = 1024 / (2 * D), NC = 64 / W / RPC;  // rows per copy, copies per wave
  const int crow = wv * (64 / W) + lane / (D / 8);  // of copy 0
  const char* kcopy = (const char*)p.ks.codes + w.kvh * p.stride_head;
  const char* vcopy = (const char*)p.vs.codes + w.kvh * p.stride_head;
  unsigned pages[NC];
  auto pages_of = [&](int tile) {
#pragma unroll
    for (int i = 0; i < NC; ++i) pages[i] = page_of(key_of(tile, crow + RPC * i));
  };
  const unsigned lds0 = lds_address((const void*)lds);
  auto copy = [&](int tile, unsigned at) {  // pages: of this tile
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int r = crow + RPC * i;
      const unsigned long long off = row_offset(p, min(pages[i], last_page), key_of(tile, r) & pmask) +
                                     16 * ((lane % (D / 8)) ^ chunk_swizzle<D>(r));
      const unsigned dst = at + (wv * (64 / W) + RPC * i) * D * 2;
      dma16_kept(kcopy + off, dst);
      dma16_kept(vcopy + off, dst + TB);
    }
  };
  // quantised: thread tid carries 1 / TPR of row tid / TPR through registers
  constexpr int TPR = W, EPT = D / TPR, WORDS = FMT == CACHE_BF16 ? 1 : ROW / TPR / 4;
  const int srow = tid / TPR, spart = tid % TPR;
  const char* kpart = kcopy + spart * (ROW / TPR);
  const char* vpart = vcopy + spart * (ROW / TPR);
  const long long shead = w.kvh * p.scale_stride_head + spart * EPT / 32;
  unsigned kw[WORDS], vw[WORDS];
  unsigned ksc = 0, vsc = 0;
  auto load_words = [](unsigned (&d)[WORDS], const char* s) {
    if constexpr (WORDS >= 4) {
#pragma unroll
      for (int i = 0; i < WORDS / 4; ++i) {
        const u32x4 u = *(const u32x4*)(s + 16 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) d[4 * i + e] = u[e];
      }
    } else if constexpr (WORDS == 2) {
      const u32x2 u = *(const u32x2*)s;
      d[0] = u[0], d[1] = u[1];
    } else {
      d[0] = *(const unsigned*)s;
    }
  };
  auto fetch = [&](int tile, unsigned page) {
    const unsigned pg = min(page, last_page), slot = key_of(tile, srow) & pmask;
    const unsigned long long off = row_offset(p, pg, slot);
    load_words(kw, kpart + off);
    load_words(vw, vpart + off);
    if constexpr (MX) {
      const unsigned long long so = scale_offset(p, pg, slot) + shead;
      ksc = ((const uint8_t*)p.ks.scale)[so];
      vsc = ((const uint8_t*)p.vs.scale)[so];
    }
  };
  constexpr int PN = EPT / 8, PW = FMT == CACHE_MXFP4 ? 1 : 2;  // chunks of a part, words of a chunk
  const unsigned turn = write_turn<D, PN>(srow, spart), pswz = chunk_swizzle<D>(srow) ^ turn;
  // chunk i of the keys' part (the values' from PN on) to the tile (K, then V) at
  // `tile`, in turn from 0 on
  auto put = [&](lds_char* tile, int i) {
    if constexpr (FMT != CACHE_BF16) {
      const bool is_v = i >= PN;
      const int ch = i % PN;
      unsigned(&x)[PN * PW] = is_v ? vw : kw;
      if (ch == 0) turn_chunks<PN, PW>(x, turn);
      const float f = MX ? block_scale(is_v ? vsc : ksc) : 1.f;
      *(__attribute__((address_space(3))) bf16x8*)(tile + (is_v ? TB : 0) + srow * D * 2 + 16 * ((spart * PN + ch) ^ pswz)) =
          expand<FMT>(x[PW * ch], x[PW * ch + PW - 1], f);
    }
  };
  auto put_all = [&](lds_char* tile) {
    if constexpr (FMT != CACHE_BF16) {
#pragma unroll
      for (int i = 0; i < 2 * PN; ++i) put(tile, i);
    }
  };

  f32x16 o[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) o[mt] = f32x16{};
  float m = -INFINITY, l = 0.f;
  unsigned koff[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) koff[ks] = (l32 * D + 8 * ((2 * ks + hh) ^ chunk_swizzle<D>(l32))) * 2;
  const ValueRead<D> vread(lane);

  // Two buffers of (K, V).  bf16: tile t + 1 is on its way while tile t is
  // worked on.  Quantised: tile t + 2 is, and t + 1 is expanded into LDS, beside
  // the score products (24 requests with a chunk of 1000 in mxfp4 60 -> 55 us;
  // but not where registers would spill: mxfp8 heads of 64, 1300 -> 1320).
  constexpr bool BESIDE = FMT != CACHE_BF16 && !(D == 64 && FMT == CACHE_MXFP8);
  unsigned page = 0;
  if (tb < te) {
    if constexpr (FMT == CACHE_BF16) {
      pages_of(tb);
      copy(tb, lds0);
      pages_of(min(tb + 1, te - 1));
      wait_vmcnt<0>();
    } else {
      fetch(tb, page_of(key_of(tb, srow)));
      put_all(lds);
      if (tb + 1 < te) {
        fetch(tb + 1, page_of(key_of(tb + 1, srow)));
        page = page_of(key_of(min(tb + 2, te - 1), srow));
      }
    }
    __syncthreads();
  }
  for (int t = tb; t < te; ++t) {
    const int cur = ((t - tb) & 1) * 2 * TB, nxt = 2 * TB - cur;
    lds_char* kt = lds + cur;
    lds_char* vt = kt + TB;
    if constexpr (FMT == CACHE_BF16) {
      if (t + 1 < te) {
        copy(t + 1, lds0 + nxt);
        pages_of(min(t + 2, te - 1));
      }
    }
    const int kb = all.lo + 64 * t;
    // which 32-key halves some row of the wave sees
    const bool on0 = wave_on && kb < own.hi && kb + 32 > own.lo, on1 = wave_on && kb + 32 < own.hi && kb + 64 > own.lo;
    const bool on = on0 && on1;
    f32x16 s[2];
    if (on) {
      // operands are read AHEAD steps before their product
      constexpr int AHEAD = 3;
      bf16x8 kf[KS][2];
      auto kread = [&](int ks) {
        kf[ks][0] = *(const __attribute__((address_space(3))) bf16x8*)(kt + koff[ks]);
        kf[ks][1] = *(const __attribute__((address_space(3))) bf16x8*)(kt + koff[ks] + 32 * D * 2);
      };
#pragma unroll
      for (int ks = 0; ks < AHEAD; ++ks) kread(ks);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if (ks + AHEAD < KS) kread(ks + AHEAD);
        s[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[ks][0], qf[ks], ks ? s[0] : f32x16{}, 0, 0, 0);
        s[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[ks][1], qf[ks], ks ? s[1] : f32x16{}, 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (BESIDE) {
          // tile t + 1 into LDS (behind the last tile nobody reads it)
#pragma unroll
          for (int i = 0; i < 2 * PN; ++i)
            if (i * KS / (2 * PN) == ks) put(lds + nxt, i);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    if (!BESIDE || !on) put_all(lds + nxt);
    if constexpr (FMT != CACHE_BF16) {
      if (t + 2 < te) {
        fetch(t + 2, page);
        page = page_of(key_of(min(t + 3, te - 1), srow));
      }
    }
    if (on) {
      if (kb < own.all_lo || kb + 64 > own.all_hi) {
        hide(s[0], kb, row_lo, row_hi, hh);
        hide(s[1], kb + 32, row_lo, row_hi, hh);
      }
      softmax_step<2, MT>(s, o, m, l, c, slack, hh);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bf16x8 pb = p_operand(s[j >> 1], j & 1);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          o[mt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vread(vt, mt, j), pb, o[mt], 0, 0, 0);
      }
    } else if (on0 || on1) {
      const int half = on1 ? 32 : 0;
      f32x16 s1[1];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const bf16x8 kf = *(const __attribute__((address_space(3))) bf16x8*)(kt + half * D * 2 + koff[ks]);
        s1[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[ks], ks ? s1[0] : f32x16{}, 0, 0, 0);
      }
      hide(s1[0], kb + half, row_lo, row_hi, hh);
      softmax_step<1, MT>(s1, o, m, l, c, slack, hh);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const bf16x8 pb = p_operand(s1[0], j);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          o[mt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vread(vt + half * D * 2, mt, j), pb, o[mt], 0, 0, 0);
      }
    }
    if constexpr (FMT == CACHE_BF16) wait_vmcnt<0>();  // this wave's copies of the next tile have landed
    __syncthreads();
  }

  if (!wave_on) return;
  float zero = 0.f;  // (NaN once a sum is not finite)
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int i = 0; i < 16; ++i) zero = fmaf(o[mt][i], 0.f, zero);
  // (no wave reads the tiles any more: the last step's barrier)
  if (__any(zero != 0.f)) tile_rows_by_key<D, FMT, SHARED>(lds, o, m, l);
  l += xor32(l, hh);
  const float lse2 = l > 0.f ? m * c + __builtin_amdgcn_logf(l) : l == 0.f ? -INFINITY : l;
  float inv = l != 0.f ? vscale / l : 0.f;
  const bool mine = wrow + l32 < w.nrows;
  if constexpr (SHARED) {
    if (w.part == PART_SHARED) {
      store_image<D>(p, w, o, inv, lse2, wrow, l32, hh);
      return;
    }
  }
  if (is_partial<SHARED>(w)) {
    if (!mine) return;
    const long long pr = w.slot + (long long)w.chunk * w.nrows + row;
    float* po = p.part_o + pr * D + 4 * hh;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *(f32x4*)(po + 32 * mt + 8 * q) = (f32x4){o[mt][4 * q] * inv, o[mt][4 * q + 1] * inv, o[mt][4 * q + 2] * inv,
                                                 o[mt][4 * q + 3] * inv};
    if (hh == 0) p.part_lse[pr] = lse2;
    return;
  }
  inv *= sink_factor(p, at.head, lse2);
  if (!mine) return;
  bf16_t* op = (bf16_t*)p.o + (long long)at.token * p.o_stride_n + (long long)at.head * p.o_stride_h;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    float acc[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = o[mt][i];
    store_row_block32(op + 32 * mt, acc, inv, hh);
  }
  if (hh == 0) p.lse[at.token * p.lse_stride_n + at.head] = p.lse_base2 ? lse2 : lse2 * kLn2;
}

// ---- token items ----
// RB row blocks of 16 packed rows, shared by all waves; v_mfma_f32_16x16x32_bf16:
// lane l holds row l % 16 of a block, and of a 16-key block the scores of keys
// 4 (l / 16) .. + 3.  PF tiles of 32 keys are in flight per wave.
template <bool STREAM, typename T>
__device__ __forceinline__ T load_kv(const T* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load(p);
  return *p;
}

// SOLO (plans with shared keys): each wave of the workgroup has rows or keys of its
// own, w is the wave's, and its state goes out as it is.
template <int D, int FMT, int W, int RB, int PF, bool STREAM, bool SHARED, bool SOLO = false>
__device__ __forceinline__ void token_item(const ChunkParams& p, const ChunkItem& w, lds_char* lds, float* stats) {
  constexpr int TW = SOLO ? 1 : W;  // waves that share the item's tiles
  constexpr int MT = D / 16, KS = D / 32, ROW = Format<D, FMT>::ROW;
  constexpr bool MX = Format<D, FMT>::MX;
  constexpr int NK = ROW / 64;                  // 16-byte pieces of a lane's quarter of a key row
  constexpr int KW = NK > 0 ? 4 : ROW / 16;     // words of a piece (half pieces where a quarter row is 8 bytes)
  constexpr int NKP = NK > 0 ? NK : 1;
  // Which pieces of a key row are a lane's: the four lanes of a row take
  // neighbouring ones, so that a load reads whole 64-byte runs; with block scales
  // a quarter of the row each, which one block covers at D = 128.
  constexpr bool SPREAD = !MX && NK > 1;
  constexpr int PE = 16 * D / ROW;              // elements of a piece
  constexpr int PPR = ROW / 16;                 // 16-byte pieces of a row
  constexpr int NV = PPR / 2;                   // value pieces per lane and tile
  constexpr int VB = 32 * D * 2;                // bytes of a wave's value tile
  const int tid = threadIdx.x, wv = tid >> 6, lane = tid & 63, l16 = lane & 15, g4 = lane >> 4;

  Span all = rows_span<SHARED>(p, w, 0, w.nrows - 1, false);
  const int tile0 = all.lo >> 5, ntiles_all = all.hi > all.lo ? ((all.hi + 31) >> 5) - tile0 : 0;
  const int tb = tile0 + (int)((long long)ntiles_all * w.chunk / w.nchunks);
  const int te = tile0 + (int)((long long)ntiles_all * (w.chunk + 1) / w.nchunks);

  int pos[RB], row_lo[RB];  // last and first key of a row
  int least = 0x7FFFFFFF;   // lowest position of the lane's rows
  bf16x8 qf[RB][KS];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int row = min(16 * rb + l16, w.nrows - 1);
    const RowOut at(p, w, row);
    pos[rb] = row_pos<SHARED>(p, w, all.pos0, row);
    row_lo[rb] = row_first<SHARED>(p, w, pos[rb]);
    if constexpr (SHARED) least = min(least, pos[rb]);
    pos[rb] = row_last<SHARED>(w, pos[rb]);
    const bf16_t* qp = (const bf16_t*)p.q + (long long)at.token * p.q_stride_n + (long long)at.head * p.q_stride_h;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      qf[rb][ks] = *(const bf16x8*)(qp + (SPREAD ? PE * (g4 + 4 * (8 * ks / PE)) + 8 * ks % PE : g4 * (D / 4) + 8 * ks));
  }
  float c = p.sm_scale * kLog2e, vscale = 1.f;
  if constexpr (FMT == CACHE_FP8) {
    c *= ((const float*)p.ks.scale)[w.kvh];
    vscale = ((const float*)p.vs.scale)[w.kvh];
  }
  const float slack = c > 0.f ? kRescaleSlack / c : 0.f;

  // keys go straight to the operand, values through the wave's LDS
  const char* kbase = (const char*)p.ks.codes + w.kvh * p.stride_head;
  const char* vbase = (const char*)p.vs.codes + w.kvh * p.stride_head;
  const uint8_t* ksbase = (const uint8_t*)p.ks.scale + w.kvh * p.scale_stride_head;
  const uint8_t* vsbase = (const uint8_t*)p.vs.scale + w.kvh * p.scale_stride_head;
  constexpr int PSTEP = SPREAD ? 64 : 16;  // bytes between a lane's pieces
  const unsigned kcol = SPREAD ? 16 * g4 : g4 * (ROW / 4), vcol = 16 * (lane % PPR), kscol = g4 * (D / 4) / 32;
  const unsigned vscol = FMT == CACHE_MXFP4 ? lane % PPR : lane % PPR / 2;
  const int pmask = (1 << p.log2_page) - 1;
  const unsigned last_page = (unsigned)p.num_pages - 1u;  // (clamped where used, as above)
  auto key_at = [&](int tile, int i) -> int { return min(max(32 * tile + i, all.lo), all.hi - 1); };
  auto page_at = [&](int key) -> unsigned { return (unsigned)p.page_table[w.page_begin + (key >> p.log2_page)]; };
  struct Raw {
    unsigned k[2][NKP][KW];
    u32x4 v[NV];
    unsigned ksc[2], vsc[NV];
    unsigned next;  // page of this lane's key (l % 32) of the tile after the next one to take these registers
  } raw[PF];
  // Where the rows of every load share a page and none is clamped, the page and
  // the address stay in scalar registers and a lane adds a constant (32 requests
  // of 8..32k tokens: bf16 475 -> 460 us, mxfp4 160 -> 156).
  constexpr int VR = 64 / PPR;  // rows of one load of values
  const bool shared_pages = (1 << p.log2_page) >= (VR > 16 ? VR : 16);
  const unsigned klane = l16 * p.stride_tok + kcol, vlane = lane / PPR * p.stride_tok + vcol;
  const unsigned kslane = l16 * p.scale_stride_tok + kscol, vslane = lane / PPR * p.scale_stride_tok + vscol;
  auto load_k = [&](unsigned (&d)[NKP][KW], const char* base, unsigned off) {
#pragma unroll
    for (int i = 0; i < NKP; ++i) {
      if constexpr (KW == 4) {
        const u32x4 u = load_kv<STREAM>((const u32x4*)(base + off + PSTEP * i));
#pragma unroll
        for (int e = 0; e < 4; ++e) d[i][e] = u[e];
      } else {
        const u32x2 u = load_kv<STREAM>((const u32x2*)(base + off));
        d[i][0] = u[0], d[i][1] = u[1];
      }
    }
  };
  // page: lane l's is the page of key l % 32 of the tile
  auto fetch = [&](Raw& x, int tile, unsigned page) {
    if (shared_pages && 32 * tile >= all.lo && 32 * tile + 32 <= all.hi) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const unsigned pg = __builtin_amdgcn_readlane(page, 16 * b), slot = (32 * tile + 16 * b) & pmask;
        load_k(x.k[b], kbase + row_offset(p, pg, slot), klane);
        if constexpr (MX) x.ksc[b] = (ksbase + scale_offset(p, pg, slot))[kslane];
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const unsigned pg = __builtin_amdgcn_readlane(page, VR * i), slot = (32 * tile + VR * i) & pmask;
        x.v[i] = load_kv<STREAM>((const u32x4*)(vbase + row_offset(p, pg, slot) + vlane));
        if constexpr (MX) x.vsc[i] = (vsbase + scale_offset(p, pg, slot))[vslane];
      }
      return;
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const unsigned pg = __shfl(page, 16 * b + l16), slot = key_at(tile, 16 * b + l16) & pmask;
      load_k(x.k[b], kbase + row_offset(p, pg, slot), kcol);
      if constexpr (MX) x.ksc[b] = (ksbase + scale_offset(p, pg, slot))[kscol];
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int kk = (64 * i + lane) / PPR;
      const unsigned pg = __shfl(page, kk), slot = key_at(tile, kk) & pmask;
      x.v[i] = load_kv<STREAM>((const u32x4*)(vbase + row_offset(p, pg, slot) + vcol));
      if constexpr (MX) x.vsc[i] = (vsbase + scale_offset(p, pg, slot))[vscol];
    }
  };

  f32x4 o[RB][MT];
  float m[RB], l[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) o[rb][mt] = f32x4{};
    m[rb] = -INFINITY, l[rb] = 0.f;
  }
  lds_char* vt = lds + wv * VB;
  // V^T operands: 16-lane group g reads keys 4g .. 4g + 3 (+ 16 for the second
  // half) of 16 head dims, the keys its lanes hold probabilities of
  auto vread = [&](int mt) -> bf16x8 {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const int r = 4 * g4 + (l16 >> 2), ch = 2 * mt + ((l16 & 3) >> 1), in = 8 * (l16 & 1);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds_piece<D>(vt, r, ch) + in));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds_piece<D>(vt, r + 16, ch) + in));
    const u32x2 x = __builtin_bit_cast(u32x2, lo), y = __builtin_bit_cast(u32x2, hi);
    return __builtin_bit_cast(bf16x8, (u32x4){x[0], x[1], y[0], y[1]});
  };
  // maximum / sum over the four lanes of a row
  auto over_row = [&](float x, auto&& f) -> float {
    x = f(x, __shfl_xor(x, 16));
    return f(x, __shfl_xor(x, 32));
  };

  auto step = [&](Raw& x, int t, auto by_key) {
    constexpr bool BY_KEY = decltype(by_key)::value;
    const int tn = t + PF * TW;  // the tile that takes these registers next
    // (page ids are loaded a round before the rows they lead to: the wait for
    // one is a wait for every load before it)
    unsigned pg = 0;
    if constexpr (!BY_KEY) {
      pg = min(x.next, last_page);
      x.next = page_at(key_at(tn + PF * TW, lane & 31));
    }
    f32x4 s[RB][2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        bf16x8 a;
        if constexpr (FMT == CACHE_BF16) {
          a = __builtin_bit_cast(bf16x8, (u32x4){x.k[b][ks][0], x.k[b][ks][1], x.k[b][ks][2], x.k[b][ks][3]});
        } else {
          const float f = MX ? block_scale(x.ksc[b]) : 1.f;
          constexpr int PER = FMT == CACHE_MXFP4 ? 1 : 2;  // words of 8 codes
          const int w0 = PER * ks;
          a = expand<FMT>(x.k[b][w0 / KW][w0 % KW], x.k[b][(w0 + PER - 1) / KW][(w0 + PER - 1) % KW], f);
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
          s[rb][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qf[rb][ks], ks ? s[rb][b] : f32x4{}, 0, 0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int kk = (64 * i + lane) / PPR, col = lane % PPR;
      if constexpr (FMT == CACHE_BF16) {
        *(__attribute__((address_space(3))) u32x4*)lds_piece<D>(vt, kk, col) = x.v[i];
      } else {
        constexpr int CH = FMT == CACHE_MXFP4 ? 4 : 2, CW = 4 / CH;  // 8-element chunks of a piece, words of a chunk
        const float f = MX ? block_scale(x.vsc[i]) : 1.f;
        const unsigned turn = write_turn<D, CH>(kk, col);
        unsigned c[4] = {x.v[i][0], x.v[i][1], x.v[i][2], x.v[i][3]};
        turn_chunks<CH, CW>(c, turn);
#pragma unroll
        for (int e = 0; e < CH; ++e)
          *(__attribute__((address_space(3))) bf16x8*)(vt + kk * D * 2 +
                                                       16 * ((CH * col + e) ^ chunk_swizzle<D>(kk) ^ turn)) =
              expand<FMT>(c[CW * e], c[CW * e + CW - 1], f);
      }
    }
    if (!BY_KEY && tn < te) {
      fetch(x, tn, pg);
    }
    const int kb = 32 * t;
    const bool edge = kb < all.all_lo || kb + 32 > all.all_hi;
    bf16x8 pb[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      if (edge) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int key = kb + 16 * (i >> 2) + 4 * g4 + (i & 3);
          s[rb][i >> 2][i & 3] = key >= row_lo[rb] && key <= pos[rb] ? s[rb][i >> 2][i & 3] : -INFINITY;
        }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = fmaxf(mx, s[rb][i >> 2][i & 3]);
      mx = over_row(mx, [](float u, float v) { return fmaxf(u, v); });
      if (__any(mx > m[rb] + slack)) {
        const float mn = fmaxf(m[rb], mx);
        const float a = m[rb] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m[rb] - mn) * c);
        l[rb] *= a;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) o[rb][mt] *= a;
        m[rb] = mn;
      }
      const float mc = m[rb] == -INFINITY ? 0.f : m[rb] * c;
      u32x4 u;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e0 = __builtin_amdgcn_exp2f(fmaf(s[rb][i >> 1][2 * (i & 1)], c, -mc));
        const float e1 = __builtin_amdgcn_exp2f(fmaf(s[rb][i >> 1][2 * (i & 1) + 1], c, -mc));
        l[rb] += e0 + e1;
        u[i] = pack_bf16x2(e0, e1);
      }
      pb[rb] = __builtin_bit_cast(bf16x8, u);
    }
    // (LDS serves a wave's accesses in order; the fences keep the compiler's order)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (BY_KEY && edge) {
#pragma unroll 1
      for (int k = 0; k < 32; ++k) {
        const u32x4 keep = one_element(4 * (k >> 4) + (k & 3), g4 == (k >> 2 & 3));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const u32x4 a = __builtin_bit_cast(u32x4, vread(mt)) & keep;
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) {
            const f32x4 y = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                __builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, pb[rb]) & keep), f32x4{}, 0,
                0, 0);
            const bool sees = kb + k >= row_lo[rb] && kb + k <= pos[rb];
#pragma unroll
            for (int i = 0; i < 4; ++i) o[rb][mt][i] = sees ? o[rb][mt][i] + y[i] : o[rb][mt][i];
          }
        }
      }
    } else {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const bf16x8 a = vread(mt);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
          o[rb][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pb[rb], o[rb][mt], 0, 0, 0);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  };

  const int t0 = tb + (SOLO ? 0 : __builtin_amdgcn_readfirstlane(wv));
  unsigned pages[PF];
#pragma unroll
  for (int i = 0; i < PF; ++i) {
    // (keys past the range are clamped to its last one; an item without keys loads nothing)
    if (te > tb) {
      raw[i].next = page_at(key_at(t0 + (PF + i) * TW, lane & 31));
      pages[i] = page_at(key_at(t0 + i * TW, lane & 31));
    }
  }
#pragma unroll
  for (int i = 0; i < PF; ++i) {
    const int t = t0 + i * TW;
    if (t < te) {
      const unsigned pg = min(pages[i], last_page);
      fetch(raw[i], t, pg);
    }
  }
  if constexpr (SHARED)  // (not before the first keys are on their way)
    if (w.part == PART_SHARED && p.window_left < 0) all.all_lo = 0, all.all_hi = min(w.bound, wave_min(least) + 1);
  for (int t = t0; t < te; t += PF * TW) {
#pragma unroll
    for (int i = 0; i < PF; ++i)
      if (t + i * TW < te) step(raw[i], t + i * TW, std::false_type{});
  }
  if (all.lo < all.all_lo || all.hi > all.all_hi) {
    float zero = 0.f;  // (NaN once a sum is not finite)
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) zero = fmaf(o[rb][mt][i], 0.f, zero);
    if (__any(zero != 0.f)) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) o[rb][mt] = f32x4{};
        m[rb] = -INFINITY, l[rb] = 0.f;
      }
#pragma unroll 1
      for (int t = t0; t < te; t += TW) {
        const unsigned pg = min(page_at(key_at(t, lane & 31)), last_page);
        fetch(raw[0], t, pg);
        step(raw[0], t, std::true_type{});
      }
    }
  }

  if constexpr (SOLO) {
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int row = 16 * rb + l16;
      const float sum = over_row(l[rb], [](float u, float v) { return u + v; });
      const float lse2 = sum > 0.f ? m[rb] * c + __builtin_amdgcn_logf(sum) : sum == 0.f ? -INFINITY : sum;
      float inv = sum != 0.f ? vscale / sum : 0.f;
      if (row >= w.nrows) continue;
      if (is_partial<SHARED>(w)) {
        const long long pr = w.slot + (long long)w.chunk * w.nrows + row;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) *(f32x4*)(p.part_o + pr * D + 16 * mt + 4 * g4) = o[rb][mt] * inv;
        if (g4 == 0) p.part_lse[pr] = lse2;
      } else {
        const RowOut at(p, w, row);
        inv *= sink_factor(p, at.head, lse2);
        bf16_t* op = (bf16_t*)p.o + (long long)at.token * p.o_stride_n + (long long)at.head * p.o_stride_h + 4 * g4;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          *(u32x2*)(op + 16 * mt) = (u32x2){pack_bf16x2(o[rb][mt][0] * inv, o[rb][mt][1] * inv),
                                            pack_bf16x2(o[rb][mt][2] * inv, o[rb][mt][3] * inv)};
        if (g4 == 0) p.lse[at.token * p.lse_stride_n + at.head] = p.lse_base2 ? lse2 : lse2 * kLn2;
      }
    }
    return;
  }

  // join the waves' states through LDS
  float* ms = stats;
  float* lw = stats + W * kTokenRows;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const float ls = over_row(l[rb], [](float u, float v) { return u + v; });
    if (g4 == 0) {
      ms[wv * kTokenRows + 16 * rb + l16] = m[rb];
      lw[wv * kTokenRows + 16 * rb + l16] = ls;
    }
  }
  const int nr = w.nrows;
  typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
  // in RB rounds, each of D / RB head dims: W states of 16 RB rows fit the waves' value tiles
  static_assert(16 * D * 4 <= VB, "the waves' states fit");
  constexpr int MR = MT / RB;
#pragma unroll
  for (int rd = 0; rd < RB; ++rd) {
    __syncthreads();  // the value tiles, or the last round's states, have been read
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
      if (16 * rb + l16 < nr)
#pragma unroll
        for (int mt = 0; mt < MR; ++mt)
          ((lds_f32x4*)lds)[(wv * 4 * MR + 4 * mt + g4) * nr + 16 * rb + l16] = o[rb][rd * MR + mt];
    __syncthreads();
    for (int i = tid; i < nr * 4 * MR; i += 64 * W) {
      const int r = i % nr, d4 = i / nr, dd = 16 * rd * MR + 4 * d4;
      float top = -INFINITY;
#pragma unroll
      for (int v = 0; v < W; ++v) top = fmaxf(top, ms[v * kTokenRows + r]);
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
      float sum = 0.f;
#pragma unroll
      for (int v = 0; v < W; ++v) {
        const float mv = ms[v * kTokenRows + r];
        const float a = mv == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mv - top) * c);
        sum += a * lw[v * kTokenRows + r];
        acc += a * ((lds_f32x4*)lds)[(v * 4 * MR + d4) * nr + r];
      }
      const float lse2 = sum > 0.f ? top * c + __builtin_amdgcn_logf(sum) : sum == 0.f ? -INFINITY : sum;
      float inv = sum != 0.f ? vscale / sum : 0.f;
      if (is_partial<SHARED>(w)) {
        const long long pr = w.slot + (long long)w.chunk * nr + r;
        *(f32x4*)(p.part_o + pr * D + dd) = acc * inv;
        if (dd == 0) p.part_lse[pr] = lse2;
      } else {
        const RowOut at(p, w, r);
        inv *= sink_factor(p, at.head, lse2);
        *(u32x2*)((bf16_t*)p.o + (long long)at.token * p.o_stride_n + (long long)at.head * p.o_stride_h + dd) =
            (u32x2){pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv)};
        if (dd == 0) p.lse[at.token * p.lse_stride_n + at.head] = p.lse_base2 ? lse2 : lse2 * kLn2;
      }
    }
  }
}

#ifdef D2SD_CHUNK_SHARED
#include "shared_tile.h"
#endif

// Tiles of 32 keys a wave of a token item has in flight (more than one does
// not help bf16, whose tiles are 16 KB)
template <int FMT>
constexpr int token_depth() {
  return FMT == CACHE_BF16 ? 1 : 2;
}

// Waves per SIMD: what the registers allow without spilling.
template <int D, int FMT, int FORM>
constexpr int chunk_occupancy() {
  return FORM >= CHUNK_TOKENS ? (FMT == CACHE_MXFP4 ? 3 : 2) : D == 64 ? 3 : 2;
}

template <int D, int FMT, int FORM, bool SHARED>
__device__ __forceinline__ void chunk_work(const ChunkParams& p) {
  constexpr int W = chunk_waves(FORM);
  constexpr bool TOKENS = FORM >= CHUNK_TOKENS;
  constexpr int VALUES = W * 32 * D * 2, STATS = 2 * W * kTokenRows * 4;  // of token items
#ifdef D2SD_CHUNK_SHARED
  constexpr int TILES = SharedRing<D, FMT, W>::bytes;
#else
  constexpr int TILES = 4 * 64 * D * 2;
#endif
  __shared__ __align__(16) char lds[TOKENS || VALUES + STATS > TILES ? VALUES + STATS : TILES];
  float* const stats = (float*)(lds + VALUES);
  const ChunkItem w = p.items[blockIdx.x];
  if constexpr (TOKENS) {
    token_item<D, FMT, W, 1, token_depth<FMT>(), FORM == CHUNK_STREAM, SHARED>(p, w, (lds_char*)lds, stats);
  } else {
    if (w.kind == CHUNK_TILE) {
#ifdef D2SD_CHUNK_SHARED
      if (w.part == PART_SHARED) {
        auto chunk_of = [&](int lo, int hi, int& from, int& to) {
          const int ntiles = max(hi - lo + 63, 0) >> 6;
          from = lo + 64 * (int)((long long)ntiles * w.chunk / w.nchunks);
          to = min(lo + 64 * (int)((long long)ntiles * (w.chunk + 1) / w.nchunks), hi);
        };
        int from, to;
        if (p.window_left < 0 && w.heads > 0 && shared_tile_takes<D, FMT, W>(p, 0)) {
          // The usual case, taken for granted: every row sees all of the chunk's keys.  The
          // lengths are looked at last, so that the first keys do not wait for them: no
          // request of the rows' ends before any row's distance to an end, or else (new
          // prompts of other lengths in one row tile, an idle request) row by row.  (64
          // prompts of 1 to 60 tokens behind 8192 bf16 keys: 264 us; looked at by the
          // first measure alone, half of the tiles came twice, 408.)
          const int lane = threadIdx.x & 63;
          const int len = lane < w.heads ? p.kv_len[w.nq + lane] : 0x7FFFFFFF;
          chunk_of(0, w.bound, from, to);
          if (from < to) {
            shared_tile<D, FMT, W>(p, w, (lds_char*)lds, from, to);
            if (!__any(len < to + w.back - 1)) return;
            if (to <= seen_by_all_rows()) return;
            __syncthreads();  // (the tiles: all waves are done with them)
          }
        } else {
          const Span all = rows_span<true>(p, w, 0, w.nrows - 1);
          chunk_of(all.lo, all.hi, from, to);
          if (from < to && from >= all.all_lo && to <= all.all_hi && shared_tile_takes<D, FMT, W>(p, from)) {
            shared_tile<D, FMT, W>(p, w, (lds_char*)lds, from, to);
            return;
          }
        }
      }
#endif
      tile_item<D, FMT, W, SHARED>(p, w, (lds_char*)lds);
      return;
    }
    if constexpr (SHARED) {
      // wave wv takes unit kvh + wv of the request's chunks x heads
      ChunkItem u = w;
      const int unit = __builtin_amdgcn_readfirstlane(w.kvh + (threadIdx.x >> 6));
      if (unit >= w.heads * w.nchunks) return;
      u.chunk = unit / w.heads;
      u.kvh = unit - u.chunk * w.heads;
      u.slot = w.slot + u.kvh * w.nchunks * w.nrows;
      if (w.nrows <= 16)
        token_item<D, FMT, W, 1, token_depth<FMT>(), false, true, true>(p, u, (lds_char*)lds, stats);
      else
        token_item<D, FMT, W, 2, 1, false, true, true>(p, u, (lds_char*)lds, stats);
    } else if (w.nrows <= 16) {
      token_item<D, FMT, W, 1, token_depth<FMT>(), FORM == CHUNK_STREAM, false>(p, w, (lds_char*)lds, stats);
    } else {
      token_item<D, FMT, W, 2, 1, false, false>(p, w, (lds_char*)lds, stats);
    }
  }
}

// (This file is compiled twice: its kernels for plans without and with shared keys.)
#ifndef D2SD_CHUNK_SHARED
#define ATTN_KERNEL chunk_attn_kernel
#define LAUNCH launch_chunk_attention
template <int D, int FMT, int FORM>
__global__ __launch_bounds__(64 * chunk_waves(FORM), (chunk_occupancy<D, FMT, FORM>())) void
chunk_attn_kernel(const ChunkParams p) {
  chunk_work<D, FMT, FORM, false>(p);
}
#else
#define ATTN_KERNEL shared_attn_kernel
#define LAUNCH launch_shared_attention
template <int D, int FMT, int FORM>
__global__ __launch_bounds__(64 * chunk_waves(FORM), (FORM < CHUNK_TOKENS ? 2 : chunk_occupancy<D, FMT, FORM>())) void
shared_attn_kernel(const ChunkParams p) {
  chunk_work<D, FMT, FORM, true>(p);
}
#endif

// Row i of a merge item from its partial states, nchunks of them, then (SHARED)
// those over the keys that it shares (IMAGE: as store_image left them): thread (i,
// d4) holds head dims 4 d4 .. 4 d4 + 3; of the images eight rows lie side by side.
// Latency bound: the sums and states of eight chunks are read at once (one token
// over 8 chunks: 3.8 -> 3.0 us against sums first), joined in chunk order whatever
// the order they were written in.
template <int D, bool SHARED, bool IMAGE, typename Merge>
__device__ __forceinline__ void merge_rows(const ChunkParams& p, const Merge& w) {
  constexpr int ROWS = 1024 / D;
  const int i = SHARED ? threadIdx.x % ROWS : threadIdx.x / (D / 4);
  const int dd = 4 * (SHARED ? threadIdx.x / ROWS : threadIdx.x % (D / 4));
  if (i >= w.nrows) return;
  constexpr int B = 8;
  float top = -INFINITY, sum = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  int nchunks = w.nchunks;
  if constexpr (SHARED) nchunks += w.shared_chunks;
  for (int c0 = 0; c0 < nchunks; c0 += B) {
    float s[B];
    f32x4 v[B];
#pragma unroll
    for (int u = 0; u < B; ++u) {
      const int c = min(c0 + u, nchunks - 1);
      long long pr = w.slot + i + (long long)c * w.stride;
      long long at = pr * D + dd;
      if constexpr (SHARED)
        if (c >= w.nchunks) {
          const int row = w.shared_row + i;
          pr = w.shared_slot + row + (long long)(c - w.nchunks) * w.shared_stride;
          at = IMAGE ? image_at<D>(pr - (row & 31), dd / 4, row & 31) : pr * D + dd;
        }
      s[u] = c0 + u < nchunks ? p.part_lse[pr] : -INFINITY;
      v[u] = *(const f32x4*)(p.part_o + at);
    }
    float mx = top;
#pragma unroll
    for (int u = 0; u < B; ++u) mx = fmaxf(mx, s[u]);
    if (mx == -INFINITY) {  // no key in any of them (or NaN, which stays)
#pragma unroll
      for (int u = 0; u < B; ++u) sum = s[u] == s[u] ? sum : s[u];
      continue;
    }
    const float a0 = __builtin_amdgcn_exp2f(top - mx);
    top = mx;
    sum *= a0;
    acc *= a0;
#pragma unroll
    for (int u = 0; u < B; ++u) {
      const float a = __builtin_amdgcn_exp2f(s[u] - top);
      sum += a;
      acc += s[u] == -INFINITY ? f32x4{0.f, 0.f, 0.f, 0.f} : a * v[u];
    }
  }
  const float lse2 = sum > 0.f ? top + __builtin_amdgcn_logf(sum) : sum == 0.f ? -INFINITY : sum;
  const int r = w.row0 + i, token = w.q0 + r / p.group, head = w.kvh * p.group + r % p.group;
  float inv = sum != 0.f ? 1.f / sum : 0.f;
  inv *= sink_factor(p, head, lse2);
  *(u32x2*)((bf16_t*)p.o + (long long)token * p.o_stride_n + (long long)head * p.o_stride_h + dd) =
      (u32x2){pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv)};
  if (dd == 0) p.lse[token * p.lse_stride_n + head] = p.lse_base2 ? lse2 : lse2 * kLn2;
}

#ifndef D2SD_CHUNK_SHARED
template <int D>
__global__ __launch_bounds__(256) void chunk_merge_kernel(const ChunkParams p) {
  merge_rows<D, false, false>(p, p.merges[blockIdx.x]);
}
#else
template <int D, bool IMAGE>
__global__ __launch_bounds__(256) void shared_merge_kernel(const ChunkParams p) {
  merge_rows<D, true, IMAGE>(p, ((const SharedMerge*)p.merges)[blockIdx.x]);
}
#endif

template <int D, int FMT>
hipError_t launch_f(const ChunkParams& p, int form, int nitems, int nmerges, hipStream_t s) {
  const dim3 grid((unsigned)nitems), block(64 * chunk_waves(form));
  if (form == CHUNK_TOKENS) {
    hipLaunchKernelGGL((ATTN_KERNEL<D, FMT, CHUNK_TOKENS>), grid, block, 0, s, p);
  } else if (form == CHUNK_STREAM) {
    hipLaunchKernelGGL((ATTN_KERNEL<D, FMT, CHUNK_STREAM>), grid, block, 0, s, p);
  } else if (form == CHUNK_WAVES4) {
#ifdef D2SD_CHUNK_SHARED
    if constexpr (!shared_waves4(D, FMT)) return hipErrorInvalidValue;
    else
#endif
    hipLaunchKernelGGL((ATTN_KERNEL<D, FMT, CHUNK_WAVES4>), grid, block, 0, s, p);
  } else {
    if constexpr (D == 64) return hipErrorInvalidValue;  // (the planner gives heads of 64 four waves)
    else hipLaunchKernelGGL((ATTN_KERNEL<D, FMT, CHUNK_WAVES8>), grid, block, 0, s, p);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (nmerges <= 0) return hipSuccess;
#ifdef D2SD_CHUNK_SHARED
  if (form >= CHUNK_TOKENS)
    hipLaunchKernelGGL((shared_merge_kernel<D, false>), dim3((unsigned)nmerges), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((shared_merge_kernel<D, true>), dim3((unsigned)nmerges), dim3(256), 0, s, p);
#else
  hipLaunchKernelGGL(chunk_merge_kernel<D>, dim3((unsigned)nmerges), dim3(256), 0, s, p);
#endif
  return hipGetLastError();
}

template <int D>
hipError_t launch_d(const ChunkParams& p, int format, int form, int nitems, int nmerges, hipStream_t s) {
  switch (format) {
    case CACHE_BF16: return launch_f<D, CACHE_BF16>(p, form, nitems, nmerges, s);
    case CACHE_FP8: return launch_f<D, CACHE_FP8>(p, form, nitems, nmerges, s);
    case CACHE_MXFP8: return launch_f<D, CACHE_MXFP8>(p, form, nitems, nmerges, s);
    case CACHE_MXFP4: return launch_f<D, CACHE_MXFP4>(p, form, nitems, nmerges, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t LAUNCH(const ChunkParams& p, int head_dim, int format, int form, int nitems, int nmerges, hipStream_t s) {
  if (nitems <= 0) return hipSuccess;
  return head_dim == 64    ? launch_d<64>(p, format, form, nitems, nmerges, s)
         : head_dim == 128 ? launch_d<128>(p, format, form, nitems, nmerges, s)
                           : hipErrorInvalidValue;
}

}  // namespace d2sd
