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
//   chunk_attn_kernel   one workgroup of 8 waves per work item: packed rows of
//                       one (request, kv head) against a chunk of their visible
//                       keys, with a running maximum and sum (one pass over the
//                       cache), state in registers
//   chunk_merge_kernel  joins the partial states of rows whose keys were split
//
// Rows are packed (token, query head of the kv head) pairs, row = token * g + j,
// so that a key is read once for all query heads that share it.  S^T = K Q^T
// and O^T += V^T P^T run on v_mfma_f32_32x32x16_bf16: lane l holds the scores
// and the output of row l % 32, so the softmax stays in a lane (and its partner
// l ^ 32), and P^T goes back as an operand without leaving the registers.  Codes
// are expanded to bf16 by the converters that apply a block's scale as they go;
// that is exact, so quantised caches cost no accuracy beyond their own.
//
// Two kinds of item, by packed rows:
//  * tile items (more than 32 rows): each wave owns 32 rows, the workgroup
//    stages tiles of 64 keys through registers into LDS (two buffers, one
//    barrier a tile).  Bound by MFMA beside the softmax's vector instructions.
//  * token items (up to 32 rows: decoding): all waves share the rows, and wave w
//    takes every 8th tile of 32 keys.  Keys go from the cache straight to the
//    MFMA operand: the sum over head dims may run in any order, so lane l takes
//    the contiguous half l / 32 of key l % 32's dims.  Values pass through the
//    wave's own LDS to be read transposed.  No barrier until the waves' states
//    are joined.  Bound by HBM.
//
// Keys outside an item's visible range are never read: their addresses are
// clamped to the range, so what lies behind a cache's end (or before its
// window) may hold anything.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

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
  int pos0;       // position of the request's query 0 (negative: it has no key yet)
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

template <int D>
__device__ __forceinline__ lds_char* lds_piece(lds_char* tile, int row, int chunk) {
  return tile + row * D * 2 + 16 * (chunk ^ chunk_swizzle<D>(row));
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

__device__ __forceinline__ float natural(const ChunkParams& p, float lse2) { return lse2 * kLn2; }

__device__ __forceinline__ float sink_factor(const ChunkParams& p, int head, float lse2) {
  if (!p.sinks) return 1.f;
  return 1.f / (1.f + __builtin_amdgcn_exp2f((p.sinks[head] - lse2 * kLn2) * kLog2e));
}

// ---- tile items ----
template <int D, int FMT>
__device__ __forceinline__ void tile_item(const ChunkParams& p, const ChunkItem& w, lds_char* lds) {
  constexpr int MT = D / 32, KS = D / 16, EPT = D / 8, ROW = Format<D, FMT>::ROW, TB = 64 * D * 2;
  constexpr bool MX = Format<D, FMT>::MX;
  constexpr int WORDS = ROW / 8 / 4;  // words of codes per thread and tile (keys; as many for values)
  const int tid = threadIdx.x, wv = tid >> 6, lane = tid & 63, l32 = lane & 31, hh = lane >> 5;

  const Span all = item_span(p, w, w.row0 / p.group, (w.row0 + w.nrows - 1) / p.group);
  const int tile0 = all.lo >> 6, ntiles_all = all.hi > all.lo ? ((all.hi + 63) >> 6) - tile0 : 0;
  const int tb = tile0 + (int)((long long)ntiles_all * w.chunk / w.nchunks);
  const int te = tile0 + (int)((long long)ntiles_all * (w.chunk + 1) / w.nchunks);

  // this wave's rows
  const int wrow = 32 * wv, row = min(wrow + l32, w.nrows - 1);
  const bool wave_on = wrow < w.nrows;
  const int t_row = (w.row0 + row) / p.group;
  const int pos = all.pos0 + t_row;
  const int row_lo = p.window_left >= 0 ? max(pos - p.window_left, 0) : 0;
  const Span own = item_span(p, w, (w.row0 + min(wrow, w.nrows - 1)) / p.group,
                             (w.row0 + min(wrow + 31, w.nrows - 1)) / p.group);
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

  // staging: thread tid carries 1/8 of key row tid / 8
  const int srow = tid >> 3, spart = tid & 7;
  const char* kb_ = (const char*)p.ks.codes + w.kvh * p.stride_head + spart * (ROW / 8);
  const char* vb_ = (const char*)p.vs.codes + w.kvh * p.stride_head + spart * (ROW / 8);
  const long long shead = w.kvh * p.scale_stride_head + spart * EPT / 32;
  auto page_of = [&](int tile) -> int {
    const int key = min(max(64 * tile + srow, all.lo), all.hi - 1);
    return min((unsigned)p.page_table[w.page_begin + (key >> p.log2_page)], (unsigned)p.num_pages - 1u);
  };
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
  auto fetch = [&](int tile, int page) {
    const int key = min(max(64 * tile + srow, all.lo), all.hi - 1);
    const int slot = key & ((1 << p.log2_page) - 1);
    const long long off = page * p.stride_page + slot * p.stride_tok;
    load_words(kw, kb_ + off);
    load_words(vw, vb_ + off);
    if constexpr (MX) {
      const long long so = page * p.scale_stride_page + slot * p.scale_stride_tok + shead;
      ksc = ((const uint8_t*)p.ks.scale)[so];
      vsc = ((const uint8_t*)p.vs.scale)[so];
    }
  };
  auto put = [&](lds_char* tile, const unsigned (&d)[WORDS], unsigned sc) {
    const float f = MX ? block_scale(sc) : 1.f;
#pragma unroll
    for (int i = 0; i < EPT / 8; ++i) {
      bf16x8 v;
      if constexpr (FMT == CACHE_BF16)
        v = __builtin_bit_cast(bf16x8, (u32x4){d[4 * i], d[4 * i + 1], d[4 * i + 2], d[4 * i + 3]});
      else if constexpr (FMT == CACHE_MXFP4)
        v = expand<FMT>(d[i], 0u, f);
      else
        v = expand<FMT>(d[2 * i], d[2 * i + 1], f);
      *(__attribute__((address_space(3))) bf16x8*)lds_piece<D>(tile, srow, spart * (EPT / 8) + i) = v;
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

  int page = 0;
  if (tb < te) {
    fetch(tb, page_of(tb));
    put(lds, kw, ksc);
    put(lds + TB, vw, vsc);
    if (tb + 1 < te) {
      fetch(tb + 1, page_of(tb + 1));
      page = page_of(min(tb + 2, te - 1));
    }
    __syncthreads();
  }
  for (int t = tb; t < te; ++t) {
    lds_char* kt = lds + ((t - tb) & 1) * 2 * TB;
    lds_char* vt = kt + TB;
    lds_char* nx = lds + ((t - tb + 1) & 1) * 2 * TB;
    const int kb = 64 * t;
    const bool on = wave_on && kb < own.hi && kb + 64 > own.lo;
    f32x16 s[2];
    if (on) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const bf16x8 a0 = *(const __attribute__((address_space(3))) bf16x8*)(kt + koff[ks]);
        const bf16x8 a1 = *(const __attribute__((address_space(3))) bf16x8*)(kt + koff[ks] + 32 * D * 2);
        s[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a0, qf[ks], ks ? s[0] : f32x16{}, 0, 0, 0);
        s[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a1, qf[ks], ks ? s[1] : f32x16{}, 0, 0, 0);
      }
    }
    if (t + 1 < te) {
      put(nx, kw, ksc);
      put(nx + TB, vw, vsc);
      if (t + 2 < te) {
        fetch(t + 2, page);
        page = page_of(min(t + 3, te - 1));
      }
    }
    if (on) {
      if (kb < own.all_lo || kb + 64 > own.all_hi) {
        hide(s[0], kb, row_lo, pos, hh);
        hide(s[1], kb + 32, row_lo, pos, hh);
      }
      softmax_step<2, MT>(s, o, m, l, c, slack, hh);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bf16x8 pb = p_operand(s[j >> 1], j & 1);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          o[mt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vread(vt, mt, j), pb, o[mt], 0, 0, 0);
      }
    }
    __syncthreads();
  }

  if (!wave_on) return;
  l += xor32(l, hh);
  const float lse2 = l > 0.f ? m * c + __builtin_amdgcn_logf(l) : l == 0.f ? -INFINITY : l;
  float inv = l != 0.f ? vscale / l : 0.f;
  const bool mine = wrow + l32 < w.nrows;
  if (w.nchunks > 1) {
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
template <int D, int FMT>
__device__ __forceinline__ void token_item(const ChunkParams& p, const ChunkItem& w, lds_char* lds, float* stats) {
  constexpr int MT = D / 32, KS = D / 16, ROW = Format<D, FMT>::ROW;
  constexpr bool MX = Format<D, FMT>::MX;
  constexpr int PPR = ROW / 16;    // 16-byte pieces of a row
  constexpr int NP = PPR / 2;      // pieces per lane and tile of 32 keys (keys; as many for values)
  constexpr int VB = 32 * D * 2;   // bytes of a wave's value tile
  const int tid = threadIdx.x, wv = tid >> 6, lane = tid & 63, l32 = lane & 31, hh = lane >> 5;

  const Span all = item_span(p, w, w.row0 / p.group, (w.row0 + w.nrows - 1) / p.group);
  const int tile0 = all.lo >> 5, ntiles_all = all.hi > all.lo ? ((all.hi + 31) >> 5) - tile0 : 0;
  const int tb = tile0 + (int)((long long)ntiles_all * w.chunk / w.nchunks);
  const int te = tile0 + (int)((long long)ntiles_all * (w.chunk + 1) / w.nchunks);

  const int row = min(l32, w.nrows - 1);
  const int pos = all.pos0 + (w.row0 + row) / p.group;
  const int row_lo = p.window_left >= 0 ? max(pos - p.window_left, 0) : 0;
  bf16x8 qf[KS];
  {
    const RowOut at(p, w, row);
    const bf16_t* qp = (const bf16_t*)p.q + (long long)at.token * p.q_stride_n + (long long)at.head * p.q_stride_h + hh * (D / 2);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *(const bf16x8*)(qp + 8 * ks);
  }
  float c = p.sm_scale * kLog2e, vscale = 1.f;
  if constexpr (FMT == CACHE_FP8) {
    c *= ((const float*)p.ks.scale)[w.kvh];
    vscale = ((const float*)p.vs.scale)[w.kvh];
  }
  const float slack = c > 0.f ? kRescaleSlack / c : 0.f;

  const char* kbase = (const char*)p.ks.codes + w.kvh * p.stride_head + hh * (ROW / 2);
  const char* vbase = (const char*)p.vs.codes + w.kvh * p.stride_head;
  const long long shead = w.kvh * p.scale_stride_head;
  const int pmask = (1 << p.log2_page) - 1;
  auto key_at = [&](int tile, int i) -> int { return min(max(32 * tile + i, all.lo), all.hi - 1); };
  auto page_at = [&](int key) -> int {
    return min((unsigned)p.page_table[w.page_begin + (key >> p.log2_page)], (unsigned)p.num_pages - 1u);
  };
  u32x4 kr[NP], vr[NP];
  unsigned ksc = 0, vsc[NP];
  // page: the page of this lane's key (l32) of the tile
  auto fetch_k = [&](int tile, int page) {
    const int slot = key_at(tile, l32) & pmask;
    const char* s = kbase + page * p.stride_page + slot * p.stride_tok;
#pragma unroll
    for (int i = 0; i < NP; ++i) kr[i] = *(const u32x4*)(s + 16 * i);
    if constexpr (MX) {
      const uint8_t* q = (const uint8_t*)p.ks.scale + page * p.scale_stride_page + slot * p.scale_stride_tok + shead;
      if constexpr (D == 128) ksc = q[2 * hh] | (unsigned)q[2 * hh + 1] << 8;
      else ksc = q[hh];
    }
  };
  auto fetch_v = [&](int tile, int page) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int idx = 64 * i + lane, kk = idx / PPR, col = idx % PPR;
      const int pg = __shfl(page, kk);
      const int slot = key_at(tile, kk) & pmask;
      vr[i] = *(const u32x4*)(vbase + pg * p.stride_page + slot * p.stride_tok + 16 * col);
      if constexpr (MX)
        vsc[i] = ((const uint8_t*)p.vs.scale)[pg * p.scale_stride_page + slot * p.scale_stride_tok + shead +
                                              (FMT == CACHE_MXFP4 ? col : col / 2)];
    }
  };

  f32x16 o[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) o[mt] = f32x16{};
  float m = -INFINITY, l = 0.f;
  lds_char* vt = lds + wv * VB;
  const ValueRead<D> vread(lane);

  int t = tb + wv;
  int page = 0, pnext = 0;
  if (t < te) {
    page = page_at(key_at(t, l32));
    fetch_k(t, page);
    fetch_v(t, page);
    pnext = page_at(key_at(min(t + kChunkWaves, te - 1), l32));
  }
  for (; t < te; t += kChunkWaves) {
    const int tn = min(t + kChunkWaves, te - 1);  // (the last round fetches its own tile again, unused)
    const int pg = pnext;
    pnext = page_at(key_at(min(t + 2 * kChunkWaves, te - 1), l32));
    f32x16 s[1];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      bf16x8 a;
      if constexpr (FMT == CACHE_BF16) {
        a = __builtin_bit_cast(bf16x8, kr[ks]);
      } else {
        const float f = MX ? block_scale(ksc >> (8 * (ks / 4)) & 255u) : 1.f;
        if constexpr (FMT == CACHE_MXFP4) a = expand<FMT>(kr[ks / 4][ks % 4], 0u, f);
        else a = expand<FMT>(kr[ks / 2][2 * (ks % 2)], kr[ks / 2][2 * (ks % 2) + 1], f);
      }
      s[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, qf[ks], ks ? s[0] : f32x16{}, 0, 0, 0);
    }
    if (t + kChunkWaves < te) fetch_k(tn, pg);
    const int kb = 32 * t;
    if (kb < all.all_lo || kb + 32 > all.all_hi) hide(s[0], kb, row_lo, pos, hh);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int idx = 64 * i + lane, kk = idx / PPR, col = idx % PPR;
      if constexpr (FMT == CACHE_BF16) {
        *(__attribute__((address_space(3))) u32x4*)lds_piece<D>(vt, kk, col) = vr[i];
      } else {
        constexpr int CH = FMT == CACHE_MXFP4 ? 4 : 2;  // 8-element chunks of a piece
        const float f = MX ? block_scale(vsc[i]) : 1.f;
#pragma unroll
        for (int e = 0; e < CH; ++e) {
          const bf16x8 v = FMT == CACHE_MXFP4 ? expand<FMT>(vr[i][e], 0u, f) : expand<FMT>(vr[i][2 * e & 3], vr[i][(2 * e + 1) & 3], f);
          *(__attribute__((address_space(3))) bf16x8*)lds_piece<D>(vt, kk, CH * col + e) = v;
        }
      }
    }
    if (t + kChunkWaves < te) fetch_v(tn, pg);
    softmax_step<1, MT>(s, o, m, l, c, slack, hh);
    // (LDS serves a wave's accesses in order; the fence keeps the compiler's order)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const bf16x8 pb = p_operand(s[0], j);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
        o[mt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vread(vt, mt, j), pb, o[mt], 0, 0, 0);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }

  // join the waves: every wave's m and l, then O in rounds that fit the LDS
  // (all head dims at once for up to 16 rows, half of them for more)
  l += xor32(l, hh);
  float* ms = stats;
  float* lw = stats + kChunkWaves * kTokenRows;
  if (hh == 0) {
    ms[wv * kTokenRows + l32] = m;
    lw[wv * kTokenRows + l32] = l;
  }
  const int nr = w.nrows;
  const int per_round = nr > 16 ? MT / 2 : MT;
  typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
  for (int mt0 = 0; mt0 < MT; mt0 += per_round) {
    __syncthreads();  // the tiles, or the last round's states, have been read
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      if (mt < mt0 || mt >= mt0 + per_round || l32 >= nr) continue;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int d4 = 8 * (mt - mt0) + 2 * q + hh;
        ((lds_f32x4*)lds)[(wv * 8 * per_round + d4) * nr + l32] =
            (f32x4){o[mt][4 * q], o[mt][4 * q + 1], o[mt][4 * q + 2], o[mt][4 * q + 3]};
      }
    }
    __syncthreads();
    for (int i = tid; i < nr * 8 * per_round; i += 64 * kChunkWaves) {
      const int r = i % nr, d4 = i / nr;
      float top = -INFINITY;
#pragma unroll
      for (int v = 0; v < kChunkWaves; ++v) top = fmaxf(top, ms[v * kTokenRows + r]);
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
      float sum = 0.f;
#pragma unroll
      for (int v = 0; v < kChunkWaves; ++v) {
        const float mv = ms[v * kTokenRows + r];
        const float a = mv == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mv - top) * c);
        sum += a * lw[v * kTokenRows + r];
        acc += a * ((lds_f32x4*)lds)[(v * 8 * per_round + d4) * nr + r];
      }
      const float lse2 = sum > 0.f ? top * c + __builtin_amdgcn_logf(sum) : sum == 0.f ? -INFINITY : sum;
      float inv = sum != 0.f ? vscale / sum : 0.f;
      const int dd = 32 * mt0 + 4 * d4;
      if (w.nchunks > 1) {
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

template <int D, int FMT>
__global__ __launch_bounds__(64 * kChunkWaves) void chunk_attn_kernel(const ChunkParams p) {
  __shared__ __align__(16) char lds[4 * 64 * D * 2];
  __shared__ float stats[2 * kChunkWaves * kTokenRows];
  const ChunkItem w = p.items[blockIdx.x];
  if (w.kind == CHUNK_TILE)
    tile_item<D, FMT>(p, w, (lds_char*)lds);
  else
    token_item<D, FMT>(p, w, (lds_char*)lds, stats);
}

// Row i of a merge item from its nchunks partial states: thread (i, d4) holds
// head dims 4 d4 .. 4 d4 + 3.  Latency bound: all of a row's sums are read first,
// then its states, in chunk order whatever the order they were written in.
template <int D>
__global__ __launch_bounds__(256) void chunk_merge_kernel(const ChunkParams p) {
  const ChunkMerge w = p.merges[blockIdx.x];
  const int i = threadIdx.x / (D / 4), dd = 4 * (threadIdx.x % (D / 4));
  if (i >= w.nrows) return;
  const float* ls = p.part_lse + w.slot + i;
  float top = -INFINITY;
  for (int c = 0; c < w.nchunks; ++c) top = fmaxf(top, ls[(long long)c * w.stride]);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f;
  for (int c = 0; c < w.nchunks; ++c) {
    const float s = ls[(long long)c * w.stride];
    const float a = s == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s - top);
    const f32x4 v = *(const f32x4*)(p.part_o + (w.slot + (long long)c * w.stride + i) * D + dd);
    sum += a;
    acc += a * v;
  }
  const float lse2 = sum > 0.f ? top + __builtin_amdgcn_logf(sum) : sum == 0.f ? -INFINITY : sum;
  const int r = w.row0 + i, token = w.q0 + r / p.group, head = w.kvh * p.group + r % p.group;
  float inv = sum != 0.f ? 1.f / sum : 0.f;
  inv *= sink_factor(p, head, lse2);
  *(u32x2*)((bf16_t*)p.o + (long long)token * p.o_stride_n + (long long)head * p.o_stride_h + dd) =
      (u32x2){pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv)};
  if (dd == 0) p.lse[token * p.lse_stride_n + head] = p.lse_base2 ? lse2 : lse2 * kLn2;
}

template <int D>
hipError_t launch_d(const ChunkParams& p, int format, int nitems, int nmerges, hipStream_t s) {
  const dim3 grid((unsigned)nitems), block(64 * kChunkWaves);
  if (nitems > 0) {
    switch (format) {
      case CACHE_BF16: hipLaunchKernelGGL((chunk_attn_kernel<D, CACHE_BF16>), grid, block, 0, s, p); break;
      case CACHE_FP8: hipLaunchKernelGGL((chunk_attn_kernel<D, CACHE_FP8>), grid, block, 0, s, p); break;
      case CACHE_MXFP8: hipLaunchKernelGGL((chunk_attn_kernel<D, CACHE_MXFP8>), grid, block, 0, s, p); break;
      case CACHE_MXFP4: hipLaunchKernelGGL((chunk_attn_kernel<D, CACHE_MXFP4>), grid, block, 0, s, p); break;
      default: return hipErrorInvalidValue;
    }
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (nmerges > 0) hipLaunchKernelGGL(chunk_merge_kernel<D>, dim3((unsigned)nmerges), dim3(256), 0, s, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_chunk_attention(const ChunkParams& p, int head_dim, int format, int nitems, int nmerges,
                                  hipStream_t s) {
  return head_dim == 64    ? launch_d<64>(p, format, nitems, nmerges, s)
         : head_dim == 128 ? launch_d<128>(p, format, nitems, nmerges, s)
                           : hipErrorInvalidValue;
}

}  // namespace d2sd
