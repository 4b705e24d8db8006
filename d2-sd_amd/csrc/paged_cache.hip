// gfx950 kernels of the paged KV cache of a ragged batch: the new tokens' keys
// and values quantised into their pages (write), and cached tokens read back
// as contiguous bf16 (read).
//
// Formats.  bf16; fp8: e4m3fn(x / scale[head]), the quotient correctly rounded
// in fp32; mxfp8 / mxfp4: blocks of 32 head dims, each a power-of-two scale 2^e
// (byte e + 127) and elements RNE(x 2^-e) in e4m3 or e2m1 (two to a byte, the
// even element low).  e is the smallest exponent with amax <= M 2^e, M = 448
// or 6: with amax = f 2^k, 1 <= f < 2, it is k - kM + (f > fM) for
// M = fM 2^kM, integer arithmetic on amax's bits, so that the codes follow from
// the inputs alone, whatever the order of work.  e stays at or above -117,
// where the smallest element (2^-9 2^e) is a normal bf16, and at or below 119
// (mxfp8) or 125 (mxfp4), where the largest is finite; there elements saturate.
// x 2^-e is exact and every element times 2^e is a bf16 value, so reading back
// is exact.  A block that holds an infinity or NaN gets the scale byte 255 and
// reads back as NaN.
//
// Both kernels move data once: bound by HBM (16 requests, 72.6k tokens in mxfp8 read
// back, 0.45 GB moved: 90 us, 5.0 TB/s, the rate of a large copy) or, for a step's few tokens, by the
// chain token -> cache length -> page id -> store (64 tokens: 3 us).  A thread
// carries 8 elements: a 16-byte bf16 load or store against 8 bytes (fp8, mxfp8)
// or 4 (mxfp4) of codes; the four threads of a block of 32 find its amax by DPP.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "d2sd_internal.h"
#include "kernel_common.h"
#include "paged_store.h"
#include "plan.h"

namespace d2sd {

namespace {

// tokens of an item that one block reads (16 requests in mxfp8, 72.6k tokens: 1, 2, 4, 8, 16:
// 127, 93, 91, 89, 95.5 us; 18.2k tokens in mxfp4 with their write, three states in turn:
// 48.5, 43.7, 43.2, 44.1, 47)
constexpr int kReadShare = 4;
constexpr int kWriteTokens = 8;         // of one block, where there are many
// (8 heads of 128 in mxfp4: 4096 tokens 7.1 and 7.2 us, 8000 tokens 13.3 one by one, 11.3 by eight)
constexpr int kWriteManyTokens = 6144;
// Results larger than half of the last-level cache are stored past it: nothing
// of them would be found there by whoever reads them from their start (16
// requests of 100..8000 tokens, 0.30 GB of results: 99 -> 94 us with 16 tokens a block).
constexpr long long kReadStreamBytes = 128ll << 20;

// 2^(byte - 127); byte 255 stands for NaN, byte 0 for 2^-127
__device__ __forceinline__ float block_scale(unsigned byte) {
  const unsigned bits = byte == 255u ? 0x7FC00000u : byte == 0u ? 0x00400000u : byte << 23;
  return __uint_as_float(bits);
}

// The places of N tokens, in scalar registers: lane i of a wave found token i's
// page (below zero: none) and slot.  Built where all lanes are active.
template <int N>
struct Places {
  int page[N], slot[N];
  __device__ __forceinline__ Places(int pg, int sl) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      page[i] = __builtin_amdgcn_readlane(pg, i);
      slot[i] = __builtin_amdgcn_readlane(sl, i);
    }
  }
  __device__ __forceinline__ bool on(int i) const { return page[i] >= 0; }
  __device__ __forceinline__ long long row(const CacheParams& p, int i) const {
    return page[i] * p.stride_page + slot[i] * p.stride_tok;
  }
  __device__ __forceinline__ long long scale_row(const CacheParams& p, int i) const {
    return page[i] * p.scale_stride_page + slot[i] * p.scale_stride_tok;
  }
};

// Block b: new tokens TOK b .., all heads, keys then values.  tokens[t] =
// (request, tokens from it to its request's end, first page table entry, page
// table end).  A thread takes the same piece of every token: TOK = 8 keeps as
// many loads in flight and starts fewer blocks (one request of 16.3k tokens, 8 heads of 128 in mxfp4: 35 -> 22 us, 84 MB at 3.8 TB/s),
// TOK = 1 spreads a step's few tokens.
template <int FMT, int TOK>
__global__ __launch_bounds__(256) void cache_write_kernel(const CacheParams p) {
  const int t0 = blockIdx.x * TOK, nt = min(TOK, p.num_items - t0);
  const int cpr = p.head_dim / 8, nch = p.num_kv_heads * cpr;
  u32x4 val[TOK];
  // the rows' loads first: they do not wait for the place they go to
  auto source = [&](bool is_v, int h, int d) {
    const uint16_t* s = (const uint16_t*)(is_v ? p.v : p.k) + (long long)t0 * p.stride_n + (long long)h * p.stride_h + d;
#pragma unroll
    for (int i = 0; i < TOK; ++i)
      if (i < nt) val[i] = *(const u32x4*)(s + i * p.stride_n);
  };
  auto head_of = [&](int c) { return (c >= nch ? c - nch : c) / cpr; };
  int c = threadIdx.x;
  int h = head_of(c), d = 8 * ((c >= nch ? c - nch : c) - h * cpr);
  if (c < 2 * nch) source(c >= nch, h, d);
  const int lane = threadIdx.x & 63;
  int page = -1, slot = 0;
  if (lane < nt) {
    const int4 w = ((const int4*)p.items)[t0 + lane];
    const int pos = p.kv_len[w.x] - w.y;
    const int at = w.z + (pos >> p.log2_page);
    slot = pos & ((1 << p.log2_page) - 1);
    // (before the cache's start, or no page is reserved for it: nothing to write)
    if (pos >= 0 && at < w.w) page = p.page_table[at];
    if (page >= p.num_pages) page = -1;
  }
  const Places<TOK> places(page, slot);
  while (c < 2 * nch) {
    const bool is_v = c >= nch;
    const CacheSide& s = is_v ? p.vs : p.ks;
    const long long row = h * p.stride_head, srow = h * p.scale_stride_head;
#pragma unroll
    for (int i = 0; i < TOK; ++i)
      if (places.on(i)) store_piece<FMT>(s, h, row + places.row(p, i), srow + places.scale_row(p, i), d, val[i]);
    c += blockDim.x;
    h = head_of(c), d = 8 * ((c >= nch ? c - nch : c) - h * cpr);
    if (c < 2 * nch) source(c >= nch, h, d);
  }
}

// 8 cached elements as bf16.
template <int FMT>
__device__ __forceinline__ u32x4 load_piece(const CacheSide& s, int h, long long row, long long srow, int d) {
  if constexpr (FMT == CACHE_BF16) {
    return *(const u32x4*)((const uint16_t*)s.codes + row + d);
  } else if constexpr (FMT == CACHE_FP8) {
    const u32x2 b = *(const u32x2*)((const uint8_t*)s.codes + row + d);
    const float sc = ((const float*)s.scale)[h];
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const u32x2 v = fp8x4_to_bf16x4(b[i]);
      o[2 * i] = pack_bf16x2(bf16_lo(v[0]) * sc, bf16_hi(v[0]) * sc);
      o[2 * i + 1] = pack_bf16x2(bf16_lo(v[1]) * sc, bf16_hi(v[1]) * sc);
    }
    return o;
  } else {
    const float sc = block_scale(((const uint8_t*)s.scale)[srow + d / 32]);
    u32x4 o;
    if constexpr (FMT == CACHE_MXFP8) {
      const u32x2 b = *(const u32x2*)((const uint8_t*)s.codes + row + d);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        o[2 * i] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b[i], sc, false));
        o[2 * i + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b[i], sc, true));
      }
    } else {
      const unsigned b = *(const unsigned*)((const uint8_t*)s.codes + row + d / 2);
      o[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(b, sc, 0));
      o[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(b, sc, 1));
      o[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(b, sc, 2));
      o[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(b, sc, 3));
    }
    return o;
  }
}

// Block (i, j): tokens kReadShare j .. of the up to kReadTokens cached tokens of one
// request that items[i] names (CacheReadItem), all heads, keys then values.  A thread takes the same piece of every
// token, or, where a token has at most 128 pieces, of every n-th one; the tokens'
// pages are found once, by one lane each.  One load, then its store: with 8 loads
// in flight a thread's stores scatter over 8 rows (99 -> 117 us).
template <int FMT, bool STREAM>
__global__ __launch_bounds__(256) void cache_read_kernel(const CacheParams p) {
  const CacheReadItem w = ((const CacheReadItem*)p.items)[blockIdx.x];
  const int from = blockIdx.y * kReadShare, count = min(w.count - from, kReadShare);
  if (count <= 0) return;
  const int len = p.kv_len[w.req];
  const int pos0 = (w.from_end ? len - w.first : w.first) + from;  // cache position of the block's first token
  const int cpr = p.head_dim / 8, nch = p.num_kv_heads * cpr;
  const int lane = threadIdx.x & 63;
  int page = -1, slot = 0;
  if (lane < count) {
    const int pos = pos0 + lane, at = w.page_begin + (pos >> p.log2_page);
    slot = pos & ((1 << p.log2_page) - 1);
    if (pos >= 0 && pos < len && at < w.page_end) page = p.page_table[at];
    if (page >= p.num_pages) page = -1;
  }
  auto piece = [&](int c, auto&& tokens) {
    const bool is_v = c >= nch;
    const int cc = is_v ? c - nch : c, h = cc / cpr, d = 8 * (cc - h * cpr);
    const long long row = h * p.stride_head, srow = h * p.scale_stride_head;
    uint16_t* out = (uint16_t*)(is_v ? p.v : p.k) + (long long)(w.row + from) * p.stride_n + (long long)h * p.stride_h + d;
    tokens(is_v ? p.vs : p.ks, h, d, row, srow, out);
  };
  // (apart from the copy: a second store in its loop takes the read of 16 requests from 90 to 112 us)
  if (p.zero_missing && __any(lane < count && page < 0)) {
    for (int i = 0; i < count; ++i) {
      if (__shfl(page, i) >= 0) continue;
      for (int c = threadIdx.x; c < 2 * nch; c += 256)
        piece(c, [&](const CacheSide&, int, int, long long, long long, uint16_t* out) {
          *(u32x4*)(out + i * p.stride_n) = u32x4{0u, 0u, 0u, 0u};
        });
    }
  }
  const int apart = 256 / (2 * nch);  // threads of a piece
  if (apart > 1) {
    const int first = threadIdx.x / (2 * nch);
    piece(threadIdx.x - first * 2 * nch, [&](const CacheSide& s, int h, int d, long long row, long long srow, uint16_t* out) {
      for (int i0 = 0; i0 < kReadShare; i0 += apart) {  // (every lane stays for the shuffles)
        const int i = i0 + first, pg = __shfl(page, i), sl = __shfl(slot, i);
        if (first < apart && i < count && pg >= 0)
          *(u32x4*)(out + i * p.stride_n) = load_piece<FMT>(s, h, row + pg * p.stride_page + sl * p.stride_tok,
                                                            srow + pg * p.scale_stride_page + sl * p.scale_stride_tok, d);
      }
    });
    return;
  }
  const Places<kReadShare> places(page, slot);
  for (int c = threadIdx.x; c < 2 * nch; c += 256) {
    piece(c, [&](const CacheSide& s, int h, int d, long long row, long long srow, uint16_t* out) {
#pragma unroll
      for (int i = 0; i < kReadShare; ++i) {
        if (!places.on(i)) continue;
        const u32x4 val = load_piece<FMT>(s, h, row + places.row(p, i), srow + places.scale_row(p, i), d);
        u32x4* at = (u32x4*)(out + i * p.stride_n);
        if constexpr (STREAM)
          __builtin_nontemporal_store(val, at);
        else
          *at = val;
      }
    });
  }
}

}  // namespace

template <int FMT>
static void launch_write(const CacheParams& p, hipStream_t s) {
  const int pieces = 2 * p.num_kv_heads * (p.head_dim / 8);
  const dim3 block((unsigned)std::min(256, (pieces + 63) / 64 * 64));
  if (p.num_items >= kWriteManyTokens)
    hipLaunchKernelGGL((cache_write_kernel<FMT, kWriteTokens>), dim3((unsigned)((p.num_items + kWriteTokens - 1) / kWriteTokens)),
                       block, 0, s, p);
  else
    hipLaunchKernelGGL((cache_write_kernel<FMT, 1>), dim3((unsigned)p.num_items), block, 0, s, p);
}

hipError_t launch_cache_write(const CacheParams& p, int format, hipStream_t s) {
  if (p.num_items <= 0) return hipSuccess;
  switch (format) {
    case CACHE_BF16: launch_write<CACHE_BF16>(p, s); break;
    case CACHE_FP8: launch_write<CACHE_FP8>(p, s); break;
    case CACHE_MXFP8: launch_write<CACHE_MXFP8>(p, s); break;
    case CACHE_MXFP4: launch_write<CACHE_MXFP4>(p, s); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

template <int FMT>
static void launch_read(const CacheParams& p, hipStream_t s) {
  const dim3 grid((unsigned)p.num_items, kReadTokens / kReadShare), block(256);
  if (4ll * p.num_kv_heads * p.head_dim * kReadTokens * p.num_items > kReadStreamBytes)
    hipLaunchKernelGGL((cache_read_kernel<FMT, true>), grid, block, 0, s, p);
  else
    hipLaunchKernelGGL((cache_read_kernel<FMT, false>), grid, block, 0, s, p);
}

hipError_t launch_cache_read(const CacheParams& p, int format, hipStream_t s) {
  if (p.num_items <= 0) return hipSuccess;
  switch (format) {
    case CACHE_BF16: launch_read<CACHE_BF16>(p, s); break;
    case CACHE_FP8: launch_read<CACHE_FP8>(p, s); break;
    case CACHE_MXFP8: launch_read<CACHE_MXFP8>(p, s); break;
    case CACHE_MXFP4: launch_read<CACHE_MXFP4>(p, s); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace d2sd
