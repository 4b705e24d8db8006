// gfx950 kernel: the new tokens of a ragged batch from their projection to the
// attention in one launch.  Query and key heads are normed (with weights given)
// and rotated at their positions, queries stored, keys and values quantised into
// their pages.
//
//   y = x / sqrt(mean(x^2) + eps) * w
//   (a, b) -> s (a cos t - b sin t, b cos t + a sin t),  t = position * f
//
// with the pairs and codes of rotary.hip and paged_cache.hip.  Everything between the
// loads and the stores is 32-bit (angles: 64-bit turns); queries and keys are rounded
// once, keys straight to the cache's elements.  (Calls of rotary_embedding and
// cache_write round a key to bf16 between them.)
//
// A wave owns one token and a run of its heads, queries, keys and values in this
// order; a lane holds eight neighbouring head dims of a head, so that a block of 32
// dims is four lanes side by side, as the quantiser wants it.  The eight that they
// are paired with are its own, or lie 1, 2, 4 or 8 lanes apart in the usual layouts
// (NEAR): one or two register moves between lanes; else they are read too (from the
// vector cache: the same lines).  The run's cosines and sines are computed once,
// lane i those of pair i, and shared through LDS.
//
// Bound by HBM: 8192 tokens of 64 + 16 heads of 128 into a bf16 cache, 336 MB, take
// 66 us, 5.1 TB/s, where a large copy reaches 5.0.  (With paired dims read, unpacked
// and normed again, library sines and each head's page address apart, vector
// instructions bounded it: 81.)  5 prompts, 11.8K tokens of 64 + 16 heads of 64, into
// mxfp4 with their read back, 247 MB, 54 us.  2500 tokens of 28 + 8 heads of 128 into
// fp8, 39 MB, 13: a round and a half of the waves that the device holds, each a chain
// of loads.  A decoding step is one launch's latency: a token 4 us (a call 5 to 6), 48
// tokens of 32 + 16 heads into mxfp8 5.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "d2sd_internal.h"
#include "kernel_common.h"
#include "paged_store.h"
#include "plan.h"

namespace d2sd {

namespace {

constexpr int kAppendWaves = 4;
// Heads of a lane: two.  (Paired dims read again, each wave its own cosines: one head
// 105 us over 8192 tokens, two 83, four 88; waves that go on from token to token 191.
// Four of 64 with register moves: 54 us over 5 prompts, as two.)
constexpr int kAppendRows = 2;
// Queries of more than this are stored past the caches, as rotary_embedding's (5
// prompts into mxfp4 58 -> 54 us, 8192 tokens 67.5 -> 66).
constexpr long long kAppendStreamBytes = 32ll << 20;

// Scaled cosine and sine of position * frequency.  32 bits hold what is left of the
// angle behind quarter turns, within 2^-28 of a turn, below what the products round.
// (Behind whole turns, 2^-26: 1.6 to 1.8 times as many keys round to another value
// than those of exact angles.)  Up to an eighth of a turn a, sin a and cos a are their
// power series up to a^9 and a^10: the next terms are 2e-9 of them.
__device__ __forceinline__ float2 fine_turn(long long pos, double f, float scale) {
  const double quarters = (double)pos * f * 0.63661977236758134307553505349;
  const double n = rint(quarters);
  const float r = (float)(quarters - n), t = r * r;
  constexpr double H = 1.57079632679489661923132169164, H2 = H * H;  // a = H r
  constexpr float S1 = (float)H, R1 = (float)(H - (double)S1), S3 = (float)(-H * H2 / 6), S5 = (float)(H * H2 * H2 / 120),
                  S7 = (float)(-H * H2 * H2 * H2 / 5040), S9 = (float)(H * H2 * H2 * H2 * H2 / 362880);
  constexpr float C2 = (float)(-H2 / 2), C4 = (float)(H2 * H2 / 24), C6 = (float)(-H2 * H2 * H2 / 720),
                  C8 = (float)(H2 * H2 * H2 * H2 / 40320), C10 = (float)(-H2 * H2 * H2 * H2 * H2 / 3628800);
  const float s = fmaf(r, S1, r * fmaf(t, fmaf(t, fmaf(t, fmaf(t, S9, S7), S5), S3), R1));  // (H is S1 + R1)
  const float c = fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, C10, C8), C6), C4), C2), 1.f);
  const int k = (int)(n - 4.0 * floor(0.25 * n));
  const float x = k & 1 ? -s : c, y = k & 1 ? c : s;
  return k & 2 ? float2{-x * scale, -y * scale} : float2{x * scale, y * scale};
}

// x of another lane of the wave's row of 16 (all lanes take part)
template <int CTRL>
__device__ __forceinline__ float lane_move(float x) {
  return __uint_as_float((unsigned)__builtin_amdgcn_mov_dpp((int)__float_as_uint(x), CTRL, 0xF, 0xF, true));
}
constexpr int kQuadXor1 = 0xB1, kQuadXor2 = 0x4E, kQuadXor3 = 0x1B, kHalfMirror = 0x141, kMirror = 0x140, kTurn8 = 0x128;

// Sum over the 2^log2_lanes lanes of a head, the same in all of them.
__device__ __forceinline__ float head_sum(float x, int log2_lanes) {
  x += lane_move<kQuadXor1>(x);
  x += lane_move<kQuadXor2>(x);
  if (log2_lanes > 2) x += lane_move<kHalfMirror>(x);
  if (log2_lanes > 3) x += lane_move<kMirror>(x);
  if (log2_lanes > 4) x += __shfl_xor(x, 16);
  return x;
}

// x of lane ^ (1, 2, 4 or 8)
__device__ __forceinline__ void across(const float (&x)[8], float (&y)[8], int lanes) {
  auto move = [&](auto f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = f(x[i]);
  };
  if (lanes == 8) move([](float v) { return lane_move<kTurn8>(v); });
  else if (lanes == 4) move([](float v) { return lane_move<kQuadXor3>(lane_move<kHalfMirror>(v)); });  // 7 - lane, 3 - lane
  else if (lanes == 2) move([](float v) { return lane_move<kQuadXor2>(v); });
  else move([](float v) { return lane_move<kQuadXor1>(v); });
}

__device__ __forceinline__ float bf16_at(const uint16_t* p) { return __uint_as_float((unsigned)*p << 16); }

// (bf16 fits eight waves on a SIMD if asked to, 8192 tokens 83 -> 80.6 us before the
// above; for the others that sets scalar registers aside, 5 prompts 58 -> 61.)
template <int FMT, bool NEAR, bool STREAM>
__global__ __launch_bounds__(64 * kAppendWaves, NEAR && FMT == CACHE_BF16 ? 8 : 1) void cache_append_kernel(const AppendParams p) {
  __shared__ float2 turns[kAppendWaves][kRotaryMaxPairs];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long unit = (long long)blockIdx.x * kAppendWaves + wv;
  const int num_tokens = p.c.num_items, hq = p.num_qo_heads, hkv = p.c.num_kv_heads, D = p.c.head_dim;
  if (unit >= (long long)num_tokens * p.runs) return;  // (no barrier below: waves are on their own)
  const int t = (int)(unit / p.runs);
  const int h0 = (int)(unit - (long long)t * p.runs) * p.heads_per_run, h1 = min(h0 + p.heads_per_run, hq + 2 * hkv);
  const int lph = 1 << p.log2_lanes;  // lanes of a head
  const int d = 8 * (lane & (lph - 1));
  const int pairs = p.pairs, turning = 2 * pairs;
  // eight pairs whose other elements are eight neighbours too
  const bool wide = !p.interleaved && (NEAR || pairs % 8 == 0);
  const int mate = d < pairs ? d + pairs : d - pairs;
  const bool turns_any = h0 < hq + hkv;

  // the rows' loads first: they do not wait for the place they go to
  u32x4 own[kAppendRows], other[kAppendRows];
  const uint16_t* row[kAppendRows];
  int head[kAppendRows];  // of q, of k plus hq, of v plus hq + hkv; -1: none
  const uint16_t* const q_row = (const uint16_t*)p.q + (long long)t * p.q_stride_n;
  const uint16_t* const k_row = (const uint16_t*)p.c.k + (long long)t * p.c.stride_n;
  const uint16_t* const v_row = (const uint16_t*)p.c.v + (long long)t * p.v_stride_n;
#pragma unroll
  for (int u = 0; u < kAppendRows; ++u) {
    const int h = h0 + (u << (6 - p.log2_lanes)) + (lane >> p.log2_lanes);
    head[u] = h < h1 && d < D ? h : -1;
    own[u] = other[u] = u32x4{0u, 0u, 0u, 0u};
    row[u] = nullptr;
    if (head[u] < 0) continue;
    row[u] = h < hq         ? q_row + (long long)h * p.q_stride_h
             : h < hq + hkv ? k_row + (long long)(h - hq) * p.c.stride_h
                            : v_row + (long long)(h - hq - hkv) * p.v_stride_h;
    own[u] = *(const u32x4*)(row[u] + d);
    if (!NEAR && wide && d < turning && h < hq + hkv) other[u] = *(const u32x4*)(row[u] + mate);
  }

  const int4 tok = ((const int4*)p.c.items)[t];
  const int place = p.c.kv_len[tok.x] - tok.y;  // the token's position in its cache
  int page = -1;
  if (h1 > hq) {
    const int behind = place >> p.c.log2_page;
    // (before the cache's start, or no page is reserved for it: nothing to write)
    if (place >= 0 && behind < tok.w - tok.z) page = p.c.page_table[tok.z + behind];
    if (page >= p.c.num_pages) page = -1;
  }
  const int slot = place & ((1 << p.c.log2_page) - 1);
  const long long cell = page * p.c.stride_page + slot * p.c.stride_tok;  // of head 0
  const long long scell = page * p.c.scale_stride_page + slot * p.c.scale_stride_tok;
  float2* turn = turns[wv];
  if (turns_any) {
    const long long pos = !p.positions ? (long long)place
                          : p.pos64    ? ((const long long*)p.positions)[t]
                                       : (long long)((const int*)p.positions)[t];
    for (int i = lane; i < pairs; i += 64) turn[i] = fine_turn(pos, p.inv_freq[i], p.scale);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();

#pragma unroll
  for (int u = 0; u < kAppendRows; ++u) {
    const int h = head[u];
    const bool is_q = h >= 0 && h < hq, is_k = h >= hq && h < hq + hkv;
    float x[8], y[8], pre = 1.f, inv = 1.f;
    if (turns_any) {
      expand8(own[u], x);
      if (!NEAR) expand8(other[u], y);
      if (p.q_norm || p.k_norm) {
        // (every lane takes part; heads without a norm drop the result)
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
        ss = head_sum(ss, p.log2_lanes);
        const uint16_t* weight = (const uint16_t*)(is_q ? p.q_norm : is_k ? p.k_norm : nullptr);
        if (__any(isinf(ss))) {  // values above 2^59: all of them 2^64 smaller
          const bool large = isinf(ss);
          float small = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) small = fmaf(x[i] * 0x1p-64f, x[i] * 0x1p-64f, small);
          small = head_sum(small, p.log2_lanes);
          if (large && weight) {
            pre = 0x1p-64f, ss = small;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] *= pre, y[i] = NEAR ? 0.f : y[i] * pre;
          }
        }
        if (weight) {
          inv = rsqrtf(ss / (float)D + p.eps * pre * pre);
          float w[8];
          expand8(*(const u32x4*)(weight + d), w);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * w[i];
          if (!NEAR && wide && d < turning) {
            expand8(*(const u32x4*)(weight + mate), w);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = y[i] * inv * w[i];
          }
        }
      }
      if (NEAR && wide) across(x, y, pairs >> 3);
    }
    if (h < 0) continue;
    if (h >= hq + hkv) {
      if (page >= 0) {
        const int hv = h - hq - hkv;
        store_piece<FMT>(p.c.vs, hv, cell + hv * p.c.stride_head, scell + hv * p.c.scale_stride_head, d, own[u]);
      }
      continue;
    }
    if (d < turning) {
      if (wide) {
        const float2* cs = turn + (d < pairs ? d : mate);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 c = cs[i];
          x[i] = fmaf(d < pairs ? -y[i] : y[i], c.y, x[i] * c.x);
        }
      } else if (p.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (d + 2 * i >= turning) continue;
          const float2 c = turn[d / 2 + i];
          const float a = x[2 * i], b = x[2 * i + 1];
          x[2 * i] = a * c.x - b * c.y;
          x[2 * i + 1] = b * c.x + a * c.y;
        }
      } else if constexpr (!NEAR) {
        // (pairs that come in no eights: one element at a time)
        const uint16_t* weight = (const uint16_t*)(is_q ? p.q_norm : p.k_norm);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int e = d + i;
          if (e >= turning) continue;
          const int m = e < pairs ? e + pairs : e - pairs;
          const float2 c = turn[e < pairs ? e : m];
          float b = bf16_at(row[u] + m);
          if (weight) b = b * pre * inv * bf16_at(weight + m);
          x[i] = x[i] * c.x + (e < pairs ? -b : b) * c.y;
        }
      }
    }
    if (is_q) {
      u32x4* at = (u32x4*)((uint16_t*)p.q_out + (long long)t * p.qo_stride_n + (long long)h * p.qo_stride_h + d);
      const u32x4 out = {pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
      if constexpr (STREAM)
        __builtin_nontemporal_store(out, at);
      else
        *at = out;
    } else {
      const int hk = h - hq;
      store_values<FMT>(p.c.ks, hk, cell + hk * p.c.stride_head, scell + hk * p.c.scale_stride_head, d, x, page >= 0);
    }
  }
}

template <int FMT, bool NEAR>
void launch_t(const AppendParams& p, bool stream, unsigned grid, hipStream_t s) {
  const dim3 g(grid), block(64 * kAppendWaves);
  if (stream)
    hipLaunchKernelGGL((cache_append_kernel<FMT, NEAR, true>), g, block, 0, s, p);
  else
    hipLaunchKernelGGL((cache_append_kernel<FMT, NEAR, false>), g, block, 0, s, p);
}

template <int FMT>
void launch_f(const AppendParams& p, bool near, bool stream, unsigned grid, hipStream_t s) {
  near ? launch_t<FMT, true>(p, stream, grid, s) : launch_t<FMT, false>(p, stream, grid, s);
}

}  // namespace

hipError_t launch_cache_append(AppendParams p, int format, hipStream_t s) {
  if (p.c.num_items <= 0) return hipSuccess;
  p.log2_lanes = 2;  // head dims come in thirty-twos
  while ((8 << p.log2_lanes) < p.c.head_dim) ++p.log2_lanes;
  p.heads_per_run = kAppendRows * (64 >> p.log2_lanes);
  p.runs = (p.num_qo_heads + 2 * p.c.num_kv_heads + p.heads_per_run - 1) / p.heads_per_run;
  const long long grid = ((long long)p.c.num_items * p.runs + kAppendWaves - 1) / kAppendWaves;
  if (grid > 0x7FFFFFFFll) return hipErrorInvalidValue;
  const bool stream = 2ll * p.c.num_items * p.num_qo_heads * p.c.head_dim > kAppendStreamBytes;
  const bool near = p.interleaved || p.pairs == 8 || p.pairs == 16 || p.pairs == 32 || p.pairs == 64;
  switch (format) {
    case CACHE_BF16: launch_f<CACHE_BF16>(p, near, stream, (unsigned)grid, s); break;
    case CACHE_FP8: launch_f<CACHE_FP8>(p, near, stream, (unsigned)grid, s); break;
    case CACHE_MXFP8: launch_f<CACHE_MXFP8>(p, near, stream, (unsigned)grid, s); break;
    case CACHE_MXFP4: launch_f<CACHE_MXFP4>(p, near, stream, (unsigned)grid, s); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace d2sd
