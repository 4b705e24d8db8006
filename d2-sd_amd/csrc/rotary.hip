// gfx950 kernel: rotary embedding of queries and keys at their positions, with
// the angles computed in the kernel (no table of cosines, no longest position).
//
//   (a, b) -> s (a cos t - b sin t, b cos t + a sin t),  t = position * f
//
// for the pairs (a, b) = (x[i], x[i + r/2]) (half layout) or (x[2i], x[2i + 1])
// (interleaved) of a head's first r dims; the other dims pass through.  t is
// taken in turns: position * (f / 2 pi) in 64 bits (off by 2^-53 of the turns
// made, 1e-9 turns at a million turns), its fraction of a turn in 32; a 32-bit
// angle would be off by 0.06 radians at a position of a million.  The products
// are 32-bit, rounded to bf16 once.
//
// A wave owns one token and a run of its heads: lane i computes the cosine and
// sine of pair i (and i + 64), through LDS all its heads share them.  A slot
// (lane) holds VEC pairs of one head: two 16-byte loads and stores for rows on
// 16-byte boundaries, else one element at a time.  Bound by HBM for prompts
// (q and k once in, once out) and by latency for a step's few tokens.  A wave
// takes only as many heads as one slot per lane covers: the sines (about 100
// instructions) cost less than a second round of loads (8192 tokens of 72 heads
// of 64, all heads in one wave: 29.5 us, this way 26.2; 1024 tokens of 40 heads
// of 128: 7.2 and 5.6).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "d2sd_internal.h"
#include "kernel_common.h"
#include "plan.h"

namespace d2sd {

namespace {

constexpr int kRotaryWaves = 4;
// Results larger than the L2s together are stored past the caches (8192 tokens of
// 72 heads of 64: 31.3 -> 26.3 us, 5.7 TB/s; the kernels that read them next take
// as long either way).
constexpr long long kRotaryStreamBytes = 32ll << 20;

// bf16 of two floats, rounded to nearest even, as one word
__device__ __forceinline__ unsigned pack2(float a, float b) { return pack_bf16x2(a, b); }

template <int VEC, bool INTER, bool STREAM>
__global__ __launch_bounds__(64 * kRotaryWaves) void rotary_kernel(const RotaryParams p) {
  __shared__ float2 turn[kRotaryWaves][kRotaryMaxPairs];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const long long unit = (long long)blockIdx.x * kRotaryWaves + wv;
  if (unit >= (long long)p.num_tokens * p.runs) return;  // (no barrier below: waves are on their own)
  const int t = (int)(unit / p.runs);
  const int run = (int)(unit - (long long)t * p.runs);
  const int h0 = run * p.heads_per_run, h1 = min(h0 + p.heads_per_run, p.num_qo_heads + p.num_kv_heads);
  const long long pos = p.pos64 ? ((const long long*)p.positions)[t] : (long long)((const int*)p.positions)[t];
  for (int i = lane; i < p.pairs; i += 64) {
    const double turns = (double)pos * p.inv_freq[i] * 0.15915494309189533576888376337251;
    const float f = (float)(turns - rint(turns));  // [-0.5, 0.5] of a turn
    float s, c;
    sincospif(2.f * f, &s, &c);
    turn[wv][i] = float2{c * p.scale, (p.inverse ? -s : s) * p.scale};
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const int slots = p.head_dim / (2 * VEC), turning = p.pairs / VEC;
  const int total = (h1 - h0) * slots;
  int h = h0 + lane / slots, slot = lane % slots;
  const int dh = 64 / slots, ds = 64 % slots;
  for (int i = lane; i < total; i += 64) {
    const bool is_k = h >= p.num_qo_heads;
    const int hh = is_k ? h - p.num_qo_heads : h;
    const uint16_t* x = (const uint16_t*)(is_k ? p.k : p.q) + (long long)t * (is_k ? p.k_stride_n : p.q_stride_n) +
                        (long long)hh * (is_k ? p.k_stride_h : p.q_stride_h);
    uint16_t* y = (uint16_t*)(is_k ? p.k_out : p.q_out) +
                  (long long)t * (is_k ? p.ko_stride_n : p.qo_stride_n) +
                  (long long)hh * (is_k ? p.ko_stride_h : p.qo_stride_h);
    const bool rot = slot < turning;
    // the slot's two runs of VEC elements
    const int a = !rot || INTER ? 2 * VEC * slot : VEC * slot;
    const int b = !rot || INTER ? a + VEC : a + p.pairs;
    if (rot || p.copy_rest) {
      if constexpr (VEC == 8) {
        const u32x4 ua = *(const u32x4*)(x + a), ub = *(const u32x4*)(x + b);
        u32x4 oa = ua, ob = ub;
        if (rot) {
          const float2* cs = &turn[wv][VEC * slot];
          if constexpr (INTER) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 c0 = cs[e], c1 = cs[4 + e];
              const float a0 = bf16_lo(ua[e]), b0 = bf16_hi(ua[e]), a1 = bf16_lo(ub[e]), b1 = bf16_hi(ub[e]);
              oa[e] = pack2(a0 * c0.x - b0 * c0.y, b0 * c0.x + a0 * c0.y);
              ob[e] = pack2(a1 * c1.x - b1 * c1.y, b1 * c1.x + a1 * c1.y);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 c0 = cs[2 * e], c1 = cs[2 * e + 1];
              const float a0 = bf16_lo(ua[e]), a1 = bf16_hi(ua[e]), b0 = bf16_lo(ub[e]), b1 = bf16_hi(ub[e]);
              oa[e] = pack2(a0 * c0.x - b0 * c0.y, a1 * c1.x - b1 * c1.y);
              ob[e] = pack2(b0 * c0.x + a0 * c0.y, b1 * c1.x + a1 * c1.y);
            }
          }
        }
        if constexpr (STREAM) {
          __builtin_nontemporal_store(oa, (u32x4*)(y + a));
          __builtin_nontemporal_store(ob, (u32x4*)(y + b));
        } else {
          *(u32x4*)(y + a) = oa;
          *(u32x4*)(y + b) = ob;
        }
      } else {
        const uint16_t wa = x[a], wb = x[b];
        unsigned o = (unsigned)wa | (unsigned)wb << 16;
        if (rot) {
          const float2 c = turn[wv][slot];
          const float fa = __uint_as_float((unsigned)wa << 16), fb = __uint_as_float((unsigned)wb << 16);
          o = pack2(fa * c.x - fb * c.y, fb * c.x + fa * c.y);
        }
        y[a] = (uint16_t)o;
        y[b] = (uint16_t)(o >> 16);
      }
    }
    h += dh;
    slot += ds;
    if (slot >= slots) {
      slot -= slots;
      ++h;
    }
  }
}

template <int VEC, bool STREAM>
hipError_t launch_t(const RotaryParams& p, bool interleaved, unsigned grid, hipStream_t s) {
  if (interleaved)
    hipLaunchKernelGGL((rotary_kernel<VEC, true, STREAM>), dim3(grid), dim3(64 * kRotaryWaves), 0, s, p);
  else
    hipLaunchKernelGGL((rotary_kernel<VEC, false, STREAM>), dim3(grid), dim3(64 * kRotaryWaves), 0, s, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_rotary(RotaryParams p, bool interleaved, hipStream_t s) {
  const int heads = p.num_qo_heads + p.num_kv_heads;
  if (p.num_tokens <= 0 || heads <= 0) return hipSuccess;
  // 16-byte slots where every row starts on a 16-byte boundary and pairs come in eights
  const uintptr_t at = (uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.q_out | (uintptr_t)p.k_out;
  const long long st = p.q_stride_n | p.q_stride_h | p.k_stride_n | p.k_stride_h | p.qo_stride_n | p.qo_stride_h |
                       p.ko_stride_n | p.ko_stride_h;
  const bool vec = (at & 15) == 0 && (st & 7) == 0 && p.head_dim % 16 == 0 && p.pairs % 8 == 0;
  const int slots = p.head_dim / (vec ? 16 : 2);
  p.heads_per_run = slots >= 64 ? 1 : 64 / slots;  // those that one pass of a wave covers
  p.runs = (heads + p.heads_per_run - 1) / p.heads_per_run;
  const long long grid = ((long long)p.num_tokens * p.runs + kRotaryWaves - 1) / kRotaryWaves;
  if (grid > 0x7FFFFFFFll) return hipErrorInvalidValue;
  if (!vec) return launch_t<1, false>(p, interleaved, (unsigned)grid, s);
  const bool stream = 2ll * p.num_tokens * heads * p.head_dim > kRotaryStreamBytes;
  return stream ? launch_t<8, true>(p, interleaved, (unsigned)grid, s) : launch_t<8, false>(p, interleaved, (unsigned)grid, s);
}

}  // namespace d2sd
