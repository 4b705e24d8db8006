// Shared keys against the rows of a whole group of requests, where every row sees
// all of them: the inner loop of chunk_attention.hip's plans with shared keys
// (included there, in the namespace of its kernels).
//
// A wave works through its keys in halves of a 64-key tile.  Two regions of MFMAs
// a half, each with other work placed between them in a pinned order:
//   1. O^T += V^T P^T of half h - 1, beside the rest of its exponentials, the reads
//      of K for half h + 1, and scaling and row maximum of half h's scores;
//   2. S^T = K Q^T of half h + 1, beside most of half h's exponentials and the reads
//      of V for half h.
// The offset of the exponents, mc, trails the true maximum by up to 2^kRescaleSlack;
// scores are scaled and offset before their maximum is taken (x = s c - mc, one
// fma), so that the maximum needs no instruction to quiet a NaN and the usual half,
// whose maximum stays below the slack, goes on to 2^x as it is.
//
// Everything reaches LDS by direct copies, several tiles ahead.  bf16 tiles go into
// rings of slots, K two steps further ahead than they are worked on, V one (W = 4;
// one more each with 8 waves).  Codes and block scales go into a ring of bundles (K
// of a tile, V of the tile before it), from which each thread expands one segment of
// K and one of V a tile into two slots each: loaded through registers instead, a tile
// and a half ahead, tiles took 2.7 us in mxfp8 where memory was busy, and registers
// spilled.  One barrier a tile.
//
// Bound by MFMA and, with all CUs at work, by the clock that power leaves: 256 rows x
// 64 keys of 128 dims take a CU 1.4 to 1.6 us while half of the others idle, 1.7 in
// bf16 and 1.9 quantised with all of them, 1.25 PFLOP/s, 92% of a large library
// product; tile_item's loop took 2.0 to 3.3.
#pragma once

// LDS of the tiles.  bf16: KST slots of K, VST of V, the LDS share of a workgroup (two
// on a CU; W = 8: one).  Quantised: two of each and RD bundles.
template <int D, int FMT, int W>
struct SharedRing {
  static constexpr bool BF16 = FMT == CACHE_BF16, MX = Format<D, FMT>::MX;
  static constexpr int KST = !BF16 ? 2 : D == 64 ? 5 : W == 8 ? 4 : 3, VST = BF16 ? KST - 1 : 2;
  static constexpr int TB = 64 * D * 2, CODES = 64 * Format<D, FMT>::ROW;  // bytes of a tile, of its codes
  static constexpr int RD = BF16 ? 0 : 4, BUNDLE = 2 * CODES + (MX ? 2 * 64 * 4 : 0);
  static constexpr int bytes = (KST + VST) * TB + RD * BUNDLE;
};

// vmcnt <= k * UNIT for a wave-uniform k in [0, MAXK]
template <int UNIT, int MAXK>
__device__ __forceinline__ void wait_copies(int k) {
  static_for<MAXK + 1>([&](auto i) {
    if (k == decltype(i)::value) wait_vmcnt<decltype(i)::value * UNIT>();
  });
}

// Whether shared_tile takes the cache's pages: the rows of a quantised copy (at most
// two runs of them) share a page, and block scales lie on boundaries of their copies.
template <int D, int FMT, int W>
__device__ __forceinline__ bool shared_tile_takes(const ChunkParams& p, int kb0) {
  if constexpr (FMT == CACHE_BF16) return true;
  constexpr int RPI = 1024 / Format<D, FMT>::ROW;
  bool ok = (kb0 & 63) == 0 && (1 << p.log2_page) >= (RPI > 16 ? RPI / 2 : RPI) && (1 << p.log2_page) >= 64 / W;
  if constexpr (Format<D, FMT>::MX) {
    constexpr unsigned A = D / 32 - 1;  // one copy a row: 4 or 2 bytes
    ok = ok && (((unsigned)(uintptr_t)p.ks.scale | (unsigned)(uintptr_t)p.vs.scale | p.scale_stride_page | p.scale_stride_tok |
                 (unsigned)p.scale_stride_head) & A) == 0;
  }
  return ok;
}

// Keys [kb0, ke) of the item's pages, kb0 < ke, all seen by all of its rows.
template <int D, int FMT, int W>
__device__ __forceinline__ void shared_tile(const ChunkParams& p, const ChunkItem& w, lds_char* lds, int kb0, int ke) {
  constexpr bool BF16 = FMT == CACHE_BF16, MX = Format<D, FMT>::MX;
  constexpr int MT = D / 32, KS = D / 16, NPV = 2 * MT, TB = 64 * D * 2;
  typedef SharedRing<D, FMT, W> Ring;
  constexpr int KST = Ring::KST, VST = Ring::VST;
  static_assert(KS == NPV, "a fragment is used up per slot");
  const int tid = threadIdx.x, wv = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l32 = lane & 31, hh = lane >> 5;
  const int nt = (ke - kb0 + 63) >> 6;
  const bool live = 32 * wv < w.nrows;  // (waves without rows copy and keep the barriers)
  const unsigned kring = lds_address((const void*)lds), vring = kring + KST * TB;
  const unsigned last_page = (unsigned)p.num_pages - 1u;
  const int pmask = (1 << p.log2_page) - 1;
  const char* kbase = (const char*)p.ks.codes + w.kvh * p.stride_head;
  const char* vbase = (const char*)p.vs.codes + w.kvh * p.stride_head;
  float c = p.sm_scale * kLog2e, vscale = 1.f;
  if constexpr (FMT == CACHE_FP8) {
    c *= ((const float*)p.ks.scale)[w.kvh];
    vscale = ((const float*)p.vs.scale)[w.kvh];
  }

  f32x16 o[MT], sc, sp;  // scores of half h; of half h - 1
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) o[mt] = f32x16{};
  bf16x8 qf[KS], kf[KS], vf[NPV];  // rows; K of half h + 1; V^T of half h - 1
  u32x4 pc[2];                     // P^T of half h - 1 (bf16)
  float l4[4] = {0.f, 0.f, 0.f, 0.f}, mc = 0.f, grow_at = -INFINITY;

  // fragment addresses in the K and V slots being read, stepped from slot to slot
  // (ValueRead has the layout of V^T)
  unsigned ka[KS], va0[MT], va1[MT];
  unsigned kstep = 0, vstep = 0;
  auto kread = [&](int kt, int ks) -> bf16x8 {
    return *(const __attribute__((address_space(3))) bf16x8*)(uintptr_t)(ka[ks] + kt * 32 * D * 2);
  };
  auto vread = [&](int mt, int j) -> bf16x8 {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(va0[mt] + j * 16 * D * 2));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(va1[mt] + j * 16 * D * 2));
    const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
    return __builtin_bit_cast(bf16x8, (u32x4){a[0], a[1], b[0], b[1]});
  };
  auto koff = [&](int ks) -> unsigned { return (l32 * D + 8 * ((2 * ks + hh) ^ chunk_swizzle<D>(l32))) * 2; };
  auto sched_fence = [] { __builtin_amdgcn_sched_barrier(0); };
  using std::false_type;
  using std::true_type;

  // A half's exponentials: eight words (pairs of keys) in two stages, word w's from
  // slot word_slot(w) on, counted from region 2's first; sums are in 32 bits, before
  // the probabilities are rounded to bf16 as the second product's operands (V is bf16 at
  // most, its product with 32-bit ones would take two MFMAs for one; outputs are 0.0020
  // to 0.0024 from 64-bit ones in the mean, 0.0017 of it their own rounding).
  constexpr auto word_slot = [](int i) { return KS == 8 ? 3 * i / 2 : 2 * i / 3; };
  static_assert(word_slot(3) + 1 < KS && word_slot(7) + 1 < KS + MT, "words ready before their PV");
  auto words = [&](auto tc, f32x16& s) {
    constexpr int T = decltype(tc)::value;
    static_for<8>([&](auto wc) {
      constexpr int i = decltype(wc)::value;
      if constexpr (word_slot(i) + 1 == T) {
        l4[(2 * i) & 3] += s[2 * i];
        l4[(2 * i + 1) & 3] += s[2 * i + 1];
        pc[i >> 2][i & 3] = pack_bf16x2(s[2 * i], s[2 * i + 1]);
      }
      if constexpr (word_slot(i) == T) {
        s[2 * i] = __builtin_amdgcn_exp2f(s[2 * i]);
        s[2 * i + 1] = __builtin_amdgcn_exp2f(s[2 * i + 1]);
      }
    });
  };
  // The next region's fragments that are read before slot i.
  constexpr auto reads_before = [](int i) {
    return KS == 8 ? (i < 2 ? i : i < 4 ? 2 * i - 2 : i < 6 ? i + 2 : KS) : (2 * i < KS ? 2 * i : KS);
  };
  // prev: half h - 1 exists; next: kload(ks) reads K of half h + 1; tail: keys of the
  // half that starts at kh may lie behind the range; aside(slot): other work
  auto region1 = [&](auto prev, auto next, auto&& kload, auto tail, int kh, auto&& aside) {
    constexpr bool PREV = decltype(prev)::value, NEXT = decltype(next)::value;
    float mx[5];
    constexpr int F0 = KS == 8 ? 1 : 0, FN = KS == 8 ? 4 : 2;  // slots that scale: FN from F0 on
    constexpr int L0 = NPV == 8 ? 5 : 2;                       // first level of the maximum
    wait_lgkm0();
    sched_fence();
    static_for<NPV>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      if constexpr (PREV)
        o[i % MT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[i], __builtin_bit_cast(bf16x8, pc[i / MT]), o[i % MT], 0, 0, 0);
      if constexpr (NEXT)
        static_for<reads_before(i + 1) - reads_before(i)>([&](auto kk) {
          constexpr int ks = reads_before(i) + decltype(kk)::value;
          kf[ks] = kload(ks);
        });
      if constexpr (PREV) words(std::integral_constant<int, KS + i>{}, sp);
      if constexpr (i >= F0 && i < F0 + FN) {
#pragma unroll
        for (int e = (i - F0) * 16 / FN; e < (i - F0 + 1) * 16 / FN; ++e) sc[e] = fmaf(sc[e], c, -mc);
      }
      if constexpr (i == F0 + FN - 1 && decltype(tail)::value) {
        if (ke - kh < 32) {
#pragma unroll
          for (int e = 0; e < 16; ++e) sc[e] = kh + 8 * (e >> 2) + 4 * hh + (e & 3) < ke ? sc[e] : -INFINITY;
        }
      }
      if constexpr (i == L0) {
#pragma unroll
        for (int m = 0; m < 5; ++m) mx[m] = fmaxf(fmaxf(sc[3 * m], sc[3 * m + 1]), sc[3 * m + 2]);
      }
      if constexpr (i == L0 + 1) {
        mx[0] = fmaxf(fmaxf(mx[0], mx[1]), mx[2]);
        mx[0] = fmaxf(mx[0], fmaxf(fmaxf(mx[3], mx[4]), sc[15]));
      }
      aside(ic);
      sched_fence();
    });
    const float top = fmaxf(mx[0], xor32(mx[0], hh));
    if (__builtin_expect(__any(top > grow_at), PREV ? 0 : 1)) {
      // (rows whose maximum is below their offset keep it; nothing to scale yet
      // where a row has none)
      const bool none = grow_at == -INFINITY;
      const float to = none ? top : mc + fmaxf(top, 0.f);
      const float d = none ? top : to - mc;
      const float a = none ? 0.f : __builtin_amdgcn_exp2f(-d);
      if (none && !(top > -INFINITY)) {
        // (no key above -inf so far)
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] -= d;
#pragma unroll
        for (int e = 0; e < 4; ++e) l4[e] *= a;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) o[mt] *= a;
        mc = to;
        grow_at = kRescaleSlack;
      }
    }
  };
  auto region2 = [&](auto next, auto&& vload, auto&& aside) {
    f32x16 sn;
    wait_lgkm0();
    sched_fence();
    static_for<KS>([&](auto ic) {
      constexpr int ks = decltype(ic)::value;
      if constexpr (decltype(next)::value)
        sn = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[ks], qf[ks], ks == 0 ? f32x16{} : sn, 0, 0, 0);
      static_for<reads_before(ks + 1) - reads_before(ks)>([&](auto vv) {
        constexpr int i = reads_before(ks) + decltype(vv)::value;
        vf[i] = vload(i % MT, i / MT);
      });
      words(ic, sc);
      aside(ic);
      sched_fence();
    });
    sp = sc;
    if constexpr (decltype(next)::value) sc = sn;
  };
  auto nothing = [](auto) {};
  // first tile's addresses, its first half's scores and its second half's K
  auto start_tiles = [&]() {
    const int row = 4 * hh + ((lane & 15) >> 2), dsub = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) ka[ks] = kring + koff(ks);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int d = 32 * mt + dsub;
      va0[mt] = vring + (row * D + 8 * ((d >> 3) ^ chunk_swizzle<D>(row)) + (d & 7)) * 2;
      va1[mt] = vring + ((row + 8) * D + 8 * ((d >> 3) ^ chunk_swizzle<D>(row + 8)) + (d & 7)) * 2;
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const bf16x8 a0 = kread(0, ks);
      kf[ks] = kread(1, ks);
      sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a0, qf[ks], ks == 0 ? f32x16{} : sc, 0, 0, 0);
    }
  };
  // in region 1 of a tile's first half: K is read in its first slots, V after it
  auto step_addresses = [&](auto ic, auto first) {
    constexpr int i = decltype(ic)::value;
    static_for<KS>([&](auto kc) {
      constexpr int ks = decltype(kc)::value;
      if constexpr (NPV / 2 + ks * (NPV / 2) / KS == i) ka[ks] += kstep;
    });
    if constexpr (!decltype(first)::value && i < MT) va0[i] += vstep, va1[i] += vstep;
  };
  auto tile_barrier = [&]() {
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __asm__ volatile("" ::: "memory");
  };
  auto half_finish = [&]() {
    static_for<NPV>([&](auto ic) { words(std::integral_constant<int, KS + decltype(ic)::value>{}, sp); });
#pragma unroll
    for (int i = 0; i < NPV; ++i)
      o[i % MT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[i], __builtin_bit_cast(bf16x8, pc[i / MT]), o[i % MT], 0, 0, 0);
  };
  // the last tile's second half, and what is left of the last half
  auto finish = [&]() {
    const int last = kb0 + (nt - 1) * 64 + 32;
    if (last < ke) {
      region1(true_type{}, false_type{}, [&](int) { return zero_bf16x8(); }, true_type{}, last, nothing);
      region2(false_type{}, [&](int mt, int j) { return vread(mt, 2 + j); }, nothing);
    }
    half_finish();
  };

  if constexpr (BF16) {
    constexpr int CH = D / 8, RPI = 64 / CH;        // chunks of a row; rows of a 1 KB copy
    constexpr int IPW = 64 / RPI / W;               // copies of a tile per wave
    constexpr int WROWS = IPW * RPI;                // rows of a tile that a wave copies
    constexpr int MAXK = 1 + (VST - 2) + (VST - 2);
    static_assert(IPW >= 1 && MAXK * IPW < 64, "vmcnt range");
    const int lrow = lane / CH, cs = lane % CH;
    // A wave's rows of a whole tile share a page: its address stays in scalar
    // registers.  (Tiles start at multiples of 64 keys but where a window moves them.)
    const bool fast = (kb0 & 63) == 0 && (1 << p.log2_page) >= WROWS;
    unsigned lane_off[IPW];
#pragma unroll
    for (int i = 0; i < IPW; ++i)
      lane_off[i] = (unsigned)(RPI * i + lrow) * p.stride_tok + 16u * (cs ^ chunk_swizzle<D>(wv * WROWS + RPI * i + lrow));
    const int last_entry = w.page_begin + ((ke - 1) >> p.log2_page);
    typedef const __attribute__((address_space(4))) int const_int;
    // page of the wave's rows of tile `it` (behind the range: its last page)
    auto wave_page = [&](int it) -> int {
      return ((const_int*)p.page_table)[min(w.page_begin + ((kb0 + it * 64 + wv * WROWS) >> p.log2_page), last_entry)];
    };
    auto tile_base = [&](const char* base, int it, int page) -> const char* {
      return base + row_offset(p, min((unsigned)page, last_page), (unsigned)(kb0 + it * 64 + wv * WROWS) & pmask);
    };
    // keys behind the range: the last one again
    auto issue = [&](int it, int page, const char* base, unsigned slot) {
      const int kb = kb0 + it * 64;
      if (__builtin_expect(fast && kb + 64 <= ke, 1)) {
        const char* at = tile_base(base, it, page);
#pragma unroll
        for (int i = 0; i < IPW; ++i) dma16s_kept(at, lane_off[i], slot + (wv * IPW + i) * 1024);
      } else {
#pragma unroll
        for (int i = 0; i < IPW; ++i) {
          const int r = wv * WROWS + RPI * i + lrow, key = min(kb + r, ke - 1);
          const unsigned pg = min((unsigned)p.page_table[w.page_begin + (key >> p.log2_page)], last_page);
          dma16_kept(base + row_offset(p, pg, key & pmask) + 16 * (cs ^ chunk_swizzle<D>(r)), slot + (wv * IPW + i) * 1024);
        }
      }
    };
    auto issue_k = [&](int it, int page) { issue(it, page, kbase, kring + it % KST * TB); };
    auto issue_v = [&](int it, int page) { issue(it, page, vbase, vring + it % VST * TB); };

    // Rows of Q to slots that the first tiles leave free (K slots 2 .., then V slots
    // 1 ..), so that nothing waits for more than Q and K(0) (a load to registers
    // would be waited for with all copies in flight).  Issue order: K(0), Q, V(0), K(1),
    // then K(2), then V(j), K(j + 2); tile s's sync issues V(s + VST - 1), K(s + KST).
    constexpr int QB = 32 * D * 2, NQI = QB / 1024, QFREE = (KST - 2) * TB, QRPI = 1024 / (D * 2);
    static_assert(W * QB <= QFREE + (VST - 1) * TB && TB % QB == 0, "Q fits free slots");
    const unsigned qdst = wv * QB < QFREE ? kring + 2 * TB + wv * QB : vring + TB + (wv * QB - QFREE);
    {
      const int pg0 = wave_page(0);
      issue_k(0, pg0);
      const int g = p.group, lr = lane / (D / 8), qcs = lane % (D / 8), rows = w.nrows;
      // row -> (token, head) by one division, then in steps of QRPI rows
      int row = 32 * wv + lr;
      int qj = (w.row0 + row) % g;
      const long long sn = p.q_stride_n, sh = p.q_stride_h;
      const char* q0 = (const char*)((const bf16_t*)p.q + (long long)w.q0 * sn + (long long)w.kvh * g * sh);
      long long qoff = (long long)((w.row0 + row) / g) * sn + (long long)qj * sh;
      const int dj = QRPI % g;
      const long long dstep = (long long)(QRPI / g) * sn + (long long)dj * sh, wrap = sn - (long long)g * sh;
      const long long safe = (long long)(w.row0 / g) * sn + (long long)(w.row0 % g) * sh;  // the item's first row
#pragma unroll
      for (int i = 0; i < NQI && live; ++i) {
        dma16_kept(q0 + 2 * ((row < rows ? qoff : safe) + 8 * (qcs ^ chunk_swizzle<D>(i * QRPI + lr))), qdst + i * 1024);
        row += QRPI;
        qoff += dstep;
        qj += dj;
        if (qj >= g) qj -= g, qoff += wrap;
      }
      issue_v(0, pg0);
    }
    if (1 < nt) issue_k(1, wave_page(1));
    wait_copies<IPW, 2>(1 < nt ? 2 : 1);  // Q and K(0) have landed
    tile_barrier();
    if (live) {
      const lds_char* qs = (const lds_char*)(uintptr_t)qdst;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[ks] = *(const __attribute__((address_space(3))) bf16x8*)(qs + koff(ks));
    }
    wait_lgkm0();  // before the slots are refilled
    tile_barrier();
    if (2 < nt) issue_k(2, wave_page(2));
#pragma clang loop unroll(disable)
    for (int j = 1; j < VST - 1; ++j) {
      if (j < nt) issue_v(j, wave_page(j));
      if (j + 2 < nt) issue_k(j + 2, wave_page(j + 2));
    }
    // page ids of tiles it + VST - 1, it + VST and it + KST at tile it's sync
    int pgq[3] = {wave_page(VST - 1), wave_page(VST), wave_page(KST)};
    auto next_page = [&](int it) {
      pgq[0] = pgq[1];
      pgq[1] = pgq[2];
      pgq[2] = wave_page(it + KST);
    };
    // Copies that may be under way when tile `it` is needed: those issued after V(it).
    auto tile_outstanding = [&](int it) -> int {
      const int r = nt - 1 - it;
      return (r >= 2 ? 1 : 0) + min(r, VST - 2) + max(0, min(VST - 2, r - 2));
    };
    // Before V(it) and K(it + 1) are read: they have landed, for all waves, and the
    // slots of K(it) and V(it - 1), whose reads each wave has ended, are refilled.
    auto tile_sync = [&](int it) {
      wait_lgkm0();
      wait_copies<IPW, MAXK>(tile_outstanding(it));
      tile_barrier();
      if (it + VST - 1 < nt) issue_v(it + VST - 1, pgq[0]);
      if (it + KST < nt) issue_k(it + KST, pgq[2]);
    };
    if (!live) {
      for (int it = 0; it < nt; ++it) {
        tile_sync(it);
        next_page(it + 1);
      }
      return;
    }
    unsigned kslot = kring, vslot = vring;
    // spread: both tiles that the sync issues are whole: their copies go out
    // between the MFMAs of the step
    auto first_half = [&](int it, auto prev, auto spread) {
      constexpr bool FIRST = !decltype(prev)::value, SPREAD = decltype(spread)::value;
      const unsigned kfree = kslot, vfree = vslot;  // slots of K(it), V(it - 1)
      kstep = kslot + TB == vring ? 0u - (KST - 1) * TB : (unsigned)TB;
      kslot += kstep;
      if constexpr (!FIRST) {
        vstep = vslot + TB == vring + VST * TB ? 0u - (VST - 1) * TB : (unsigned)TB;
        vslot += vstep;
      }
      const char *sv = nullptr, *sk = nullptr;
      region1(prev, prev, [&](int ks) { return kread(1, ks); }, std::integral_constant<bool, !SPREAD>{}, kb0 + it * 64,
              [&](auto ic) {
                step_addresses(ic, std::integral_constant<bool, FIRST>{});
                if constexpr (SPREAD && decltype(ic)::value == 1) sv = tile_base(vbase, it + VST - 1, pgq[0]);
                if constexpr (SPREAD && decltype(ic)::value == 2) sk = tile_base(kbase, it + KST, pgq[2]);
              });
      if constexpr (SPREAD) {
        wait_lgkm0();
        wait_vmcnt<(1 + 2 * (VST - 2)) * IPW>();
        tile_barrier();
        region2(true_type{}, vread, [&](auto sc_) {
          static_for<2 * IPW>([&](auto ic) {
            constexpr int i = decltype(ic)::value % IPW;
            if constexpr (decltype(ic)::value * KS / (2 * IPW) == decltype(sc_)::value) {
              if constexpr (decltype(ic)::value < IPW)
                dma16s_kept(sv, lane_off[i], vfree + (wv * IPW + i) * 1024);
              else
                dma16s_kept(sk, lane_off[i], kfree + (wv * IPW + i) * 1024);
            }
          });
        });
      } else {
        tile_sync(it);
        region2(true_type{}, vread, nothing);
      }
    };
    auto second_half = [&](int it) {
      region1(true_type{}, true_type{}, [&](int ks) { return kread(0, ks); }, false_type{}, kb0 + it * 64 + 32, nothing);
      // (the next tile's page: a scalar load, waited for with the region's LDS reads)
      region2(true_type{}, [&](int mt, int j) { return vread(mt, 2 + j); }, [&](auto ic) {
        if constexpr (decltype(ic)::value == 0) next_page(it + 1);
      });
    };
    start_tiles();
    first_half(0, false_type{}, false_type{});
    const int whole = fast ? (ke - kb0) >> 6 : 0;
    int it = 1;
    for (; it + KST < whole; ++it) {
      second_half(it - 1);
      first_half(it, true_type{}, true_type{});
    }
    for (; it < nt; ++it) {
      second_half(it - 1);
      first_half(it, true_type{}, false_type{});
    }
    finish();
  } else {
    // A thread's segment of a tile: 16 elements, column `col` of row `row`, expanded
    // to two chunks.  Eight lanes beside each other hold four columns of a row and of
    // the fourth row behind it, whose chunks the swizzle moves to the odd places: they
    // write eight different 16-byte columns of the 128 bytes that LDS takes at a time.
    constexpr int ROW = Format<D, FMT>::ROW, SEG = D / 16, WORDS = FMT == CACHE_MXFP4 ? 2 : 4, SB = 4 * WORDS;
    static_assert(64 * SEG == 64 * W, "a segment of K and one of V for each thread");
    constexpr int RD = Ring::RD, BUNDLE = Ring::BUNDLE, CODES = Ring::CODES;
    const int col = (tid & 3) | (SEG == 8 ? tid >> 1 & 4 : 0);
    const int rest = SEG == 8 ? tid >> 4 : tid >> 3;
    const int row = (rest & 3) | (tid & 4) | (rest & ~3) << 1;
    const unsigned put0 = row * D * 2 + 16 * ((2 * col) ^ chunk_swizzle<D>(row)), put1 = put0 ^ 16;
    // Codes lie in a bundle as in their rows, rows of 128 bytes with their halves
    // exchanged in every other four, so that those eight lanes read from all of them.
    const unsigned half = ROW == 128 ? (row & 4) << 4 : 0;
    const unsigned raw = row * ROW + (col * SB ^ half);
    // dwords of scales: each wave's rows of K, then of V
    constexpr int SROWS = 64 / W;
    const unsigned sraw = 2 * CODES + (row / SROWS * 2 * SROWS + row % SROWS) * 4 + (col >> 1);
    const unsigned bundles = vring + VST * TB;

    // Copies of a bundle: NI of codes, K's first (one: the first waves K, the others
    // V), two of scales.
    constexpr int RPI = 1024 / ROW, CPR = ROW / 16, NI = ROW / 8 / W, NC = NI + (MX ? 2 : 0);
    static_assert(NI == 1 || NI == 2, "copies of a wave");
    const int lrow = lane / CPR;
    const int first = RPI * (NI == 2 ? wv : wv & (W / 2 - 1));  // row of a wave's copies
    const unsigned lane_off = (unsigned)(RPI > 16 ? lrow & (RPI / 2 - 1) : lrow) * p.stride_tok +
                              16u * (lane % CPR ^ (ROW == 128 && (first + lrow & 4) ? 4 : 0));
    const char* ksbase = (const char*)p.ks.scale + w.kvh * p.scale_stride_head;
    const char* vsbase = (const char*)p.vs.scale + w.kvh * p.scale_stride_head;
    const int last_entry = w.page_begin + ((ke - 1) >> p.log2_page);
    typedef const __attribute__((address_space(4))) int const_int;
    auto page_of = [&](int key) -> unsigned {  // (behind the range: its last page)
      return min((unsigned)((const_int*)p.page_table)[min(w.page_begin + (key >> p.log2_page), last_entry)], last_page);
    };
    auto copy_codes = [&](const char* base, int kb, unsigned dst) {
      const int k0 = kb + first;
      if (__builtin_expect(k0 + RPI <= ke, 1)) {
        const unsigned long long at = row_offset(p, page_of(k0), k0 & pmask);
        if constexpr (RPI > 16) {
          // two runs of rows, by the halves of the wave
          const int k1 = k0 + RPI / 2;
          const unsigned long long at1 = row_offset(p, page_of(k1), k1 & pmask);
          dma16_kept(base + (hh ? at1 : at) + lane_off, dst);
        } else {
          dma16s_kept(base + at, lane_off, dst);
        }
      } else {
        // rows behind the range: its last one again
        const int key = min(k0 + lrow, ke - 1);
        const unsigned pa = page_of(min(k0, ke - 1)), pb = page_of(ke - 1), pm = page_of(min(k0 + RPI / 2, ke - 1));
        const unsigned pg = key >> p.log2_page == (ke - 1) >> p.log2_page ? pb : key >> p.log2_page == k0 >> p.log2_page ? pa : pm;
        dma16_kept(base + row_offset(p, pg, key & pmask) + 16u * (lane % CPR ^ (ROW == 128 && (first + lrow & 4) ? 4 : 0)), dst);
      }
    };
    auto copy_scales = [&](const char* base, int kb, unsigned dst) {
      if (lane >= SROWS) return;
      const int k0 = min(kb + wv * SROWS, ke - 1);
      const unsigned long long at = scale_offset(p, page_of(k0), k0 & pmask);
      // (rows behind the range: of the same page, their scales are never used but with
      // the codes of the last row: any but NaN; so take the last row's)
      const unsigned off = min(lane, ke - 1 - k0) * p.scale_stride_tok;
      dma_scale<D / 32>(base + at, off, dst);
    };
    // bundle b: K of tile b + 1 (behind the last tile: nothing reads it), V of tile b
    auto issue = [&](int b) {
      const unsigned at = bundles + (unsigned)(b + RD) % RD * BUNDLE;
      const int kk = kb0 + 64 * min(b + 1, nt - 1), kv = kb0 + 64 * max(b, 0);
      if constexpr (NI == 2) {
        copy_codes(kbase, kk, at + wv * 1024);
        copy_codes(vbase, kv, at + CODES + wv * 1024);
      } else {
        if (wv < W / 2)
          copy_codes(kbase, kk, at + wv * 1024);
        else
          copy_codes(vbase, kv, at + CODES + (wv - W / 2) * 1024);
      }
      if constexpr (MX) {
        copy_scales(ksbase, kk, at + 2 * CODES + wv * 2 * SROWS * 4);
        copy_scales(vsbase, kv, at + 2 * CODES + wv * 2 * SROWS * 4 + SROWS * 4);
      }
    };
    // The same for bundles of whole tiles, in steps: page ids first, a tile ahead
    // (scalar loads, waited for with a region's LDS reads), then the addresses, then the
    // copies between MFMAs.
    int page_k = 0, page_v = 0, page_c[2] = {0, 0};  // of the wave's scale rows; of its codes (two: as they are copied)
    auto load_ids = [&](int b) {
      auto id = [&](int key) -> int { return ((const_int*)p.page_table)[w.page_begin + (key >> p.log2_page)]; };
      const int kk = kb0 + 64 * (b + 1);
      page_v = page_k;
      page_k = id(kk + wv * SROWS);
      if constexpr (NI == 1) {
        const int kc = (wv < W / 2 ? kk : kk - 64) + first;
        page_c[0] = id(kc);
        if constexpr (RPI > 16) page_c[1] = id(kc + RPI / 2);
      }
    };
    struct Bases {
      unsigned long long k, v, c, c1, sk, sv;
    } bases;
    auto find = [&](int b) {
      const int kk = kb0 + 64 * (b + 1);
      auto at = [&](int id, int key) { return row_offset(p, min((unsigned)id, last_page), key & pmask); };
      if constexpr (NI == 2) {
        bases.k = at(page_k, kk + first);
        bases.v = at(page_v, kk - 64 + first);
      } else {
        const int kc = (wv < W / 2 ? kk : kk - 64) + first;
        bases.c = at(page_c[0], kc);
        if constexpr (RPI > 16) bases.c1 = at(page_c[1], kc + RPI / 2);
      }
      if constexpr (MX) {
        bases.sk = scale_offset(p, min((unsigned)page_k, last_page), (kk + wv * SROWS) & pmask);
        bases.sv = scale_offset(p, min((unsigned)page_v, last_page), (kk - 64 + wv * SROWS) & pmask);
      }
    };
    const unsigned scale_off = (lane & (SROWS - 1)) * p.scale_stride_tok;
    auto copy_step = [&](int b, auto step) {  // of NC
      constexpr int i = decltype(step)::value;
      const unsigned at = bundles + (unsigned)b % RD * BUNDLE;
      if constexpr (i < NI && NI == 2) {
        if constexpr (i == 0)
          dma16s_kept(kbase + bases.k, lane_off, at + wv * 1024);
        else
          dma16s_kept(vbase + bases.v, lane_off, at + CODES + wv * 1024);
      } else if constexpr (i < NI) {
        const unsigned dst = at + (wv < W / 2 ? wv * 1024 : CODES + (wv - W / 2) * 1024);
        const char* base = wv < W / 2 ? kbase : vbase;
        if constexpr (RPI > 16)
          dma16_kept(base + (hh ? bases.c1 : bases.c) + lane_off, dst);
        else
          dma16s_kept(base + bases.c, lane_off, dst);
      } else if (lane < SROWS) {
        const unsigned dst = at + 2 * CODES + wv * 2 * SROWS * 4;
        if constexpr (i == NI)
          dma_scale<D / 32>(ksbase + bases.sk, scale_off, dst);
        else
          dma_scale<D / 32>(vsbase + bases.sv, scale_off, dst + SROWS * 4);
      }
    };
    {
      const RowOut at(p, w, min(32 * wv + l32, w.nrows - 1));
      const bf16_t* qp = (const bf16_t*)p.q + (long long)at.token * p.q_stride_n + (long long)at.head * p.q_stride_h + 8 * hh;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[ks] = *(const bf16x8*)(qp + 16 * ks);
      // (landed before the copies, which the compiler does not see, are under way)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        u32x4 u = __builtin_bit_cast(u32x4, qf[ks]);
        __asm__ volatile("" : "+v"(u));
        qf[ks] = __builtin_bit_cast(bf16x8, u);
      }
    }
    // a segment's codes and scale from bundle b, side V: 1
    struct Segment {
      unsigned code[WORDS];
      unsigned scale;
    };
    auto read_segment = [&](int b, int side) -> Segment {
      const unsigned at = bundles + (unsigned)(b + RD) % RD * BUNDLE;
      Segment x;
      if constexpr (WORDS == 4) {
        const u32x4 u = *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)(at + side * CODES + raw);
#pragma unroll
        for (int e = 0; e < 4; ++e) x.code[e] = u[e];
      } else {
        const u32x2 u = *(const __attribute__((address_space(3))) u32x2*)(uintptr_t)(at + side * CODES + raw);
        x.code[0] = u[0], x.code[1] = u[1];
      }
      x.scale = MX ? *(const __attribute__((address_space(3))) uint8_t*)(uintptr_t)(at + sraw + side * SROWS * 4) : 0u;
      return x;
    };
    auto store_segment = [&](const Segment& x, unsigned slot) {
      const float f = MX ? block_scale(x.scale) : 1.f;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *(__attribute__((address_space(3))) bf16x8*)(uintptr_t)(slot + (h ? put1 : put0)) =
            expand<FMT>(x.code[WORDS / 2 * h], WORDS == 4 ? x.code[WORDS / 2 * h + 1] : 0u, f);
    };
    // K(j) in slot j % 2, V(j) likewise.  At tile it's barrier K(it + 1), V(it) and, raw,
    // bundle it + 1 are there, K(it), V(it - 1) and bundle it no longer read.
#pragma unroll
    for (int b = -1; b < RD - 1; ++b)
      if (b < nt) issue(b);
    // bundles that may be under way when bundle b is needed, `ahead` issued behind it
    auto wait_bundle = [&](int b, int ahead) { wait_copies<NC, RD - 2>(max(0, min(ahead, nt - 1 - b))); };
    wait_bundle(0, RD - 2);
    tile_barrier();
    store_segment(read_segment(-1, 0), kring);
    store_segment(read_segment(0, 0), kring + TB);
    store_segment(read_segment(0, 1), vring);
    wait_lgkm0();
    tile_barrier();
    if (RD - 1 < nt) issue(RD - 1);
    auto sync = [&](int it) {
      wait_lgkm0();
      wait_bundle(it + 1, RD - 2);
      tile_barrier();
    };
    Segment seg;
    // before tile it, in six steps: K(it + 1), then V(it), to their slots
    auto put = [&](int it, auto step) {
      constexpr int i = decltype(step)::value;
      if constexpr (i == 0) seg = read_segment(it, 0);
      if constexpr (i == 1) store_segment(seg, kring + ((it + 1) & 1) * TB);
      if constexpr (i == 2) seg = read_segment(it, 1);
      if constexpr (i == 3) store_segment(seg, vring + (it & 1) * TB);
    };
    if (!live) {
      sync(0);
      if (RD < nt) issue(RD);
      for (int it = 1; it < nt; ++it) {
        static_for<4>([&](auto i) { put(it, i); });
        sync(it);
        if (it + RD < nt) issue(it + RD);
      }
      return;
    }
    start_tiles();
    auto first_half = [&](int it, auto prev, auto spread) {
      constexpr bool FIRST = !decltype(prev)::value, SPREAD = decltype(spread)::value;
      kstep = (it & 1) ? 0u - TB : TB;
      vstep = (it & 1) ? TB : 0u - TB;
      region1(prev, prev, [&](int ks) { return kread(1, ks); }, std::integral_constant<bool, !SPREAD>{}, kb0 + it * 64,
              [&](auto ic) {
                step_addresses(ic, std::integral_constant<bool, FIRST>{});
                if constexpr (SPREAD && decltype(ic)::value == 1) find(it + RD);
              });
      if constexpr (SPREAD) {
        wait_lgkm0();
        wait_vmcnt<(RD - 2) * NC>();
        tile_barrier();
        region2(true_type{}, vread, [&](auto sc_) {
          static_for<NC>([&](auto ic) {
            if constexpr (decltype(ic)::value * KS / NC == decltype(sc_)::value) copy_step(it + RD, ic);
          });
        });
      } else {
        sync(it);
        if (it + RD < nt) issue(it + RD);
        region2(true_type{}, vread, nothing);
      }
    };
    auto second_half = [&](int it, auto spread) {
      region1(true_type{}, true_type{}, [&](int ks) { return kread(0, ks); }, false_type{}, kb0 + it * 64 + 32, [&](auto ic) {
        // (a read two slots before its use)
        constexpr int i = decltype(ic)::value;
        static_for<4>([&](auto step) {
          if constexpr (decltype(step)::value * NPV / 4 == i) put(it + 1, step);
        });
      });
      region2(true_type{}, [&](int mt, int j) { return vread(mt, 2 + j); }, [&](auto ic) {
        if constexpr (decltype(spread)::value && decltype(ic)::value == 0) load_ids(it + 1 + RD);
      });
    };
    first_half(0, false_type{}, false_type{});
    // (tile it + RD + 1 is whole)
    const int whole = (ke - kb0) >> 6;
    int it = 1;
    if (it + RD + 1 < whole) {
      load_ids(RD);  // (for the V of bundle RD + 1)
      for (; it + RD + 1 < whole; ++it) {
        second_half(it - 1, true_type{});
        first_half(it, true_type{}, true_type{});
      }
    }
    for (; it < nt; ++it) {
      second_half(it - 1, false_type{});
      first_half(it, true_type{}, false_type{});
    }
    finish();
  }

  // the rows' partial state: normalised, base-2 log of the sum
  float l = (l4[0] + l4[1]) + (l4[2] + l4[3]);
  l += xor32(l, hh);
  const float lse2 = l > 0.f ? mc + __builtin_amdgcn_logf(l) : l == 0.f ? -INFINITY : l;
  store_image<D>(p, w, o, l != 0.f ? vscale / l : 0.f, lse2, 32 * wv, l32, hh);
}
