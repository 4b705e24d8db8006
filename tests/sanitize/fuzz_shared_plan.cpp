// Randomized inputs to the chunk attention's planner with shared keys
// (d2-sd_amd/csrc/chunk_plan.cpp), built with AddressSanitizer and UBSan on the host by
// tests/test_shared_plan_sanitize.py: items name requests, rows, heads and pages of the
// batch, and every partial row is written by one item and joined by one merge, whose
// row it is.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>
#include <tuple>
#include <vector>
#include "plan.h"
using namespace d2sd;
#define NEED(...) do { if (!(__VA_ARGS__)) { printf("batch %d: %s\n", t, #__VA_ARGS__); return 1; } } while (0)
int main(int argc, char** argv) {
  const int iters = argc > 1 ? atoi(argv[1]) : 2000;
  std::mt19937_64 rng(4242);
  auto U = [&](int a, int b) { return (int)std::uniform_int_distribution<int>(a, b)(rng); };
  int apart = 0, few = 0, waves[2] = {0, 0};
  for (int t = 0; t < iters; ++t) {
    const int R = U(0, 70), page = 1 << U(0, 8), style = U(0, 3);  // tokens, mixed, chunks, anything
    std::vector<int> qo(R + 1, 0), kv(R), pi(R + 1, 0), first{0}, bound;
    while (first.back() < R) first.push_back(std::min(R, first.back() + (U(0, 4) ? U(1, 40) : U(0, 2))));
    if (R == 0 && U(0, 1)) first.push_back(0);
    const int G = (int)first.size() - 1;
    for (int i = 0; i < G; ++i) {
      bound.push_back(U(0, 5) == 0 ? 0 : U(0, 3) ? U(1, 9000) : U(1, 64));
      for (int r = first[i]; r < first[i + 1]; ++r) {
        const int n = style == 0 ? U(0, 2) : style == 1 ? (U(0, 9) ? 1 : U(1, 700)) : style == 2 ? U(30, 700) : U(0, 100);
        qo[r + 1] = qo[r] + n;
        kv[r] = U(0, 9) == 0 ? U(0, n + bound[i]) : bound[i] + n + U(0, U(0, 3) ? 900 : 20000);
        // (pages of its own for what the others hold elsewhere, or not; the first one's hold all)
        const int need = (std::max(kv[r], r == first[i] ? bound[i] : 0) + page - 1) / page;
        pi[r + 1] = pi[r] + (r > first[i] && U(0, 5) == 0 ? need / 2 : need + U(0, 2));
      }
    }
    const int hkv = U(1, 9), g = U(0, 3) ? 1 << U(0, 4) : U(1, 20);
    ChunkPlanInput in{};
    in.num_reqs = R;
    in.qo_indptr = qo.data();
    in.kv_len = kv.data();
    in.page_indptr = pi.data();
    in.num_qo_heads = hkv * g;
    in.num_kv_heads = hkv;
    in.head_dim = U(0, 1) ? 64 : 128;
    in.format = U(0, 3);
    in.page_size = page;
    in.window_left = U(0, 2) ? -1 : U(0, 5000);
    in.num_cus = std::vector<int>{1, 4, 64, 256, 1024}[U(0, 4)];
    in.max_splits = U(0, 2) ? 0 : U(1, 100);
    in.num_groups = G;
    in.shared_indptr = first.data();
    in.shared_len = bound.data();
    in.keep_shared = U(0, 2) != 0;
    ChunkPlanOutput out;
    plan_chunk(in, out);
    if (!(out.form & CHUNK_SHARED)) {
      ++apart;
      NEED(out.tokens.empty() && out.shared_merges.empty());
      continue;
    }
    const int form = out.form & ~CHUNK_SHARED;
    NEED(form >= 0 && form <= CHUNK_STREAM && out.merges.empty() && (int)out.tokens.size() == qo[R]);
    NEED(!(form == CHUNK_WAVES8 && in.head_dim == 64) && !(form == CHUNK_WAVES4 && !shared_waves4(in.head_dim, in.format)));
    form >= CHUNK_TOKENS ? ++few : ++waves[form == CHUNK_WAVES4];
    for (int r = 0; r < R; ++r)
      for (int i = qo[r]; i < qo[r + 1]; ++i)
        NEED(out.tokens[i].req == r && out.tokens[i].back == qo[r + 1] - i && out.tokens[i].room == (pi[r + 1] - pi[r]) * page);
    typedef std::tuple<long long, int> Row;  // row of q x heads of a kv head + head, kv head
    std::vector<Row> slots((size_t)out.partial_rows, Row{-1, 0});
    std::set<Row> direct;
    auto put = [&](const ChunkItem& i, int kvh, int chunk, long long slot, int stride) {
      if (i.nchunks == 1 && i.part == PART_ALONE) {
        for (int r = 0; r < i.nrows; ++r)
          if (!direct.insert({(long long)i.q0 * g + i.row0 + r, kvh}).second) return false;
        return true;
      }
      for (int r = 0; r < i.nrows; ++r) {
        const long long at = slot + (long long)chunk * stride + r;
        if (at < 0 || at >= out.partial_rows || std::get<0>(slots[at]) >= 0) return false;
        slots[at] = {(long long)i.q0 * g + i.row0 + r, kvh};
      }
      return true;
    };
    for (const ChunkItem& i : out.items) {
      NEED(i.req >= 0 && i.req < R && i.q0 == qo[i.req] && i.page_begin == pi[i.req] && i.page_end == pi[i.req + 1]);
      NEED(i.nchunks >= 1 && i.nchunks <= kChunkMaxSplits && (in.max_splits == 0 || i.nchunks <= in.max_splits));
      NEED(i.nrows > 0 && i.row0 >= 0 && i.q0 * (long long)g + i.row0 + i.nrows <= (long long)qo[R] * g);
      NEED(i.bound == 0 || i.bound <= (i.part == PART_SHARED ? (pi[i.req + 1] - pi[i.req]) * page : 1 << 30));
      if (form < CHUNK_TOKENS && i.kind == CHUNK_TOKEN) {  // units of waves
        NEED(i.heads == hkv && i.kvh >= 0 && i.kvh % chunk_waves(form) == 0 && i.kvh < i.nchunks * hkv && i.nrows <= kTokenRows);
        for (int u = i.kvh; u < std::min(i.kvh + chunk_waves(form), i.nchunks * hkv); ++u)
          NEED(put(i, u % hkv, u / hkv, i.slot + (long long)(u % hkv) * i.nchunks * i.nrows, i.nrows));
        continue;
      }
      NEED(i.kvh >= 0 && i.kvh < hkv && i.chunk >= 0 && i.chunk < i.nchunks && (form < CHUNK_TOKENS || i.kind == CHUNK_TOKEN));
      NEED(i.nrows <= (i.kind == CHUNK_TOKEN ? kTokenRows : chunk_rows(form)));
      NEED(i.kind == CHUNK_TOKEN || i.part != PART_SHARED || (i.heads >= 0 && i.heads <= 64 && i.nq >= i.req && i.nq + i.heads <= R));
      NEED(put(i, i.kvh, i.chunk, i.slot, i.part == PART_SHARED && i.kind == CHUNK_TILE ? (i.nrows + 31) / 32 * 32 : i.nrows));
    }
    auto take = [&](long long at, const Row& row) {
      if (at < 0 || at >= out.partial_rows || slots[at] != row) return false;
      slots[at] = {-1, 0};
      return true;
    };
    for (const SharedMerge& m : out.shared_merges) {
      NEED(m.nrows > 0 && m.nrows <= 1024 / in.head_dim && m.nchunks >= 1 && m.shared_chunks >= 0);
      for (int r = 0; r < m.nrows; ++r) {
        const Row row{(long long)m.q0 * g + m.row0 + r, m.kvh};
        for (int c = 0; c < m.nchunks; ++c) NEED(take(m.slot + (long long)c * m.stride + r, row));
        for (int c = 0; c < m.shared_chunks; ++c)
          NEED(take(m.shared_slot + (long long)c * m.shared_stride + m.shared_row + r, row));
        NEED(direct.insert(row).second);
      }
    }
    for (const Row& x : slots) NEED(std::get<0>(x) < 0);
    NEED((long long)direct.size() == (long long)qo[R] * g * hkv);
  }
  if (iters >= 200 && (!apart || !few || !waves[0] || !waves[1])) return printf("a kind of plan never came\n"), 1;
  printf("ok: %d plans; %d apart, %d of few rows, %d and %d of 8 and 4 waves\n", iters, apart, few, waves[0], waves[1]);
  return 0;
}
