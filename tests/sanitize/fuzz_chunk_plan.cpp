// Randomized inputs to the chunk attention's planner (d2-sd_amd/csrc/chunk_plan.cpp),
// built with AddressSanitizer and UBSan on the host by
// tests/test_chunk_plan_sanitize.py: every (request, kv head) has each of its
// packed rows in exactly one row tile, every tile all of its key chunks, chunks
// of split tiles slots of their own, and every row of a split tile one merge.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>
#include <tuple>
#include <vector>
#include "plan.h"
using namespace d2sd;
#define NEED(...) do { if (!(__VA_ARGS__)) { printf("batch %d: %s\n", t, #__VA_ARGS__); return 1; } } while (0)
int main(int argc, char** argv) {
  const int iters = argc > 1 ? atoi(argv[1]) : 2000;
  std::mt19937_64 rng(777);
  auto U = [&](int a, int b) { return (int)std::uniform_int_distribution<int>(a, b)(rng); };
  int forms[4] = {0, 0, 0, 0}, split = 0;
  for (int t = 0; t < iters; ++t) {
    const int R = U(0, 40), page = 1 << U(0, 8);
    const int style = U(0, 3);  // tokens, mixed, chunks, anything
    std::vector<int> qo(R + 1, 0), kv(R + 1, 0), pi(R + 1, 0);
    for (int r = 0; r < R; ++r) {
      const int n = style == 0 ? U(0, 2) : style == 1 ? (U(0, 9) ? 1 : U(1, 1500)) : style == 2 ? U(100, 2500) : U(0, 300);
      qo[r + 1] = qo[r] + n;
      kv[r] = U(0, 9) == 0 ? U(0, n) : n + U(0, U(0, 3) ? 6000 : 200000);
      pi[r + 1] = pi[r] + (kv[r] + page - 1) / page + U(0, 2);
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
    in.window_left = U(0, 2) ? -1 : U(0, 3000);
    in.num_cus = std::vector<int>{1, 4, 64, 256, 1024}[U(0, 4)];
    in.max_splits = U(0, 2) ? 0 : U(1, 100);
    ChunkPlanOutput out;
    plan_chunk(in, out);
    NEED(out.form >= 0 && out.form <= CHUNK_STREAM && !(out.form == CHUNK_WAVES8 && in.head_dim == 64));
    ++forms[out.form];
    std::map<std::tuple<int, int, int>, std::vector<ChunkItem>> tiles;  // request, kv head, first row
    std::set<long long> slots;
    for (const ChunkItem& i : out.items) {
      NEED(i.req >= 0 && i.req < R && i.kvh >= 0 && i.kvh < hkv && i.q0 == qo[i.req] && i.nq == qo[i.req + 1] - qo[i.req]);
      NEED(i.page_begin == pi[i.req] && i.page_end == pi[i.req + 1]);
      NEED(i.nrows > 0 && i.row0 >= 0 && i.row0 + i.nrows <= (long long)i.nq * g);
      NEED(i.nrows <= (i.kind == CHUNK_TOKEN ? kTokenRows : chunk_rows(out.form)));
      NEED(out.form < CHUNK_TOKENS || (i.kind == CHUNK_TOKEN && i.nrows <= 16));
      NEED(i.nchunks >= 1 && i.nchunks <= kChunkMaxSplits && i.chunk >= 0 && i.chunk < i.nchunks);
      NEED(in.max_splits == 0 || i.nchunks <= in.max_splits);
      if (i.nchunks > 1)
        for (int r = 0; r < i.nrows; ++r) NEED(slots.insert(i.slot + (long long)i.chunk * i.nrows + r).second);
      tiles[{i.req, i.kvh, i.row0}].push_back(i);
    }
    NEED((long long)slots.size() == out.partial_rows && (slots.empty() || (*slots.begin() == 0 && *slots.rbegin() + 1 == out.partial_rows)));
    std::map<std::pair<int, int>, long long> rows;
    std::map<std::tuple<int, int, int>, const ChunkItem*> want;  // rows to merge: first query row, kv head, row
    for (auto& [k, v] : tiles) {
      std::set<int> chunks;
      for (const ChunkItem& i : v) {
        NEED(i.nrows == v[0].nrows && i.nchunks == v[0].nchunks && i.slot == v[0].slot);
        chunks.insert(i.chunk);
      }
      NEED((int)chunks.size() == v[0].nchunks && (int)v.size() == v[0].nchunks);
      long long& at = rows[{std::get<0>(k), std::get<1>(k)}];
      NEED(at == std::get<2>(k));  // (tiles come in row order)
      at += v[0].nrows;
      if (v[0].nchunks > 1)
        for (int r = 0; r < v[0].nrows; ++r) want[{v[0].q0, v[0].kvh, v[0].row0 + r}] = &v[0];
    }
    for (int r = 0; r < R; ++r)
      for (int h = 0; h < hkv; ++h) {
        const long long n = (long long)(qo[r + 1] - qo[r]) * g;
        NEED(n == 0 ? !rows.count({r, h}) : rows[{r, h}] == n);
      }
    split += !want.empty();
    for (const ChunkMerge& m : out.merges) {
      NEED(m.nrows > 0 && m.nrows <= 1024 / in.head_dim);
      for (int r = 0; r < m.nrows; ++r) {
        auto it = want.find({m.q0, m.kvh, m.row0 + r});
        NEED(it != want.end());
        const ChunkItem& i = *it->second;
        NEED(m.nchunks == i.nchunks && m.stride == i.nrows && m.slot == i.slot + m.row0 - i.row0);
        want.erase(it);
      }
    }
    NEED(want.empty());
  }
  if (iters >= 200 && (!forms[0] || !forms[1] || !forms[2] || !forms[3] || !split)) return printf("a kind of plan never came\n"), 1;
  printf("ok: %d plans, %d with split keys; forms %d %d %d %d\n", iters, split, forms[0], forms[1], forms[2], forms[3]);
  return 0;
}
