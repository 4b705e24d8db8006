// Work planner of the chunk attention (chunk_attention.hip): which workgroup
// takes which rows and which share of their keys.
#include <algorithm>
#include <cstdint>
#include <queue>
#include <vector>

#include "plan.h"

namespace d2sd {

namespace {

// Times of a workgroup on a CU of its own, in us (measured at D = 128; half at
// D = 64): an item's start and end, a 64-key tile of a tile item, a round of
// 8 x 32 keys of a token item, the share of HBM of one CU (bytes per us), a
// partial state's extra and the merge launch.
constexpr double kItemUs = 4.0, kTileUs = 1.4, kRoundUs = 0.8, kCuBytesPerUs = 19500.0, kMergeUs = 4.0;

struct Group {
  int req, kvh, row0, nrows, kind, units;  // units: 64-key tiles (tile items), 32-key tiles (token items)
  double unit_us, cost;
};

int row_bytes(int format, int d) {
  return format == CACHE_BF16 ? 2 * d : format == CACHE_FP8 ? d : format == CACHE_MXFP8 ? d + d / 32 : d / 2 + d / 32;
}

int chunks_of(const Group& g, double limit, int max_splits) {
  const int least = g.kind == CHUNK_TOKEN ? kChunkWaves : 4;  // units of the shortest chunk
  const int most = std::max(1, std::min({g.units / least, max_splits, kChunkMaxSplits}));
  const double work = g.cost - kItemUs;
  const int want = work <= limit ? 1 : (int)std::min<double>(most, (work + limit - 1e-9) / limit);
  return std::max(1, std::min(most, want));
}

// Time until the last workgroup ends when the longest start first, one per CU.
double span_us(const std::vector<Group>& groups, double limit, int max_splits, int cus) {
  std::vector<double> times;
  bool split = false;
  for (const Group& g : groups) {
    const int n = chunks_of(g, limit, max_splits);
    split = split || n > 1;
    for (int c = 0; c < n; ++c) times.push_back((g.cost - kItemUs) / n + kItemUs);
  }
  std::sort(times.begin(), times.end(), std::greater<double>());
  std::priority_queue<double, std::vector<double>, std::greater<double>> ends;
  double last = 0.0;
  for (double t : times) {
    double at = 0.0;
    if ((int)ends.size() >= cus) {
      at = ends.top();
      ends.pop();
    }
    ends.push(at + t);
    last = std::max(last, at + t);
  }
  return last + (split ? kMergeUs : 0.0);
}

}  // namespace

void plan_chunk(const ChunkPlanInput& in, ChunkPlanOutput& out) {
  out = ChunkPlanOutput{};
  const int group = in.num_qo_heads / in.num_kv_heads;
  const double scale = in.head_dim == 64 ? 0.5 : 1.0;
  const int max_splits = in.max_splits > 0 ? in.max_splits : kChunkMaxSplits;
  std::vector<Group> groups;
  double total = 0.0, longest = 0.0;
  for (int r = 0; r < in.num_reqs; ++r) {
    const int nq = in.qo_indptr[r + 1] - in.qo_indptr[r];
    const long long rows = (long long)nq * group;
    const int kind = rows <= kTokenRows ? CHUNK_TOKEN : CHUNK_TILE;
    const int step = kind == CHUNK_TOKEN ? kTokenRows : kChunkRows, keys_per_unit = kind == CHUNK_TOKEN ? 32 : 64;
    for (long long row0 = 0; row0 < rows; row0 += step) {
      Group g{};
      g.req = r;
      g.row0 = (int)row0;
      g.nrows = (int)std::min<long long>(step, rows - row0);
      g.kind = kind;
      const long long pos0 = (long long)in.kv_len[r] - nq;
      const long long first = pos0 + row0 / group, last = pos0 + (row0 + g.nrows - 1) / group;
      const long long hi = std::max(last + 1, 0ll);
      const long long lo = in.window_left >= 0 ? std::max(first - in.window_left, 0ll) : 0;
      g.units = hi > lo ? (int)((hi + keys_per_unit - 1) / keys_per_unit - lo / keys_per_unit) : 0;
      if (kind == CHUNK_TOKEN) {
        const double bytes = 2.0 * 32 * row_bytes(in.format, in.head_dim);
        g.unit_us = std::max(kRoundUs * scale / kChunkWaves, bytes / kCuBytesPerUs);
      } else {
        g.unit_us = kTileUs * scale;
      }
      g.cost = kItemUs + g.units * g.unit_us;
      for (int h = 0; h < in.num_kv_heads; ++h) {
        g.kvh = h;
        groups.push_back(g);
        total += g.cost - kItemUs;
        longest = std::max(longest, g.cost - kItemUs);
      }
    }
  }
  // the longest chunk: the one whose schedule ends first, among no split and
  // shares of an even load
  double limit = longest + 1.0;
  if (!groups.empty()) {
    double best = span_us(groups, limit, max_splits, in.num_cus);
    const double even = total / in.num_cus;
    for (double f : {1.0, 0.75, 0.5, 0.34, 0.25}) {
      const double t = span_us(groups, even * f, max_splits, in.num_cus);
      if (t < best) best = t, limit = even * f;
    }
  }
  struct Timed {
    double us;
    ChunkItem item;
  };
  std::vector<Timed> items;
  const int merge_rows = 1024 / in.head_dim;  // rows of one merge workgroup: 256 threads, 4 head dims each
  long long slot = 0;
  for (const Group& g : groups) {
    const int n = chunks_of(g, limit, max_splits);
    ChunkItem it{};
    it.req = g.req;
    it.kvh = g.kvh;
    it.q0 = in.qo_indptr[g.req];
    it.nq = in.qo_indptr[g.req + 1] - it.q0;
    it.row0 = g.row0;
    it.nrows = g.nrows;
    it.page_begin = in.page_indptr[g.req];
    it.page_end = in.page_indptr[g.req + 1];
    it.nchunks = n;
    it.slot = n > 1 ? (int)slot : 0;
    it.kind = g.kind;
    for (int c = 0; c < n; ++c) {
      it.chunk = c;
      items.push_back({(g.cost - kItemUs) / n, it});
    }
    if (n > 1) {
      for (int i = 0; i < g.nrows; i += merge_rows)
        out.merges.push_back(ChunkMerge{it.q0, g.kvh, g.row0 + i, std::min(merge_rows, g.nrows - i), (int)slot + i,
                                        g.nrows, n, 0});
      slot += (long long)n * g.nrows;
    }
  }
  // Longest first; among equals the kv heads of one key chunk side by side, so
  // that with 8 (or 16, ..) kv heads each XCD (workgroups are dealt to the 8 of
  // them in turn) keeps a head's keys in its own L2 for all row tiles.
  std::stable_sort(items.begin(), items.end(), [](const Timed& a, const Timed& b) {
    if (a.us != b.us) return a.us > b.us;
    if (a.item.req != b.item.req) return a.item.req < b.item.req;
    if (a.item.row0 != b.item.row0) return a.item.row0 < b.item.row0;
    if (a.item.chunk != b.item.chunk) return a.item.chunk < b.item.chunk;
    return a.item.kvh < b.item.kvh;
  });
  out.items.reserve(items.size());
  for (const Timed& t : items) out.items.push_back(t.item);
  out.partial_rows = slot;
}

}  // namespace d2sd
