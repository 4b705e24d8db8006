// Work planner of the chunk attention (chunk_attention.hip): which workgroup
// takes which rows and which share of their keys.
#include <algorithm>
#include <cstdint>
#include <queue>
#include <vector>

#include "plan.h"

namespace d2sd {

namespace {

// Measured times in us: a workgroup's start and end; a 64-key tile of a tile
// item (D = 64: of half the rows, three workgroups on a CU); a 32-key tile of one
// wave of a token item (half as long at D = 64); a merge launch; and rates in bytes per us: what one CU reads at
// most, what all of them read together, what a merge moves.
constexpr double kItemUs = 5.0, kTileUs = 1.9, kTileUs64 = 2.0, kTokenTileUs = 0.9, kMergeUs = 3.0;
constexpr double kCuBytes = 57e3, kHbmBytes = 5.4e6, kMergeBytes = 3.0e6;

int row_bytes(int format, int d) {
  return format == CACHE_BF16 ? 2 * d : format == CACHE_FP8 ? d : format == CACHE_MXFP8 ? d + d / 32 : d / 2 + d / 32;
}

struct Group {         // one row tile of a request, for every kv head
  int req, row0, nrows, kind;
  int units, least;    // key tiles, and those of the shortest chunk
  double unit_us;      // of a tile, alone
  double unit_read_us; // of that, its bytes at a workgroup's highest rate
  double work() const { return units * unit_us; }
  double read_us() const { return units * unit_read_us; }
};

struct Planner {
  const ChunkPlanInput& in;
  std::vector<Group> groups;
  int places = 1;      // workgroups resident on the device
  double place_bytes = 0.0;  // highest rate of one of them
  int most;            // chunks of a group

  int chunks(const Group& g, double limit) const {
    const int top = std::max(1, std::min(most, g.units / g.least));
    return g.work() <= limit ? 1 : (int)std::min<double>(top, g.work() / limit + 0.999);
  }

  // Time until the last workgroup ends when the longest start first.  Token
  // items that read at the same time share the HBM's rate.
  double span(double limit) const {
    std::vector<double> times;
    double partial = 0.0, readers = 0.0;
    for (const Group& g : groups)
      if (g.kind == CHUNK_TOKEN) readers += (double)chunks(g, limit) * in.num_kv_heads;
    const double slower = std::max(1.0, std::min(readers, (double)places) * place_bytes / kHbmBytes);
    for (const Group& g : groups) {
      const int n = chunks(g, limit);
      if (n > 1) partial += (double)n * g.nrows * in.num_kv_heads * in.head_dim * 8.0;  // written and read
      const double us = g.kind == CHUNK_TOKEN ? std::max(g.work(), g.read_us() * slower) : g.work();
      times.insert(times.end(), (size_t)n * in.num_kv_heads, us / n + kItemUs);
    }
    double last = 0.0;
    if ((int)times.size() <= places) {
      for (double t : times) last = std::max(last, t);
    } else {
      std::sort(times.begin(), times.end(), std::greater<double>());
      std::priority_queue<double, std::vector<double>, std::greater<double>> ends;
      for (double t : times) {
        double at = 0.0;
        if ((int)ends.size() >= places) {
          at = ends.top();
          ends.pop();
        }
        ends.push(at + t);
        last = std::max(last, at + t);
      }
    }
    return last + (partial > 0.0 ? kMergeUs + partial / kMergeBytes : 0.0);
  }
};

}  // namespace

void plan_chunk(const ChunkPlanInput& in, ChunkPlanOutput& out) {
  out = ChunkPlanOutput{};
  const int group = in.num_qo_heads / in.num_kv_heads;
  const double scale = in.head_dim == 64 ? 0.5 : 1.0, tile_us = in.head_dim == 64 ? kTileUs64 : kTileUs;
  out.tokens_only = true;
  for (int r = 0; r < in.num_reqs; ++r)
    if ((long long)(in.qo_indptr[r + 1] - in.qo_indptr[r]) * group > 16) out.tokens_only = false;
  // (register bound: chunk_attn_kernel)
  const int per_cu = in.head_dim == 64 ? 3 : !out.tokens_only ? 1 : in.format == CACHE_MXFP4 ? 3 : 2;
  const int waves = out.tokens_only ? kTokenWaves : chunk_waves(in.head_dim);
  Planner pl{in, {}, in.num_cus * per_cu, kCuBytes / per_cu, in.max_splits > 0 ? std::min(in.max_splits, kChunkMaxSplits) : kChunkMaxSplits};
  double longest = 0.0, total = 0.0;
  long long count = 0;
  for (int r = 0; r < in.num_reqs; ++r) {
    const int nq = in.qo_indptr[r + 1] - in.qo_indptr[r];
    const long long rows = (long long)nq * group;
    const int kind = rows <= kTokenRows ? CHUNK_TOKEN : CHUNK_TILE;
    const int step = kind == CHUNK_TOKEN ? kTokenRows : chunk_rows(in.head_dim), keys_per_unit = kind == CHUNK_TOKEN ? 32 : 64;
    const double unit_bytes = 2.0 * keys_per_unit * row_bytes(in.format, in.head_dim);
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
        g.unit_read_us = unit_bytes / pl.place_bytes;
        g.unit_us = std::max(kTokenTileUs * scale / waves, g.unit_read_us);
        g.least = waves;
      } else {
        g.unit_us = tile_us;
        g.least = 4;
      }
      pl.groups.push_back(g);
      longest = std::max(longest, g.work());
      total += g.work() * in.num_kv_heads;
      count += in.num_kv_heads;
    }
  }
  // The longest chunk: of no split and of ever shorter ones, the one whose
  // schedule ends first.  Batches of many groups need only be evened out.
  double limit = longest + 1.0;
  if (count > 0) {
    double best = pl.span(limit);
    const double even = total / pl.places;
    const double shortest = count > 4ll * pl.places ? even * 0.5 : even / 16.0;
    for (double x = longest * 0.7072; x > shortest && x > 1.0; x *= 0.7072) {
      if (count > 4ll * pl.places && x > 2.0 * even) continue;
      const double t = pl.span(x);
      if (t < best * 0.99) best = t, limit = x;
    }
  }
  struct Timed {
    double us;
    ChunkItem item;
  };
  std::vector<Timed> items;
  const int merge_rows = 1024 / in.head_dim;  // rows of one merge workgroup: 256 threads, 4 head dims each
  long long slot = 0;
  for (const Group& g : pl.groups) {
    const int n = pl.chunks(g, limit);
    ChunkItem it{};
    it.req = g.req;
    it.q0 = in.qo_indptr[g.req];
    it.nq = in.qo_indptr[g.req + 1] - it.q0;
    it.row0 = g.row0;
    it.nrows = g.nrows;
    it.page_begin = in.page_indptr[g.req];
    it.page_end = in.page_indptr[g.req + 1];
    it.nchunks = n;
    it.kind = g.kind;
    for (int h = 0; h < in.num_kv_heads; ++h) {
      it.kvh = h;
      it.slot = n > 1 ? (int)slot : 0;
      for (int c = 0; c < n; ++c) {
        it.chunk = c;
        items.push_back({g.work() / n, it});
      }
      if (n > 1) {
        for (int i = 0; i < g.nrows; i += merge_rows)
          out.merges.push_back(ChunkMerge{it.q0, h, g.row0 + i, std::min(merge_rows, g.nrows - i), (int)slot + i, g.nrows,
                                          n, 0});
        slot += (long long)n * g.nrows;
      }
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
