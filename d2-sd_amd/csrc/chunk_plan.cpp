// Work planner of the chunk attention (chunk_attention.hip): which workgroup
// takes which rows and which share of their keys.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <queue>
#include <vector>

#include "plan.h"

namespace d2sd {

namespace {

// Measured times in us: a workgroup's start and end; a 32-key tile of one wave
// of a token item (D = 128; half as long at D = 64); a merge launch; and rates in
// bytes per us: what one CU reads at most, what all of them read together, what
// a merge moves.
constexpr double kItemUs = 5.0, kTokenTileUs = 1.2, kMergeUs = 5.0;
constexpr double kStreamBytes = 128 << 20;
constexpr double kCuBytes = 57e3, kHbmBytes = 5.4e6, kMergeBytes = 3.0e6;

int row_bytes(int format, int d) {
  return format == CACHE_BF16 ? 2 * d : format == CACHE_FP8 ? d : format == CACHE_MXFP8 ? d + d / 32 : d / 2 + d / 32;
}

// A 64-key tile of a tile item, with n workgroups on its CU (D = 128: 8 waves
// alone 2.0; 4 waves, half the rows, 1.35 alone and 2.35 of two; D = 64, 4
// waves: 1.0, 1.5, 2.0).
double tile_us(int form, int head_dim, double n) {
  if (head_dim == 64) return 0.5 + 0.5 * n;
  return form == CHUNK_WAVES8 ? 2.0 : 0.35 + n;
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
  int form;
  std::vector<Group> groups;
  int per_cu, places;   // workgroups resident on a CU, on the device
  double place_bytes;   // highest rate of one of them
  int most;             // chunks of a group
  double limit = 0.0;   // the longest chunk, in us of one workgroup alone on its CU
  double token_share = 1.0;  // of that, a token item's longest

  Planner(const ChunkPlanInput& input, int f) : in(input), form(f) {
    // (by registers: chunk_attn_kernel; the token kernels of heads of 64 would fit four
    // but for mxfp8, the schedule counts three)
    per_cu = form == CHUNK_WAVES8 ? 1 : in.head_dim == 64 ? 3 : form == CHUNK_TOKENS && in.format == CACHE_MXFP4 ? 3 : 2;
    places = in.num_cus * per_cu;
    place_bytes = kCuBytes / per_cu;
    most = in.max_splits > 0 ? std::min(in.max_splits, kChunkMaxSplits) : kChunkMaxSplits;
  }

  void take(Planner&& other) {
    form = other.form;
    groups = std::move(other.groups);
    limit = other.limit;
    token_share = other.token_share;
  }

  int chunks(const Group& g) const {
    const int top = std::max(1, std::min(most, g.units / g.least));
    const double us = g.kind == CHUNK_TOKEN ? limit * token_share : limit;
    return g.work() <= us ? 1 : (int)std::min<double>(top, g.work() / us + 0.999);
  }

  // Time until the last workgroup ends when the longest start first.  Tile items
  // slow each other down on a CU; token items that read at the same time share
  // the HBM's rate.
  double span() const {
    std::vector<std::pair<double, int>> times;  // of a workgroup, and how many are alike
    times.reserve(groups.size());
    long long items = 0;
    double partial = 0.0, readers = 0.0, work = 0.0, longest = 0.0;
    for (const Group& g : groups) {
      const int n = chunks(g);
      items += (long long)n * in.num_kv_heads;
      work += g.work() * in.num_kv_heads;
      longest = std::max(longest, g.work() / n);
      if (g.kind == CHUNK_TOKEN) readers += (double)n * in.num_kv_heads;
    }
    // Workgroups on a CU beside each other: those of the longest one's time, by CUs;
    // with some more than CUs a few share theirs, and end last.
    const double per = longest > 0.0 ? work / longest / in.num_cus : 0.0;
    const double sharing = std::min<double>(per_cu, std::max(1.0, 0.6 * per + 0.4 * std::ceil(per - 0.02)));
    const double slower_tile = tile_us(form, in.head_dim, sharing) / tile_us(form, in.head_dim, 1.0);
    const double slower_read = std::max(1.0, std::min(readers, (double)places) * place_bytes / kHbmBytes);
    for (const Group& g : groups) {
      const int n = chunks(g);
      if (n > 1) partial += (double)n * g.nrows * in.num_kv_heads * in.head_dim * 8.0;  // written and read
      const double us = g.kind == CHUNK_TOKEN ? std::max(g.work(), g.read_us() * slower_read) : g.work() * slower_tile;
      times.push_back({us / n + kItemUs, n * in.num_kv_heads});
    }
    double last = 0.0;
    if (items <= places) {
      for (const auto& x : times) last = std::max(last, x.first);
    } else {
      std::sort(times.begin(), times.end(), std::greater<std::pair<double, int>>());
      // places by the time they are free, those alike together
      std::priority_queue<std::pair<double, int>, std::vector<std::pair<double, int>>, std::greater<std::pair<double, int>>> free;
      free.push({0.0, places});
      for (const auto& x : times) {
        for (int left = x.second; left > 0;) {
          const auto at = free.top();
          free.pop();
          const int k = std::min(left, at.second);
          free.push({at.first + x.first, k});
          if (k < at.second) free.push({at.first, at.second - k});
          left -= k;
          last = std::max(last, at.first + x.first);
        }
      }
    }
    return last + (partial > 0.0 ? kMergeUs + partial / kMergeBytes : 0.0);
  }

  // Row tiles, then the longest chunk: of no split and of ever shorter ones, the
  // one whose schedule ends first.  Batches of many groups need only be evened
  // out.  Returns its time.
  double plan() {
    const int group = in.num_qo_heads / in.num_kv_heads, waves = chunk_waves(form);
    const double token_us = kTokenTileUs * (in.head_dim == 64 ? 0.5 : 1.0) / waves;
    double longest = 0.0, total = 0.0;
    bool tiles = false, tokens = false;
    for (int r = 0; r < in.num_reqs; ++r) {
      const int nq = in.qo_indptr[r + 1] - in.qo_indptr[r];
      const long long rows = (long long)nq * group;
      const int kind = rows <= kTokenRows ? CHUNK_TOKEN : CHUNK_TILE;
      const int step = kind == CHUNK_TOKEN ? kTokenRows : chunk_rows(form), keys_per_unit = kind == CHUNK_TOKEN ? 32 : 64;
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
        // (a tile item's tiles start at its first key, a token item's at multiples)
        const long long from = kind == CHUNK_TOKEN ? lo / keys_per_unit * keys_per_unit : lo;
        g.units = hi > lo ? (int)((hi - from + keys_per_unit - 1) / keys_per_unit) : 0;
        (kind == CHUNK_TOKEN ? tokens : tiles) = true;
        if (kind == CHUNK_TOKEN) {
          g.unit_read_us = unit_bytes / place_bytes;
          g.unit_us = std::max(token_us, g.unit_read_us);
          g.least = waves;
        } else {
          g.unit_us = tile_us(form, in.head_dim, 1.0);
          g.least = 4;
        }
        groups.push_back(g);
        longest = std::max(longest, g.work());
        total += g.work() * in.num_kv_heads;
      }
    }
    limit = longest + 1.0;
    if (groups.empty()) return 0.0;
    const bool many = (double)groups.size() * in.num_kv_heads > 4.0 * places;
    double best = span(), best_limit = limit;
    const double even = total / places, shortest = many ? even * 0.5 : even / 16.0;
    for (double x = longest * 0.8409; x > shortest && x > 1.0; x *= 0.8409) {
      if (many && x > 2.0 * even) continue;
      limit = x;
      const double t = span();
      if (t < best * 0.99) best = t, best_limit = x;
    }
    limit = best_limit;
    // beside tile items, shorter chunks for the token items alone (their partial
    // states are small)
    double best_share = 1.0;
    if (tiles && tokens) {
      for (double share : {0.7, 0.5, 0.35}) {
        token_share = share;
        const double t = span();
        if (t < best * 0.99) best = t, best_share = share;
      }
    }
    token_share = best_share;
    return best;
  }
};

}  // namespace

void plan_chunk(const ChunkPlanInput& in, ChunkPlanOutput& out) {
  out = ChunkPlanOutput{};
  const int group = in.num_qo_heads / in.num_kv_heads;
  bool tokens_only = true;
  for (int r = 0; r < in.num_reqs; ++r)
    if ((long long)(in.qo_indptr[r + 1] - in.qo_indptr[r]) * group > 16) tokens_only = false;
  // Heads of 128: workgroups of 8 waves share a tile's staging among more rows
  // (2 x 2048 tokens at 16384 bf16 keys: 953 us against 1045), those of 4 fill
  // the device with fewer rows (1000 tokens at 2100: 47 us against 50 split in two
  // and 60 unsplit).  Heads of 64: 4 waves, three workgroups on a CU (before tiles
  // were kept in L2, 4 x 1024 tokens, window 128: 39 us against 44; 8 x 300 at 1000:
  // 66 against 74; but 2 x 2048 at 16384: 1340 against 1259 in bf16, 1201 against
  // 1217 in mxfp4; now 28, 55, 1200 and 1145 of 4 waves, 8 were not measured again).
  Planner pl(in, tokens_only ? CHUNK_TOKENS : CHUNK_WAVES4);
  const double us = pl.plan();
  if (!tokens_only && in.head_dim == 128) {
    Planner other(in, CHUNK_WAVES8);
    if (other.plan() < us) pl.take(std::move(other));
  }
  out.form = pl.form;
  // Token items alone that read more than half of the last-level cache (256 MB):
  // what they read is not there when the next call reads it, and goes past the
  // caches (32 requests of 8..32k tokens: bf16 452 -> 425 us, fp8 248 -> 224,
  // mxfp4 149 -> 134).  Smaller reads may be found there (8 x 4000 tokens in bf16:
  // 27 us, 30 past the caches).
  double bytes = 0.0;
  for (const Group& g : pl.groups) bytes += 64.0 * g.units * row_bytes(in.format, in.head_dim) * in.num_kv_heads;
  if (tokens_only && bytes > kStreamBytes) out.form = CHUNK_STREAM;
  const int merge_rows = 1024 / in.head_dim;  // rows of one merge workgroup: 256 threads, 4 head dims each
  struct Placed {
    double us;   // of a chunk
    int group, chunks;
    long long slot;
  };
  std::vector<Placed> order;
  order.reserve(pl.groups.size());
  long long slot = 0, items = 0;
  for (int i = 0; i < (int)pl.groups.size(); ++i) {
    const Group& g = pl.groups[i];
    const int n = pl.chunks(g);
    order.push_back({g.work() / n, i, n, slot});
    items += (long long)n * in.num_kv_heads;
    if (n == 1) continue;
    const int q0 = in.qo_indptr[g.req];
    for (int h = 0; h < in.num_kv_heads; ++h, slot += (long long)n * g.nrows)
      for (int r = 0; r < g.nrows; r += merge_rows)
        out.merges.push_back(ChunkMerge{q0, h, g.row0 + r, std::min(merge_rows, g.nrows - r), (int)slot + r, g.nrows, n, 0});
  }
  // Longest first; among equals the kv heads of one key chunk side by side, so
  // that with 8 (or 16, ..) kv heads each XCD (workgroups are dealt to the 8 of
  // them in turn) keeps a head's keys in its own L2 for all row tiles.
  std::stable_sort(order.begin(), order.end(), [](const Placed& a, const Placed& b) { return a.us > b.us; });
  out.items.reserve((size_t)items);
  for (const Placed& x : order) {
    const Group& g = pl.groups[x.group];
    ChunkItem it{};
    it.req = g.req;
    it.q0 = in.qo_indptr[g.req];
    it.nq = in.qo_indptr[g.req + 1] - it.q0;
    it.row0 = g.row0;
    it.nrows = g.nrows;
    it.page_begin = in.page_indptr[g.req];
    it.page_end = in.page_indptr[g.req + 1];
    it.nchunks = x.chunks;
    it.kind = g.kind;
    for (it.chunk = 0; it.chunk < x.chunks; ++it.chunk)
      for (it.kvh = 0; it.kvh < in.num_kv_heads; ++it.kvh) {
        it.slot = x.chunks > 1 ? (int)(x.slot + (long long)it.kvh * x.chunks * g.nrows) : 0;
        out.items.push_back(it);
      }
  }
  out.partial_rows = slot;
}

}  // namespace d2sd
