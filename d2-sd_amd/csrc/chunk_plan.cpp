// Work planner of the chunk attention (chunk_attention.hip): which workgroup
// takes which rows and which share of their keys.
#include <algorithm>
#include <array>
#include <cmath>
#include <cstdint>
#include <functional>
#include <map>
#include <memory>
#include <optional>
#include <queue>
#include <tuple>
#include <utility>
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

// Rows that are packed together: a request's, or, over the keys that they share,
// those of all requests of a group.
struct Rows {
  int part, req;        // PART_*; the (first) request
  int q0, nq;           // first row of q, their number
  int last_req;         // behind the last of its requests
  int bound;            // keys [0, bound) are shared
};

// Keys [lo, hi) that packed rows [row0, row0 + nrows) of a set see.  req: of shared
// keys, a request at or before that of the first row (moved on to it).
void seen_keys(const ChunkPlanInput& in, const Rows& set, int group, long long row0, int nrows, int& req, long long& lo,
               long long& hi) {
  if (set.part == PART_SHARED) {
    lo = 0, hi = set.bound;
    if (in.window_left < 0) return;
    const int t0 = set.q0 + (int)(row0 / group), t1 = set.q0 + (int)((row0 + nrows - 1) / group);
    while (in.qo_indptr[req + 1] <= t0) ++req;
    long long first = 1ll << 40, last = -1;
    for (int r = req; r < set.last_req && in.qo_indptr[r] <= t1; ++r) {
      if (in.qo_indptr[r + 1] <= std::max(in.qo_indptr[r], t0)) continue;
      const long long end = (long long)in.kv_len[r] - in.qo_indptr[r + 1];
      first = std::min(first, end + std::max(in.qo_indptr[r], t0));
      last = std::max(last, end + std::min(in.qo_indptr[r + 1] - 1, t1));
    }
    lo = std::max(first - in.window_left, 0ll);
    hi = std::min<long long>(set.bound, std::max(last + 1, 0ll));
    return;
  }
  const long long pos0 = (long long)in.kv_len[set.req] - set.nq;
  const long long first = pos0 + row0 / group, last = pos0 + (row0 + nrows - 1) / group;
  hi = std::max(last + 1, 0ll);
  lo = std::max<long long>(in.window_left >= 0 ? std::max(first - in.window_left, 0ll) : 0, set.bound);
}

struct Group {         // one row tile of a request, for every kv head
  int rows;            // index of its Rows
  int row0, nrows, kind;
  int units, least;    // key tiles, and those of the shortest chunk
  double unit_us;      // of a tile, alone
  double unit_read_us; // of that, its bytes at a workgroup's highest rate
  bool partial;        // its state is joined with another's whatever its chunks
  double work() const { return units * unit_us; }
  double read_us() const { return units * unit_read_us; }
};

struct Planner {
  const ChunkPlanInput& in;
  const std::vector<Rows>& rows_list;
  int form;
  std::vector<Group> groups;
  int per_cu, places;   // workgroups resident on a CU, on the device
  double place_bytes;   // highest rate of one of them
  int most;             // chunks of a group
  double limit = 0.0;   // the longest chunk, in us of one workgroup alone on its CU
  double token_share = 1.0;  // of that, a token item's longest
  // Beside a plan with shared keys: what is read again comes from L2, and rows of token
  // items beyond 16 are waited for (their loads no longer are).
  double read_rate = kHbmBytes, wide_tokens = 1.0;

  Planner(const ChunkPlanInput& input, const std::vector<Rows>& rows, int f) : in(input), rows_list(rows), form(f) {
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

  // Bytes of the partial states.
  double states() const {
    double rows = 0.0;
    for (const Group& g : groups)
      if (const int n = chunks(g); n > 1 || g.partial) rows += (double)n * g.nrows;
    return rows * in.num_kv_heads * (in.head_dim + 1) * 4.0;
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
    const double slower_read = std::max(1.0, std::min(readers, (double)places) * place_bytes / read_rate);
    for (const Group& g : groups) {
      const int n = chunks(g);
      if (n > 1 || g.partial) partial += (double)n * g.nrows * in.num_kv_heads * in.head_dim * 8.0;  // written and read
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
  // out.  Returns its time.  Not `fine`: for an estimate, in a quarter of the looks.
  double plan(bool fine = true) {
    const int group = in.num_qo_heads / in.num_kv_heads, waves = chunk_waves(form);
    const double token_us = kTokenTileUs * (in.head_dim == 64 ? 0.5 : 1.0) / waves;
    double longest = 0.0, total = 0.0;
    bool tiles = false, tokens = false;
    for (int at = 0; at < (int)rows_list.size(); ++at) {
      const Rows& set = rows_list[at];
      const long long rows = (long long)set.nq * group;
      const int kind = rows <= kTokenRows ? CHUNK_TOKEN : CHUNK_TILE;
      const int step = kind == CHUNK_TOKEN ? kTokenRows : chunk_rows(form), keys_per_unit = kind == CHUNK_TOKEN ? 32 : 64;
      const double unit_bytes = 2.0 * keys_per_unit * row_bytes(in.format, in.head_dim);
      int req = set.req;  // (of shared keys: that of the row tile's first token)
      for (long long row0 = 0; row0 < rows; row0 += step) {
        Group g{};
        g.rows = at;
        g.row0 = (int)row0;
        g.nrows = (int)std::min<long long>(step, rows - row0);
        g.kind = kind;
        g.partial = set.part != PART_ALONE;
        long long lo, hi;
        seen_keys(in, set, group, row0, g.nrows, req, lo, hi);
        // (a tile item's tiles start at its first key, a token item's at multiples)
        const long long from = kind == CHUNK_TOKEN ? lo / keys_per_unit * keys_per_unit : lo;
        g.units = hi > lo ? (int)((hi - from + keys_per_unit - 1) / keys_per_unit) : 0;
        (kind == CHUNK_TOKEN ? tokens : tiles) = true;
        if (kind == CHUNK_TOKEN) {
          g.unit_read_us = unit_bytes / place_bytes;
          g.unit_us = std::max(rows > 16 ? token_us * wide_tokens : token_us, g.unit_read_us);
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
    const double step = fine ? 0.8409 : 0.5;
    for (double x = longest * step; x > shortest && x > 1.0; x *= step) {
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

// Workgroup items and merges of plans with shared keys for workgroups of `form`'s
// waves: group i in chunks[i] chunks of keys.
struct SharedGroup {
  int rows, row0, nrows, kind;
  int units;    // 64-key tiles (CHUNK_TILE) or 32-key tiles
  int chunks;
};

// ---- plans with shared keys (but for those of a few rows, which stay above) ----
// Row tiles of a group's rows over the shared keys (tile items, whatever their rows),
// and each request's own keys: tile items where it brings more than 32 rows, else
// units of one wave (a request, kv head and chunk of keys each), which fill
// workgroups of as many waves.  Chunk lengths are those that end soonest by the times
// below, all measured.  (A wave's 32-key tile takes 1.3; one of eight on a CU, which
// wait for memory beside tile items, 1.7: 96 requests behind 32K mxfp8 keys 186 us
// planned by 1.3, 158 by 1.7, 168 by 2; 64 behind 16K in bf16, of four waves, 42.8 by
// 1.3, 44.1 by 1.7.  By themselves, in 24 to 144 workgroups at 0.2 to 5 TB/s: 1.1 to 1.7
// of four waves in bf16, 1.2 to 1.8 of eight in mxfp4 and mxfp8; heads of 64 0.6 to 1.1
// in bf16, 0.6 to 0.9 quantised, taken as 0.7 of those of 128.  Without what reads and
// work cost beside each other, chunks come out long where reads bound them: 48 behind 8K
// in bf16, heads of 64, 43 -> 35.)
constexpr double kSharedItemUs = 6.0, kWaveItemUs = 6.0;  // a workgroup's start and end
constexpr double kWaveTileUs = 1.3, kWaveTile8Us = 1.7;  // a 32-key tile of one of 4 waves, of 8
constexpr double kReadBeside = 0.2;      // of reads and work, how much of the shorter is not hidden
constexpr double kSharedMergeUs = 3.0, kPartialBytes = 2.6e6;  // the merge's launch; partial states written and read, per us
constexpr double kAgainBytes = 13e6, kWideTokens = 2.0;  // keys that other requests read too, per us; 17 to 32 rows to 16

struct SharedPlanner {
  const ChunkPlanInput& in;
  const std::vector<Rows>& rows_list;
  int form, waves, per_cu;
  std::vector<SharedGroup> groups;
  double tile_limit, wave_limit;  // longest chunks, in tiles
  double own_bytes, shared_bytes; // of the keys and values
  int most_units, most_own;       // tiles of the longest tile item, of the longest wave's
  // Groups that a schedule need not tell apart: those of about the same tiles (units: of
  // four bits, rounded up), all of them of the planner's waves.
  struct Alike {
    int kind, units;
    bool partial;
    double tile_us, tile_us_beside;  // of a tile, alone on a CU and not
    long long count, rows;
  };
  std::vector<Alike> alike;
  mutable std::vector<std::pair<double, long long>> tiles, solo;  // items: time of each, how many
  mutable std::vector<std::pair<double, long long>> free;         // places: when they are free, how many

  SharedPlanner(const ChunkPlanInput& input, const std::vector<Rows>& rows, int f) : in(input), rows_list(rows), form(f) {
    waves = chunk_waves(form);
    per_cu = form == CHUNK_WAVES8 ? 1 : 2;
    const int group = in.num_qo_heads / in.num_kv_heads;
    for (int at = 0; at < (int)rows_list.size(); ++at) {
      const Rows& set = rows_list[at];
      const long long rows = (long long)set.nq * group;
      const int kind = set.part == PART_SHARED || rows > kTokenRows ? CHUNK_TILE : CHUNK_TOKEN;
      const int step = kind == CHUNK_TOKEN ? kTokenRows : chunk_rows(form), keys = kind == CHUNK_TOKEN ? 32 : 64;
      int req = set.req;
      for (long long row0 = 0; row0 < rows; row0 += step) {
        SharedGroup g{at, (int)row0, (int)std::min<long long>(step, rows - row0), kind, 0, 1};
        long long lo, hi;
        seen_keys(in, set, group, row0, g.nrows, req, lo, hi);
        const long long from = kind == CHUNK_TOKEN ? lo / keys * keys : lo;
        g.units = hi > lo ? (int)((hi - from + keys - 1) / keys) : 0;
        groups.push_back(g);
      }
    }
    own_bytes = shared_bytes = 0.0;
    most_units = most_own = 0;
    std::map<std::tuple<int, int, bool, bool, bool>, std::pair<long long, long long>> same;  // groups and rows
    for (const SharedGroup& g : groups) {
      const bool over_shared = rows_list[g.rows].part == PART_SHARED;
      // (row tiles of a set read the same keys, from L2 but for the first)
      if (g.row0 == 0 || !over_shared)
        (over_shared ? shared_bytes : own_bytes) +=
            2.0 * (g.kind == CHUNK_TILE ? 64 : 32) * g.units * row_bytes(in.format, in.head_dim) * in.num_kv_heads;
      int fine = 0;
      while (g.units >> fine >= 16) ++fine;
      const int units = (g.units + (1 << fine) - 1) >> fine << fine;
      int& most = g.kind == CHUNK_TILE ? most_units : most_own;
      most = std::max(most, units);
      auto& m = same[{g.kind, units, over_shared, g.nrows * 2 > chunk_rows(form), rows_list[g.rows].part != PART_ALONE}];
      ++m.first;
      m.second += g.nrows;
    }
    const double wave_us = (waves == 8 ? kWaveTile8Us : kWaveTileUs) * (in.head_dim == 64 ? 0.7 : 1.0);
    for (const auto& [x, m] : same) {
      const auto [kind, units, over_shared, full, partial] = x;
      const bool tile = kind == CHUNK_TILE;
      alike.push_back({kind, units, partial, tile ? step_us(over_shared, true, full) : wave_us,
                       tile ? step_us(over_shared, false, full) : wave_us, m.first, m.second});
    }
  }

  void take(SharedPlanner&& other) {
    form = other.form;
    waves = other.waves;
    groups = std::move(other.groups);
  }

  // Bytes of the partial states (planned).
  double states() const {
    double rows = 0.0;
    for (const SharedGroup& g : groups)
      if (g.chunks > 1 || rows_list[g.rows].part != PART_ALONE) rows += (double)g.chunks * g.nrows;
    return rows * in.num_kv_heads * (in.head_dim + 1) * 4.0;
  }

  int most() const { return in.max_splits > 0 ? std::min(in.max_splits, kChunkMaxSplits) : kChunkMaxSplits; }
  int chunks_of(int kind, int units, double tiles, double own) const {
    return std::max(1, std::min(most(), (int)std::ceil(units / (kind == CHUNK_TILE ? tiles : own) - 1e-6)));
  }

  // Time until the last workgroup ends, those of tile items first, the longest before
  // the others, and the merge of the partial states.  At `enough` or more: some bound
  // below it, not less than that.
  double span(double tile_limit, double own_limit, double enough) const {
    tiles.clear(), solo.clear(), free.clear();
    double partial = 0.0, work = 0.0, last = 0.0;
    const long long heads = in.num_kv_heads, places = (long long)in.num_cus * per_cu;
    bool alone = per_cu == 1;
    if (!alone) {
      long long count = 0;
      for (const Alike& g : alike)
        if (g.kind == CHUNK_TILE) count += g.count * chunks_of(CHUNK_TILE, g.units, tile_limit, own_limit) * heads;
      alone = count <= in.num_cus;
    }
    for (const Alike& g : alike) {
      const int n = chunks_of(g.kind, g.units, tile_limit, own_limit);
      if (n > 1 || g.partial) partial += (double)n * g.rows * heads * in.head_dim * 4.0;
      const double us = (g.kind == CHUNK_TILE ? kSharedItemUs : kWaveItemUs) + (double)g.units / n * (alone ? g.tile_us : g.tile_us_beside);
      const long long items = g.count * (g.kind == CHUNK_TILE ? n * heads : (n * heads + waves - 1) / waves);
      (g.kind == CHUNK_TILE ? tiles : solo).push_back({us, items});
      work += us * items;
      last = std::max(last, us);
    }
    if (partial > 0.0) partial = kSharedMergeUs + partial / kPartialBytes;
    const double read = (own_bytes + shared_bytes) / kHbmBytes;
    auto total = [&](double us) {
      us -= kSharedItemUs;
      return kSharedItemUs + std::max(us, read) + kReadBeside * std::min(us, read) + partial;
    };
    const double bound = total(std::max(last, work / places));
    if (bound >= enough) return bound;
    std::sort(tiles.begin(), tiles.end(), std::greater<>());
    std::sort(solo.begin(), solo.end(), std::greater<>());
    const auto later = std::greater<std::pair<double, long long>>();
    free.push_back({0.0, places});
    for (const auto* list : {&tiles, &solo})
      for (const auto& x : *list)
        for (long long left = x.second; left > 0;) {
          std::pop_heap(free.begin(), free.end(), later);
          const auto at = free.back();
          free.pop_back();
          // (rounds in which the same places take items of the same length again and again)
          const long long rounds = free.empty() ? std::max(1ll, left / at.second) : 1, k = rounds > 1 ? at.second : std::min(left, at.second);
          const double end = at.first + rounds * x.first;
          free.push_back({end, k});
          std::push_heap(free.begin(), free.end(), later);
          if (k < at.second) {
            free.push_back({at.first, at.second - k});
            std::push_heap(free.begin(), free.end(), later);
          }
          left -= rounds * k;
          last = std::max(last, end);
        }
    return total(last);
  }

  // The longest chunks whose schedule ends first: a coarse search over all of them, then
  // (`fine`) one around what it found.  (Of 689 batches none comes out more than 0.5%
  // above a fine search over all; within a factor of 1.6 of n instead, 11%.)
  double plan(bool fine = true) {
    double best = 1e30;
    tile_limit = wave_limit = 1.0;
    const double longest = std::max(1, most_units), longest_own = std::max(4, most_own);
    auto search = [&](double n0, double n1, double n_step, double o0, double o1, double o_step) {
      for (double n = n0; n == n0 || (n <= std::min<double>(n1, most()) && longest / n >= 2.0); n = std::max(n + 1.0, std::floor(n * n_step)))
        for (double t = longest / n, o = o0;; o = std::max(o1, o * o_step)) {
          const double us = span(t, o, best * 0.995);
          if (us < best * 0.995) best = us, tile_limit = t, wave_limit = o;
          if (o <= o1) break;
        }
    };
    search(1.0, most(), 1.6, longest_own, 4.0, 0.4);
    if (fine) {
      const double n = std::round(longest / tile_limit), o = wave_limit;
      search(std::max(1.0, std::floor(n / 2.6)), std::ceil(n * 2.6), 1.08, std::min(longest_own, o / 0.16),
             std::max(4.0, o * 0.16), 0.62);
    }
    for (SharedGroup& g : groups) g.chunks = chunks_of(g.kind, g.units, tile_limit, wave_limit);
    return best;
  }

  // A 64-key tile of a tile item, alone on its CU or beside another.  Over shared keys
  // the inner loop of shared_tile, else that of tile_item.
  double step_us(bool over_shared, bool alone, bool full) const {
    if (in.head_dim == 64) return over_shared ? (alone ? 0.7 : 1.15) : (alone ? 1.0 : 1.5);
    if (form == CHUNK_WAVES8) return over_shared ? (!full ? 1.4 : in.format == CACHE_BF16 ? 1.75 : 1.9) : 2.0;
    return over_shared ? (alone ? 1.1 : 1.75) : (alone ? 1.35 : 2.35);
  }
};

// Plans of the waves that end soonest by their schedule, and that time.
double plan_waves(Planner& pl, bool fine = true) {
  double us = pl.plan(fine);
  if (pl.form == CHUNK_WAVES4 && pl.in.head_dim == 128) {
    Planner other(pl.in, pl.rows_list, CHUNK_WAVES8);
    other.read_rate = pl.read_rate, other.wide_tokens = pl.wide_tokens;
    const double o = other.plan(fine);
    if (o < us) pl.take(std::move(other)), us = o;
  }
  return us;
}
double plan_waves(SharedPlanner& pl, bool fine = true) {
  double us = pl.plan(fine);
  if (pl.form == CHUNK_WAVES4 && pl.in.head_dim == 128) {
    SharedPlanner other(pl.in, pl.rows_list, CHUNK_WAVES8);
    const double o = other.plan(fine);
    if (o < us) pl.take(std::move(other)), us = o;
  }
  return us;
}

// Waves to begin with: two workgroups on a CU where their rings fit.
int shared_form(const ChunkPlanInput& in) { return shared_waves4(in.head_dim, in.format) ? CHUNK_WAVES4 : CHUNK_WAVES8; }

// Rows of one chunk's partial states: those over shared keys in blocks of 32.
int partial_rows(const Rows& set, const SharedGroup& g) {
  return set.part == PART_SHARED ? (g.nrows + 31) & ~31 : g.nrows;
}

void shared_tokens(const ChunkPlanInput& in, ChunkPlanOutput& out) {
  for (int r = 0; r < in.num_reqs; ++r)
    for (int t = in.qo_indptr[r]; t < in.qo_indptr[r + 1]; ++t)
      out.tokens.push_back({r, in.qo_indptr[r + 1] - t, (in.page_indptr[r + 1] - in.page_indptr[r]) * in.page_size, 0});
}

// Items and merges of the planned groups.  shared_rows: of a request, the Rows of what it
// shares.
void plan_shared(const ChunkPlanInput& in, const std::vector<Rows>& rows, const std::vector<int>& shared_rows,
                 const SharedPlanner& pl, ChunkPlanOutput& out) {
  const int group = in.num_qo_heads / in.num_kv_heads, heads = in.num_kv_heads;
  out.form = pl.form | CHUNK_SHARED;
  const int merge_rows = 1024 / in.head_dim;
  long long slot = 0;
  std::vector<long long> slots(pl.groups.size());
  std::vector<int> first_group(rows.size(), -1);
  size_t merges = 0;  // (some more where a merge would cross the border of two row tiles)
  for (const SharedGroup& g : pl.groups)
    if (const int part = rows[g.rows].part; part == PART_OWN || (part == PART_ALONE && g.chunks > 1))
      merges += (size_t)(g.nrows / merge_rows + 2) * heads;
  out.shared_merges.reserve(merges);
  for (int i = 0; i < (int)pl.groups.size(); ++i) {
    const SharedGroup& g = pl.groups[i];
    const Rows& set = rows[g.rows];
    if (first_group[g.rows] < 0) first_group[g.rows] = i;
    if (g.chunks == 1 && set.part == PART_ALONE) continue;
    slots[i] = slot;
    slot += (long long)g.chunks * partial_rows(set, g) * heads;
    if (set.part == PART_SHARED) continue;
    // (kv heads side by side: a merge on the XCD whose L2 has the head's partial states)
    for (int r = 0, take; r < g.nrows; r += take) {
      for (int h = 0; h < heads; ++h) {
        const long long at = slots[i] + (long long)h * g.chunks * g.nrows;
        take = std::min(merge_rows, g.nrows - r);
        SharedMerge m{set.q0, h, g.row0 + r, take, (int)at + r, g.nrows, g.chunks, 0, 0, 0, 0, 0};
        if (set.part == PART_OWN) {
          // its rows among those of the group, within one of their row tiles
          const int sh = shared_rows[set.req], from = (set.q0 - rows[sh].q0) * group + g.row0 + r;
          const int k = first_group[sh] + from / chunk_rows(pl.form);
          const SharedGroup& sg = pl.groups[k];
          take = m.nrows = std::min(take, sg.row0 + sg.nrows - from);
          const int stride = partial_rows(rows[sh], sg);
          m.shared_slot = (int)(slots[k] + (long long)h * sg.chunks * stride);
          m.shared_row = from - sg.row0;
          m.shared_stride = stride;
          m.shared_chunks = sg.chunks;
        }
        out.shared_merges.push_back(m);
      }
    }
  }
  auto item_of = [&](int i) {
    const SharedGroup& g = pl.groups[i];
    const Rows& set = rows[g.rows];
    ChunkItem it{};
    it.req = set.req;
    it.q0 = set.q0;
    it.nq = set.nq;
    it.row0 = g.row0;
    it.nrows = g.nrows;
    it.page_begin = in.page_indptr[set.req];
    it.page_end = in.page_indptr[set.req + 1];
    it.nchunks = g.chunks;
    it.kind = g.kind;
    it.part = set.part;
    it.bound = set.bound;
    it.heads = heads;
    it.slot = (int)slots[i];
    if (set.part == PART_SHARED) {
      // The row tile's requests, where a wave's lanes can hold their lengths, their pages
      // hold all that is shared and the tokens behind it, and their rows see all of it
      // (under the lengths planned for; others are found out at the end).
      const int t0 = set.q0 + g.row0 / group, t1 = set.q0 + (g.row0 + g.nrows - 1) / group;
      int first = set.req;
      while (in.qo_indptr[first + 1] <= t0) ++first;
      int last = first;
      long long room = 1ll << 40;
      bool all = true;
      for (; last < set.last_req && in.qo_indptr[last] <= t1; ++last) {
        if (in.qo_indptr[last + 1] == in.qo_indptr[last]) continue;
        const int back = in.qo_indptr[last + 1] - std::max(in.qo_indptr[last], t0);  // of the request's first row here
        it.back = std::max(it.back, back);
        all = all && in.kv_len[last] - back + 1 >= set.bound;
        room = std::min(room, (long long)(in.page_indptr[last + 1] - in.page_indptr[last]) * in.page_size);
      }
      it.nq = first;
      it.heads = all && last - first <= 64 && room >= (long long)set.bound + it.back ? last - first : 0;
    }
    return it;
  };
  std::vector<ChunkItem> tiles, solo;
  std::vector<int> order(pl.groups.size());
  for (int i = 0; i < (int)order.size(); ++i) order[i] = i;
  std::stable_sort(order.begin(), order.end(), [&](int a, int b) {
    return (double)pl.groups[a].units / pl.groups[a].chunks > (double)pl.groups[b].units / pl.groups[b].chunks;
  });
  for (int i : order) {
    const SharedGroup& g = pl.groups[i];
    const Rows& set = rows[g.rows];
    ChunkItem it = item_of(i);
    if (g.kind == CHUNK_TILE) {
      for (it.chunk = 0; it.chunk < g.chunks; ++it.chunk)
        for (it.kvh = 0; it.kvh < heads; ++it.kvh) {
          it.slot = (int)(slots[i] + (long long)it.kvh * g.chunks * partial_rows(set, g));
          tiles.push_back(it);
        }
    } else {
      for (it.kvh = 0; it.kvh < g.chunks * heads; it.kvh += pl.waves) solo.push_back(it);
    }
  }
  // Tile items first, the longest before the others: what they leave free takes the waves' units.
  out.items = std::move(tiles);
  out.items.insert(out.items.end(), solo.begin(), solo.end());
  out.partial_rows = slot;
  shared_tokens(in, out);
}

// The rows of requests [r0, r1).  use: groups whose keys are shared.  shared_rows: of a
// request, the Rows of what it shares (-1: nothing).  Returns whether any shares.
bool batch_rows(const ChunkPlanInput& in, const std::vector<char>& use, int r0, int r1, std::vector<Rows>& rows,
                std::vector<int>& shared_rows) {
  rows.clear();
  shared_rows.assign(in.num_reqs, -1);
  for (int i = 0; i < in.num_groups; ++i) {
    const int a = in.shared_indptr[i], b = in.shared_indptr[i + 1];
    if (!use[i] || a < r0 || b > r1) continue;
    for (int r = a; r < b; ++r) shared_rows[r] = (int)rows.size();
    rows.push_back({PART_SHARED, a, in.qo_indptr[a], in.qo_indptr[b] - in.qo_indptr[a], b, in.shared_len[i]});
  }
  const bool shared = !rows.empty();
  for (int r = r0; r < r1; ++r) {
    const int q0 = in.qo_indptr[r], nq = in.qo_indptr[r + 1] - q0, s = shared_rows[r];
    rows.push_back({s < 0 ? PART_ALONE : PART_OWN, r, q0, nq, r + 1, s < 0 ? 0 : rows[s].bound});
  }
  return shared;
}

bool tokens_only(const ChunkPlanInput& in, const std::vector<Rows>& rows) {
  const int group = in.num_qo_heads / in.num_kv_heads;
  for (const Rows& x : rows)
    if ((long long)x.nq * group > 16) return false;
  return true;
}

// What requests [r0, r1) cost with the keys of these groups shared.
struct Cost {
  double us, states;  // time; bytes of the partial states
};
// A plan of tile items with shared keys, as far as it is one.
struct SharedPlan {
  std::vector<Rows> rows;
  std::vector<int> shared_rows;
  std::optional<SharedPlanner> planner;
};
// `fine`: what a plan comes to; else an estimate in fewer looks.  keep: takes the plan.
Cost batch_cost(const ChunkPlanInput& in, const std::vector<char>& use, int r0, int r1, bool fine = true,
                SharedPlan* keep = nullptr) {
  SharedPlan own, &plan = keep ? *keep : own;
  std::vector<Rows>& rows = plan.rows;
  const bool shared = batch_rows(in, use, r0, r1, rows, plan.shared_rows), few = tokens_only(in, rows);
  if (shared && !few) {
    SharedPlanner& pl = plan.planner.emplace(in, rows, shared_form(in));
    const double us = plan_waves(pl, fine);
    return {us, pl.states()};
  }
  Planner pl(in, rows, few ? CHUNK_TOKENS : CHUNK_WAVES4);
  if (!shared) {
    double keys = 1.0, again = 0.0;  // of those that are read, those that another request read before
    for (int i = 0; i < in.num_groups; ++i)
      for (int r = in.shared_indptr[i]; r < in.shared_indptr[i + 1]; ++r) {
        if (r < r0 || r >= r1) continue;
        const int nq = in.qo_indptr[r + 1] - in.qo_indptr[r];
        const long long lo = in.window_left >= 0 ? std::max(0ll, (long long)in.kv_len[r] - nq - in.window_left) : 0;
        keys += std::max(0ll, in.kv_len[r] - lo);
        if (r > in.shared_indptr[i]) again += std::max(0ll, std::min(in.kv_len[r], in.shared_len[i]) - lo);
      }
    pl.read_rate = 1.0 / (again / keys / kAgainBytes + (1.0 - again / keys) / kHbmBytes);
    pl.wide_tokens = kWideTokens;
  }
  const double us = plan_waves(pl, fine);
  return {us, pl.states()};
}

// Groups whose keys are read once for all of their rows.  Sharing costs partial states
// and a launch that joins them, so that it is not worth a few keys, nor many rows that
// are bound by their products either way: all of the groups share, or those that gain
// by themselves, or none, whichever ends soonest by the schedules' times.
//
// What is shared has to gain 1%, and 1% more for each 128 MB that its partial states are
// larger: the caller holds them.  (330 batches of 2 to 64 requests of 1 to 400 tokens
// behind 64 to 16384 keys took, shared, 0.26 to 2.5 times what they took apart; all of
// them 31.5 ms apart, 25.8 shared, 24.73 as chosen and 24.64 by the better of the two.
// Estimated ratios are off by 14%, to either side: with a margin of 5% the choice took
// 24.96.  8 prompts of 8192 tokens behind 16384 bf16 keys would gain 1% by the
// estimate, 6% measured, with 2.2 GB of states: apart; 1024 requests in 128 groups, 1.1
// GB, 20% and 25%: shared.)
constexpr double kShareGain = 0.01, kShareGainByte = 0.01 / (128 << 20);
bool worth_sharing(const Cost& shared, const Cost& apart) {
  return shared.us < apart.us * (1.0 - kShareGain - kShareGainByte * std::max(0.0, shared.states - apart.states));
}
// plan: that of the groups returned, if one was made.
std::vector<char> sharing(const ChunkPlanInput& in, std::unique_ptr<SharedPlan>& plan) {
  std::vector<char> use(in.num_groups, 0);
  int groups = 0;
  for (int i = 0; i < in.num_groups; ++i) {
    const int a = in.shared_indptr[i], b = in.shared_indptr[i + 1];
    use[i] = b - a > 1 && in.shared_len[i] > 0 && in.qo_indptr[b] > in.qo_indptr[a];
    groups += use[i];
  }
  if (groups == 0 || in.keep_shared) return use;
  const std::vector<char> none(in.num_groups, 0);
  auto of_all = std::make_unique<SharedPlan>();
  const Cost apart = batch_cost(in, none, 0, in.num_reqs), all = batch_cost(in, use, 0, in.num_reqs, true, of_all.get());
  double best = apart.us;
  std::vector<char> kept = none;
  if (worth_sharing(all, apart)) best = all.us, kept = use, plan = std::move(of_all);
  // (groups of about the same sizes are looked at once; of very many kinds, none is)
  std::map<std::array<int, 4>, char> kinds;
  auto kind_of = [&](int i) {
    const int a = in.shared_indptr[i], b = in.shared_indptr[i + 1];
    long long keys = 0;
    for (int r = a; r < b; ++r) keys += in.kv_len[r];
    auto about = [](long long x) {
      int e = 0;
      while (x >> e >= 8) ++e;
      return (int)(x >> e << e);
    };
    return std::array<int, 4>{about(b - a), about(in.qo_indptr[b] - in.qo_indptr[a]), about(in.shared_len[i]), about(keys / (b - a))};
  };
  for (int i = 0; i < in.num_groups; ++i)
    if (use[i]) kinds[kind_of(i)] = 2;
  if (kinds.size() == 1 || kinds.size() > 32) return kept;
  std::vector<char> gain = use;
  for (int i = 0; i < in.num_groups; ++i) {
    if (!use[i]) continue;
    char& known = kinds[kind_of(i)];
    const int a = in.shared_indptr[i], b = in.shared_indptr[i + 1];
    if (known == 2) known = worth_sharing(batch_cost(in, use, a, b, false), batch_cost(in, none, a, b, false));
    gain[i] = known;
  }
  if (gain == use || gain == none) return kept;
  auto of_some = std::make_unique<SharedPlan>();
  const Cost some = batch_cost(in, gain, 0, in.num_reqs, true, of_some.get());
  if (some.us < best && worth_sharing(some, apart)) kept = gain, plan = std::move(of_some);
  return kept;
}

}  // namespace

void plan_chunk(const ChunkPlanInput& in, ChunkPlanOutput& out) {
  out = ChunkPlanOutput{};
  const int group = in.num_qo_heads / in.num_kv_heads;
  std::unique_ptr<SharedPlan> plan;
  const std::vector<char> use = sharing(in, plan);
  if (plan && plan->planner) {
    plan_shared(in, plan->rows, plan->shared_rows, *plan->planner, out);
    return;
  }
  std::vector<Rows> rows;
  std::vector<int> shared_rows;  // of a request: the Rows of what it shares
  const bool shared = batch_rows(in, use, 0, in.num_reqs, rows, shared_rows), few = tokens_only(in, rows);
  if (shared && !few) {
    SharedPlanner pl(in, rows, shared_form(in));
    plan_waves(pl);
    plan_shared(in, rows, shared_rows, pl, out);
    return;
  }
  // Heads of 128: workgroups of 8 waves share a tile's staging among more rows
  // (2 x 2048 tokens at 16384 bf16 keys: 953 us against 1045), those of 4 fill
  // the device with fewer rows (1000 tokens at 2100: 47 us against 50 split in two
  // and 60 unsplit).  Heads of 64: 4 waves, three workgroups on a CU (before tiles
  // were kept in L2, 4 x 1024 tokens, window 128: 39 us against 44; 8 x 300 at 1000:
  // 66 against 74; but 2 x 2048 at 16384: 1340 against 1259 in bf16, 1201 against
  // 1217 in mxfp4; now 28, 55, 1200 and 1145 of 4 waves, 8 were not measured again).
  Planner pl(in, rows, few ? CHUNK_TOKENS : CHUNK_WAVES4);
  plan_waves(pl);
  out.form = pl.form;
  // Token items alone that read more than half of the last-level cache (256 MB):
  // what they read is not there when the next call reads it, and goes past the
  // caches (32 requests of 8..32k tokens: bf16 452 -> 425 us, fp8 248 -> 224,
  // mxfp4 149 -> 134).  Smaller reads may be found there (8 x 4000 tokens in bf16:
  // 27 us, 30 past the caches).
  double bytes = 0.0;
  for (const Group& g : pl.groups) bytes += 64.0 * g.units * row_bytes(in.format, in.head_dim) * in.num_kv_heads;
  if (few && bytes > kStreamBytes) out.form = CHUNK_STREAM;
  const int merge_rows = 1024 / in.head_dim;  // rows of one merge workgroup: 256 threads, 4 head dims each
  struct Placed {
    double us;   // of a chunk
    int group, chunks;
    long long slot;
  };
  std::vector<Placed> order;
  order.reserve(pl.groups.size());
  long long slot = 0, items = 0;
  std::vector<long long> slots(pl.groups.size());  // of head 0
  std::vector<int> first_group(rows.size(), -1);   // of a Rows' row tiles, which follow each other
  for (int i = 0; i < (int)pl.groups.size(); ++i) {
    const Group& g = pl.groups[i];
    const int n = pl.chunks(g);
    order.push_back({g.work() / n, i, n, slot});
    items += (long long)n * in.num_kv_heads;
    if (first_group[g.rows] < 0) first_group[g.rows] = i;
    if (n == 1 && !g.partial) continue;
    slots[i] = slot;
    slot += (long long)n * g.nrows * in.num_kv_heads;
    const Rows& set = rows[g.rows];
    if (set.part == PART_SHARED) continue;
    for (int h = 0; h < in.num_kv_heads; ++h) {
      const long long at = slots[i] + (long long)h * n * g.nrows;
      if (!shared) {
        for (int r = 0; r < g.nrows; r += merge_rows)
          out.merges.push_back(ChunkMerge{set.q0, h, g.row0 + r, std::min(merge_rows, g.nrows - r), (int)at + r, g.nrows, n, 0});
        continue;
      }
      for (int r = 0, take; r < g.nrows; r += take) {
        take = std::min(merge_rows, g.nrows - r);
        SharedMerge m{set.q0, h, g.row0 + r, take, (int)at + r, g.nrows, n, 0, 0, 0, 0, 0};
        if (set.part == PART_OWN) {
          // its rows among those of the group, within one of their row tiles
          const int sh = shared_rows[set.req], from = (set.q0 - rows[sh].q0) * group + g.row0 + r;
          const int k = first_group[sh] + from / chunk_rows(pl.form);
          const Group& sg = pl.groups[k];
          const int sn = pl.chunks(sg);
          take = m.nrows = std::min(take, sg.row0 + sg.nrows - from);
          m.shared_slot = (int)(slots[k] + (long long)h * sn * sg.nrows);
          m.shared_row = from - sg.row0;
          m.shared_stride = sg.nrows;
          m.shared_chunks = sn;
        }
        out.shared_merges.push_back(m);
      }
    }
  }
  // Longest first; among equals the kv heads of one key chunk side by side, so
  // that with 8 (or 16, ..) kv heads each XCD (workgroups are dealt to the 8 of
  // them in turn) keeps a head's keys in its own L2 for all row tiles.
  std::stable_sort(order.begin(), order.end(), [](const Placed& a, const Placed& b) { return a.us > b.us; });
  out.items.reserve((size_t)items);
  for (const Placed& x : order) {
    const Group& g = pl.groups[x.group];
    ChunkItem it{};
    const Rows& set = rows[g.rows];
    it.req = set.req;
    it.q0 = set.q0;
    it.nq = set.nq;
    it.row0 = g.row0;
    it.nrows = g.nrows;
    it.page_begin = in.page_indptr[set.req];
    it.page_end = in.page_indptr[set.req + 1];
    it.nchunks = x.chunks;
    it.kind = g.kind;
    it.part = set.part;
    it.bound = set.bound;
    for (it.chunk = 0; it.chunk < x.chunks; ++it.chunk)
      for (it.kvh = 0; it.kvh < in.num_kv_heads; ++it.kvh) {
        it.slot = x.chunks > 1 || g.partial ? (int)(x.slot + (long long)it.kvh * x.chunks * g.nrows) : 0;
        out.items.push_back(it);
      }
  }
  out.partial_rows = slot;
  if (!shared) return;
  out.form |= CHUNK_SHARED;
  shared_tokens(in, out);
}

}  // namespace d2sd
