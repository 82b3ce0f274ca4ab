// Host-built work plan of the shared-prefix attention (csrc/prefix.cuh).
//
// A group is a run of consecutive requests that read one shared prefix; the keys of
// request i are, in this order, its group's prefix rows, its own cached rows and its
// new rows. The plan cuts the queries into tiles and every tile's key chain into
// pieces, and assigns the pieces to persistent CTAs:
//
//   shared tiles   up to 128 consecutive query rows of a group, of any requests,
//                  against the prefix: its rows are read once per tile instead of
//                  once per request, and a tile of 8-row requests fills the MMA;
//   private tiles  up to 128 query rows of one request against its own + new rows;
//   chain tiles    up to 128 query rows of one request against all of its keys, for
//                  groups whose requests fill tiles by themselves (one request, or
//                  kChainRows query rows on average): nothing to merge then.
//
// A tile whose chain is one piece and holds every key of its rows writes the output;
// any other piece leaves normalised fp32 partial rows with their maximum m and sum l, which
// the merge kernel combines (out = sum_c w_c o_c / sum_c w_c, w_c = l_c 2^(m_c - max m)).
#pragma once
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <numeric>
#include <queue>
#include <utility>
#include <vector>

namespace dspark {
namespace prefix {

constexpr int kPlanMagic = 0x44535046;     // "DSPF"
constexpr int kHeadWords = 32;
constexpr int kItemWords = 20;
constexpr int kRunWords = 12;
constexpr int kHeads = 8;                  // KV heads
constexpr int kHalfTile = 64;              // query rows of one MMA tile (x 2 heads = 128 rows)
constexpr int kTileRows = 2 * kHalfTile;   // query rows of an item: two MMA tiles sharing the keys
constexpr int kBlock = 128;                // keys per block
constexpr int kMaxSegs = 3;
constexpr int kAllVisible = 1 << 30;

enum Head {
  kHMagic = 0, kHTotalQ = 2, kHGrid, kHItems, kHCtaAt, kHItemsAt, kHSlots = 8, kHRuns, kHRunsAt, kHTokenRunAt,
  kHPrefixRows, kHOwnRows, kHNewRows, kHCheck = 18, kHMaxItemRows = 20, kHPartRows, kHPartsAt
};
// Item record: a tile, a KV head and a piece of the tile's key chain. Query row t of
// the item sees the keys whose chain position is below kIVisible + t.
enum ItemField {
  kIQ0 = 0, kINq, kIHead, kISlot /* -1: write the output */, kIVisible, kISegs,
  kIDual /* one MMA tile's rows, even key blocks on tile A and odd ones on tile B */,
  kIPart /* workspace row at which the item's first slot begins */, kISeg0 = 8,
  kISegWords = 4 /* source (0 prefix, 1 own, 2 new), first row, keys, chain position of the first key */
};
// Run record: query rows [kRunQ0, + kRunNq) merge the same tiles' partials.
enum RunField {
  kRunQ0 = 0, kRunNq, kRunTiles, kRunTile0 = 4,
  kRunTileWords = 4 /* slot, pieces, slots per (piece, head): 1, 2 or kDualSlots, q0 */
};
constexpr int kDualSlots = 3;              // two slots, both holding (part of) every row
// Behind the runs, the workspace of a run's tiles: (first row of the tile's slots, rows of a
// slot) for each of the two. Slots follow one another as (piece, head, slot).
constexpr int kPartWords = 4;

// Workspace rows of a slot: an MMA tile's rows (query row, head). An even number, so every slot
// starts on 16 bytes. (128 rows throughout took 1.1 GB for 1024 one-row requests.)
__host__ __device__ inline int part_pitch(int nq) { return 2 * (nq > kHalfTile ? kHalfTile : nq); }

// Whether an item's own words are in range: its rows, its head, and its slots among the
// plan's (a direct item, slot -1, needs none; a wide or dual one needs two) and in the
// workspace. The kernels skip an item that fails, so build_plan hands out none.
__host__ __device__ inline bool item_fits(int q0, int nq, int head, int slot, int part, int nsegs, bool dual,
                                          int total_q, int slots, int part_rows) {
  const bool rows = nq >= 1 && nq <= kTileRows && q0 >= 0 && q0 <= total_q - nq;
  const int need = nq > kHalfTile || dual ? 2 : 1;
  const bool store = slot < 0 ? slot == -1 && !dual
                              : slot <= slots - need && (!dual || nq <= kHalfTile) && part >= 0 &&
                                    part <= part_rows - need * part_pitch(nq);
  return rows && store && head >= 0 && head < kHeads && nsegs >= 0 && nsegs <= kMaxSegs;
}

// Costs the schedule balances, in units of one two-tile key block.
constexpr double kCostPair = 1.0;
constexpr double kCostSingle = 0.9;
constexpr double kCostDual = 0.6;
constexpr double kCostItem = 1.6;
constexpr double kCostPartial = 0.5;       // writing one MMA tile's partial rows (and reading them back)
// Mean query rows from which a group's requests get chain tiles instead of a share of the
// group's. Behind 8192 shared keys, chain against shared: 16 requests of 64 rows 115 / 91 us,
// 96 139 / 129, 112 140 / 153, 128 139 / 155; behind 1024: 64 rows 37 / 43, 96 31 / 46. With
// few requests the shared tiles spread better (4 x 128 rows behind 1024: 35 / 27).
constexpr int kChainRows = 96;

struct Seg {
  int src, row, len;
};

struct PlanTile {
  int q0, nq;
  int visible;        // kIVisible
  Seg segs[kMaxSegs];
  int nsegs;
  bool complete;      // holds every key of its rows
  int blocks;
  int pieces, slot, part;
  bool dual;
  int slots() const { return dual || nq > kHalfTile ? 2 : 1; }
};

// Whether a one-tile piece runs its blocks on both MMA tiles: a single tile's chain
// (product, softmax, product) is bound by its latency, two of them overlap. A complete
// tile pays with a merge, which is worth it from kDualBlocks blocks (400 requests of 8 rows
// and no prefix, on both tiles against one: 2 blocks 201 / 181 us, 3 248 / 236, 4 263 / 279,
// 8 377 / 455; 40 requests: 2 32 / 31, 4 39 / 45).
constexpr int kDualBlocks = 4;
inline bool dual_piece(int nq, bool complete, int blocks, int pieces) {
  return nq <= kHalfTile && blocks / pieces >= 2 && (!complete || pieces > 1 || blocks >= kDualBlocks);
}

inline int blocks_of(const Seg& s) { return (s.len + kBlock - 1) / kBlock; }

// Adds tiles of query rows [q0, + nq) (rows rel0.. of a request with q_len rows, or of a
// group) over the chain `segs`; causal >= 0: chain positions visible to row 0.
inline void add_tiles(std::vector<PlanTile>& tiles, int q0, int nq, const Seg* segs, int nsegs, bool causal,
                      long long keys, int q_len, bool complete) {
  for (int t = 0; t < nq; t += kTileRows) {
    PlanTile tile{};
    tile.q0 = q0 + t;
    tile.nq = std::min(kTileRows, nq - t);
    tile.visible = kAllVisible;
    long long left = keys;
    if (causal) {
      tile.visible = static_cast<int>(keys - q_len + t + 1);
      left = std::min(keys, static_cast<long long>(tile.visible) + tile.nq - 1);
    }
    for (int s = 0; s < nsegs; ++s) {
      Seg x = segs[s];
      x.len = static_cast<int>(std::max(0ll, std::min<long long>(x.len, left)));
      left -= x.len;
      if (x.len > 0) {
        tile.segs[tile.nsegs++] = x;
        tile.blocks += blocks_of(x);
      }
    }
    tile.complete = complete;
    tiles.push_back(tile);
  }
}

inline double piece_cost(const PlanTile& t, int blocks, bool direct, bool dual) {
  const bool pair = t.nq > kHalfTile;
  return kCostItem + blocks * (pair ? kCostPair : (dual ? kCostDual : kCostSingle)) +
         (direct ? 0.0 : kCostPartial * (pair ? 2 : 1));
}

// Largest-first assignment of the pieces' costs to `grid` CTAs; returns the makespan.
inline double assign(const std::vector<double>& cost, int grid, std::vector<int>* cta) {
  std::vector<int> order(cost.size());
  std::iota(order.begin(), order.end(), 0);
  std::stable_sort(order.begin(), order.end(), [&](int a, int b) { return cost[a] > cost[b]; });
  using Load = std::pair<double, int>;
  std::priority_queue<Load, std::vector<Load>, std::greater<Load>> heap;
  for (int c = 0; c < grid; ++c) heap.push({0.0, c});
  double worst = 0.0;
  if (cta) cta->assign(cost.size(), 0);
  for (int i : order) {
    Load l = heap.top();
    heap.pop();
    l.first += cost[i];
    worst = std::max(worst, l.first);
    if (cta) (*cta)[i] = l.second;
    heap.push(l);
  }
  return worst;
}

struct PlanInput {
  int groups;
  const int32_t *group_size, *prefix_start, *prefix_len;
  int requests;
  const int32_t *q_len, *own_start, *own_len, *new_start, *new_len;   // new_*: null without new rows
  bool causal;
  int grid_limit;
};

enum PlanStatus { kPlanOk = 0, kPlanInvalid = 1, kPlanTooLarge = 2 };

inline int32_t plan_check(const std::vector<int32_t>& plan) {
  uint32_t h = 2166136261u;                      // FNV-1a over the words, the check word itself as zero
  for (size_t i = 0; i < plan.size(); ++i) {
    h ^= i == kHCheck ? 0u : static_cast<uint32_t>(plan[i]);
    h *= 16777619u;
  }
  return static_cast<int32_t>(h & 0x7fffffffu);
}

inline int build_plan(const PlanInput& in, std::vector<int32_t>& plan) {
  constexpr long long kLimit = 1ll << 30;        // rows, keys of a request and plan offsets stay below
  std::vector<PlanTile> tiles;
  struct Req { int q0, nq, first_tile, n_tiles; };
  struct Group { bool shared; int first_tile, n_tiles, q0, nq, req0, nreq; };
  std::vector<Req> reqs(in.requests);
  std::vector<Group> groups(in.groups);
  long long q0 = 0, prefix_rows = 0, own_rows = 0, new_rows = 0;
  int r = 0;
  for (int g = 0; g < in.groups; ++g) {
    const int n = in.group_size[g];
    if (n < 1 || n > in.requests - r || in.prefix_len[g] < 0 || in.prefix_start[g] < 0) return kPlanInvalid;
    const long long pl = in.prefix_len[g];
    if (in.prefix_start[g] + pl > kLimit) return kPlanTooLarge;
    if (pl > 0) prefix_rows = std::max(prefix_rows, in.prefix_start[g] + pl);
    long long tokens = 0;
    for (int i = r; i < r + n; ++i) {
      const long long q = in.q_len[i], al = in.own_len[i], bl = in.new_len ? in.new_len[i] : 0;
      const long long as = in.own_start[i], bs = in.new_len ? in.new_start[i] : 0;
      if (q < 0 || al < 0 || bl < 0 || as < 0 || bs < 0 || (in.causal && al + bl < q)) return kPlanInvalid;
      if (as + al > kLimit || bs + bl > kLimit || pl + al + bl > kLimit || q0 + tokens + q > kLimit)
        return kPlanTooLarge;
      if (al > 0) own_rows = std::max(own_rows, as + al);
      if (bl > 0) new_rows = std::max(new_rows, bs + bl);
      reqs[i] = Req{static_cast<int>(q0 + tokens), static_cast<int>(q), 0, 0};
      tokens += q;
    }
    Group& gr = groups[g];
    gr = Group{n > 1 && pl > 0 && tokens < static_cast<long long>(kChainRows) * n, 0, 0, static_cast<int>(q0),
               static_cast<int>(tokens), r, n};
    const Seg ps{0, in.prefix_start[g], in.prefix_len[g]};
    if (gr.shared) {
      bool only = true;                          // no request has keys besides the prefix
      for (int i = r; i < r + n; ++i) only = only && in.own_len[i] + (in.new_len ? in.new_len[i] : 0) == 0;
      gr.first_tile = static_cast<int>(tiles.size());
      add_tiles(tiles, gr.q0, gr.nq, &ps, 1, false, pl, 0, only);
      gr.n_tiles = static_cast<int>(tiles.size()) - gr.first_tile;
    }
    for (int i = r; i < r + n; ++i) {
      Seg segs[kMaxSegs] = {ps, {1, in.own_start[i], in.own_len[i]},
                            {2, in.new_len ? in.new_start[i] : 0, in.new_len ? in.new_len[i] : 0}};
      const int skip = gr.shared ? 1 : 0;
      const long long keys = (gr.shared ? 0 : pl) + segs[1].len + segs[2].len;
      reqs[i].first_tile = static_cast<int>(tiles.size());
      if (!gr.shared || keys > 0)
        add_tiles(tiles, reqs[i].q0, reqs[i].nq, segs + skip, kMaxSegs - skip, in.causal, keys, reqs[i].nq,
                  !gr.shared);
      reqs[i].n_tiles = static_cast<int>(tiles.size()) - reqs[i].first_tile;
    }
    q0 += tokens;
    r += n;
  }
  if (r != in.requests) return kPlanInvalid;
  if (tiles.size() > 500000) return kPlanTooLarge;

  // Cut the chains: try several piece lengths and keep the shortest schedule. Pieces
  // are the same for the 8 KV heads, so a slot index is computed from (piece, head).
  double total = 0.0;
  for (const PlanTile& t : tiles) total += kHeads * piece_cost(t, t.blocks, t.complete, dual_piece(t.nq, t.complete, t.blocks, 1));
  auto cut = [&](double target, std::vector<int>& pieces) {
    pieces.resize(tiles.size());
    for (size_t i = 0; i < tiles.size(); ++i) {
      const PlanTile& t = tiles[i];
      const double per = t.nq > kHalfTile ? kCostPair : kCostDual;
      const double room = std::max(per, target - kCostItem);
      pieces[i] = static_cast<int>(std::max(1.0, std::min<double>(t.blocks, std::ceil(t.blocks * per / room))));
    }
  };
  auto costs = [&](const std::vector<int>& pieces, std::vector<double>& cost) {
    cost.clear();
    for (size_t i = 0; i < tiles.size(); ++i)
      for (int h = 0; h < kHeads; ++h)
        for (int p = 0; p < pieces[i]; ++p) {
          const int b0 = static_cast<int>(static_cast<long long>(tiles[i].blocks) * p / pieces[i]);
          const int b1 = static_cast<int>(static_cast<long long>(tiles[i].blocks) * (p + 1) / pieces[i]);
          const bool dual = dual_piece(tiles[i].nq, tiles[i].complete, tiles[i].blocks, pieces[i]);
          cost.push_back(piece_cost(tiles[i], b1 - b0, tiles[i].complete && pieces[i] == 1 && !dual, dual));
        }
  };
  std::vector<int> pieces, best;
  std::vector<double> cost;
  double best_span = 1e300;
  const double share = total / in.grid_limit;
  for (double f : {1e30, 1.0, 1.05, 1.12, 1.25, 1.4, 0.75, 0.6, 0.51, 0.4, 0.34}) {
    cut(std::max(share * f, kCostItem + kCostPair), pieces);
    costs(pieces, cost);
    if (cost.size() > 4000000) return kPlanTooLarge;
    const double span = assign(cost, in.grid_limit, nullptr);
    if (span < best_span - 1e-9) {
      best_span = span;
      best = pieces;
    }
  }
  long long slots = 0, part_rows = 0;
  for (size_t i = 0; i < tiles.size(); ++i) {
    PlanTile& t = tiles[i];
    t.pieces = best[i];
    t.slot = -1;
    t.dual = dual_piece(t.nq, t.complete, t.blocks, t.pieces);
    if (!(t.complete && t.pieces == 1 && !t.dual)) {
      const long long n = static_cast<long long>(t.pieces) * kHeads * t.slots();
      t.slot = static_cast<int>(slots);
      t.part = static_cast<int>(part_rows);
      slots += n;
      part_rows += n * part_pitch(t.nq);
      if (part_rows > kLimit) return kPlanTooLarge;
    }
  }
  costs(best, cost);
  const int n_items = static_cast<int>(cost.size());
  const int grid = std::max(1, std::min(in.grid_limit, n_items));
  std::vector<int> cta;
  assign(cost, grid, &cta);
  std::vector<std::vector<std::pair<double, int>>> per_cta(grid);
  std::vector<int32_t> items(static_cast<size_t>(n_items) * kItemWords, 0);
  int idx = 0;
  for (const PlanTile& t : tiles)
    for (int h = 0; h < kHeads; ++h)
      for (int p = 0; p < t.pieces; ++p, ++idx) {
        int32_t* it = items.data() + static_cast<size_t>(idx) * kItemWords;
        const int b0 = static_cast<int>(static_cast<long long>(t.blocks) * p / t.pieces);
        const int b1 = static_cast<int>(static_cast<long long>(t.blocks) * (p + 1) / t.pieces);
        it[kIQ0] = t.q0;
        it[kINq] = t.nq;
        it[kIHead] = h;
        it[kISlot] = t.slot < 0 ? -1 : t.slot + (p * kHeads + h) * t.slots();
        it[kIDual] = t.dual ? 1 : 0;
        it[kIPart] = t.slot < 0 ? 0 : t.part + (p * kHeads + h) * t.slots() * part_pitch(t.nq);
        it[kIVisible] = t.visible;
        int at = 0, pos = 0, n = 0;
        for (int s = 0; s < t.nsegs; ++s) {
          const int nb = blocks_of(t.segs[s]);
          const int lo = std::max(b0 - at, 0), hi = std::min(b1 - at, nb);
          if (lo < hi) {
            int32_t* w = it + kISeg0 + n * kISegWords;
            w[0] = t.segs[s].src;
            w[1] = t.segs[s].row + lo * kBlock;
            w[2] = std::min(t.segs[s].len, hi * kBlock) - lo * kBlock;
            w[3] = pos + lo * kBlock;
            ++n;
          }
          at += nb;
          pos += t.segs[s].len;
        }
        it[kISegs] = n;
        if (!item_fits(it[kIQ0], it[kINq], h, it[kISlot], it[kIPart], n, t.dual, static_cast<int>(q0),
                       static_cast<int>(slots), static_cast<int>(part_rows)))
          return kPlanInvalid;
        per_cta[cta[idx]].push_back({cost[idx], idx});
      }

  // Merge runs: maximal row ranges whose rows merge the same tiles.
  std::vector<int32_t> runs, parts, token_run;
  if (slots > 0) {
    token_run.assign(q0, -1);
    auto add_run = [&](int a, int b, const PlanTile* x, const PlanTile* y) {
      if (a >= b) return;
      const int id = static_cast<int>(runs.size()) / kRunWords;
      runs.resize(runs.size() + kRunWords, 0);
      parts.resize(parts.size() + kPartWords, 0);
      int32_t* w = runs.data() + static_cast<size_t>(id) * kRunWords;
      w[kRunQ0] = a;
      w[kRunNq] = b - a;
      int n = 0;
      for (const PlanTile* t : {x, y})
        if (t) {
          int32_t* k = w + kRunTile0 + kRunTileWords * n++;
          k[0] = t->slot;
          k[1] = t->pieces;
          k[2] = t->dual ? kDualSlots : t->slots();
          k[3] = t->q0;
          parts[parts.size() - kPartWords + 2 * n - 2] = t->part;
          parts[parts.size() - kPartWords + 2 * n - 1] = part_pitch(t->nq);
        }
      w[kRunTiles] = n;
      std::fill(token_run.begin() + a, token_run.begin() + b, id);
    };
    for (const Group& g : groups)
      for (int i = g.req0; i < g.req0 + g.nreq; ++i) {
        // walk the request's rows over the boundaries of its private and the group's shared tiles
        const int end = reqs[i].q0 + reqs[i].nq;
        for (int a = reqs[i].q0; a < end;) {
          int b = end;
          const PlanTile *x = nullptr, *y = nullptr;
          if (g.shared) {
            x = &tiles[g.first_tile + (a - g.q0) / kTileRows];
            b = std::min(b, x->q0 + x->nq);
          }
          if (reqs[i].n_tiles > 0) {
            y = &tiles[reqs[i].first_tile + (a - reqs[i].q0) / kTileRows];
            b = std::min(b, y->q0 + y->nq);
          }
          if (x && x->slot < 0) x = nullptr;
          if (y && y->slot < 0) y = nullptr;
          if (x || y) add_run(a, b, x, y);
          a = b;
        }
      }
  }

  auto round4 = [](long long v) { return (v + 3) & ~3ll; };
  const long long cta_at = kHeadWords, items_at = round4(cta_at + grid + 1),
                  runs_at = items_at + static_cast<long long>(items.size()),
                  parts_at = runs_at + static_cast<long long>(runs.size()),
                  token_at = parts_at + static_cast<long long>(parts.size()),
                  words = round4(token_at + static_cast<long long>(token_run.size()));
  if (words > kLimit) return kPlanTooLarge;
  plan.assign(words, 0);
  plan[kHMagic] = kPlanMagic;
  plan[kHTotalQ] = static_cast<int32_t>(q0);
  plan[kHGrid] = grid;
  plan[kHItems] = n_items;
  plan[kHCtaAt] = static_cast<int32_t>(cta_at);
  plan[kHItemsAt] = static_cast<int32_t>(items_at);
  plan[kHSlots] = static_cast<int32_t>(slots);
  plan[kHRuns] = static_cast<int32_t>(runs.size() / kRunWords);
  plan[kHRunsAt] = static_cast<int32_t>(runs_at);
  plan[kHPartsAt] = static_cast<int32_t>(parts_at);
  plan[kHPartRows] = static_cast<int32_t>(part_rows);
  plan[kHTokenRunAt] = static_cast<int32_t>(token_at);
  plan[kHPrefixRows] = static_cast<int32_t>(prefix_rows);
  plan[kHOwnRows] = static_cast<int32_t>(own_rows);
  plan[kHNewRows] = static_cast<int32_t>(new_rows);
  for (const PlanTile& t : tiles) plan[kHMaxItemRows] = std::max(plan[kHMaxItemRows], t.nq);
  int next = 0;
  for (int c = 0; c < grid; ++c) {
    plan[cta_at + c] = next;
    std::stable_sort(per_cta[c].begin(), per_cta[c].end(),
                     [](const std::pair<double, int>& a, const std::pair<double, int>& b) { return a.first > b.first; });
    for (const auto& e : per_cta[c])
      std::copy_n(items.begin() + static_cast<size_t>(e.second) * kItemWords, kItemWords,
                  plan.begin() + items_at + static_cast<long long>(next++) * kItemWords);
  }
  plan[cta_at + grid] = next;
  std::copy(runs.begin(), runs.end(), plan.begin() + runs_at);
  std::copy(parts.begin(), parts.end(), plan.begin() + parts_at);
  std::copy(token_run.begin(), token_run.end(), plan.begin() + token_at);
  plan[kHCheck] = plan_check(plan);
  return kPlanOk;
}

}  // namespace prefix
}  // namespace dspark
