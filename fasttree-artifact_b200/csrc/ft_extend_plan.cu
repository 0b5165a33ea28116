// Host-side schedule of an extend-attention step (no device code).
//
// The step's query tokens are laid out request by request and packed, with their GQA group, into query tiles of
// rows_per_tile rows.  A block is one query tile, or two that read mostly the same K/V.  Its K/V is the union of what
// its tokens may see, as a list of segments - runs of entries of the row-id table - each with the block's tokens that
// see it: a prefix that the block's requests share stands there once.  The segments are numbered through (virtual
// positions) and cut into tiles of tile_tokens.
//
// A block whose K/V is long for the machine is cut into items along the virtual positions; items leave partial rows,
// which a second launch merges.  Every (item, KV head) is a task; tasks are dealt to the SMs longest first, each to the
// SM that is free first by the cost model below, and of several cuts the one whose simulated schedule ends first is
// taken.
//
// Layout of the table, in ints.
// CTA (16): its first task in sm_tasks, one past its last, the first task itself, 0, that task's first and last K/V tile, its block's
//   first record in the tile table, 0, the first four ints of its first tile's record, then 4 zeros.
// Item (32): first and last K/V tile, step, query tiles, virtual length, the block's first record in the tile table, 0, 0, then two
//   streams of {first token, tokens, first tile, last tile, -1 if the tokens' rows go to the output itself, else the place in the
//   extra table of each token's partial row (-2: it sees nothing there and has none), query tile of the item,
//   first token within the block, query tile of the block}, then the record of its first tile.  Two streams are two query tiles
//   over the same K/V tiles (step 1), or one query tile whose even and odd K/V tiles run as two streams with partial rows of
//   their own (step 2).
// Tile (8): table offset of its first token (low, high), tokens, -1 if the tokens' offsets are consecutive, else the place of
//   their offsets (low, high each) in the extra table; per query tile of the block -1 if each of its tokens sees the whole tile of
//   tile_tokens, else the place of the bits of those that the block's tokens see, a word per 32 and token; 0, 0.
// Token (2): row of q, position.  Merged token (4): row of q, first entry of its list of partial rows, entries, 0.
//
// Plans of drafted tokens (a tree per request, whose parents only the device knows) are made for every tree of their sizes: a
// token may see any drafted token before it and, behind a window, any cached one that depth 0 would show it, and tiles where that
// differs from tree to tree have bits for ft_draft_tree to fill in.  Until then the tokens are chains.
// Draft (8), one per request with tokens: first row of q, tokens, cached tokens, start of its entries of the row-id table (low, high),
// its number, its first span, spans.  Span (8), a stretch of a tile that some tokens of one request see differently from tree to
// tree: place of the first token's bits in the extra table, tokens, the first one's number among the request's, first and last bit,
// position of the first bit less the cached tokens, 0, 0.
#include <algorithm>
#include <climits>
#include <cstdint>
#include <cstring>
#include <memory>
#include <new>
#include <queue>
#include <vector>

#include "fasttree_b200.h"
#include "ft_draft_span.cuh"

struct ft_extend_plan {
  std::vector<int32_t> table;
  ft_extend_plan_info info;
};

namespace {

constexpr int ITEM_INTS = 32;

struct Segment {
  int64_t kv_off;
  int32_t len, pos0, tok_lo, tok_hi, voff;
};

struct Token {
  int32_t q_row, pos, cached, req;
};

struct Block {
  int tok0 = 0, ntok = 0, split = 0;  // its tokens; those from `split` on belong to the second query tile (split == ntok: none)
  int seg0 = 0, nseg = 0, len = 0;    // virtual length
  int req_lo = 0, req_hi = 0;
};

struct Item {
  int block, t0, t1;
  bool alternate;    // one query tile, two streams
  int which;         // bit w: query tile w takes part
  int lo[2], hi[2];  // tiles of the streams
  double cost;
};

struct Costs {  // microseconds, B200: per K/V tile of two query tiles, of one in two streams or in one, and per item
  double pair, load, alternate, single, item;
};

struct Problem {
  const int64_t *seq, *ext, *start, *qstart, *shared;
  const int32_t* ids;  // of drafts: the requests' numbers
  int batch, group, kv_heads, head_dim, rows, tile;
  int64_t window;
  bool draft;
  bool two_tiles, streams;
  int tokens_per_tile;
  int slots;
  Costs cost;
};

// The positions that a token may see, and those that it sees whatever its request's tree is.
struct Sight {
  int64_t from, to, sure_from, sure_to;
  Sight(const Problem& p, const Token& t) {
    to = t.pos + 1;
    sure_to = p.draft ? t.cached : to;
    from = sure_from = 0;
    if (p.window > 0) {
      from = std::max<int64_t>((p.draft ? t.cached : t.pos) - p.window + 1, 0);
      sure_from = std::max<int64_t>(t.pos - p.window + 1, 0);
    }
  }
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
uint32_t bits_below(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

class Builder {
 public:
  explicit Builder(const Problem& p) : p_(p) {}
  double end = 0;  // of the simulated schedule, in microseconds

  void run() {
    place_tokens();
    pack_blocks();
    choose_items();
  }

  std::vector<Token> tokens;
  std::vector<Segment> segs;
  std::vector<Block> blocks;
  std::vector<Item> items;
  std::vector<int> task_order;  // items x heads dealt to the slots: slot s takes sm_tasks[sm_offs[s] ..]
  std::vector<int32_t> sm_offs, sm_tasks;

 private:
  const Problem p_;
  std::vector<int> req_of_, first_tok_;

  int64_t prefix(int i) const { return p_.seq[i] - p_.ext[i]; }

  void place_tokens() {
    first_tok_.resize(p_.batch + 1, 0);
    for (int i = 0; i < p_.batch; ++i) {
      first_tok_[i] = (int)tokens.size();
      for (int64_t t = 0; t < p_.ext[i]; ++t) {
        tokens.push_back({(int32_t)(p_.qstart[i] + t), (int32_t)(prefix(i) + t), (int32_t)prefix(i), i});
        req_of_.push_back(i);
      }
    }
    first_tok_[p_.batch] = (int)tokens.size();
  }

  // Query tiles: a request joins the tile that the one before it has not filled where that costs less K/V than a tile of
  // its own - whole if it fits and does not read long stretches alone (those would only become tiles with masks), in part if
  // what it shares is the most of what it reads.
  void pack_blocks() {
    std::vector<std::pair<int, int>> tiles;  // [first, last) token
    const int cap = p_.tokens_per_tile;
    int cur = 0, room = 0, last = -1;  // tokens [cur, end) are in the open tile
    int end = 0;
    for (int i = 0; i < p_.batch; ++i) {
      int64_t e = p_.ext[i];
      if (e == 0) continue;
      int at = first_tok_[i];
      if (room > 0) {
        int64_t common = INT64_MAX;  // with the request before it that has tokens
        for (int k = last + 1; k <= i; ++k) common = std::min(common, p_.shared[k]);
        const int64_t part = std::min<int64_t>(e, room), own = prefix(i) - common + part;
        const bool alone = own > 4 * p_.tile && own > 4 * common;
        const bool join = (e <= room && !alone) || (common > 0 && own * cap < part * p_.seq[i]);
        if (join) {
          end = at + (int)part;
          at = end;
          e -= part;
          room -= (int)part;
        }
        if (e > 0 || room == 0) {
          tiles.push_back({cur, end});
          room = 0;
        }
      }
      while (e > 0) {
        const int take = (int)std::min<int64_t>(e, cap);
        cur = at;
        end = at += take;
        e -= take;
        room = cap - take;
        if (e > 0 || room == 0) {
          tiles.push_back({cur, end});
          room = 0;
        }
      }
      last = i;
    }
    if (room > 0) tiles.push_back({cur, end});

    for (size_t i = 0; i < tiles.size(); ++i) {
      Block one = make_block(tiles[i].first, tiles[i].second, tiles[i].second);
      if (p_.two_tiles && i + 1 < tiles.size()) {
        // two tiles together where they read mostly the same
        const size_t mark = segs.size();
        const Block other = make_block(tiles[i + 1].first, tiles[i + 1].second, tiles[i + 1].second);
        segs.resize(mark);
        Block both = make_block(tiles[i].first, tiles[i + 1].second, tiles[i].second);
        if (both.len * 100ll <= 80ll * ((int64_t)one.len + other.len)) {
          segs.erase(segs.begin() + one.seg0, segs.begin() + both.seg0);
          both.seg0 = one.seg0;
          blocks.push_back(both);
          ++i;
          continue;
        }
        segs.resize(mark);
      }
      blocks.push_back(one);
    }
  }

  Block make_block(int tok0, int tok1, int split) {
    Block b;
    b.tok0 = tok0;
    b.ntok = tok1 - tok0;
    b.split = split - tok0;
    b.req_lo = req_of_[tok0];
    b.req_hi = req_of_[tok1 - 1];
    b.seg0 = (int)segs.size();
    emit(b, b.req_lo, b.req_hi, 0);
    b.nseg = (int)segs.size() - b.seg0;
    return b;
  }

  // the tokens of requests lo .. hi that are in the block
  std::pair<int, int> toks(const Block& b, int lo, int hi) const {
    return {std::max(first_tok_[lo], b.tok0), std::min(first_tok_[hi + 1], b.tok0 + b.ntok)};
  }

  void emit(Block& b, int lo, int hi, int64_t depth) {
    const std::pair<int, int> tk = toks(b, lo, hi);
    if (tk.first >= tk.second) return;
    int64_t first = INT64_MAX, common = INT64_MAX;
    for (int t = tk.first; t < tk.second; ++t) first = std::min(first, Sight(p_, tokens[t]).from);
    if (lo == hi) common = tokens[tk.second - 1].pos + 1;
    for (int k = lo + 1; k <= hi; ++k) common = std::min(common, p_.shared[k]);
    const int64_t begin = std::max(depth, first);
    if (begin < common) {
      segs.push_back({p_.start[lo] + begin, (int32_t)(common - begin), (int32_t)begin, tk.first - b.tok0, tk.second - b.tok0, b.len});
      b.len += (int32_t)(common - begin);
    }
    if (lo == hi) return;
    const int64_t next = std::max(depth, common);
    for (int k = lo, from = lo; k <= hi; ++k)
      if (k == hi || p_.shared[k + 1] <= common) {
        emit(b, from, k, next);
        from = k + 1;
      }
  }

  int tiles_of(const Block& b) const { return (int)ceil_div(b.len, p_.tile); }

  // per K/V tile of the block: which of its query tiles see a token of it
  std::vector<uint8_t> activity(const Block& b) const {
    std::vector<uint8_t> act(tiles_of(b), 0);
    for (int s = b.seg0; s < b.seg0 + b.nseg; ++s) {
      const Segment& g = segs[s];
      for (int w = 0; w < 2; ++w) {
        const int lo = std::max(g.tok_lo, w == 0 ? 0 : b.split), hi = std::min(g.tok_hi, w == 0 ? b.split : b.ntok);
        if (lo >= hi) continue;
        int64_t from = INT64_MAX, to = 0;
        for (int t = lo; t < hi; ++t) {
          const Sight see(p_, tokens[b.tok0 + t]);
          from = std::min(from, see.from);
          to = std::max(to, see.to);
        }
        from = std::max<int64_t>(from - g.pos0, 0);
        to = std::min<int64_t>(to - g.pos0, g.len);
        if (from >= to) continue;
        for (int64_t t = (g.voff + from) / p_.tile; t <= (g.voff + to - 1) / p_.tile; ++t) act[t] |= (uint8_t)(1 << w);
      }
    }
    return act;
  }

  // tiles [t0, t1) of a block as one item; streams: whether one query tile may run as two streams
  Item make_item(int block, const std::vector<uint8_t>& act, int t0, int t1, bool streams) const {
    Item it;
    it.block = block;
    it.which = 0;
    int n = 0;
    for (int w = 0; w < 2; ++w) {
      int lo = t1, hi = t0;
      for (int t = t0; t < t1; ++t)
        if (act[t] & (1 << w)) {
          lo = std::min(lo, t);
          hi = t + 1;
        }
      it.lo[w] = it.hi[w] = t0;
      if (lo < hi) {
        it.which |= 1 << w;
        it.lo[w] = lo;
        it.hi[w] = hi;
        n += hi - lo;
      }
    }
    it.t0 = t1;
    it.t1 = t0;
    for (int w = 0; w < 2; ++w)
      if (it.which & (1 << w)) {
        it.t0 = std::min(it.t0, it.lo[w]);
        it.t1 = std::max(it.t1, it.hi[w]);
      }
    it.alternate = streams && it.which != 3 && it.t1 - it.t0 >= 2;
    const Costs& c = p_.cost;
    const int loaded = it.t1 - it.t0;
    it.cost = c.item + (it.which == 3 ? c.pair * n + c.load * loaded : it.alternate ? c.alternate * loaded : c.single * loaded);
    return it;
  }

  // Deals the tasks, longest first, to the slot that is free first; returns when the last one is done.
  double deal(const std::vector<Item>& its, std::vector<int>* order, std::vector<int>* slot_of) const {
    std::vector<int> by(its.size());
    for (size_t i = 0; i < by.size(); ++i) by[i] = (int)i;
    std::stable_sort(by.begin(), by.end(), [&](int a, int b) { return its[a].cost > its[b].cost; });
    typedef std::pair<double, int> Free;
    std::priority_queue<Free, std::vector<Free>, std::greater<Free>> free;
    for (int s = 0; s < p_.slots; ++s) free.push({0.0, s});
    double end = 0;
    for (int i : by)
      for (int h = 0; h < p_.kv_heads; ++h) {
        Free f = free.top();
        free.pop();
        f.first += its[i].cost;
        end = std::max(end, f.first);
        if (order != nullptr) {
          order->push_back(i * p_.kv_heads + h);
          slot_of->push_back(f.second);
        }
        free.push(f);
      }
    return end;
  }

  // about how many of the block's tokens see something of an item
  int seen_by(const Item& it) const {
    const Block& b = blocks[it.block];
    int n = 0;
    for (int s = b.seg0; s < b.seg0 + b.nseg; ++s)
      if (segs[s].voff < it.t1 * p_.tile && segs[s].voff + segs[s].len > it.t0 * p_.tile) n += segs[s].tok_hi - segs[s].tok_lo;
    return std::min(n, it.which == 3 ? b.ntok : it.which == 1 ? b.split : b.ntok - b.split);
  }

  void choose_items() {
    const int nb = (int)blocks.size();
    std::vector<std::vector<uint8_t>> act(nb);
    std::vector<std::vector<int>> cuts(nb);  // section borders
    for (int b = 0; b < nb; ++b) {
      act[b] = activity(blocks[b]);
      const int n = (int)act[b].size();
      // a block of two query tiles is cut where a long run of K/V is seen by one of them alone
      std::vector<int>& c = cuts[b];
      c.push_back(0);
      for (int t = 0; t < n;) {
        int e = t;
        while (e < n && act[b][e] == act[b][t]) ++e;
        if (e - t >= 6 && act[b][t] != 3 && blocks[b].split < blocks[b].ntok) {
          if (c.back() != t) c.push_back(t);
          if (e < n) c.push_back(e);
        }
        t = e;
      }
      c.push_back(n);
    }
    double total = 0;
    auto cut = [&](double most, std::vector<Item>& out, int from_block = 0, bool remainder = false) {
      out.clear();
      double parts = 0;  // partial rows of the cut
      for (int b = 0; b < nb; ++b) {
        const double limit = b < from_block ? 0 : most;
        const size_t from = out.size();
        for (size_t s = 0; s + 1 < cuts[b].size(); ++s) {
          const int t0 = cuts[b][s], t1 = cuts[b][s + 1];
          const bool whole = cuts[b].size() == 2;
          const Item one = make_item(b, act[b], t0, t1, p_.streams && !(whole && limit <= 0));
          if (one.which == 0) continue;
          int n = 1;
          if (limit > 0) {
            const double work = one.cost - p_.cost.item;
            n = (int)std::min<int64_t>(std::max<int64_t>((int64_t)((work + limit - 1e-9) / limit), 1), one.t1 - one.t0);
            // a short block of one query tile stays one item that writes the output itself
            if (whole && n == 1 && one.alternate && one.t1 - one.t0 <= 6) {
              out.push_back(make_item(b, act[b], t0, t1, false));
              continue;
            }
          }
          for (int k = 0; k < n; ++k) {
            const int all = one.t1 - one.t0;
            int a = one.t0 + (int)((int64_t)all * k / n), e = one.t0 + (int)((int64_t)all * (k + 1) / n);
            if (remainder && n > 1) {  // pieces as long as the limit allows, and what is left
              const int len = std::max(1, (int)(limit * all / (one.cost - p_.cost.item)));
              a = std::min(one.t1, one.t0 + k * len);
              e = k + 1 == n ? one.t1 : std::min(one.t1, a + len);
              if (a >= e) continue;
            }
            const Item it = make_item(b, act[b], a, e, p_.streams && !(whole && limit <= 0));
            if (it.which != 0) out.push_back(it);
          }
        }
        if (out.size() - from > 1 || (out.size() > from && out[from].alternate))
          for (size_t i = from; i < out.size(); ++i) parts += (out[i].alternate ? 2.0 : 1.0) * seen_by(out[i]);
      }
      return parts;
    };
    std::vector<Item> trial;
    cut(0, trial);
    for (const Item& it : trial) total += it.cost * p_.kv_heads;
    const double even = total / p_.slots;
    auto merge_cost = [&](double parts) {  // a launch, and the partial rows written and read back
      return parts > 0 ? 4.0 + parts * p_.kv_heads * p_.group * 8.0 * p_.head_dim / 4e6 : 0.0;
    };
    // no schedule of these items ends sooner: their work spread evenly, the dearest of them, the merge
    auto at_least = [&](const std::vector<Item>& its, double parts) {
      double sum = 0, dearest = 0;
      for (const Item& it : its) {
        sum += it.cost * p_.kv_heads;
        dearest = std::max(dearest, it.cost);
      }
      return std::max(sum / p_.slots, dearest) + merge_cost(parts);
    };
    double best = -1;
    static const double pieces[] = {0, 2.0, 1.5, 1.25, 1.15, 1.08, 1.04, 1.0, 0.75, 0.5, 0.34, 0.25};
    for (int form = 0; form < 2 * (int)(sizeof(pieces) / sizeof(pieces[0])); ++form) {
      const double f = pieces[form / 2];
      if (form % 2 == 1 && (f < 1.0 || f > 1.3)) continue;  // in equal pieces, or long ones and a remainder
      const double parts = cut(f * even, trial, 0, form % 2 == 1);
      if (best >= 0 && at_least(trial, parts) >= best * 0.99) continue;
      const double finish = deal(trial, nullptr, nullptr) + merge_cost(parts);
      if (best < 0 || finish < best * 0.99) {
        best = end = finish;
        items = trial;
      }
      if (f == 0 && finish <= 1.04 * even + 1.0) break;  // nothing to gain
    }
    // Tasks that fill some rounds of the slots and leave a part of one: only the blocks of that part are cut.
    const int64_t tasks = (int64_t)nb * p_.kv_heads, left = tasks % p_.slots;
    if (best > 1.04 * even + 1.0 && tasks > p_.slots && tasks < 16 * p_.slots && left > 0) {
      const int few = (int)std::min<int64_t>(nb, ceil_div(left, p_.kv_heads));
      double typical = 0;
      for (int b = nb - few; b < nb; ++b) typical += make_item(b, act[b], 0, (int)act[b].size(), false).cost / few;
      static const int ways[] = {2, 3, 4, 6};
      for (int n : ways) {
        const double parts = cut(typical / n, trial, nb - few);
        if (at_least(trial, parts) >= best * 0.98) continue;
        const double finish = deal(trial, nullptr, nullptr) + merge_cost(parts);
        if (finish < best * 0.98) {
          best = end = finish;
          items = trial;
        }
      }
    }
    std::vector<int> order, slot;
    deal(items, &order, &slot);
    sm_offs.assign(p_.slots + 1, 0);
    for (int s : slot) ++sm_offs[s + 1];
    for (int s = 0; s < p_.slots; ++s) sm_offs[s + 1] += sm_offs[s];
    sm_tasks.resize(order.size());
    std::vector<int32_t> at(sm_offs.begin(), sm_offs.end() - 1);
    for (size_t i = 0; i < order.size(); ++i) sm_tasks[at[slot[i]]++] = order[i];
  }
};

// Where the step is bound by the distinct K/V rows that come from memory rather than by products, a tile costs an SM its share of
// the copy rate.
void memory_bound_costs(Problem& p, int elem_bytes, int num_sms) {
  double distinct = 0, pairs = 0;
  for (int i = 0; i < p.batch; ++i) {
    if (p.ext[i] == 0) continue;
    const int64_t cached = p.seq[i] - p.ext[i], reach = p.window > 0 ? std::min(p.seq[i], p.window + p.ext[i]) : p.seq[i];
    distinct += (double)std::min(reach, p.seq[i] - p.shared[i]);
    pairs += (double)p.ext[i] * (double)std::min(reach, cached + (p.ext[i] + 1) / 2);
  }
  const double bytes = distinct * p.kv_heads * 2.0 * p.head_dim * elem_bytes, flops = pairs * p.kv_heads * p.group * 4.0 * p.head_dim;
  if (bytes / 6.2e6 <= flops / 1.0e9) return;
  const double share = p.tile * 2.0 * p.head_dim * elem_bytes / (6.2e6 / num_sms);
  p.cost.alternate = std::max(p.cost.alternate, share);
  p.cost.single = std::max(p.cost.single, share);
  p.cost.load = std::max(p.cost.load, share - 2 * p.cost.pair);
}

// The stretches of the tile [v0, v1) of a block that tokens of a request see differently from tree to tree.
void add_spans(const Problem& p, const Builder& b, const Block& blk, int sg, int v0, int v1, int bits_at,
               std::vector<std::vector<DraftSpan>>& spans_of) {
  const int words = p.tile / 32;
  for (int s = sg; s < blk.seg0 + blk.nseg && b.segs[s].voff < v1; ++s) {
    const Segment& g = b.segs[s];
    const int lo = std::max(v0, (int)g.voff), hi = std::min(v1, g.voff + g.len);
    const int64_t pos_lo = g.pos0 + (lo - g.voff), pos_hi = g.pos0 + (hi - g.voff);
    for (int t = g.tok_lo; t < g.tok_hi;) {
      const Token& first = b.tokens[blk.tok0 + t];
      int e = t;
      bool differs = false;
      for (; e < g.tok_hi && b.tokens[blk.tok0 + e].req == first.req; ++e) {
        const Sight see(p, b.tokens[blk.tok0 + e]);
        differs |= std::max(pos_lo, see.from) < std::min(pos_hi, see.to) && (pos_lo < see.sure_from || pos_hi > see.sure_to);
      }
      if (differs && lo < hi)
        spans_of[first.req].push_back({bits_at + t * words, e - t, first.pos - first.cached, lo - v0, hi - v0, (int32_t)(pos_lo - first.cached), 0, 0});
      t = e;
    }
  }
}

void pack(const Problem& p, const Builder& b, ft_extend_plan* out) {
  ft_extend_plan_info& info = out->info;
  std::vector<int32_t>& t = out->table;
  auto align = [&] { t.resize((t.size() + 3) / 4 * 4, 0); };
  // partial rows: every stream of an item of a block with more than one of them has its tokens' rows
  std::vector<int> streams(b.blocks.size(), 0);
  for (const Item& it : b.items) streams[it.block] += it.alternate ? 2 : 1;
  std::vector<char> partial(b.blocks.size(), 0);
  {
    std::vector<int> n_items(b.blocks.size(), 0);
    for (const Item& it : b.items) ++n_items[it.block];
    for (const Item& it : b.items) partial[it.block] |= (char)(n_items[it.block] > 1 || it.alternate);
  }
  std::vector<std::vector<int32_t>> rows_of(b.tokens.size());  // per token its partial rows
  int64_t rows = 0;
  // records of the blocks' tiles
  std::vector<int32_t> tiles, extra, tile0(b.blocks.size(), 0);
  const int words = p.tile / 32;
  std::vector<std::vector<DraftSpan>> spans_of(p.draft ? p.batch : 0);  // per request
  info.kv_entries_len = 0;
  for (size_t k = 0; k < b.blocks.size(); ++k) {
    const Block& blk = b.blocks[k];
    tile0[k] = (int32_t)(tiles.size() / 8);
    // what token t of the block may see of segment g, and what it surely does, as virtual positions
    auto sight = [&](const Segment& g, int t, int64_t& from, int64_t& to) {
      const Sight see(p, b.tokens[blk.tok0 + t]);
      from = g.voff + std::max<int64_t>(see.from - g.pos0, 0);
      to = g.voff + std::min<int64_t>(g.len, see.to - g.pos0);
    };
    auto sure = [&](const Segment& g, int t, int64_t& from, int64_t& to) {
      const Sight see(p, b.tokens[blk.tok0 + t]);
      from = g.voff + std::max<int64_t>(see.sure_from - g.pos0, 0);
      to = g.voff + std::min<int64_t>(g.len, see.sure_to - g.pos0);
    };
    int sg = blk.seg0, sg_known = -1;
    int64_t all_lo[2] = {0, 0}, all_hi[2] = {0, 0};  // what all tokens of query tile w see of segment sg
    for (int v0 = 0; v0 < blk.len; v0 += p.tile) {
      while (b.segs[sg].voff + b.segs[sg].len <= v0) ++sg;
      const int v1 = std::min(v0 + p.tile, blk.len);
      const Segment& g = b.segs[sg];
      const int64_t off = g.kv_off + (v0 - g.voff);
      const bool single = g.voff + g.len >= v1;
      int32_t x[8] = {(int32_t)(uint32_t)(off & 0xffffffffll), (int32_t)(off >> 32), v1 - v0, -1, -1, -1, 0, 0};
      if (!single) {
        x[3] = (int32_t)extra.size();
        extra.resize(extra.size() + 2 * p.tile, 0);
        for (int s = sg; s < blk.seg0 + blk.nseg && b.segs[s].voff < v1; ++s)
          for (int v = std::max(v0, (int)b.segs[s].voff); v < std::min(v1, b.segs[s].voff + b.segs[s].len); ++v) {
            const int64_t e = b.segs[s].kv_off + (v - b.segs[s].voff);
            extra[x[3] + 2 * (v - v0)] = (int32_t)(uint32_t)(e & 0xffffffffll);
            extra[x[3] + 2 * (v - v0) + 1] = (int32_t)(e >> 32);
          }
      } else if (sg != sg_known) {
        sg_known = sg;
        for (int w = 0; w < 2; ++w) {
          const int lo = w == 0 ? 0 : blk.split, hi = w == 0 ? blk.split : blk.ntok;
          all_lo[w] = 0;
          all_hi[w] = g.tok_lo <= lo && g.tok_hi >= hi ? INT64_MAX : 0;
          for (int t = lo; t < hi && all_hi[w] > 0; ++t) {
            int64_t from, to;
            sure(g, t, from, to);
            all_lo[w] = std::max(all_lo[w], from);
            all_hi[w] = std::min(all_hi[w], to);
          }
        }
      }
      int32_t bits_at = -1;
      for (int w = 0; w < 2; ++w) {
        if (single && v1 - v0 == p.tile && v0 >= all_lo[w] && v1 <= all_hi[w]) continue;
        if (bits_at < 0) {
          bits_at = (int32_t)extra.size();
          extra.resize(extra.size() + (size_t)(blk.ntok * words + 3) / 4 * 4, 0);
          for (int s = sg; s < blk.seg0 + blk.nseg && b.segs[s].voff < v1; ++s)
            for (int t = b.segs[s].tok_lo; t < b.segs[s].tok_hi; ++t) {
              int64_t from, to;
              sight(b.segs[s], t, from, to);
              const int lo = (int)(std::max<int64_t>(from, v0) - v0), hi = (int)(std::min<int64_t>(to, v1) - v0);
              for (int wd = 0; wd < words && lo < hi; ++wd)
                extra[bits_at + t * words + wd] |= (int32_t)(bits_below(hi - 32 * wd) & ~bits_below(lo - 32 * wd));
            }
        }
        x[4 + w] = bits_at;
      }
      if (p.draft && bits_at >= 0) add_spans(p, b, blk, sg, v0, v1, bits_at, spans_of);
      tiles.insert(tiles.end(), x, x + 8);
      if (extra.size() > (size_t)INT32_MAX / 2) throw std::bad_alloc();
    }
  }
  for (const Segment& g : b.segs) info.kv_entries_len = std::max(info.kv_entries_len, g.kv_off + g.len);
  if (p.draft)  // (a window may hide all but the newest entries, which ft_draft_accept writes)
    for (int i = 0; i < p.batch; ++i)
      if (p.ext[i] > 0) info.kv_entries_len = std::max(info.kv_entries_len, p.start[i] + p.seq[i]);
  info.items_off = 0;
  for (const Item& it : b.items) {
    const Block& blk = b.blocks[it.block];
    int32_t x[ITEM_INTS] = {it.t0, it.t1, it.alternate ? 2 : 1, it.which == 3 ? 2 : 1, blk.len, tile0[it.block], 0, 0};
    std::memcpy(x + 24, tiles.data() + 8 * ((size_t)tile0[it.block] + it.t0), 8 * sizeof(int32_t));
    int q_tile = 0;
    for (int w = 0; w < 2; ++w) {
      const int of = it.alternate ? (it.which == 1 ? 0 : 1) : w;  // the query tile of this stream
      if (!(it.which & (1 << of))) continue;
      const int first = of == 0 ? 0 : blk.split, n = of == 0 ? blk.split : blk.ntok - blk.split;
      // one query tile is always tile 0 of its item, and one stream stream 0
      int32_t* s = x + 8 + 8 * (it.alternate ? w : q_tile);
      s[0] = blk.tok0 + first;
      s[1] = n;
      s[2] = it.alternate ? it.t0 + w : it.lo[of];
      s[3] = it.alternate ? it.t1 : it.hi[of];
      s[4] = -1;
      s[5] = it.alternate ? 0 : q_tile;
      s[6] = first;
      s[7] = of;
      if (partial[it.block]) {
        s[4] = (int32_t)extra.size();
        for (int i = first; i < first + n; ++i) {
          bool sees = false;
          for (int k = s[2]; k < s[3] && !sees; k += x[2]) {
            const int32_t at = tiles[8 * ((size_t)tile0[it.block] + k) + 4 + of];
            sees = at < 0;
            for (int wd = 0; wd < words && !sees; ++wd) sees = extra[(size_t)at + i * words + wd] != 0;
          }
          extra.push_back(sees ? (int32_t)rows : -2);
          if (sees) rows_of[blk.tok0 + i].push_back((int32_t)rows++);
        }
      }
      ++q_tile;
    }
    t.insert(t.end(), x, x + ITEM_INTS);
  }
  if (p.draft) {  // until the trees are known
    std::vector<int16_t> chain, depth;
    for (int i = 0; i < p.batch; ++i) {
      while ((int64_t)chain.size() < p.ext[i]) {
        chain.push_back((int16_t)chain.size() - 1);
        depth.push_back((int16_t)depth.size());
      }
      for (const DraftSpan& s : spans_of[i])
        for (int k = 0; k < s.tokens; ++k)
          draft_span_words(s, k, (int)p.window, chain.data(), depth.data(), [&](int word, uint32_t mask, uint32_t bits) {
            int32_t& x = extra[(size_t)s.bits + k * words + word];
            x = (int32_t)(((uint32_t)x & ~mask) | bits);
          });
    }
  }
  align();
  info.tokens_off = (int64_t)t.size();
  info.q_rows = 0;
  for (const Token& k : b.tokens) {
    t.push_back(k.q_row);
    t.push_back(k.pos);
    info.q_rows = std::max<int64_t>(info.q_rows, (int64_t)k.q_row + 1);
  }
  align();
  info.tiles_off = (int64_t)t.size();
  t.insert(t.end(), tiles.begin(), tiles.end());
  info.extra_off = (int64_t)t.size();
  t.insert(t.end(), extra.begin(), extra.end());
  // ft_extend's kernels read sms before the kernel ahead of them, which may be ft_draft_tree's, has ended: a cache line of 128 bytes,
  // wherever the table starts, lies between those ints and the words that it writes
  if (p.draft) t.insert(t.end(), 32, 0);
  align();
  info.sms_off = (int64_t)t.size();
  for (int c = 0; c < p.slots; ++c) {
    int32_t x[16] = {b.sm_offs[c], b.sm_offs[c + 1], -1, 0};
    if (x[0] < x[1]) {
      x[2] = b.sm_tasks[x[0]];
      const Item& it = b.items[x[2] / p.kv_heads];
      x[4] = it.t0, x[5] = it.t1, x[6] = tile0[it.block];
      std::memcpy(x + 8, tiles.data() + 8 * ((size_t)tile0[it.block] + it.t0), 4 * sizeof(int32_t));
    }
    t.insert(t.end(), x, x + 16);
  }
  info.sm_tasks_off = (int64_t)t.size();
  t.insert(t.end(), b.sm_tasks.begin(), b.sm_tasks.end());
  align();
  // merged tokens: {row of q, first entry of its list of partial rows, entries, 0}, then the lists
  std::vector<int32_t> merged, lists;
  for (size_t k = 0; k < b.blocks.size(); ++k) {
    if (!partial[k]) continue;
    for (int i = b.blocks[k].tok0; i < b.blocks[k].tok0 + b.blocks[k].ntok; ++i) {
      const int32_t x[4] = {b.tokens[i].q_row, (int32_t)lists.size(), (int32_t)rows_of[i].size(), 0};
      lists.insert(lists.end(), rows_of[i].begin(), rows_of[i].end());
      merged.insert(merged.end(), x, x + 4);
    }
  }
  info.merge_off = (int64_t)t.size();
  t.insert(t.end(), merged.begin(), merged.end());
  info.merge_rows_off = (int64_t)t.size();
  t.insert(t.end(), lists.begin(), lists.end());
  align();
  if (p.draft) {
    info.draft = 1;
    std::vector<DraftSpan> spans;
    info.drafts_off = (int64_t)t.size();
    for (int i = 0; i < p.batch; ++i) {
      const int32_t x[8] = {(int32_t)p.qstart[i], (int32_t)p.ext[i], (int32_t)(p.seq[i] - p.ext[i]), (int32_t)(uint32_t)(p.start[i] & 0xffffffffll),
                            (int32_t)(p.start[i] >> 32), p.ids[i], (int32_t)spans.size(), (int32_t)spans_of[i].size()};
      t.insert(t.end(), x, x + 8);
      spans.insert(spans.end(), spans_of[i].begin(), spans_of[i].end());
      info.longest_draft = std::max(info.longest_draft, (int32_t)p.ext[i]);
    }
    info.num_drafts = p.batch;
    info.num_spans = (int32_t)spans.size();
    info.spans_off = (int64_t)t.size();
    static_assert(sizeof(DraftSpan) == 8 * sizeof(int32_t), "a span is eight ints of the table");
    const int32_t* raw = reinterpret_cast<const int32_t*>(spans.data());
    t.insert(t.end(), raw, raw + 8 * spans.size());
  }
  info.table_ints = (int64_t)t.size();
  info.num_items = (int32_t)b.items.size();
  info.num_tiles = (int32_t)(tiles.size() / 8);
  info.num_tokens = (int32_t)b.tokens.size();
  info.num_merged = (int32_t)(merged.size() / 4);
  info.partial_rows = (int32_t)rows;
  info.num_sms = p.slots;
}

int build(const int64_t* seq_lens, const int64_t* extend_lens, const int64_t* kv_starts, const int64_t* q_starts,
          const int64_t* shared_with_previous, const int32_t* draft_ids, int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads,
          int32_t head_dim, int32_t elem_bytes, int64_t window, int32_t num_sms, ft_extend_plan** out) {
  if (out == nullptr) return FT_ERR_INVALID_ARGUMENT;
  *out = nullptr;
  if (batch < 0 || num_qo_heads <= 0 || num_kv_heads <= 0 || num_qo_heads % num_kv_heads != 0 || num_sms <= 0 || window < 0 ||
      (elem_bytes != 2 && elem_bytes != 4))
    return FT_ERR_INVALID_ARGUMENT;
  if (batch > 0 && (!seq_lens || !extend_lens || !kv_starts || !q_starts || !shared_with_previous)) return FT_ERR_INVALID_ARGUMENT;
  if (!(head_dim == 16 || head_dim == 32 || head_dim == 64 || head_dim == 128 || head_dim == 256)) return FT_ERR_UNSUPPORTED;
  int64_t total = 0, most = 0;
  for (int i = 0; i < batch; ++i) {
    if (extend_lens[i] < 0 || seq_lens[i] < extend_lens[i] || kv_starts[i] < 0 || q_starts[i] < 0 || shared_with_previous[i] < 0)
      return FT_ERR_INVALID_ARGUMENT;
    const int64_t cached = seq_lens[i] - extend_lens[i];
    if (shared_with_previous[i] > cached || (shared_with_previous[i] > 0 && (i == 0 || shared_with_previous[i] > seq_lens[i - 1] - extend_lens[i - 1])))
      return FT_ERR_INVALID_ARGUMENT;
    if (seq_lens[i] > INT32_MAX / 2 || q_starts[i] > INT32_MAX / 2 || q_starts[i] + extend_lens[i] > INT32_MAX / 2 || kv_starts[i] > INT64_MAX / 2)
      return FT_ERR_TOO_LARGE;
    if (draft_ids != nullptr && (draft_ids[i] < 0 || draft_ids[i] >= batch)) return FT_ERR_INVALID_ARGUMENT;
    if (draft_ids != nullptr && extend_lens[i] > FT_MAX_DRAFT) return FT_ERR_TOO_LARGE;
    total += extend_lens[i];
    most = std::max(most, seq_lens[i]);
  }
  if (total > INT32_MAX / 64 || window > INT32_MAX) return FT_ERR_TOO_LARGE;
  try {
    // a row of q is one request's: two writers of a row of o would race
    std::vector<std::pair<int64_t, int64_t>> q_rows;
    for (int i = 0; i < batch; ++i)
      if (extend_lens[i] > 0) q_rows.push_back({q_starts[i], q_starts[i] + extend_lens[i]});
    std::sort(q_rows.begin(), q_rows.end());
    for (size_t i = 1; i < q_rows.size(); ++i)
      if (q_rows[i].first < q_rows[i - 1].second) return FT_ERR_INVALID_ARGUMENT;
    Problem p;
    p.seq = seq_lens, p.ext = extend_lens, p.start = kv_starts, p.qstart = q_starts, p.shared = shared_with_previous;
    p.draft = draft_ids != nullptr;
    p.ids = draft_ids;
    p.batch = batch;
    p.group = num_qo_heads / num_kv_heads;
    p.kv_heads = num_kv_heads;
    p.head_dim = head_dim;
    p.window = window > most ? 0 : window;  // a window that hides nothing is none
    const bool tensor = elem_bytes == 2 && head_dim >= 64 && p.group <= 128;
    p.two_tiles = p.streams = tensor && head_dim <= 128;
    p.tile = tensor && head_dim <= 128 ? 128 : 64;
    p.slots = tensor ? num_sms : elem_bytes == 4 && head_dim == 256 ? num_sms : 2 * num_sms;
    // Query tiles: 128 rows on the tensor cores; 64 or 16 on the CUDA cores, whichever schedule ends first.
    const double d = head_dim / 128.0;
    // (The tensor-core costs for head_dim 64 are those measured at 128, and a cap is not known here, although a capped tile costs half
    // as much again: such steps are cut as if their tiles cost the same, so only the tasks' order and number can suffer.)
    const Costs tc = head_dim == 256 ? Costs{1.0, 0, 1.0, 1.0, 3.0} : Costs{0.6, 0.15, 0.75, 1.1, 2.5};
    const Costs many = {0, 0, 0, 1.0 + 13.0 * d, 4.0}, few = {0, 0, 0, 1.0 + 4.0 * d, 3.0};
    struct Form {
      int rows;
      Costs cost;
    };
    const Form forms[2] = {{tensor ? 128 : 64, tensor ? tc : many}, {16, few}};
    std::unique_ptr<Builder> built;
    Problem best_p = p;
    for (int f = 0; f < (tensor ? 1 : 2); ++f) {
      Problem trial = p;
      trial.rows = forms[f].rows;
      trial.cost = forms[f].cost;
      trial.tokens_per_tile = std::max(1, trial.rows / p.group);
      if (tensor) memory_bound_costs(trial, elem_bytes, num_sms);
      std::unique_ptr<Builder> b(new Builder(trial));
      b->run();
      if (!built || b->end < built->end) {
        best_p = trial;
        built = std::move(b);
      }
    }
    p = best_p;
    const Builder& b = *built;
    // what the tables' 32-bit fields hold
    int64_t virt = 0, rows = 0;
    for (const Block& blk : b.blocks) virt = std::max<int64_t>(virt, blk.len);
    for (const Item& it : b.items) rows += 2 * (int64_t)b.blocks[it.block].ntok;
    if (virt > INT32_MAX / 2 || rows > INT32_MAX || (int64_t)b.items.size() * num_kv_heads > INT32_MAX / 2) return FT_ERR_TOO_LARGE;
    ft_extend_plan* plan = new ft_extend_plan();
    std::memset(&plan->info, 0, sizeof(plan->info));
    plan->info.num_qo_heads = num_qo_heads;
    plan->info.num_kv_heads = num_kv_heads;
    plan->info.head_dim = head_dim;
    plan->info.window = (int32_t)p.window;
    plan->info.elem_bytes = elem_bytes;
    plan->info.rows_per_tile = p.rows;
    plan->info.tile_tokens = p.tile;
    try {
      pack(p, b, plan);
    } catch (...) {
      delete plan;
      throw;
    }
    *out = plan;
  } catch (const std::bad_alloc&) {
    return FT_ERR_TOO_LARGE;
  } catch (...) {
    return FT_ERR_INVALID_ARGUMENT;
  }
  return FT_OK;
}

}  // namespace

extern "C" {

int ft_extend_plan_build(const int64_t* seq_lens, const int64_t* extend_lens, const int64_t* kv_starts, const int64_t* q_starts,
                         const int64_t* shared_with_previous, int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads,
                         int32_t head_dim, int32_t elem_bytes, int64_t window, int32_t num_sms, ft_extend_plan** out) {
  return build(seq_lens, extend_lens, kv_starts, q_starts, shared_with_previous, nullptr, batch, num_qo_heads, num_kv_heads, head_dim,
               elem_bytes, window, num_sms, out);
}

int ft_draft_plan_build(const int64_t* seq_lens, const int64_t* draft_lens, const int64_t* kv_starts, const int64_t* q_starts,
                        const int64_t* shared_with_previous, const int32_t* request_ids, int32_t batch, int32_t num_qo_heads,
                        int32_t num_kv_heads, int32_t head_dim, int32_t elem_bytes, int64_t window, int32_t num_sms, ft_extend_plan** out) {
  static const int32_t none = 0;
  if (out != nullptr) *out = nullptr;
  if (batch > 0 && request_ids == nullptr) return FT_ERR_INVALID_ARGUMENT;
  return build(seq_lens, draft_lens, kv_starts, q_starts, shared_with_previous, batch > 0 ? request_ids : &none, batch, num_qo_heads,
               num_kv_heads, head_dim, elem_bytes, window, num_sms, out);
}

int ft_extend_plan_get_info(const ft_extend_plan* plan, ft_extend_plan_info* info) {
  if (plan == nullptr || info == nullptr) return FT_ERR_INVALID_ARGUMENT;
  *info = plan->info;
  return FT_OK;
}

int ft_extend_plan_copy(const ft_extend_plan* plan, int32_t* table) {
  if (plan == nullptr || table == nullptr) return FT_ERR_INVALID_ARGUMENT;
  if (!plan->table.empty()) std::memcpy(table, plan->table.data(), plan->table.size() * sizeof(int32_t));
  return FT_OK;
}

void ft_extend_plan_free(ft_extend_plan* plan) { delete plan; }

}  // extern "C"
