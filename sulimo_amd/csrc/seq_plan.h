// seq_plan.h - the sequences of a step on the host: the checks of their arrays and what the
// kernels read of them. Host arithmetic only, so that a CPU test can compile it.
//
// Sequence s has start[s] positions in the cache and n_new[s] new rows; the new rows of all
// sequences lie one behind the other (row off[s] is the first of sequence s). Position p of
// sequence s is cache row pages[page_off[s] + p / page_size] * page_size + p % page_size.
#pragma once

#include <limits.h>
#include <stddef.h>
#include <stdint.h>

#include <math.h>

#include <algorithm>
#include <string>
#include <vector>

namespace sulimo {

struct SeqShape {  // a batch's geometry; 0: none given
  int n_head = 0, n_head_kv = 0, head_dim = 0, window = 0, page_size = 0, n_pages = 0;
};

struct Seqs {
  int n_seqs = 0, rows = 0, positions = 0;  // positions: the sum of start + n_new
  bool paged = false;                       // a page table was given
  std::vector<int32_t> start, n_new, off, pages, page_off;
};

// Up to kLoadTile consecutive positions of one sequence, going to rows out_row .. of a
// packed output.
constexpr int kLoadTile = 16;
struct LoadTile {
  int32_t page_off, pos, out_row, count;
};

// Why the geometry is refused; empty: it is not.
inline std::string check_seq_shape(size_t head_count, size_t head_count_kv, size_t head_dim, size_t window,
                                   size_t page_size, size_t n_pages) {
  if (head_count || head_count_kv || head_dim) {
    if (head_count_kv == 0 || head_count == 0 || head_count % head_count_kv != 0 || head_count > 1024)
      return "head_count must be a multiple of head_count_kv, 1 to 1024";
    if (head_dim != 64 && head_dim != 128) return "a batch's head_dim is 64 or 128";
  } else if (page_size || n_pages || window) {
    return "pages and a window need a head layout";
  }
  if ((page_size == 0) != (n_pages == 0)) return "page_size and n_pages go together";
  if (page_size > (size_t)INT_MAX || n_pages > (size_t)INT_MAX || page_size * n_pages > (size_t)INT_MAX)
    return "the cache has more than 2^31 - 1 positions";
  if (window > (size_t)INT_MAX) return "window too large";
  return "";
}

// Why the sequences are refused; empty: *out holds them. The pages of every sequence are
// pages of the cache, and a page that receives new positions stands in no other place of the
// batch: two sequences may read a page, but one that is written has one owner.
inline std::string plan_seqs(const SeqShape &g, size_t n_seqs, const uint32_t *n_new, const uint32_t *start_pos,
                             const uint32_t *page_table, size_t max_pages, Seqs *out) {
  if (n_seqs > 65535) return "more than 65535 sequences";
  if (n_seqs && !n_new) return "n_new is null";
  if (page_table && !g.page_size) return "a page table needs a batch with pages";
  const size_t P = g.page_size, heads = std::max(1, g.n_head);
  size_t rows = 0, positions = 0;
  for (size_t s = 0; s < n_seqs; s++) {
    const size_t end = (size_t)n_new[s] + (start_pos ? start_pos[s] : 0);
    if (end > (size_t)INT_MAX - 4096) return "sequence " + std::to_string(s) + " is too long";
    rows += n_new[s];
    positions += end;
  }
  // rows and positions are counted in 32 bits, work items of them for every head too
  if (rows * heads > (size_t)INT_MAX / 2 || positions > (size_t)INT_MAX / 2)
    return "the batch's sequences are too long together";
  Seqs q;
  q.n_seqs = (int)n_seqs;
  q.rows = (int)rows;
  q.positions = (int)positions;
  q.paged = page_table != nullptr;
  q.start.resize(n_seqs);
  q.n_new.resize(n_seqs);
  q.page_off.resize(n_seqs);
  q.off.assign(n_seqs + 1, 0);
  std::vector<uint8_t> written(page_table ? g.n_pages : 0, 0);
  for (size_t s = 0; s < n_seqs; s++) {
    q.start[s] = start_pos ? (int32_t)start_pos[s] : 0;
    q.n_new[s] = (int32_t)n_new[s];
    q.off[s + 1] = q.off[s] + q.n_new[s];
    q.page_off[s] = (int32_t)q.pages.size();
    if (!page_table) continue;
    const size_t end = ((size_t)q.start[s] + q.n_new[s] + P - 1) / P, first = n_new[s] ? q.start[s] / P : end;
    if (end > max_pages)
      return "sequence " + std::to_string(s) + " needs " + std::to_string(end) + " pages, its table has " +
             std::to_string(max_pages);
    const uint32_t *t = page_table + s * max_pages;
    for (size_t i = 0; i < end; i++) {
      if (t[i] >= (uint32_t)g.n_pages)
        return "page " + std::to_string(t[i]) + " of sequence " + std::to_string(s) + " >= n_pages";
      if (i < first) continue;
      if (written[t[i]]) return "page " + std::to_string(t[i]) + " receives new positions twice";
      written[t[i]] = 1;
    }
    q.pages.insert(q.pages.end(), t, t + end);
  }
  if (page_table)
    for (size_t s = 0; s < n_seqs; s++) {
      const size_t end = ((size_t)q.start[s] + q.n_new[s] + P - 1) / P, first = n_new[s] ? q.start[s] / P : end;
      for (size_t i = 0; i < first; i++)
        if (written[q.pages[q.page_off[s] + i]])
          return "page " + std::to_string(q.pages[q.page_off[s] + i]) + " of sequence " + std::to_string(s) +
                 " receives new positions elsewhere in the batch";
    }
  *out = std::move(q);
  return "";
}

// Offsets of the parts of a batch's device array (int32 elements): off [n_seqs + 1] | start
// [n_seqs] | page_off [n_seqs] | row_seq [rows] | row_slot [rows], the cache row of each new
// row (paged only) | pages.
struct SeqBlob {
  size_t start = 0, page_off = 0, row_seq = 0, row_slot = 0, pages = 0;
  std::vector<int32_t> data;
};
inline SeqBlob seq_blob(const SeqShape &g, const Seqs &q) {
  SeqBlob b;
  b.data.reserve(3 * (size_t)q.n_seqs + 1 + 2 * (size_t)q.rows + q.pages.size());
  auto add = [&](const std::vector<int32_t> &v) { b.data.insert(b.data.end(), v.begin(), v.end()); };
  add(q.off);
  b.start = b.data.size();
  add(q.start);
  b.page_off = b.data.size();
  add(q.page_off);
  b.row_seq = b.data.size();
  for (int s = 0; s < q.n_seqs; s++) b.data.insert(b.data.end(), (size_t)q.n_new[s], s);
  b.row_slot = b.data.size();
  if (q.paged) {
    const size_t P = g.page_size;
    for (int s = 0; s < q.n_seqs; s++)
      for (int32_t i = 0; i < q.n_new[s]; i++) {
        const size_t p = (size_t)q.start[s] + i;
        b.data.push_back((int32_t)((size_t)q.pages[q.page_off[s] + p / P] * P + p % P));
      }
  }
  b.pages = b.data.size();
  add(q.pages);
  return b;
}

// Positions lo .. end - 1 of sequence s, to rows row .. of the output.
inline void add_load_tiles(const Seqs &q, int s, int lo, int end, int row, std::vector<LoadTile> *t) {
  for (int p = lo; p < end; p += kLoadTile)
    t->push_back(LoadTile{q.page_off[s], p, row + p - lo, std::min(kLoadTile, end - p)});
}
inline std::vector<LoadTile> load_tiles(const Seqs &q) {
  std::vector<LoadTile> t;
  int row = 0;
  for (int s = 0; s < q.n_seqs; s++) {
    const int len = q.start[s] + q.n_new[s];
    add_load_tiles(q, s, 0, len, row, &t);
    row += len;
  }
  return t;
}

// ---- attention: row tiles, and how their keys are cut ----
// A row tile is some query rows of one KV head, row r = token r / G, head kvh * G + r % G with
// G = n_head / n_head_kv query heads a KV head. A workgroup takes `heads` KV heads of a row tile
// and `sub` key tiles a step, for a run of key tiles: a piece. Pieces of a row tile leave
// records that the last one to finish joins.
struct AttnPiece {
  int32_t seq, row0;          // row tile: rows row0 .. of the sequence's n_new * G
  int32_t tile0, tile1;       // key tiles of this piece (tile t: positions t * key tile ..)
  int32_t piece, n_pieces;
  int32_t rec;                // first record row of the tile (piece p, head h, row r at rec + (p Hk + h) live + r)
  int32_t counter;            // index of the tile's arrival counters (one per head group)
};
struct AttnSplit {
  int rows;      // of a row tile
  int key_tile;  // positions
  int heads, sub;
  int slots;     // workgroups that run at once
  int threads;   // of a workgroup
  // microseconds: a piece's start and end, what it takes longer with records, a step of sub key
  // tiles where the slots are full and where few are taken, and one round of a join (8 pieces of
  // two times four values a thread)
  double piece, record, step, alone, join;
};
struct AttnPlan {
  std::vector<AttnPiece> pieces;
  int heads = 1;        // KV heads of a workgroup
  int counters = 0;     // arrival counters (head groups of every split tile)
  size_t rec_rows = 0;  // record rows, each head_dim floats and (m, l)
  double cost = 0;      // the time the cut was chosen for
};
inline int first_seen(const SeqShape &g, int pos) { return g.window && pos >= g.window ? pos - g.window + 1 : 0; }

// The row tiles of the sequences in `which`, cut into pieces of at most C steps. Pieces that all
// run at once take the longest one's time; more of them, at best their share of the slots, and
// half a piece for the last ones' unevenness. A cut tile's join comes behind that. C is the one
// of least time.
inline AttnPlan plan_attention_pieces(const SeqShape &g, const Seqs &q, const std::vector<int> &which, const AttnSplit &a) {
  AttnPlan plan;
  plan.heads = a.heads;
  const int G = g.n_head / g.n_head_kv, groups = g.n_head_kv / a.heads;
  struct Tile {
    int seq, row0, live, t0, t1, steps;
  };
  std::vector<Tile> tiles;
  int most = 1;
  for (int s : which) {
    const int total = q.n_new[s] * G;
    for (int r0 = 0; r0 < total; r0 += a.rows) {
      const int live = std::min(a.rows, total - r0);
      const int first = q.start[s] + r0 / G, last = q.start[s] + (r0 + live - 1) / G;
      Tile t{s, r0, live, first_seen(g, first) / a.key_tile, last / a.key_tile + 1, 0};
      t.steps = (t.t1 - t.t0 + a.sub - 1) / a.sub;
      most = std::max(most, t.steps);
      tiles.push_back(t);
    }
  }
  if (tiles.empty()) return plan;
  const int slots = std::max(1, a.slots / groups);
  auto cost = [&](int C) {
    long n = 0, records = 0;
    double total = 0, join = 0;
    for (const Tile &t : tiles) {
      const int np = (t.steps + C - 1) / C;
      n += np;
      total += np * (a.piece + (np > 1 ? a.record : 0)) + t.steps * a.step;
      if (np > 1) records += (long)np * g.n_head_kv * t.live;
      if (np > 1)
        join = std::max(join, a.join * ((np + 7) / 8) * std::ceil(a.heads * t.live * (g.head_dim / 4) / (2.0 * a.threads)));
    }
    if (records > INT32_MAX) return HUGE_VAL;  // (AttnPiece.rec)
    const double one = a.piece + (C < most ? a.record : 0) + std::max(a.alone, a.step * std::min(1.0, (double)n / slots)) * C;
    return (n <= slots ? one : std::max(one, total / slots) + one / 2) + join;
  };
  int C = most;
  plan.cost = cost(most);
  auto consider = [&](int c) {
    const double t = cost(c);
    if (t < plan.cost) {
      plan.cost = t;
      C = c;
    }
  };
  // the longest tile in 2 .. 64 equal pieces (eighths apart), and the shortest pieces that all run at once
  for (int np = 2, last = most; np <= 64 && last > 1; np += 1 + np / 8) {
    const int c = (most + np - 1) / np;
    if (c != last) consider(c);
    last = c;
  }
  int lo = 1, hi = most;
  while (lo < hi) {
    const int c = (lo + hi) / 2;
    long n = 0;
    for (const Tile &t : tiles) n += (t.steps + c - 1) / c;
    if (n <= slots) hi = c;
    else lo = c + 1;
  }
  if (lo < most) consider(lo);
  for (const Tile &t : tiles) {
    const int np = (t.steps + C - 1) / C;
    AttnPiece p{t.seq, t.row0, 0, 0, 0, np, (int32_t)plan.rec_rows, plan.counters};
    for (int i = 0; i < np; i++) {
      p.piece = i;
      p.tile0 = t.t0 + (int)((long)i * t.steps / np) * a.sub;
      p.tile1 = std::min(t.t1, t.t0 + (int)((long)(i + 1) * t.steps / np) * a.sub);
      plan.pieces.push_back(p);
    }
    if (np > 1) {
      plan.counters += groups;
      plan.rec_rows += (size_t)np * g.n_head_kv * t.live;
    }
  }
  // longest first: what starts last is short
  std::stable_sort(plan.pieces.begin(), plan.pieces.end(), [](const AttnPiece &x, const AttnPiece &y) {
    return x.tile1 - x.tile0 > y.tile1 - y.tile0;
  });
  return plan;
}

// Few rows read the Q8_0 cache directly (attention_cache.hip): 8 waves, of which 8 / heads share
// a KV head and take every (8 / heads)th key tile, row_tiles times 16 rows each.
constexpr int kCacheWaves = 8;
inline AttnSplit cache_split(const SeqShape &g, int row_tiles, int heads, int cus) {
  return AttnSplit{16 * row_tiles, g.head_dim == 128 ? 32 : 64, heads, kCacheWaves / heads, cus, 64 * kCacheWaves,
                   5.5, 0.0, row_tiles == 1 ? 2.8 : 4.0, row_tiles == 1 ? 2.8 : 4.0, 1.8};
}
// The KV heads of a workgroup: eight keep every line of the cache's rows in one workgroup; fewer,
// with more waves a head, have less to join where there is little to do.
inline AttnPlan plan_cache_attention(const SeqShape &g, const Seqs &q, const std::vector<int> &which, int row_tiles, int cus) {
  AttnPlan best;
  bool any = false;
  for (int heads = 8; heads >= 1; heads /= 2) {
    if (g.n_head_kv % heads) continue;
    AttnPlan p = plan_attention_pieces(g, q, which, cache_split(g, row_tiles, heads, cus));
    if (!any || p.cost < best.cost) best = std::move(p);
    any = true;
  }
  return best;
}
// The direct lists of a step: sequences of at most 16 rows a KV head (few) and of more. Tiles of
// 16 rows suit the first and tiles of 32 the second, in a launch each; one launch of either kind
// over both can be quicker, as where a step has little work: a piece of 16 rows starts and ends
// sooner. Measured, 24 heads over 8, 18 rows a KV head in tiles of 16 and of 32: one sequence
// behind 1000 positions 13.3 and 15.4 us, 64 behind 2000 119 and 95 us.
inline void plan_direct(const SeqShape &g, const Seqs &q, const std::vector<int> &few, const std::vector<int> &more,
                        int cus, AttnPlan (&out)[3]) {
  constexpr double kLaunch = 3.0;  // of a second kernel behind the first
  out[0] = plan_cache_attention(g, q, few, 1, cus);
  out[1] = AttnPlan();
  if (more.empty()) return;
  out[1] = plan_cache_attention(g, q, more, 2, cus);
  double best = out[0].cost + out[1].cost + (few.empty() ? 0.0 : kLaunch);
  std::vector<int> all(few);
  all.insert(all.end(), more.begin(), more.end());
  for (int row_tiles = 1; row_tiles <= 2; row_tiles++) {
    AttnPlan p = plan_cache_attention(g, q, all, row_tiles, cus);
    if (p.cost >= best) continue;
    best = p.cost;
    out[row_tiles - 1] = std::move(p);
    out[2 - row_tiles] = AttnPlan();
  }
}
// Many rows read f16 keys and values (attention_rows.hip), the cache's read back first.
// A cut tile of 128 rows stores and joins 64 KiB a piece and head, which costs more than the
// slots that it fills: 1000 tokens 27 us uncut and 49 in pieces of 2 tiles, 4096 tokens 126 and
// 206, the eight prompts of 677 to 4000 tokens 285 and 420. A tile is cut where a chunk is short
// and its history long.
constexpr int kRowTile = 128, kRowKeys = 64;
// exact: keys and weights in two f16 parts each, for which a workgroup of 128-wide heads takes a
// CU's registers alone.
inline AttnSplit row_split(const SeqShape &g, bool exact, int cus) {
  if (exact && g.head_dim == 128) return AttnSplit{kRowTile, kRowKeys, 1, 1, cus, 256, 4.0, 24.0, 2.3, 2.3, 1.8};
  return AttnSplit{kRowTile, kRowKeys, 1, 1, 2 * cus, 256, 4.0, 24.0, 2.1, 1.2, 1.8};
}

// Where a sequence's f16 keys and values lie: position p in [lo, lo + len) is row row0 + p - lo.
struct SeqKv {
  int32_t row0, lo, len;
};

// p / d = p * magic >> shift for every p < 2^31 (d >= 1): magic = floor(2^(31 + b) / d) + 1 with
// 2^b >= d is off by less than 2^-b <= 1 / d of the quotient.
struct FastDiv {
  uint32_t magic, shift, d;
};
inline FastDiv fast_div(uint32_t d) {
  uint32_t b = 0;
  while ((1ull << b) < d) b++;
  return FastDiv{(uint32_t)(((1ull << (31 + b)) / d) + 1), 31 + b, d};
}

}  // namespace sulimo
