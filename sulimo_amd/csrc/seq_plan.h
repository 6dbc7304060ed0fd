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
constexpr int kLoadTile = 64;
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

inline std::vector<LoadTile> load_tiles(const Seqs &q) {
  std::vector<LoadTile> t;
  int row = 0;
  for (int s = 0; s < q.n_seqs; s++) {
    const int len = q.start[s] + q.n_new[s];
    for (int p = 0; p < len; p += kLoadTile)
      t.push_back(LoadTile{q.page_off[s], p, row + p, std::min(kLoadTile, len - p)});
    row += len;
  }
  return t;
}

}  // namespace sulimo
