// attention_step.hip - which kernels a step's attention runs, and their work lists.
//
// A list depends on the batch's sequences only; it is built by the first call after a set and
// serves every layer of the step. Records of split row tiles and the part of the cache that is
// read back live in the context's workspace, whose users run one after the other.
#include <string.h>

#include "step_attn.h"

namespace sulimo {
namespace {

#define STEP_TRY(call)          \
  do {                          \
    const int32_t rc_ = (call); \
    if (rc_) return rc_;        \
  } while (0)

constexpr size_t align_up(size_t v) { return (v + 255) & ~(size_t)255; }

// Rows a KV head up to which a sequence's rows read the Q8_0 cache directly.
constexpr int kDirectRows = 128;

int32_t plan(sulimo_hip_seq_batch *b, bool packed) {
  StepPlan &p = packed ? b->packed_plan : b->paged_plan;
  if (p.ready) return SULIMO_HIP_OK;
  const int cus = device_cu_count(), G = b->g.n_head / b->g.n_head_kv;
  std::vector<int> few, many;
  for (int s = 0; s < b->q.n_seqs; s++) {
    if (b->q.n_new[s] == 0) continue;
    (!packed && (long)b->q.n_new[s] * G <= kDirectRows ? few : many).push_back(s);
  }
  const AttnPlan c = plan_attention_pieces(b->g, b->q, few, cache_split(b->g, cus));
  const AttnPlan r = plan_attention_pieces(b->g, b->q, many, row_split(cus));
  std::vector<SeqKv> kv(b->q.n_seqs, SeqKv{0, 0, 0});
  std::vector<LoadTile> tiles;
  long rows = 0;
  for (int s : many) {
    const int end = b->q.start[s] + b->q.n_new[s];
    const int lo = first_seen(b->g, b->q.start[s]) / kRowKeys * kRowKeys;
    kv[s] = packed ? SeqKv{b->q.off[s], 0, end} : SeqKv{(int32_t)rows, lo, end - lo};
    // the kernel's offsets inside a sequence are 32-bit (a tile may start at its last row)
    if ((size_t)(end - lo + kRowKeys) * b->g.n_head_kv * b->g.head_dim * 2 > 0xFFFFFFFFull)
      return fail(SULIMO_HIP_ERR_INVALID_ARGUMENT,
                  "sequence " + std::to_string(s) + " has over 4 GiB of f16 keys in sight of a long chunk");
    if (!packed) {
      add_load_tiles(b->q, s, lo, end, (int)rows, &tiles);
      rows += end - lo;
    }
  }
  // one array: pieces, pieces, where the keys are, load tiles, counters (zero)
  p.n_cache = (int)c.pieces.size();
  p.n_rows = (int)r.pieces.size();
  p.n_tiles = (int)tiles.size();
  p.read_rows = rows;
  p.cache_rec = c.rec_rows;
  p.rec_rows = c.rec_rows + r.rec_rows;
  p.at_rows = align_up(c.pieces.size() * sizeof(AttnPiece));
  p.at_kv = p.at_rows + align_up(r.pieces.size() * sizeof(AttnPiece));
  p.at_tiles = p.at_kv + align_up(kv.size() * sizeof(SeqKv));
  p.at_cache_counters = p.at_tiles + align_up(tiles.size() * sizeof(LoadTile));
  p.at_row_counters = p.at_cache_counters + align_up((size_t)c.counters * 4);
  std::vector<char> blob(p.at_row_counters + align_up((size_t)r.counters * 4), 0);
  auto put = [&](size_t at, const void *src, size_t n) {
    if (n) memcpy(blob.data() + at, src, n);
  };
  put(0, c.pieces.data(), c.pieces.size() * sizeof(AttnPiece));
  put(p.at_rows, r.pieces.data(), r.pieces.size() * sizeof(AttnPiece));
  put(p.at_kv, kv.data(), kv.size() * sizeof(SeqKv));
  put(p.at_tiles, tiles.data(), tiles.size() * sizeof(LoadTile));
  if (blob.empty()) blob.resize(256, 0);
  STEP_TRY(step_array(b, &p.lists, blob.size()));
  SULIMO_HIP_TRY(hipMemcpyAsync(p.lists.dev, blob.data(), blob.size(), hipMemcpyHostToDevice, b->ctx->stream));
  p.ready = true;
  return SULIMO_HIP_OK;
}

int32_t attend(sulimo_hip_seq_batch *b, StepPlan &p, const uint16_t *q, const uint8_t *k_cache, const uint8_t *v_cache,
               const uint16_t *k, const uint16_t *v, uint16_t *out) {
  sulimo_hip_ctx *ctx = b->ctx;
  const size_t hd = b->g.head_dim, width = (size_t)b->g.n_head_kv * hd;
  const size_t o_bytes = align_up(p.rec_rows * hd * 4), ml_bytes = align_up(p.rec_rows * 8);
  const size_t kv_bytes = align_up((size_t)p.read_rows * width * 2);
  STEP_TRY(ensure_workspace(ctx, o_bytes + ml_bytes + 2 * kv_bytes));
  char *ws = reinterpret_cast<char *>(ctx->ws), *lists = reinterpret_cast<char *>(p.lists.dev);
  float *rec_o = reinterpret_cast<float *>(ws);
  float2 *rec_ml = reinterpret_cast<float2 *>(ws + o_bytes);
  const StepAttnArgs base{seq_view(b), nullptr, 0, reinterpret_cast<const _Float16 *>(q),
                          reinterpret_cast<_Float16 *>(out), b->g.n_head, b->g.n_head_kv, b->g.head_dim, Join{}};
  if (p.n_cache) {
    StepAttnArgs c = base;
    c.pieces = reinterpret_cast<const AttnPiece *>(lists);
    c.n_pieces = p.n_cache;
    c.join = Join{rec_o, rec_ml, reinterpret_cast<int *>(lists + p.at_cache_counters)};
    STEP_TRY(launch_cache_attention(c, k_cache, v_cache, ctx->stream));
  }
  if (p.n_rows) {
    uint16_t *kr = reinterpret_cast<uint16_t *>(ws + o_bytes + ml_bytes);
    uint16_t *vr = reinterpret_cast<uint16_t *>(ws + o_bytes + ml_bytes + kv_bytes);
    if (p.n_tiles) {
      STEP_TRY(launch_kv_load_paged(reinterpret_cast<const LoadTile *>(lists + p.at_tiles), p.n_tiles, seq_view(b).pages,
                                    b->g.page_size, (int)width, k_cache, v_cache, kr, vr, ctx->stream));
      k = kr;
      v = vr;
    }
    StepAttnArgs r = base;
    r.pieces = reinterpret_cast<const AttnPiece *>(lists + p.at_rows);
    r.n_pieces = p.n_rows;
    r.join = Join{rec_o + p.cache_rec * hd, rec_ml + p.cache_rec, reinterpret_cast<int *>(lists + p.at_row_counters)};
    STEP_TRY(launch_row_attention(r, reinterpret_cast<const SeqKv *>(lists + p.at_kv), reinterpret_cast<const _Float16 *>(k),
                                  reinterpret_cast<const _Float16 *>(v), ctx->stream));
  }
  return SULIMO_HIP_OK;
}

}  // namespace

int32_t attention_paged(sulimo_hip_seq_batch *b, const uint16_t *q, const uint8_t *k_cache, const uint8_t *v_cache,
                        uint16_t *out) {
  STEP_TRY(plan(b, false));
  return attend(b, b->paged_plan, q, k_cache, v_cache, nullptr, nullptr, out);
}

int32_t attention_packed(sulimo_hip_seq_batch *b, const uint16_t *q, const uint16_t *k, const uint16_t *v,
                         uint16_t *out) {
  STEP_TRY(plan(b, true));
  return attend(b, b->packed_plan, q, nullptr, nullptr, k, v, out);
}

}  // namespace sulimo
