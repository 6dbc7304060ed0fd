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

// Rows a KV head up to which a sequence's rows read the Q8_0 cache directly; more have it read
// back and go to the row kernel. Measured, 24 heads over 8, directly and by read-back: 192 rows of
// one sequence behind 8000 positions 44 and 73 us, of 16 behind 4000 229 and 277, of 64 behind
// 2000 486 and 621; 255 rows 50 and 77, 281 and 289, 697 and 645; 384 rows of one 72 and 76, of
// 16 behind 1000 133 and 118, behind 4000 434 and 435; 768 rows 126 and 99, 245 and 188, 971 and
// 652.
constexpr int kDirectRows = 256;

int32_t plan(sulimo_hip_seq_batch *b, bool packed) {
  StepPlan &p = packed ? b->packed_plan : b->paged_plan;
  if (p.ready) return SULIMO_HIP_OK;
  const int cus = device_cu_count(), G = b->g.n_head / b->g.n_head_kv;
  std::vector<int> which[3];
  for (int s = 0; s < b->q.n_seqs; s++) {
    const long rows = (long)b->q.n_new[s] * G;
    if (rows) which[packed || rows > kDirectRows ? 2 : rows > 16 ? 1 : 0].push_back(s);
  }
  AttnPlan a[3];
  plan_direct(b->g, b->q, which[0], which[1], cus, a);
  a[2] = plan_attention_pieces(b->g, b->q, which[2], row_split(b->g, !packed, cus));
  std::vector<SeqKv> kv(b->q.n_seqs, SeqKv{0, 0, 0});
  std::vector<LoadTile> tiles;
  long rows = 0;
  for (int s : which[2]) {
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
  // one array: the pieces of each list, where the keys are, load tiles, counters (zero)
  std::vector<char> blob;
  auto put = [&](const void *src, size_t n) {
    const size_t at = blob.size();
    blob.resize(at + align_up(n), 0);
    if (src && n) memcpy(blob.data() + at, src, n);
    return at;
  };
  p.rec_rows = 0;
  for (int i = 0; i < 3; i++) {
    p.list[i].n = (int)a[i].pieces.size();
    p.list[i].at = put(a[i].pieces.data(), a[i].pieces.size() * sizeof(AttnPiece));
    p.list[i].counters = put(nullptr, (size_t)a[i].counters * 4);
    p.list[i].rec = p.rec_rows;
    p.list[i].heads = a[i].heads;
    p.rec_rows += a[i].rec_rows;
  }
  p.at_kv = put(kv.data(), kv.size() * sizeof(SeqKv));
  p.at_tiles = put(tiles.data(), tiles.size() * sizeof(LoadTile));
  p.n_tiles = (int)tiles.size();
  p.read_rows = rows;
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
  STEP_TRY(ensure_workspace(ctx, o_bytes + ml_bytes + 3 * kv_bytes));
  char *ws = reinterpret_cast<char *>(ctx->ws), *lists = reinterpret_cast<char *>(p.lists.dev);
  auto args = [&](const StepPlan::List &l) {
    return StepAttnArgs{seq_view(b), reinterpret_cast<const AttnPiece *>(lists + l.at), l.n,
                        reinterpret_cast<const _Float16 *>(q), reinterpret_cast<_Float16 *>(out), b->g.n_head,
                        b->g.n_head_kv, b->g.head_dim, l.heads,
                        Join{reinterpret_cast<float *>(ws) + l.rec * hd, reinterpret_cast<float2 *>(ws + o_bytes) + l.rec,
                             reinterpret_cast<int *>(lists + l.counters)}};
  };
  for (int i = 0; i < 2; i++)
    if (p.list[i].n) STEP_TRY(launch_cache_attention(args(p.list[i]), i + 1, k_cache, v_cache, ctx->stream));
  if (p.list[2].n) {
    uint16_t *k_rest = nullptr;
    if (p.n_tiles) {
      uint16_t *kr = reinterpret_cast<uint16_t *>(ws + o_bytes + ml_bytes), *vr = kr + kv_bytes / 2;
      k_rest = vr + kv_bytes / 2;
      STEP_TRY(launch_kv_load_paged(reinterpret_cast<const LoadTile *>(lists + p.at_tiles), p.n_tiles, seq_view(b).pages,
                                    b->g.page_size, (int)width, k_cache, v_cache, kr, vr, k_rest, ctx->stream));
      k = kr;
      v = vr;
    }
    STEP_TRY(launch_row_attention(args(p.list[2]), reinterpret_cast<const SeqKv *>(lists + p.at_kv),
                                  reinterpret_cast<const _Float16 *>(k), reinterpret_cast<const _Float16 *>(k_rest),
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
