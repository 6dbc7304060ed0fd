// seq_batch.h - the batch handle of a step, and what its kernels take.
#pragma once

#include "common.h"
#include "seq_plan.h"

namespace sulimo {
// A grown-on-demand device array that the calls of one context fill in stream order.
struct StepArray {
  void *dev = nullptr;
  size_t bytes = 0;
};
// The work lists of a step's attention (attention_step.hip), for the paged or the packed form:
// pieces over the cache by 16 rows and by 32, and over f16 rows.
struct StepPlan {
  struct List {
    int n = 0, heads = 1;         // pieces, KV heads of a workgroup
    size_t at = 0, counters = 0;  // where in `lists` the pieces and their counters are
    size_t rec = 0;               // first record row
  };
  bool ready = false;
  StepArray lists;
  List list[3];
  size_t rec_rows = 0;
  int n_tiles = 0;     // load tiles
  long read_rows = 0;  // cache rows that are read back
  size_t at_kv = 0, at_tiles = 0;
};
}  // namespace sulimo

struct sulimo_hip_seq_batch {
  sulimo_hip_ctx *ctx = nullptr;
  int device = 0;
  sulimo::SeqShape g;
  sulimo::Seqs q;
  sulimo::SeqBlob at;  // where the parts are in `seqs`
  sulimo::StepArray seqs;
  // position tiles of kv_load_paged, built by its first call after a set
  sulimo::StepArray load_tiles;
  int n_load_tiles = 0;
  bool load_ready = false;
  sulimo::StepPlan paged_plan, packed_plan;
  sulimo::StepArray verify_counters;
};

namespace sulimo {

// Device pointers of a batch's sequences.
struct SeqView {
  const int32_t *off, *start, *page_off, *row_seq, *row_slot, *pages;
  int n_seqs, rows, page_size, window;
};
SeqView seq_view(const sulimo_hip_seq_batch *b);

// Grows a to at least `bytes` (after the context's queued work, before its next).
int32_t step_array(sulimo_hip_seq_batch *b, StepArray *a, size_t bytes);

// Kernel launchers of a step's operators.
int32_t launch_kv_store_paged(const SeqView &v, int width, const uint16_t *k, const uint16_t *vv, uint8_t *k_cache,
                              uint8_t *v_cache, uint16_t *k_values, uint16_t *v_values, hipStream_t s);
// k_rest: what the rounding of k_out to f16 dropped, or null.
int32_t launch_kv_load_paged(const LoadTile *tiles, int n_tiles, const int32_t *pages, int page_size, int width,
                             const uint8_t *k_cache, const uint8_t *v_cache, uint16_t *k_out, uint16_t *v_out,
                             uint16_t *k_rest, hipStream_t s);

// Attention of the batch's new rows: over the paged Q8_0 cache (k_cache, v_cache bytes), or
// over the rows' own f16 keys and values.
int32_t attention_paged(sulimo_hip_seq_batch *b, const uint16_t *q, const uint8_t *k_cache, const uint8_t *v_cache,
                        uint16_t *out);
int32_t attention_packed(sulimo_hip_seq_batch *b, const uint16_t *q, const uint16_t *k, const uint16_t *v,
                         uint16_t *out);

struct VerifyArgs {
  const float *logits;       // [rows][vocab]
  const int32_t *tokens;     // [rows]
  const float *draft_probs;  // [rows - n_seqs][vocab], or null: each draft was certain
  const float *uniforms;     // [rows]; not read at temperature 0
  int vocab;
  double temperature;
  int32_t *accepted;  // [n_seqs]
  int32_t *answer;    // [rows]
};
int32_t verify_drafts(sulimo_hip_seq_batch *b, const VerifyArgs &a);

}  // namespace sulimo
