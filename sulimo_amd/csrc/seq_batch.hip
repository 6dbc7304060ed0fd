// seq_batch.hip - C ABI of a step of several sequences: the batch handle and the checks of
// the calls that take it. Nothing of the reference corresponds to it (its engine runs one
// sequence, crates/sulimo-engine/src/engine.rs:152-422); the cache rows are its Q8_0 ring's
// (crates/sulimo-core/src/kv_cache.rs:27-90).
#include <limits.h>

#include <algorithm>
#include <initializer_list>
#include <new>
#include <string>

#include "seq_batch.h"

using namespace sulimo;

namespace sulimo {

SeqView seq_view(const sulimo_hip_seq_batch *b) {
  const int32_t *d = reinterpret_cast<const int32_t *>(b->seqs.dev);
  return SeqView{d, d + b->at.start, d + b->at.page_off, d + b->at.row_seq, d + b->at.row_slot, d + b->at.pages,
                 b->q.n_seqs, b->q.rows, b->g.page_size, b->g.window};
}

int32_t step_array(sulimo_hip_seq_batch *b, StepArray *a, size_t bytes) {
  if (a->bytes >= bytes) return SULIMO_HIP_OK;
  StepArray next;
  next.bytes = (bytes + bytes / 4 + 4095) & ~(size_t)4095;  // a decoding batch grows by a row a step
  SULIMO_HIP_TRY(hipMalloc(&next.dev, next.bytes));
  const StepArray old = *a;
  *a = next;
  if (old.dev) {
    SULIMO_HIP_TRY(hipStreamSynchronize(b->ctx->stream));
    SULIMO_HIP_TRY(hipFree(old.dev));
  }
  return SULIMO_HIP_OK;
}

}  // namespace sulimo

namespace {

constexpr int32_t kInval = SULIMO_HIP_ERR_INVALID_ARGUMENT;

// Runs a call's body; what it throws (the host arrays' allocation) becomes an error code.
template <typename F>
int32_t guarded(F &&body) {
  try {
    return body();
  } catch (const std::bad_alloc &) {
    return fail(SULIMO_HIP_ERR_DRIVER, "out of host memory");
  } catch (const std::exception &e) {
    return fail(SULIMO_HIP_ERR_DRIVER, e.what());
  }
}

// The context, the batch and the device of a step's call.
int32_t begin_step(sulimo_hip_ctx *ctx, const sulimo_hip_seq_batch *b) {
  if (!ctx) return fail(kInval, "ctx is null");
  if (!b) return fail(kInval, "batch is null");
  if (b->ctx != ctx) return fail(kInval, "the batch belongs to another context");
  SULIMO_HIP_TRY(hipSetDevice(ctx->device));
  return SULIMO_HIP_OK;
}

int32_t need(const sulimo_hip_ctx *ctx, const sulimo_hip_buffer *b, size_t bytes, const char *name) {
  if (!b) return fail(kInval, std::string(name) + " buffer is null");
  if (b->device != ctx->device) return fail(kInval, std::string(name) + " buffer is on another device");
  if (b->bytes < bytes)
    return fail(kInval, std::string(name) + " buffer holds " + std::to_string(b->bytes) + " bytes, needs " +
                            std::to_string(bytes));
  return SULIMO_HIP_OK;
}

// A buffer that a call writes is none of its others.
int32_t alone(const sulimo_hip_buffer *b, std::initializer_list<const sulimo_hip_buffer *> others, const char *name) {
  for (const sulimo_hip_buffer *o : others)
    if (b && b == o) return fail(kInval, std::string(name) + " is also another buffer of the call");
  return SULIMO_HIP_OK;
}

#define STEP_TRY(call)              \
  do {                              \
    const int32_t rc_ = (call);     \
    if (rc_) return rc_;            \
  } while (0)

int32_t need_heads(const sulimo_hip_seq_batch *b) {
  return b->g.n_head ? SULIMO_HIP_OK : fail(kInval, "the batch was created without a head layout");
}
int32_t need_pages(const sulimo_hip_seq_batch *b) {
  STEP_TRY(need_heads(b));
  return b->q.paged ? SULIMO_HIP_OK : fail(kInval, "the batch's sequences have no page table");
}
size_t row_width(const sulimo_hip_seq_batch *b) { return (size_t)b->g.n_head_kv * b->g.head_dim; }
size_t cache_bytes(const sulimo_hip_seq_batch *b) {
  return (size_t)b->g.n_pages * b->g.page_size * (row_width(b) / 32) * 34;
}
template <typename T>
T *dp(const sulimo_hip_buffer *b) {
  return b ? reinterpret_cast<T *>(b->dev) : nullptr;
}

}  // namespace

extern "C" {

int32_t sulimo_hip_seq_batch_create(sulimo_hip_ctx *ctx, size_t head_count, size_t head_count_kv, size_t head_dim,
                                    size_t window, size_t page_size, size_t n_pages, sulimo_hip_seq_batch **out) {
  return guarded([&]() -> int32_t {
    if (!out) return fail(kInval, "out is null");
    const std::string why = check_seq_shape(head_count, head_count_kv, head_dim, window, page_size, n_pages);
    if (!why.empty()) return fail(kInval, why);
    if (!ctx) return fail(kInval, "ctx is null");
    sulimo_hip_seq_batch *b = new sulimo_hip_seq_batch();
    b->ctx = ctx;
    b->device = ctx->device;
    b->g = SeqShape{(int)head_count, (int)head_count_kv, (int)head_dim, (int)window, (int)page_size, (int)n_pages};
    *out = b;
    return SULIMO_HIP_OK;
  });
}

int32_t sulimo_hip_seq_batch_release(sulimo_hip_seq_batch *b) {
  if (!b) return SULIMO_HIP_OK;
  hipError_t e = hipSetDevice(b->device);
  for (StepArray *a : {&b->seqs, &b->load_tiles, &b->paged_plan.lists, &b->packed_plan.lists, &b->verify_counters}) {
    // hipFree waits for work that may still use the allocation
    const hipError_t f = a->dev ? hipFree(a->dev) : hipSuccess;
    if (e == hipSuccess) e = f;
  }
  delete b;
  return e == hipSuccess ? SULIMO_HIP_OK : hip_fail(e, "batch release");
}

int32_t sulimo_hip_seq_batch_set(sulimo_hip_seq_batch *b, size_t n_seqs, const uint32_t *n_new,
                                 const uint32_t *start_pos, const uint32_t *page_table, size_t max_pages) {
  return guarded([&]() -> int32_t {
    if (!b) return fail(kInval, "batch is null");
    Seqs q;
    const std::string why = plan_seqs(b->g, n_seqs, n_new, start_pos, page_table, max_pages, &q);
    if (!why.empty()) return fail(kInval, why);
    SeqBlob at = seq_blob(b->g, q);
    SULIMO_HIP_TRY(hipSetDevice(b->device));
    STEP_TRY(step_array(b, &b->seqs, at.data.size() * 4));
    b->q = Seqs();  // nothing to run on should the copy fail
    // Pageable source: staged before the call returns; ordered behind the calls that read
    // the last step's arrays.
    SULIMO_HIP_TRY(hipMemcpyAsync(b->seqs.dev, at.data.data(), at.data.size() * 4, hipMemcpyHostToDevice, b->ctx->stream));
    at.data = std::vector<int32_t>();
    b->at = std::move(at);
    b->q = std::move(q);
    b->load_ready = b->paged_plan.ready = b->packed_plan.ready = false;
    return SULIMO_HIP_OK;
  });
}

int32_t sulimo_hip_enqueue_kv_store_paged(sulimo_hip_ctx *ctx, const sulimo_hip_seq_batch *b,
                                          const sulimo_hip_buffer *k, const sulimo_hip_buffer *v,
                                          sulimo_hip_buffer *k_cache, sulimo_hip_buffer *v_cache,
                                          sulimo_hip_buffer *k_values, sulimo_hip_buffer *v_values) {
  return guarded([&]() -> int32_t {
    STEP_TRY(begin_step(ctx, b));
    STEP_TRY(need_pages(b));
    const size_t bytes = (size_t)b->q.rows * row_width(b) * 2;
    STEP_TRY(need(ctx, k, bytes, "k"));
    STEP_TRY(need(ctx, v, bytes, "v"));
    STEP_TRY(need(ctx, k_cache, cache_bytes(b), "k_cache"));
    STEP_TRY(need(ctx, v_cache, cache_bytes(b), "v_cache"));
    if (k_values) STEP_TRY(need(ctx, k_values, bytes, "k_values"));
    if (v_values) STEP_TRY(need(ctx, v_values, bytes, "v_values"));
    STEP_TRY(alone(k_cache, {k, v, v_cache}, "k_cache"));
    STEP_TRY(alone(v_cache, {k, v}, "v_cache"));
    // (a thread reads its elements of k before it writes them)
    STEP_TRY(alone(k_values, {v, k_cache, v_cache, v_values}, "k_values"));
    STEP_TRY(alone(v_values, {k, k_cache, v_cache}, "v_values"));
    if (b->q.rows == 0) return SULIMO_HIP_OK;
    wrote(k_cache);
    wrote(v_cache);
    wrote(k_values);
    wrote(v_values);
    return launch_kv_store_paged(seq_view(b), (int)row_width(b), dp<const uint16_t>(k), dp<const uint16_t>(v),
                                 dp<uint8_t>(k_cache), dp<uint8_t>(v_cache), dp<uint16_t>(k_values),
                                 dp<uint16_t>(v_values), ctx->stream);
  });
}

int32_t sulimo_hip_enqueue_kv_load_paged(sulimo_hip_ctx *ctx, sulimo_hip_seq_batch *b,
                                         const sulimo_hip_buffer *k_cache, const sulimo_hip_buffer *v_cache,
                                         sulimo_hip_buffer *k_out, sulimo_hip_buffer *v_out) {
  return guarded([&]() -> int32_t {
    STEP_TRY(begin_step(ctx, b));
    STEP_TRY(need_pages(b));
    const size_t bytes = (size_t)b->q.positions * row_width(b) * 2;
    STEP_TRY(need(ctx, k_cache, cache_bytes(b), "k_cache"));
    STEP_TRY(need(ctx, v_cache, cache_bytes(b), "v_cache"));
    STEP_TRY(need(ctx, k_out, bytes, "k_out"));
    STEP_TRY(need(ctx, v_out, bytes, "v_out"));
    STEP_TRY(alone(k_out, {k_cache, v_cache, v_out}, "k_out"));
    STEP_TRY(alone(v_out, {k_cache, v_cache}, "v_out"));
    if (b->q.positions == 0) return SULIMO_HIP_OK;
    if (!b->load_ready) {
      const std::vector<LoadTile> tiles = load_tiles(b->q);
      STEP_TRY(step_array(b, &b->load_tiles, tiles.size() * sizeof(LoadTile)));
      SULIMO_HIP_TRY(hipMemcpyAsync(b->load_tiles.dev, tiles.data(), tiles.size() * sizeof(LoadTile),
                                    hipMemcpyHostToDevice, ctx->stream));
      b->n_load_tiles = (int)tiles.size();
      b->load_ready = true;
    }
    wrote(k_out);
    wrote(v_out);
    return launch_kv_load_paged(reinterpret_cast<const LoadTile *>(b->load_tiles.dev), b->n_load_tiles,
                                seq_view(b).pages, b->g.page_size, (int)row_width(b), dp<const uint8_t>(k_cache),
                                dp<const uint8_t>(v_cache), dp<uint16_t>(k_out), dp<uint16_t>(v_out), nullptr,
                                ctx->stream);
  });
}

int32_t sulimo_hip_enqueue_attention_paged(sulimo_hip_ctx *ctx, sulimo_hip_seq_batch *b, const sulimo_hip_buffer *q,
                                           const sulimo_hip_buffer *k_cache, const sulimo_hip_buffer *v_cache,
                                           sulimo_hip_buffer *out) {
  return guarded([&]() -> int32_t {
    STEP_TRY(begin_step(ctx, b));
    STEP_TRY(need_pages(b));
    const size_t bytes = (size_t)b->q.rows * b->g.n_head * b->g.head_dim * 2;
    STEP_TRY(need(ctx, q, bytes, "q"));
    STEP_TRY(need(ctx, k_cache, cache_bytes(b), "k_cache"));
    STEP_TRY(need(ctx, v_cache, cache_bytes(b), "v_cache"));
    STEP_TRY(need(ctx, out, bytes, "out"));
    STEP_TRY(alone(out, {q, k_cache, v_cache}, "out"));
    if (b->q.rows == 0) return SULIMO_HIP_OK;
    wrote(out);
    return attention_paged(b, dp<const uint16_t>(q), dp<const uint8_t>(k_cache), dp<const uint8_t>(v_cache),
                           dp<uint16_t>(out));
  });
}

int32_t sulimo_hip_enqueue_attention_packed(sulimo_hip_ctx *ctx, sulimo_hip_seq_batch *b, const sulimo_hip_buffer *q,
                                            const sulimo_hip_buffer *k, const sulimo_hip_buffer *v,
                                            sulimo_hip_buffer *out) {
  return guarded([&]() -> int32_t {
    STEP_TRY(begin_step(ctx, b));
    STEP_TRY(need_heads(b));
    const size_t bytes = (size_t)b->q.rows * b->g.n_head * b->g.head_dim * 2;
    const size_t kv = (size_t)b->q.rows * row_width(b) * 2;
    for (int s = 0; s < b->q.n_seqs; s++)
      if (b->q.start[s]) return fail(kInval, "packed attention takes whole prompts: sequence " + std::to_string(s) + " has cached positions");
    STEP_TRY(need(ctx, q, bytes, "q"));
    STEP_TRY(need(ctx, k, kv, "k"));
    STEP_TRY(need(ctx, v, kv, "v"));
    STEP_TRY(need(ctx, out, bytes, "out"));
    STEP_TRY(alone(out, {q, k, v}, "out"));
    if (b->q.rows == 0) return SULIMO_HIP_OK;
    wrote(out);
    return attention_packed(b, dp<const uint16_t>(q), dp<const uint16_t>(k), dp<const uint16_t>(v),
                            dp<uint16_t>(out));
  });
}

int32_t sulimo_hip_enqueue_verify_drafts(sulimo_hip_ctx *ctx, sulimo_hip_seq_batch *b,
                                         const sulimo_hip_buffer *logits, const sulimo_hip_buffer *tokens,
                                         const sulimo_hip_buffer *draft_probs, const sulimo_hip_buffer *uniforms,
                                         size_t vocab, float temperature, sulimo_hip_buffer *accepted,
                                         sulimo_hip_buffer *answer) {
  return guarded([&]() -> int32_t {
    STEP_TRY(begin_step(ctx, b));
    if (vocab == 0 || vocab > (size_t)INT_MAX / 2) return fail(kInval, "bad vocab size");
    if (!(temperature >= 0.0f) || temperature > 3.0e38f) return fail(kInval, "temperature must be finite and >= 0");
    for (int s = 0; s < b->q.n_seqs; s++)
      if (b->q.n_new[s] == 0) return fail(kInval, "sequence " + std::to_string(s) + " has no row to answer from");
    const size_t rows = b->q.rows;
    STEP_TRY(need(ctx, logits, rows * vocab * 4, "logits"));
    STEP_TRY(need(ctx, tokens, rows * 4, "tokens"));
    if (draft_probs && temperature > 0.0f)
      STEP_TRY(need(ctx, draft_probs, (rows - b->q.n_seqs) * vocab * 4, "draft_probs"));
    if (temperature > 0.0f) STEP_TRY(need(ctx, uniforms, rows * 4, "uniforms"));
    STEP_TRY(need(ctx, accepted, (size_t)b->q.n_seqs * 4, "accepted"));
    STEP_TRY(need(ctx, answer, rows * 4, "answer"));
    STEP_TRY(alone(accepted, {logits, tokens, draft_probs, uniforms, answer}, "accepted"));
    STEP_TRY(alone(answer, {logits, tokens, draft_probs, uniforms}, "answer"));
    if (rows == 0) return SULIMO_HIP_OK;
    wrote(accepted);
    wrote(answer);
    VerifyArgs a{};
    a.logits = dp<const float>(logits);
    a.tokens = dp<const int32_t>(tokens);
    a.draft_probs = temperature > 0.0f ? dp<const float>(draft_probs) : nullptr;
    a.uniforms = temperature > 0.0f ? dp<const float>(uniforms) : nullptr;
    a.vocab = (int)vocab;
    a.temperature = temperature;
    a.accepted = dp<int32_t>(accepted);
    a.answer = dp<int32_t>(answer);
    return verify_drafts(b, a);
  });
}

}  // extern "C"
