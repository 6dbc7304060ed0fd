// attention_step.hip - causal grouped attention of a step's sequences.
//
// Query row t of sequence s is position P = start[s] + t and sees positions
// max(0, P - window + 1) .. P of its own sequence (window 0: all):
//   out = sum_p softmax_p(q . K_p / sqrt(d)) V_p
// with K, V = code * f16(scale) of the paged Q8_0 cache, or f16 rows of the batch.
#include <math.h>

#include "seq_batch.h"

namespace sulimo {
namespace {

struct StepAttn {
  SeqView v;
  const _Float16 *q;  // [rows][n_head][HD]
  _Float16 *out;
  const uint8_t *k_cache, *v_cache;  // paged
  const _Float16 *k, *vv;            // packed [rows][n_head_kv][HD]
  int n_head, n_head_kv;
};

// One wave per (row, head): 64 keys at a time, one per lane.
template <int HD, bool PAGED>
__global__ __launch_bounds__(64) void step_attn_simple_kernel(StepAttn a) {
  constexpr int DL = HD / 64;  // output elements of a lane
  __shared__ float qs[HD];
  const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
  const int s = a.v.row_seq[row], kvh = h / (a.n_head / a.n_head_kv);
  const int P = a.v.start[s] + row - a.v.off[s];
  const _Float16 *q = a.q + ((size_t)row * a.n_head + h) * HD;
  for (int i = lane; i < HD; i += 64) qs[i] = (float)q[i];
  __syncthreads();
  const int lo = a.v.window ? max(0, P - a.v.window + 1) : 0;
  const int32_t *pt = a.v.pages + a.v.page_off[s];
  const size_t width = (size_t)a.n_head_kv * HD, bytes = width / 32 * 34;
  auto slot = [&](int p) { return (size_t)pt[p / a.v.page_size] * a.v.page_size + p % a.v.page_size; };
  auto value = [&](const uint8_t *cache, const _Float16 *rows, size_t r, int i) {
    if constexpr (PAGED) {
      const uint8_t *b = cache + r * bytes + (size_t)(kvh * (HD / 32) + i / 32) * 34;
      return (float)(int8_t)b[2 + i % 32] * (float)*reinterpret_cast<const _Float16 *>(b);
    } else {
      return (float)rows[r * width + kvh * HD + i];
    }
  };
  float m = -INFINITY, l = 0.0f, o[DL] = {};
  for (int p0 = lo; p0 <= P; p0 += 64) {
    const int p = p0 + lane;
    size_t r = 0;
    float x = -INFINITY;
    if (p <= P) {
      r = PAGED ? slot(p) : (size_t)a.v.off[s] + p;
      float acc = 0.0f;
      for (int i = 0; i < HD; i++) acc += qs[i] * value(a.k_cache, a.k, r, i);
      x = acc / sqrtf((float)HD);
    }
    float mx = x;
    for (int e = 32; e >= 1; e >>= 1) mx = fmaxf(mx, __shfl_xor(mx, e, 64));
    const float mn = fmaxf(m, mx);
    const float w = expf(x - mn), al = expf(m - mn);
    float sum = w;
    for (int e = 32; e >= 1; e >>= 1) sum += __shfl_xor(sum, e, 64);
    l = l * al + sum;
    m = mn;
    for (int e = 0; e < DL; e++) o[e] *= al;
    const int cnt = min(64, P - p0 + 1);
    for (int j = 0; j < cnt; j++) {
      const float wj = __shfl(w, j, 64);
      const size_t rj = __shfl((long)r, j, 64);
      for (int e = 0; e < DL; e++) o[e] += wj * value(a.v_cache, a.vv, rj, lane + 64 * e);
    }
  }
  for (int e = 0; e < DL; e++) a.out[((size_t)row * a.n_head + h) * HD + lane + 64 * e] = (_Float16)(o[e] / l);
}

template <bool PAGED>
int32_t run(const StepAttn &a, int hd, hipStream_t s) {
  const dim3 grid(a.v.rows, a.n_head);
  if (hd == 64) hipLaunchKernelGGL((step_attn_simple_kernel<64, PAGED>), grid, dim3(64), 0, s, a);
  else hipLaunchKernelGGL((step_attn_simple_kernel<128, PAGED>), grid, dim3(64), 0, s, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SULIMO_HIP_OK : hip_fail(e, "step_attn_simple_kernel launch");
}

}  // namespace

int32_t attention_paged(sulimo_hip_seq_batch *b, const uint16_t *q, const uint8_t *k_cache, const uint8_t *v_cache,
                        uint16_t *out) {
  StepAttn a{seq_view(b), reinterpret_cast<const _Float16 *>(q), reinterpret_cast<_Float16 *>(out), k_cache, v_cache,
             nullptr, nullptr, b->g.n_head, b->g.n_head_kv};
  return run<true>(a, b->g.head_dim, b->ctx->stream);
}

int32_t attention_packed(sulimo_hip_seq_batch *b, const uint16_t *q, const uint16_t *k, const uint16_t *v,
                         uint16_t *out) {
  StepAttn a{seq_view(b), reinterpret_cast<const _Float16 *>(q), reinterpret_cast<_Float16 *>(out), nullptr, nullptr,
             reinterpret_cast<const _Float16 *>(k), reinterpret_cast<const _Float16 *>(v), b->g.n_head, b->g.n_head_kv};
  return run<false>(a, b->g.head_dim, b->ctx->stream);
}

}  // namespace sulimo
