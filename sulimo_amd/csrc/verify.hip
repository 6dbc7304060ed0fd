// verify.hip - drafted tokens against the target's probabilities, from given randoms.
//
// Rows off .. off + k of a sequence hold the target's logits behind its last token and behind
// each of its k drafts. With p = softmax(logits / temperature) of row off + i - 1, q the draft
// model's distribution and u the row's uniform, draft d (token off + i) is accepted while
// u q(d) < p(d); the first one that is not is replaced by a token of max(p - q, 0), normalised,
// and behind k accepted drafts comes a token of p of the last row: the lowest j whose running
// sum exceeds the last row's uniform times the total (a refused draft's own uniform is known to
// be great, so it cannot choose its replacement). So the tokens are distributed as the target's
// alone.
#include <math.h>

#include "seq_batch.h"

namespace sulimo {
namespace {

// One workgroup per sequence.
__global__ __launch_bounds__(256) void verify_simple_kernel(SeqView v, VerifyArgs a) {
  __shared__ double sd[256];
  __shared__ int si[256];
  const int s = blockIdx.x, off = v.off[s], n = v.off[s + 1] - off, tid = threadIdx.x;
  const int V = a.vocab;
  auto reduce_max = [&](double x, int i, int *arg) {  // the highest index of the greatest value
    sd[tid] = x;
    si[tid] = i;
    __syncthreads();
    for (int o = 128; o >= 1; o >>= 1) {
      if (tid < o && (sd[tid + o] > sd[tid] || (sd[tid + o] == sd[tid] && si[tid + o] > si[tid]))) {
        sd[tid] = sd[tid + o];
        si[tid] = si[tid + o];
      }
      __syncthreads();
    }
    const double r = sd[0];
    *arg = si[0];
    __syncthreads();
    return r;
  };
  auto reduce_sum = [&](double x) {
    sd[tid] = x;
    __syncthreads();
    for (int o = 128; o >= 1; o >>= 1) {
      if (tid < o) sd[tid] += sd[tid + o];
      __syncthreads();
    }
    const double r = sd[0];
    __syncthreads();
    return r;
  };
  for (int i = 0; i < n; i++) {
    const float *x = a.logits + (size_t)(off + i) * V;
    const float *q = a.draft_probs && i < n - 1 ? a.draft_probs + (size_t)(off - s + i) * V : nullptr;
    const int d = i < n - 1 ? a.tokens[off + i + 1] : -1;
    const bool valid = d >= 0 && d < V;
    double bm = -INFINITY;
    int bi = -1;
    for (int j = tid; j < V; j += 256)
      if ((double)x[j] >= bm && x[j] > -INFINITY) bm = x[j], bi = j;
    int top;
    const double m = reduce_max(bm, bi, &top);
    int answer = -1;
    bool accept;
    if (a.temperature == 0.0) {
      accept = valid && d == top;
      answer = top;
    } else {
      auto drafted = [&](int j) { return q[j] > 0.0f ? (double)q[j] : 0.0; };
      auto weight = [&](int j) {
        const double y = x[j];
        return y == m ? 1.0 : y > -INFINITY ? exp((y - m) / a.temperature) : 0.0;
      };
      double part = 0.0;
      if (top >= 0)
        for (int j = tid; j < V; j += 256) part += weight(j);
      const double W = reduce_sum(part);
      auto uniform = [&](int r) { return a.uniforms[r] >= 0.0f ? (double)a.uniforms[r] : 0.0; };
      accept = valid && top >= 0 && uniform(off + i) * (q ? drafted(d) : 1.0) < weight(d) / W;
      if (!accept && top >= 0) {
        // chunks of consecutive tokens, one a thread; a rejected draft leaves max(p - q, 0)
        const int per = (V + 255) / 256, j0 = min(V, tid * per), j1 = min(V, j0 + per);
        bool rest = i < n - 1;
        auto mass = [&](int j) {
          const double p = weight(j) / W;
          if (!rest) return p;
          if (!q) return j == d ? 0.0 : p;
          return fmax(p - drafted(j), 0.0);
        };
        const double u = uniform(off + n - 1);
        double c = 0.0, total;
        for (int j = j0; j < j1; j++) c += mass(j);
        total = reduce_sum(c);
        if (!(total > 0.0)) {
          rest = false;
          c = 0.0;
          for (int j = j0; j < j1; j++) c += mass(j);
          total = reduce_sum(c);
        }
        sd[tid] = c;
        si[tid] = -1;
        __syncthreads();
        double before = 0.0;
        for (int t = 0; t < tid; t++) before += sd[t];
        // the first token whose running sum exceeds u * total, else the last with any mass
        int hit = V, last = -1;
        for (int j = j0; j < j1; j++) {
          const double w = mass(j);
          before += w;
          if (w > 0.0) last = j;
          if (hit == V && w > 0.0 && before > u * total) hit = j;
        }
        __syncthreads();
        int lastest;
        reduce_max(last, last, &lastest);
        int first;
        reduce_max(-(double)hit, hit, &first);
        answer = first < V ? first : lastest;
      }
    }
    if (accept) {
      if (tid == 0) a.answer[off + i] = d;
      continue;
    }
    if (tid == 0) {
      a.accepted[s] = i;
      a.answer[off + i] = answer;
      for (int j = i + 1; j < n; j++) a.answer[off + j] = -1;
    }
    return;
  }
}

}  // namespace

int32_t verify_drafts(sulimo_hip_seq_batch *b, const VerifyArgs &a) {
  hipLaunchKernelGGL(verify_simple_kernel, dim3(b->q.n_seqs), dim3(256), 0, b->ctx->stream, seq_view(b), a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SULIMO_HIP_OK : hip_fail(e, "verify_simple_kernel launch");
}

}  // namespace sulimo
