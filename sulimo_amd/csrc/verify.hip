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
//
// What it must read is every logit once, and one row of draft probabilities for a refused
// draft. Two launches:
//   1. row_stats_kernel, a workgroup per (row, 4096 logits): the chunk's greatest logit, its last
//      index, and the sum of exp((x - max) / temperature), the logits held in registers between.
//   2. choose_kernel, a workgroup per (sequence, chunk): every one joins its sequence's chunks
//      and judges the drafts, eight rows at a time. Where one was refused, each adds up max(p -
//      q, 0) over its chunk (the row comes from the caches) and the last to arrive finds the
//      token; else the first finds it from the sums of launch 1. Only the chunk that holds the
//      token is walked.
// Sums and exponentials are f64: a token of 1e-5 of the mass is missed with f32 sums over 150000
// of them now and then, and the answers would depend on the order of the sum. An exponential
// costs some 16 f64 instructions, less than the loads of its logit take.
#include <math.h>

#include "seq_batch.h"

namespace sulimo {
namespace {

typedef float float4a4 __attribute__((ext_vector_type(4), aligned(4)));  // rows of any vocabulary

constexpr int kChunk = 4096;

struct ChunkStat {
  double sum;  // of exp((x - max) / temperature); 0 if nothing is above -infinity
  float max;
  int32_t arg;  // last index of max, -1 if nothing is above -infinity
};

// e^x for x <= 0 (0 below the smallest normal number): 2^n e^f, |f| <= ln 2 / 2, by its series to
// f^11 (off by less than 4e-15 of the value).
__device__ __forceinline__ double exp_neg(double x) {
  x = fmax(x, -1000.0);
  const double n = rint(x * 1.4426950408889634074);
  double f = __builtin_fma(n, -0.6931471805599453, x);  // ln 2 as f64, one rounding
  f = __builtin_fma(n, -2.3190468138462996e-17, f);      // and what is left of ln 2
  double r = 1.0 / 39916800.0;
  r = __builtin_fma(r, f, 1.0 / 3628800.0);
  r = __builtin_fma(r, f, 1.0 / 362880.0);
  r = __builtin_fma(r, f, 1.0 / 40320.0);
  r = __builtin_fma(r, f, 1.0 / 5040.0);
  r = __builtin_fma(r, f, 1.0 / 720.0);
  r = __builtin_fma(r, f, 1.0 / 120.0);
  r = __builtin_fma(r, f, 1.0 / 24.0);
  r = __builtin_fma(r, f, 1.0 / 6.0);
  r = __builtin_fma(r, f, 0.5);
  r = __builtin_fma(r, f, 1.0);
  r = __builtin_fma(r, f, 1.0);
  return ldexp(r, (int)n);
}

// Weight of logit x beside the row's greatest one, m (above -infinity): NaN counts as -infinity,
// and several +infinities are equal.
__device__ __forceinline__ double weight(float x, float m, double inv_t) {
  if (x == m) return 1.0;
  return x > -INFINITY ? exp_neg(((double)x - (double)m) * inv_t) : 0.0;
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// Greatest value and its highest index over the wave (arg -1: none).
__device__ __forceinline__ void wave_max(float &m, int &arg) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const float m2 = __shfl_xor(m, o, 64);
    const int a2 = __shfl_xor(arg, o, 64);
    if (m2 > m || (m2 == m && a2 > arg)) m = m2, arg = a2;
  }
}

// N elements of a row from j0 on, elements past the vocabulary as `past`.
template <int N>
__device__ __forceinline__ void load_row(const float *row, int j0, int vocab, float past, float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    if (j0 + i + 4 <= vocab) {
      const float4a4 v = *reinterpret_cast<const float4a4 *>(row + j0 + i);
#pragma unroll
      for (int e = 0; e < 4; e++) x[i + e] = v[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) x[i + e] = j0 + i + e < vocab ? row[j0 + i + e] : past;
    }
  }
}

__global__ __launch_bounds__(256) void row_stats_kernel(const float *logits, int vocab, int chunks, double inv_t,
                                                        ChunkStat *stats) {
  __shared__ float sm[4];
  __shared__ int sa[4];
  __shared__ double ss[4];
  const int chunk = blockIdx.x % chunks, row = blockIdx.x / chunks, wave = threadIdx.x >> 6;
  const float *x = logits + (size_t)row * vocab;
  float v[16];
  float m = -INFINITY;
  int arg = -1;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int j0 = chunk * kChunk + i * 1024 + threadIdx.x * 4;
    float w[4];
    load_row(x, j0, vocab, -INFINITY, w);
#pragma unroll
    for (int e = 0; e < 4; e++) v[4 * i + e] = w[e];
  }
#pragma unroll
  for (int i = 0; i < 16; i++)
    if (v[i] >= m && v[i] > -INFINITY) m = v[i], arg = chunk * kChunk + (i >> 2) * 1024 + threadIdx.x * 4 + (i & 3);
  wave_max(m, arg);
  if ((threadIdx.x & 63) == 0) sm[wave] = m, sa[wave] = arg;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; w++)
    if (sm[w] > m || (sm[w] == m && sa[w] > arg)) m = sm[w], arg = sa[w];
  double s = 0.0;
  if (arg >= 0 && inv_t > 0.0) {
#pragma unroll
    for (int i = 0; i < 16; i++) s += weight(v[i], m, inv_t);
  }
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) ss[wave] = s;
  __syncthreads();
  if (threadIdx.x == 0) stats[blockIdx.x] = ChunkStat{ss[0] + ss[1] + ss[2] + ss[3], m, arg};
}

struct Row {  // a row's softmax: p_j = weight(x_j) / sum
  float max;
  int arg;
  double sum;
};
// Joins a row's chunks: one wave, every lane gets the row.
__device__ __forceinline__ Row join_row(const ChunkStat *stats, int chunks, double inv_t) {
  const int lane = threadIdx.x & 63;
  Row r{-INFINITY, -1, 0.0};
  for (int c = lane; c < chunks; c += 64) {
    const ChunkStat s = stats[c];
    if (s.arg < 0) continue;
    if (s.max >= r.max) r.max = s.max, r.arg = s.arg;
  }
  wave_max(r.max, r.arg);
  if (r.arg >= 0 && inv_t > 0.0)
    for (int c = lane; c < chunks; c += 64) {
      const ChunkStat s = stats[c];
      if (s.arg >= 0) r.sum += s.sum * weight(s.max, r.max, inv_t);
    }
  r.sum = wave_sum(r.sum);
  return r;
}

constexpr int kChoose = 512, kWaves = kChoose / 64;

// The first index whose value is above the target by running sum over threads and each thread's
// 8 values (starting at `before` of the block), else the last with any; every thread gets it.
__device__ __forceinline__ int find_token(const double (&w)[8], int j0, double before, double target, double *wsum,
                                          int *found) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double mine = 0.0;
#pragma unroll
  for (int e = 0; e < 8; e++) mine += w[e];
  double scan = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(scan, o, 64);
    if (lane >= o) scan += y;
  }
  if (lane == 63) wsum[wave] = scan;
  if (threadIdx.x == 0) found[0] = INT_MAX, found[1] = -1;
  __syncthreads();
  double run = before + (scan - mine);
  for (int v = 0; v < wave; v++) run += wsum[v];
  int hit = INT_MAX, last = -1;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    run += w[e];
    if (w[e] > 0.0) {
      last = j0 + e;
      if (hit == INT_MAX && run > target) hit = j0 + e;
    }
  }
  if (hit != INT_MAX) atomicMin(&found[0], hit);
  if (last >= 0) atomicMax(&found[1], last);
  __syncthreads();
  return found[0] != INT_MAX ? found[0] : found[1];
}

// grid.x: sequence * chunks + chunk. mass: [n_seqs][chunks] f64, counters: [n_seqs], zero.
__global__ __launch_bounds__(kChoose) void choose_kernel(SeqView v, VerifyArgs a, int chunks, double inv_t,
                                                         const ChunkStat *stats, double *mass, int *counters) {
  __shared__ double wsum[kWaves];
  __shared__ int found[2], judged[kWaves];
  __shared__ Row srow[kWaves];
  __shared__ double sbefore;
  __shared__ int schunk, slast, srest;
  const int s = blockIdx.x / chunks, chunk = blockIdx.x % chunks, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int off = v.off[s], n = v.off[s + 1] - off, V = a.vocab;
  const bool greedy = inv_t == 0.0;
  auto uniform = [&](int r) { return a.uniforms[r] >= 0.0f ? (double)a.uniforms[r] : 0.0; };
  auto drafted = [&](float q) { return q > 0.0f ? (double)q : 0.0; };

  // ---- judge the drafts: a wave a row ----
  int acc = n - 1;
  Row row{};
  for (int i0 = 0; i0 < n; i0 += kWaves) {
    const int i = i0 + wave;
    if (i < n) {
      const Row r = join_row(stats + (size_t)(off + i) * chunks, chunks, inv_t);
      bool ok = false;
      if (i < n - 1 && r.arg >= 0) {
        const int d = a.tokens[off + i + 1];
        if (greedy) {
          ok = d == r.arg;
        } else if (d >= 0 && d < V) {
          const double q = a.draft_probs ? drafted(a.draft_probs[(size_t)(off - s + i) * V + d]) : 1.0;
          ok = uniform(off + i) * q < weight(a.logits[(size_t)(off + i) * V + d], r.max, inv_t) / r.sum;
        }
      }
      if (lane == 0) judged[wave] = ok, srow[wave] = r;
    }
    __syncthreads();
    const int m = min(kWaves, n - i0);
    int w = 0;
    while (w < m && judged[w]) w++;
    if (w < m) {
      acc = i0 + w;
      row = srow[w];
      break;
    }
    __syncthreads();
  }
  const bool refused = acc < n - 1;
  auto finish = [&](int token) {  // one workgroup of a sequence ends here
    if (tid == 0) a.accepted[s] = acc;
    for (int j = tid; j < n; j += kChoose) a.answer[off + j] = j < acc ? a.tokens[off + j + 1] : j == acc ? token : -1;
  };
  if (greedy || row.arg < 0) {
    if (chunk == 0) finish(row.arg);
    return;
  }
  const float *x = a.logits + (size_t)(off + acc) * V;
  const float *q = refused && a.draft_probs ? a.draft_probs + (size_t)(off - s + acc) * V : nullptr;
  const int d = refused ? a.tokens[off + acc + 1] : -1;
  // this thread's 8 tokens of chunk c: p, or what a refused draft leaves of it
  auto masses = [&](int c, bool rest, double (&w)[8]) {
    const int j0 = c * kChunk + tid * 8;
    float l[8], qv[8];
    load_row(x, j0, V, -INFINITY, l);
    if (rest && q) load_row(q, j0, V, 0.0f, qv);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      w[e] = weight(l[e], row.max, inv_t) / row.sum;
      if (rest) w[e] = q ? fmax(w[e] - drafted(qv[e]), 0.0) : j0 + e == d ? 0.0 : w[e];
    }
    return j0;
  };
  double w[8];
  if (refused) {
    masses(chunk, true, w);
    double t = 0.0;
#pragma unroll
    for (int e = 0; e < 8; e++) t += w[e];
    t = wave_sum(t);
    if (lane == 0) wsum[wave] = t;
    __syncthreads();
    if (tid == 0) {
      t = 0.0;
#pragma unroll
      for (int e = 0; e < kWaves; e++) t += wsum[e];
      // device-scope store and count: coherent across the XCDs' L2 caches
      __hip_atomic_store(reinterpret_cast<uint64_t *>(mass + blockIdx.x), __builtin_bit_cast(uint64_t, t),
                         __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      slast = __hip_atomic_fetch_add(counters + s, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == chunks - 1;
      if (slast) __hip_atomic_store(counters + s, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next call
    }
    __syncthreads();
    if (!slast) return;
  } else if (chunk) {
    return;
  }

  // ---- the chunk of the token: wave 0, sixty-four chunks at a time, in order ----
  auto chunk_mass = [&](int c, bool rest) {
    if (c >= chunks) return 0.0;
    if (rest)
      return __builtin_bit_cast(double, __hip_atomic_load(reinterpret_cast<uint64_t *>(mass + (size_t)s * chunks + c),
                                                          __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    const ChunkStat st = stats[(size_t)(off + acc) * chunks + c];
    return st.arg >= 0 ? st.sum * weight(st.max, row.max, inv_t) / row.sum : 0.0;
  };
  const double u = uniform(off + n - 1);
  bool rest = refused;
  double total = 0.0;
  if (wave == 0) {
    for (int pass = 0; pass < 2; pass++) {  // nothing left of p - q: p itself
      total = 0.0;
      for (int c0 = 0; c0 < chunks; c0 += 64) total += wave_sum(chunk_mass(c0 + lane, rest));
      if (total > 0.0 || !rest) break;
      rest = false;
    }
    const double target = u * total;
    double before = 0.0;
    int at = -1;
    double at_before = 0.0;
    for (int c0 = 0; c0 < chunks; c0 += 64) {
      const double m = chunk_mass(c0 + lane, rest);
      double scan = m;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const double y = __shfl_up(scan, o, 64);
        if (lane >= o) scan += y;
      }
      const uint64_t over = __ballot(m > 0.0 && before + scan > target), any = __ballot(m > 0.0);
      if (over || any) {  // the first above the target, else the last with any so far
        const int l = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(any);
        at = c0 + l;
        at_before = before + __shfl(scan - m, l, 64);
      }
      if (over) break;
      before += __shfl(scan, 63, 64);
    }
    if (lane == 0) schunk = at, sbefore = at_before, srest = rest, wsum[0] = target;
  }
  __syncthreads();
  const int at = schunk;
  const double before = sbefore, target = wsum[0];
  rest = srest != 0;
  __syncthreads();
  const int j0 = masses(at, rest, w);
  finish(find_token(w, j0, before, target, wsum, found));
}

}  // namespace

int32_t verify_drafts(sulimo_hip_seq_batch *b, const VerifyArgs &a) {
  sulimo_hip_ctx *ctx = b->ctx;
  const int chunks = (a.vocab + kChunk - 1) / kChunk, S = b->q.n_seqs;
  if ((size_t)b->q.rows * chunks > (size_t)INT_MAX)
    return fail(SULIMO_HIP_ERR_INVALID_ARGUMENT, "too many rows and tokens together");
  if (b->verify_counters.bytes < (size_t)S * 4) {  // zero between calls
    if (const int32_t rc = step_array(b, &b->verify_counters, (size_t)S * 4)) return rc;
    const std::vector<char> zero(b->verify_counters.bytes, 0);
    SULIMO_HIP_TRY(hipMemcpyAsync(b->verify_counters.dev, zero.data(), zero.size(), hipMemcpyHostToDevice, ctx->stream));
  }
  const size_t stat_bytes = ((size_t)b->q.rows * chunks * sizeof(ChunkStat) + 255) & ~(size_t)255;
  if (const int32_t rc = ensure_workspace(ctx, stat_bytes + (size_t)S * chunks * 8)) return rc;
  ChunkStat *stats = reinterpret_cast<ChunkStat *>(ctx->ws);
  double *mass = reinterpret_cast<double *>(reinterpret_cast<char *>(ctx->ws) + stat_bytes);
  const double inv_t = a.temperature > 0.0 ? 1.0 / a.temperature : 0.0;
  hipLaunchKernelGGL(row_stats_kernel, dim3((unsigned)b->q.rows * chunks), dim3(256), 0, ctx->stream, a.logits, a.vocab,
                     chunks, inv_t, stats);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return hip_fail(e, "row_stats_kernel launch");
  hipLaunchKernelGGL(choose_kernel, dim3((unsigned)S * chunks), dim3(kChoose), 0, ctx->stream, seq_view(b), a, chunks,
                     inv_t, stats, mass, reinterpret_cast<int *>(b->verify_counters.dev));
  e = hipGetLastError();
  return e == hipSuccess ? SULIMO_HIP_OK : hip_fail(e, "choose_kernel launch");
}

}  // namespace sulimo
