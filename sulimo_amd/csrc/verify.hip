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
//   1. row_stats_kernel, a wave per (row, 1024 logits): the chunk's greatest logit, its last index
//      where that is asked for, and the sum of exp((x - max) / temperature), the logits held in
//      registers between. Waves need nothing of each other.
//   2. choose_kernel, eight waves per (sequence, 8 chunks): every workgroup joins its sequence's
//      chunks and judges the drafts, a wave a row, eight rows at a time. Where one was refused,
//      each wave adds up max(p - q, 0) over its chunk (the row comes from the caches) and the
//      last workgroup to arrive finds the token; else the first finds it from the sums of launch
//      1. Only the chunk that holds the token is walked.
// Sums and exponentials are f64: a token of 1e-5 of the mass is missed with f32 sums over 150000
// of them now and then, and the answers would depend on the order of the sum. An exponential
// costs some 20 f64 instructions (a third of the time that 24 sequences of up to 9 rows take).
// Reductions go by DPP, whose steps wait for no LDS.
#include <math.h>

#include "seq_batch.h"

namespace sulimo {
namespace {

typedef float float4a4 __attribute__((ext_vector_type(4), aligned(4)));  // rows of any vocabulary

constexpr int kChunk = 1024;  // 16 logits a lane

struct ChunkStat {
  double sum;  // of exp((x - max) / temperature); 0 if nothing is above -infinity
  float max;
  int32_t arg;  // last index of max, -1 if nothing is above -infinity
};

// 2^t for t <= 0, zero below 2^-1021: 2^n times the series of e^(f ln 2), |f| <= 1/2, to f^10 (off by
// less than 3e-13 of the value). n comes out of the low bits of t + 1.5 2^52 and goes into the
// exponent as an integer: the conversions, roundings and ldexp of f64 take four times an fma.
__device__ __forceinline__ double exp2_neg(double t) {
  constexpr double kShift = 6755399441055744.0, L = 0.69314718055994530942;  // 1.5 2^52, ln 2
  const double at = fmax(t, -1021.0) + kShift;
  const double f = fmax(t, -1021.0) - (at - kShift);
  constexpr double c2 = L * L / 2, c3 = c2 * L / 3, c4 = c3 * L / 4, c5 = c4 * L / 5, c6 = c5 * L / 6, c7 = c6 * L / 7,
                   c8 = c7 * L / 8, c9 = c8 * L / 9, c10 = c9 * L / 10;
  double r = __builtin_fma(c10, f, c9);
  r = __builtin_fma(r, f, c8);
  r = __builtin_fma(r, f, c7);
  r = __builtin_fma(r, f, c6);
  r = __builtin_fma(r, f, c5);
  r = __builtin_fma(r, f, c4);
  r = __builtin_fma(r, f, c3);
  r = __builtin_fma(r, f, c2);
  r = __builtin_fma(r, f, L);
  r = __builtin_fma(r, f, 1.0);
  typedef int int2v __attribute__((ext_vector_type(2)));
  int2v x = __builtin_bit_cast(int2v, r);
  x[1] += __builtin_bit_cast(int2v, at)[0] << 20;
  return t < -1021.0 ? 0.0 : __builtin_bit_cast(double, x);
}

// Weight of logit x beside the row's greatest one, m (above -infinity): NaN counts as -infinity,
// and several +infinities are equal. c = log2(e) / temperature.
__device__ __forceinline__ double weight(float x, float m, double c) {
  double r = exp2_neg(((double)x - (double)m) * c);  // (no branch: each would wait for the one before)
  r = x > -INFINITY ? r : 0.0;
  return x == m ? 1.0 : r;
}

// v of the lane that the DPP control names, `none` where there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp(float v, float none) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v),
                                                               CTRL, ROWS, 0xf, false));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp0(double v) {
  typedef int int2v __attribute__((ext_vector_type(2)));
  int2v x = __builtin_bit_cast(int2v, v);
  x[0] = __builtin_amdgcn_update_dpp(0, x[0], CTRL, ROWS, 0xf, false);
  x[1] = __builtin_amdgcn_update_dpp(0, x[1], CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, x);
}
// Steps of a scan over the wave: 1, 2, 4, 8 lanes up inside rows of 16, then the rows' last lanes.
// Inclusive sum of lanes 0 .. lane.
__device__ __forceinline__ double wave_scan(double v) {
  v += dpp0<0x111, 0xf>(v);
  v += dpp0<0x112, 0xf>(v);
  v += dpp0<0x114, 0xf>(v);
  v += dpp0<0x118, 0xf>(v);
  v += dpp0<0x142, 0xa>(v);
  v += dpp0<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ double lane_value(double v, int lane) {
  typedef int int2v __attribute__((ext_vector_type(2)));
  int2v x = __builtin_bit_cast(int2v, v);
  x[0] = __builtin_amdgcn_readlane(x[0], lane);
  x[1] = __builtin_amdgcn_readlane(x[1], lane);
  return __builtin_bit_cast(double, x);
}
__device__ __forceinline__ double wave_sum(double v) { return lane_value(wave_scan(v), 63); }
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp<0x111, 0xf>(v, v));
  v = fmaxf(v, dpp<0x112, 0xf>(v, v));
  v = fmaxf(v, dpp<0x114, 0xf>(v, v));
  v = fmaxf(v, dpp<0x118, 0xf>(v, v));
  v = fmaxf(v, dpp<0x142, 0xa>(v, v));
  v = fmaxf(v, dpp<0x143, 0xc>(v, v));
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ __forceinline__ int wave_max(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x111, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x112, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x114, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x118, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x142, 0xa, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(v, 63);
}

// A lane's 16 elements of chunk c, four at each of c * kChunk + 256 i + 4 lane; elements past the
// vocabulary as `past`. Whole chunks load without a branch, so that the loads go out together.
__device__ __forceinline__ void load_chunk(const float *row, int c, int vocab, float past, float (&x)[16]) {
  const int j0 = c * kChunk + 4 * (threadIdx.x & 63);
  if ((c + 1) * kChunk <= vocab) {
    float4a4 v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = *reinterpret_cast<const float4a4 *>(row + j0 + 256 * i);
#pragma unroll
    for (int i = 0; i < 16; i++) x[i] = v[i >> 2][i & 3];
  } else {
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const int j = j0 + 256 * (i >> 2) + (i & 3);
      x[i] = j < vocab ? row[j] : past;
    }
  }
}

// total: rows * chunks, a wave each. scale: log2(e) / temperature, 0: greedy
__global__ __launch_bounds__(256) void row_stats_kernel(const float *logits, int vocab, int chunks, int total,
                                                        double scale, ChunkStat *stats) {
  const int id = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (id >= total) return;
  const int row = id / chunks, chunk = id - row * chunks;
  const float *x = logits + (size_t)row * vocab;
  float v[16], m = -INFINITY;
  load_chunk(x, chunk, vocab, -INFINITY, v);
#pragma unroll
  for (int i = 0; i < 16; i++) m = fmaxf(m, v[i]);  // (NaN is not taken)
  m = wave_max(m);
  double s = 0.0;
  int arg = -1;
  if (m > -INFINITY) {
    arg = chunk * kChunk;
    if (scale > 0.0) {
#pragma unroll
      for (int i = 0; i < 16; i++) s += weight(v[i], m, scale);
      s = wave_sum(s);
    } else {
#pragma unroll
      for (int i = 0; i < 16; i++)
        if (v[i] == m) arg = max(arg, chunk * kChunk + (i >> 2) * 256 + lane * 4 + (i & 3));
      arg = wave_max(arg);
    }
  }
  if (lane == 0) stats[id] = ChunkStat{s, m, arg};
}

struct Row {  // a row's softmax: p_j = weight(x_j) * inv
  float max;
  int arg;  // -1: nothing is above -infinity
  double inv;
};
// Joins a row's chunks: one wave, every lane gets the row. kHeld chunks a lane stay in registers.
constexpr int kHeld = 3;
__device__ __forceinline__ Row join_row(const ChunkStat *stats, int chunks, double scale) {
  const int lane = threadIdx.x & 63;
  ChunkStat held[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; i++) held[i] = lane + 64 * i < chunks ? stats[lane + 64 * i] : ChunkStat{0.0, -INFINITY, -1};
  auto each = [&](auto &&f) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kHeld; i++) f(held[i]);
    for (int c = lane + 64 * kHeld; c < chunks; c += 64) f(stats[c]);
  };
  Row r{-INFINITY, -1, 0.0};
  each([&](const ChunkStat &s) { r.max = fmaxf(r.max, s.max); });
  r.max = wave_max(r.max);
  if (r.max > -INFINITY) {
    each([&](const ChunkStat &s) {
      if (s.max == r.max) r.arg = max(r.arg, s.arg);
    });
    r.arg = wave_max(r.arg);
    if (scale > 0.0) {
      double sum = 0.0;
      each([&](const ChunkStat &s) {
        if (s.arg >= 0) sum += s.sum * weight(s.max, r.max, scale);
      });
      r.inv = 1.0 / wave_sum(sum);
    }
  }
  return r;
}

constexpr int kChoose = 512, kWaves = kChoose / 64;

// grid.x: sequence * groups + group of kWaves chunks. mass: [n_seqs][chunks] f64, counters:
// [n_seqs], zero.
__global__ __launch_bounds__(kChoose) void choose_kernel(SeqView v, VerifyArgs a, int chunks, int groups, double scale,
                                                         const ChunkStat *stats, double *mass, int *counters) {
  __shared__ int judged[kWaves], last_one, token;
  __shared__ Row srow[kWaves];
  const int s = blockIdx.x / groups, group = blockIdx.x % groups, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int off = v.off[s], n = v.off[s + 1] - off, V = a.vocab;
  const bool greedy = scale == 0.0;
  auto uniform = [&](int r) { return a.uniforms[r] >= 0.0f ? (double)a.uniforms[r] : 0.0; };
  auto drafted = [&](float q) { return q > 0.0f ? (double)q : 0.0; };

  // ---- judge the drafts: a wave a row ----
  int acc = n - 1;
  Row row{};
  for (int i0 = 0; i0 < n; i0 += kWaves) {
    const int i = i0 + wave;
    if (i < n) {
      // what the judgement reads is asked for before the row's chunks are joined
      const int d = i < n - 1 ? a.tokens[off + i + 1] : -1;
      const bool valid = d >= 0 && d < V && !greedy;
      const float x = valid ? a.logits[(size_t)(off + i) * V + d] : 0.0f;
      const double q = valid && a.draft_probs ? drafted(a.draft_probs[(size_t)(off - s + i) * V + d]) : 1.0;
      const double u = valid ? uniform(off + i) : 0.0;
      const Row r = join_row(stats + (size_t)(off + i) * chunks, chunks, scale);
      bool ok = false;
      if (i < n - 1 && r.arg >= 0) ok = greedy ? d == r.arg : valid && u * q < weight(x, r.max, scale) * r.inv;
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
  auto finish = [&](int t) {  // one workgroup of a sequence ends here
    if (tid == 0) a.accepted[s] = acc;
    for (int j = tid; j < n; j += kChoose) a.answer[off + j] = j < acc ? a.tokens[off + j + 1] : j == acc ? t : -1;
  };
  if (greedy || row.arg < 0) {
    if (group == 0) finish(row.arg);
    return;
  }
  const float *x = a.logits + (size_t)(off + acc) * V;
  const float *q = refused && a.draft_probs ? a.draft_probs + (size_t)(off - s + acc) * V : nullptr;
  const int d = refused ? a.tokens[off + acc + 1] : -1;
  // the lane's tokens of chunk c: p, or what a refused draft leaves of it
  auto masses = [&](int c, bool rest, double (&w)[16]) __attribute__((always_inline)) {
    float l[16], qv[16];
    load_chunk(x, c, V, -INFINITY, l);
    if (rest && q) load_chunk(q, c, V, 0.0f, qv);
#pragma unroll
    for (int e = 0; e < 16; e++) {
      w[e] = weight(l[e], row.max, scale) * row.inv;
      if (rest) w[e] = q ? fmax(w[e] - drafted(qv[e]), 0.0) : c * kChunk + 256 * (e >> 2) + 4 * lane + (e & 3) == d ? 0.0 : w[e];
    }
  };
  if (refused) {
    const int c = group * kWaves + wave;
    if (c < chunks) {
      double t = 0.0, w[16];
      masses(c, true, w);
#pragma unroll
      for (int e = 0; e < 16; e++) t += w[e];
      t = wave_sum(t);
      // device-scope store and count: past this XCD's L2 cache
      if (lane == 0)
        __hip_atomic_store(reinterpret_cast<uint64_t *>(mass + (size_t)s * chunks + c), __builtin_bit_cast(uint64_t, t),
                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) {
      last_one = __hip_atomic_fetch_add(counters + s, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == groups - 1;
      if (last_one) __hip_atomic_store(counters + s, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next call
    }
    __syncthreads();
    if (!last_one) return;
  } else if (group) {
    return;
  }

  // ---- the token, by wave 0: its chunk, then its place in it ----
  if (wave == 0) {
    auto chunk_mass = [&](int c, bool rest) {
      if (c >= chunks) return 0.0;
      if (rest)
        return __builtin_bit_cast(double, __hip_atomic_load(reinterpret_cast<uint64_t *>(mass + (size_t)s * chunks + c),
                                                            __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
      const ChunkStat st = stats[(size_t)(off + acc) * chunks + c];
      return st.arg >= 0 ? st.sum * weight(st.max, row.max, scale) * row.inv : 0.0;
    };
    const double u = uniform(off + n - 1);
    bool rest = refused;
    double held[kHeld], total = 0.0;
    for (int pass = 0; pass < 2; pass++) {  // nothing left of p - q: p itself
#pragma unroll
      for (int i = 0; i < kHeld; i++) held[i] = chunk_mass(lane + 64 * i, rest);
      total = 0.0;
#pragma unroll
      for (int i = 0; i < kHeld; i++) total += held[i];
      for (int c = lane + 64 * kHeld; c < chunks; c += 64) total += chunk_mass(c, rest);
      total = wave_sum(total);
      if (total > 0.0 || !rest) break;
      rest = false;
    }
    const double target = u * total;
    double before = 0.0, at_before = 0.0;
    int at = 0;
    for (int c0 = 0; c0 < chunks; c0 += 64) {
      double m = 0.0;
#pragma unroll
      for (int i = 0; i < kHeld; i++)
        if (c0 == 64 * i) m = held[i];
      if (c0 >= 64 * kHeld) m = chunk_mass(c0 + lane, rest);
      const double scan = wave_scan(m);
      const uint64_t over = __ballot(m > 0.0 && before + scan > target), any = __ballot(m > 0.0);
      if (over || any) {  // the first above the target, else the last with any so far
        const int l = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(any);
        at = c0 + l;
        at_before = before + (lane_value(scan, l) - lane_value(m, l));
      }
      if (over) break;
      before += lane_value(scan, 63);
    }
    // 256 tokens at a time, four a lane, in order
    double w[16], run = at_before;
    masses(at, rest, w);
    int hit = INT_MAX, last = -1;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const double mine = (w[4 * i] + w[4 * i + 1]) + (w[4 * i + 2] + w[4 * i + 3]);
      const double scan = wave_scan(mine);
      double r = run + (scan - mine);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int j = at * kChunk + i * 256 + lane * 4 + e;
        r += w[4 * i + e];
        if (w[4 * i + e] > 0.0) {
          last = j;
          if (hit == INT_MAX && r > target) hit = j;
        }
      }
      run += lane_value(scan, 63);
    }
    const int first = -wave_max(-hit);  // the lowest above the target, else the last with any mass
    last = wave_max(last);
    if (lane == 0) token = first != INT_MAX ? first : last;
  }
  __syncthreads();
  finish(token);
}

}  // namespace

int32_t verify_drafts(sulimo_hip_seq_batch *b, const VerifyArgs &a) {
  sulimo_hip_ctx *ctx = b->ctx;
  const int chunks = (a.vocab + kChunk - 1) / kChunk, groups = (chunks + kWaves - 1) / kWaves, S = b->q.n_seqs;
  if ((size_t)b->q.rows * chunks > (size_t)INT_MAX - 8)
    return fail(SULIMO_HIP_ERR_INVALID_ARGUMENT, "too many rows and tokens together");
  const int total = b->q.rows * chunks;
  if (b->verify_counters.bytes < (size_t)S * 4) {  // zero between calls
    if (const int32_t rc = step_array(b, &b->verify_counters, (size_t)S * 4)) return rc;
    const std::vector<char> zero(b->verify_counters.bytes, 0);
    SULIMO_HIP_TRY(hipMemcpyAsync(b->verify_counters.dev, zero.data(), zero.size(), hipMemcpyHostToDevice, ctx->stream));
  }
  const size_t stat_bytes = ((size_t)b->q.rows * chunks * sizeof(ChunkStat) + 255) & ~(size_t)255;
  if (const int32_t rc = ensure_workspace(ctx, stat_bytes + (size_t)S * chunks * 8)) return rc;
  ChunkStat *stats = reinterpret_cast<ChunkStat *>(ctx->ws);
  double *mass = reinterpret_cast<double *>(reinterpret_cast<char *>(ctx->ws) + stat_bytes);
  const double scale = a.temperature > 0.0 ? 1.4426950408889634074 / a.temperature : 0.0;
  hipLaunchKernelGGL(row_stats_kernel, dim3((unsigned)(total + 3) / 4), dim3(256), 0, ctx->stream, a.logits, a.vocab,
                     chunks, total, scale, stats);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return hip_fail(e, "row_stats_kernel launch");
  hipLaunchKernelGGL(choose_kernel, dim3((unsigned)S * groups), dim3(kChoose), 0, ctx->stream, seq_view(b), a, chunks,
                     groups, scale, stats, mass, reinterpret_cast<int *>(b->verify_counters.dev));
  e = hipGetLastError();
  return e == hipSuccess ? SULIMO_HIP_OK : hip_fail(e, "choose_kernel launch");
}

}  // namespace sulimo
