// step_attn.h - what the attention kernels of a step share: lane helpers, and the records by
// which workgroups that split a row tile's keys join their sums.
#pragma once

#include <math.h>

#include "seq_batch.h"

namespace sulimo {

// Records of split row tiles: f32 O (not yet divided) and (running max in log2 units, sum) per
// (piece, KV head, row), and an arrival counter per (row tile, head group), zero between calls.
struct Join {
  float *o;  // [record rows][head_dim]
  float2 *ml;
  int *counters;
};

struct StepAttnArgs {
  SeqView v;
  const AttnPiece *pieces;
  int n_pieces;
  const _Float16 *q;  // [rows][n_head][head_dim]
  _Float16 *out;
  int n_head, n_head_kv, head_dim;
  int heads;  // KV heads of a workgroup
  Join join;
};
int32_t launch_cache_attention(const StepAttnArgs &c, int row_tiles, const uint8_t *k_cache, const uint8_t *v_cache, hipStream_t s);
// kv: where each sequence's f16 keys and values lie in k and v ([rows][n_head_kv][head_dim]).
// k_rest: what the keys' rounding to f16 dropped, or null: the keys are f16 numbers.
int32_t launch_row_attention(const StepAttnArgs &c, const SeqKv *kv, const _Float16 *k, const _Float16 *k_rest,
                             const _Float16 *v, hipStream_t s);

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) short4v lds_short4;

constexpr float kLazy = 8.0f;  // log2 growth of the running max before O is rescaled

__device__ __forceinline__ half2v as_h2(uint32_t v) { return __builtin_bit_cast(half2v, v); }

// Device-scope (sc1) stores and loads: past this XCD's L2 cache, where the other XCDs see them.
// (An acquire fence before plain loads empties the cache instead, and took 6 to 17 us.)
__device__ __forceinline__ void st_dev(float2 *p, float2 v) {
  __hip_atomic_store(reinterpret_cast<uint64_t *>(p), __builtin_bit_cast(uint64_t, v), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ float2 ld_dev(const float2 *p) {
  return __builtin_bit_cast(float2, __hip_atomic_load(reinterpret_cast<uint64_t *>(const_cast<float2 *>(p)),
                                                      __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}
// The store of four floats at a 16-byte aligned address; whoever waits for it waits for vmcnt.
__device__ __forceinline__ void st_dev4(float *p, floatx4 v) {
  asm volatile("global_store_dwordx4 %0, %1, off sc1" : : "v"(p), "v"(v) : "memory");
}

// max over lanes l and l ^ 32
__device__ __forceinline__ float half_swap_max(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}

// Eight keys of one dimension a lane (A operand of O^T += V^T P^T) from row-major f16 rows in
// LDS: the keys of rows p .. p + 3 and q .. q + 3 as the lanes' addresses name them.
__device__ __forceinline__ half8 read_tr(const char *p, const char *q) {
  const short4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)p);
  const short4v y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)q);
  const short8v z = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_bit_cast(half8, z);
}

// After a workgroup stored its piece's records: whether it is the tile's last one (for head
// group `group`). Every thread of the workgroup calls it.
__device__ __forceinline__ bool arrived_last(const Join &j, const AttnPiece &pc, int group, int *shared) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the device-scope stores are acknowledged
  __syncthreads();
  if (threadIdx.x == 0) {
    int *ctr = j.counters + pc.counter + group;
    const int prev = __hip_atomic_fetch_add(ctr, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *shared = prev == pc.n_pieces - 1;
    if (*shared) __hip_atomic_store(ctr, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next call
  }
  __syncthreads();
  return *shared;
}

// Joins the pieces of a row tile for heads KV heads from head0 on, in piece order: four values
// of one (head, row) a job, kJobs jobs of a thread at a time with kPieces pieces' loads of each in
// flight. out: the sequence's first row.
template <int HD, int THREADS>
__device__ __forceinline__ void join_pieces(const Join &j, const AttnPiece &pc, int head0, int heads, int live,
                                            int n_head, int n_head_kv, _Float16 *out) {
  constexpr int kJobs = 2, kPieces = 8;
  const int G = n_head / n_head_kv, jobs = heads * live * (HD / 4);
  const size_t stride = (size_t)n_head_kv * live;
  for (int job0 = threadIdx.x; job0 < jobs; job0 += THREADS * kJobs) {
    float m[kJobs], l[kJobs];
    float4 acc[kJobs];
    size_t r0[kJobs];
#pragma unroll
    for (int x = 0; x < kJobs; x++) {
      m[x] = -INFINITY;
      l[x] = 0.0f;
      acc[x] = float4{0.0f, 0.0f, 0.0f, 0.0f};
      r0[x] = (size_t)pc.rec + (size_t)head0 * live + min(job0 + x * THREADS, jobs - 1) / (HD / 4);  // (head, row)
    }
    const int e = job0 % (HD / 4);  // the same for all: THREADS is a multiple
    static_assert(THREADS % (HD / 4) == 0, "jobs of a thread are at one place of their rows");
    for (int p0 = 0; p0 < pc.n_pieces; p0 += kPieces) {
      float2 ml[kJobs][kPieces];
      float4 v[kJobs][kPieces];
#pragma unroll
      for (int x = 0; x < kJobs; x++)
#pragma unroll
        for (int b = 0; b < kPieces; b++) {
          const size_t rr = r0[x] + min(p0 + b, pc.n_pieces - 1) * stride;
          ml[x][b] = ld_dev(j.ml + rr);
          const float2 *o = reinterpret_cast<const float2 *>(j.o + rr * HD) + 2 * e;
          const float2 o0 = ld_dev(o), o1 = ld_dev(o + 1);
          v[x][b] = float4{o0.x, o0.y, o1.x, o1.y};
        }
#pragma unroll
      for (int x = 0; x < kJobs; x++) {
        float mn = m[x];
#pragma unroll
        for (int b = 0; b < kPieces; b++) mn = fmaxf(mn, ml[x][b].x);
        const float ms = mn == -INFINITY ? 0.0f : mn;
        const float old = __builtin_amdgcn_exp2f(m[x] - ms);
        m[x] = mn;
        l[x] *= old;
        acc[x].x *= old;
        acc[x].y *= old;
        acc[x].z *= old;
        acc[x].w *= old;
#pragma unroll
        for (int b = 0; b < kPieces; b++) {
          if (p0 + b >= pc.n_pieces) continue;
          const float w = __builtin_amdgcn_exp2f(ml[x][b].x - ms);
          l[x] += ml[x][b].y * w;
          acc[x].x += v[x][b].x * w;
          acc[x].y += v[x][b].y * w;
          acc[x].z += v[x][b].z * w;
          acc[x].w += v[x][b].w * w;
        }
      }
    }
#pragma unroll
    for (int x = 0; x < kJobs; x++) {
      const int job = job0 + x * THREADS;
      if (job >= jobs) continue;
      const float inv = 1.0f / l[x];
      const int hr = job / (HD / 4), row = pc.row0 + hr % live;
      const int t = row / G, head = (head0 + hr / live) * G + row % G;
      *reinterpret_cast<half4 *>(out + ((size_t)t * n_head + head) * HD + 4 * e) = half4{
          (_Float16)(acc[x].x * inv), (_Float16)(acc[x].y * inv), (_Float16)(acc[x].z * inv), (_Float16)(acc[x].w * inv)};
    }
  }
}

}  // namespace
}  // namespace sulimo
