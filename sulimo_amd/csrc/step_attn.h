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
  Join join;
};
int32_t launch_cache_attention(const StepAttnArgs &c, const uint8_t *k_cache, const uint8_t *v_cache, hipStream_t s);
// kv: where each sequence's f16 keys and values lie in k and v ([rows][n_head_kv][head_dim])
int32_t launch_row_attention(const StepAttnArgs &c, const SeqKv *kv, const _Float16 *k, const _Float16 *v, hipStream_t s);

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) short4v lds_short4;

constexpr float kLazy = 8.0f;  // log2 growth of the running max before O is rescaled

__device__ __forceinline__ half2v as_h2(uint32_t v) { return __builtin_bit_cast(half2v, v); }

// Device-scope (sc1) stores and loads: coherent across the XCDs' L2 caches by themselves.
__device__ __forceinline__ void st_dev(float2 *p, float2 v) {
  __hip_atomic_store(reinterpret_cast<uint64_t *>(p), __builtin_bit_cast(uint64_t, v), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 ld_dev(const float2 *p) {
  return __builtin_bit_cast(float2, __hip_atomic_load(reinterpret_cast<uint64_t *>(const_cast<float2 *>(p)),
                                                      __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
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

// O^T tile i (dimensions 32 i .. + 31) of a lane's row to record row rr.
template <int HD>
__device__ __forceinline__ void record_tile(const Join &j, size_t rr, int i, int lg, const floatx16 &o) {
  float2 *dst = reinterpret_cast<float2 *>(j.o + rr * HD) + 16 * i + 2 * lg;
#pragma unroll
  for (int g = 0; g < 4; g++) {
    st_dev(dst + 4 * g, float2{o[4 * g], o[4 * g + 1]});
    st_dev(dst + 4 * g + 1, float2{o[4 * g + 2], o[4 * g + 3]});
  }
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
// of one (head, row) a thread. out: the sequence's first row.
template <int HD, int THREADS>
__device__ __forceinline__ void join_pieces(const Join &j, const AttnPiece &pc, int head0, int heads, int live,
                                            int n_head, int n_head_kv, _Float16 *out) {
  const int G = n_head / n_head_kv, rows = heads * live;
  for (int job = threadIdx.x; job < rows * (HD / 4); job += THREADS) {
    const int hr = job / (HD / 4), e = job % (HD / 4);
    const int hh = head0 + hr / live, row = pc.row0 + hr % live;
    const size_t r0 = (size_t)pc.rec + (size_t)hh * live + hr % live, stride = (size_t)n_head_kv * live;
    float m = -INFINITY, l = 0.0f;
    float4 acc{0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int B = 8;  // pieces whose loads are in flight together
    for (int p0 = 0; p0 < pc.n_pieces; p0 += B) {
      float2 ml[B], x[B], y[B];
#pragma unroll
      for (int b = 0; b < B; b++) {
        const size_t rr = r0 + min(p0 + b, pc.n_pieces - 1) * stride;
        const float2 *src = reinterpret_cast<const float2 *>(j.o + rr * HD) + 2 * e;
        ml[b] = ld_dev(j.ml + rr);
        x[b] = ld_dev(src);
        y[b] = ld_dev(src + 1);
      }
      float mn = m;
#pragma unroll
      for (int b = 0; b < B; b++) mn = fmaxf(mn, ml[b].x);
      const float ms = mn == -INFINITY ? 0.0f : mn;
      const float old = __builtin_amdgcn_exp2f(m - ms);
      m = mn;
      l *= old;
      acc.x *= old;
      acc.y *= old;
      acc.z *= old;
      acc.w *= old;
#pragma unroll
      for (int b = 0; b < B; b++) {
        if (p0 + b >= pc.n_pieces) continue;
        const float w = __builtin_amdgcn_exp2f(ml[b].x - ms);
        l += ml[b].y * w;
        acc.x += x[b].x * w;
        acc.y += x[b].y * w;
        acc.z += y[b].x * w;
        acc.w += y[b].y * w;
      }
    }
    const float inv = 1.0f / l;
    const int t = row / G, head = hh * G + row % G;
    *reinterpret_cast<half4 *>(out + ((size_t)t * n_head + head) * HD + 4 * e) =
        half4{(_Float16)(acc.x * inv), (_Float16)(acc.y * inv), (_Float16)(acc.z * inv), (_Float16)(acc.w * inv)};
  }
}

}  // namespace
}  // namespace sulimo
