// paged_cache.hip - a step's keys and values into the pages of the Q8_0 cache, and back.
//
// Block of 32 values x: d = max|x| / 127, scale f16(d), code = round(x * (1 / d)) halves away
// from zero, in -128 .. 127 (quantize_f32_to_q8_0, crates/sulimo-core/src/kv_cache.rs:162-193:
// the ring's bytes, so a page can be copied to and from the host cache); it stands for
// code * f16(d). Both kernels move bytes: 2 read and 34/32 written per value, or the reverse,
// and 2 more per value where the store also hands back what the cache now stands for.
//
// A thread takes 16 values, four threads the 68 bytes of two blocks:
//   dword  0: d0 and codes 0, 1     1 .. 7: codes 2 .. 29     8: codes 30, 31 and d1
//   dwords 9 .. 16: codes of the second block
// so every access is a whole dword at a 4-byte aligned address: the halves that neighbours
// share pass between lanes.
#include "seq_batch.h"

namespace sulimo {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
// four dwords at any 4-byte aligned address
typedef uint32_t u32x4a4 __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ uint32_t pack4(const float *c) {
  uint32_t r = 0;
#pragma unroll
  for (int e = 0; e < 4; e++) r |= (uint32_t)(uint8_t)(int8_t)(int)c[e] << (8 * e);
  return r;
}

// grid.x covers rows * width / 16 threads, grid.y: keys, values
__global__ __launch_bounds__(256) void kv_store_paged_kernel(const int32_t *row_slot, int rows, int width,
                                                             const _Float16 *k, const _Float16 *v, uint8_t *k_cache,
                                                             uint8_t *v_cache, _Float16 *k_values, _Float16 *v_values) {
  const _Float16 *src = blockIdx.y ? v : k;
  uint8_t *cache = blockIdx.y ? v_cache : k_cache;
  _Float16 *values = blockIdx.y ? v_values : k_values;
  const uint32_t per_row = (uint32_t)width / 16;
  const uint64_t gid = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint64_t row64 = gid / per_row;
  // the four threads of a pair of blocks are in one row, and stay or leave together
  if (row64 >= (uint64_t)rows) return;
  const uint32_t part = (uint32_t)(gid - row64 * per_row);
  const _Float16 *x = src + row64 * width + part * 16;
  const half8 a = *reinterpret_cast<const half8 *>(x), b = *reinterpret_cast<const half8 *>(x + 8);
  float f[16];
#pragma unroll
  for (int e = 0; e < 8; e++) {
    f[e] = (float)a[e];
    f[8 + e] = (float)b[e];
  }
  float amax = fabsf(f[0]);  // (a block of nothing but NaN has a NaN scale, as in the ring)
#pragma unroll
  for (int e = 1; e < 16; e++) amax = fmaxf(amax, fabsf(f[e]));
  amax = fmaxf(amax, __shfl_xor(amax, 1, 64));
  const float d = amax / 127.0f;
  const float id = d != 0.0f ? 1.0f / d : 0.0f;
#pragma unroll
  for (int e = 0; e < 16; e++) f[e] = fminf(fmaxf(roundf(f[e] * id), -128.0f), 127.0f);
  const _Float16 dh = (_Float16)d;
  const uint32_t dbits = __builtin_bit_cast(uint16_t, dh);
  uint32_t c[4];
#pragma unroll
  for (int j = 0; j < 4; j++) c[j] = pack4(f + 4 * j);
  const uint32_t prev = __shfl_up(c[3], 1, 64);       // the 4 codes before this thread's
  const uint32_t next_d = __shfl_down(dbits, 1, 64);  // the next block's scale
  const int j = part & 3;
  // dword 0 of the pair of blocks
  uint32_t *dst = reinterpret_cast<uint32_t *>(cache + ((size_t)row_slot[row64] * (width / 32) + part / 2 - (j >> 1)) * 34);
  u32x4a4 o;
  if (j < 2) {
    o[0] = (j ? prev >> 16 : dbits) | c[0] << 16;
    o[1] = c[0] >> 16 | c[1] << 16;
    o[2] = c[1] >> 16 | c[2] << 16;
    o[3] = c[2] >> 16 | c[3] << 16;
    if (j) dst[8] = c[3] >> 16 | next_d << 16;
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = c[e];
  }
  *reinterpret_cast<u32x4a4 *>(dst + 4 * j + (j >> 1)) = o;
  if (values) {
    const float dv = (float)dh;
    half8 lo, hi;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      lo[e] = (_Float16)((f[e] + 0.0f) * dv);  // code 0 has no sign
      hi[e] = (_Float16)((f[8 + e] + 0.0f) * dv);
    }
    _Float16 *y = values + row64 * width + part * 16;
    *reinterpret_cast<half8 *>(y) = lo;
    *reinterpret_cast<half8 *>(y + 8) = hi;
  }
}

// grid.x: tiles of kLoadTile positions, grid.y: keys, values. The tile's cache rows are looked up
// once, and four loads of a thread are in flight at a time (one at a time, each behind its own
// look-up, read 12 conversations of 2000 to 8000 positions at 4.0 TB/s).
__global__ __launch_bounds__(256) void kv_load_paged_kernel(const LoadTile *tiles, const int32_t *pages, int page_size,
                                                            int width, const uint8_t *k_cache, const uint8_t *v_cache,
                                                            _Float16 *k_out, _Float16 *v_out, _Float16 *k_rest) {
  __shared__ uint32_t slots[kLoadTile];
  constexpr int kDeep = 4;
  const LoadTile t = tiles[blockIdx.x];
  const uint8_t *cache = blockIdx.y ? v_cache : k_cache;
  _Float16 *out = blockIdx.y ? v_out : k_out, *rest = blockIdx.y ? nullptr : k_rest;
  if ((int)threadIdx.x < t.count) {
    const uint32_t p = (uint32_t)t.pos + threadIdx.x, pg = p / (uint32_t)page_size;
    slots[threadIdx.x] = (uint32_t)pages[t.page_off + pg] * (uint32_t)page_size + (p - pg * (uint32_t)page_size);
  }
  __syncthreads();
  const uint32_t per_row = (uint32_t)width / 16, count = (uint32_t)t.count;
  const size_t row_bytes = (size_t)(width / 32) * 34;
  const uint32_t step_row = 256 / per_row, step_part = 256 % per_row;
  uint32_t row = threadIdx.x / per_row, part = threadIdx.x % per_row;
  // the four threads of a pair of blocks have one row, and end together
  for (;;) {
    uint32_t r[kDeep], pt[kDeep], mid[kDeep];
    u32x4a4 w[kDeep];
    if (row >= count) break;
#pragma unroll
    for (int e = 0; e < kDeep; e++) {
      r[e] = row;
      pt[e] = part;
      const int j = part & 3;
      const uint32_t *src = reinterpret_cast<const uint32_t *>(cache + slots[min(row, count - 1)] * row_bytes +
                                                               (size_t)(part / 2 - (j >> 1)) * 34);
      w[e] = *reinterpret_cast<const u32x4a4 *>(src + 4 * j + (j >> 1));
      mid[e] = src[8];
      row += step_row;
      part += step_part;
      if (part >= per_row) {
        part -= per_row;
        row++;
      }
    }
#pragma unroll
    for (int e = 0; e < kDeep; e++) {
      const int j = pt[e] & 3;
      const uint32_t next = __shfl_down(w[e][0], 1, 64);
      const uint32_t after = j ? mid[e] : next;  // dword 4 for the first thread, 8 for the second
      const uint32_t first = __shfl(w[e][0], (threadIdx.x & 63) & ~3, 64);
      const float d = (float)__builtin_bit_cast(_Float16, (uint16_t)(j < 2 ? first : mid[e] >> 16));
      uint32_t c[4];
      if (j < 2) {
        c[0] = w[e][0] >> 16 | w[e][1] << 16;
        c[1] = w[e][1] >> 16 | w[e][2] << 16;
        c[2] = w[e][2] >> 16 | w[e][3] << 16;
        c[3] = w[e][3] >> 16 | after << 16;
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++) c[i] = w[e][i];
      }
      half8 o[2], low[2];
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const float x = (float)(int8_t)(c[i >> 2] >> (8 * (i & 3))) * d;
        const _Float16 hi = (_Float16)x;
        o[i >> 3][i & 7] = hi;
        low[i >> 3][i & 7] = fabsf((float)hi) < INFINITY ? (_Float16)(x - (float)hi) : (_Float16)0.0f;
      }
      if (r[e] < count) {
        _Float16 *y = out + ((size_t)t.out_row + r[e]) * width + pt[e] * 16;
        *reinterpret_cast<half8 *>(y) = o[0];
        *reinterpret_cast<half8 *>(y + 8) = o[1];
        if (rest) {
          _Float16 *z = rest + (y - out);
          *reinterpret_cast<half8 *>(z) = low[0];
          *reinterpret_cast<half8 *>(z + 8) = low[1];
        }
      }
    }
  }
}

int32_t launched(const char *what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SULIMO_HIP_OK : hip_fail(e, what);
}

}  // namespace

int32_t launch_kv_store_paged(const SeqView &v, int width, const uint16_t *k, const uint16_t *vv, uint8_t *k_cache,
                              uint8_t *v_cache, uint16_t *k_values, uint16_t *v_values, hipStream_t s) {
  const size_t threads = (size_t)v.rows * (width / 16);
  hipLaunchKernelGGL(kv_store_paged_kernel, dim3((unsigned)((threads + 255) / 256), 2), dim3(256), 0, s, v.row_slot,
                     v.rows, width, reinterpret_cast<const _Float16 *>(k), reinterpret_cast<const _Float16 *>(vv),
                     k_cache, v_cache, reinterpret_cast<_Float16 *>(k_values), reinterpret_cast<_Float16 *>(v_values));
  return launched("kv_store_paged_kernel");
}

int32_t launch_kv_load_paged(const LoadTile *tiles, int n_tiles, const int32_t *pages, int page_size, int width,
                             const uint8_t *k_cache, const uint8_t *v_cache, uint16_t *k_out, uint16_t *v_out,
                             uint16_t *k_rest, hipStream_t s) {
  hipLaunchKernelGGL(kv_load_paged_kernel, dim3(n_tiles, 2), dim3(256), 0, s, tiles, pages, page_size, width, k_cache,
                     v_cache, reinterpret_cast<_Float16 *>(k_out), reinterpret_cast<_Float16 *>(v_out),
                     reinterpret_cast<_Float16 *>(k_rest));
  return launched("kv_load_paged_kernel");
}

}  // namespace sulimo
