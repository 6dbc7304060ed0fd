// attention_cache.hip - attention of a step's short runs of rows over the paged Q8_0 cache.
//
// Query row t of sequence s is position P = start[s] + t and sees positions
// max(0, P - window + 1) .. P of its own sequence (window 0: all):
//   out = sum_p softmax_p(q . K_p / sqrt(d)) V_p,   K, V = code * f16(scale).
// The work is the cache's bytes, 34 per 32 values and read once for all query heads of a KV
// head and all rows of a tile; 4 d flops per (row, key) are few next to them.
//
// A wave takes one KV head and 32 query rows (kCacheRows, rows past the sequence's are
// computed on and dropped) and runs over key tiles of 32 (head_dim 128) or 64 (64) positions:
//   - A lane loads 68 bytes, two Q8_0 blocks, as whole dwords (block pairs start at 4-byte
//     aligned addresses): half a key of 128, or a whole key of 64. The loads of the next tile
//     are issued before this one is computed, the page-table entries two tiles ahead and
//     before the loads, so that waiting for an entry does not wait for data behind it.
//   - Codes become f16 exactly: byte ^ 0x80 under the exponent of 1024 is 1152 + code; minus
//     1152, times the block's scale (one f16 rounding, as the ring's window has it).
//   - S^T = K Q^T by v_mfma_f32_32x32x16_f16 with K from registers as A; the contraction runs
//     over the head dimensions in whatever order the lanes hold them, and Q^T has the same.
//     (A 64-wide head: lane l holds key l, and lane halves exchange chunks so that either half
//     of the wave holds dimensions of the same 32 keys.)
//   - softmax: running max and sum per lane (a lane's scores belong to one row), the max moved
//     only when a tile exceeds it by 2^8 (P <= 256: exact to f16 precision), sums in f32.
//   - V goes through the wave's own LDS rows (f16, padded by 32 bytes: neither the writes nor the
//     reads meet in a bank) and comes back transposed by ds_read_tr16, 4 keys of one dimension
//     a lane: O^T += V^T P^T with P^T straight from the registers of S^T.
// Waves of a head add up through LDS; pieces of a row tile (several workgroups, few rows over
// a long cache) leave f32 records, and the workgroup that arrives last joins them in piece
// order, so the result does not depend on who that is.
#include <math.h>

#include "step_attn.h"

namespace sulimo {
namespace {

typedef uint32_t u32x4a4 __attribute__((ext_vector_type(4), aligned(4)));

struct CacheAttn {
  SeqView v;
  const AttnPiece *pieces;
  const _Float16 *q;  // [rows][n_head][HD]
  _Float16 *out;
  const uint8_t *k, *vc;  // the cache
  int n_head, n_head_kv;
  FastDiv page;
  Join join;
};

// A lane's two blocks of one key: dwords 0 .. 16 from the pair's start.
struct Raw {
  uint32_t w[17];
};
__device__ __forceinline__ Raw load_raw(const uint8_t *p) {
  Raw r;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const u32x4a4 v = *reinterpret_cast<const u32x4a4 *>(p + 16 * i);
#pragma unroll
    for (int e = 0; e < 4; e++) r.w[4 * i + e] = v[e];
  }
  r.w[16] = *reinterpret_cast<const uint32_t *>(p + 64);
  return r;
}
// Codes 8c .. 8c + 7 of the 64 as f16(code * scale); codes in the sign-flipped form.
template <int C>
__device__ __forceinline__ half8 chunk(const uint32_t (&x)[17], half2v d0, half2v d1) {
  const half2v off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
  const half2v d = C < 4 ? d0 : d1;
  half8 o;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    // halfword of the pair: block 0's codes start at halfword 1, block 1's at 18
    const int h = C < 4 ? 1 + 4 * C + e : 18 + 4 * (C - 4) + e;
    const half2v v = (as_h2(__builtin_amdgcn_perm(0x64646464u, x[h >> 1], h & 1 ? 0x04030402u : 0x04010400u)) + off) * d;
    o[2 * e] = v[0];
    o[2 * e + 1] = v[1];
  }
  return o;
}

template <int HD>
__global__ __launch_bounds__(512, 2) void cache_attn_kernel(CacheAttn a) {
  constexpr int KT = HD == 128 ? 32 : 64, NS = KT / 32;  // keys of a tile, S^T tiles
  constexpr int OT = HD / 32, QS = HD / 16;
  constexpr int ROW = HD * 2 + 32, WB = KT * ROW;        // LDS bytes of a V row and of a wave
  static_assert(WB >= 4096, "a wave's LDS also passes one O^T tile");
  __shared__ __attribute__((aligned(16))) char lds[kCacheWaves][WB];
  __shared__ float2 lml[kCacheWaves][32];
  __shared__ int last_one;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l32 = lane & 31, lg = lane >> 5;
  const AttnPiece pc = a.pieces[blockIdx.x];
  const int heads = a.n_head_kv % 8 == 0 ? 8 : a.n_head_kv % 4 == 0 ? 4 : a.n_head_kv % 2 == 0 ? 2 : 1;
  const int sub = kCacheWaves / heads;
  const int kvh = blockIdx.y * heads + wave / sub, sw = wave % sub;
  const int G = a.n_head / a.n_head_kv;
  const int off = a.v.off[pc.seq], n = a.v.off[pc.seq + 1] - off, start = a.v.start[pc.seq];
  const int live = min(kCacheRows, n * G - pc.row0);
  const int r = pc.row0 + min(l32, live - 1);  // dead rows repeat the last one
  const int t = r / G, h = kvh * G + r % G;
  const int P = start + t, Pmin = start + pc.row0 / G, Pmax = start + (pc.row0 + live - 1) / G;
  const int win = a.v.window ? a.v.window : INT_MAX;
  const float c = 1.4426950408889634f / sqrtf((float)HD);

  // Q^T (B operand) in the lanes' order of dimensions
  half8 qf[QS];
  {
    const _Float16 *src = a.q + ((size_t)(off + t) * a.n_head + h) * HD;
#pragma unroll
    for (int s = 0; s < QS; s++) qf[s] = *reinterpret_cast<const half8 *>(src + (HD == 128 ? 64 * lg + 8 * s : 16 * s + 8 * lg));
  }

  const int32_t *table = a.v.pages + a.v.page_off[pc.seq];
  const uint32_t row_bytes = (uint32_t)a.n_head_kv * (HD / 32) * 34;
  const uint32_t col = (uint32_t)kvh * (HD / 32) * 34 + (HD == 128 ? 68 * lg : 0);
  const int klane = HD == 128 ? l32 : lane;  // the tile's key of this lane
  auto page_of = [&](int tile, uint32_t *in_page) __attribute__((always_inline)) {
    const uint32_t p = (uint32_t)min(tile * KT + klane, Pmax);  // tiles end inside a page or past the last position
    const uint32_t pg = (uint32_t)((uint64_t)p * a.page.magic >> a.page.shift);
    *in_page = p - pg * a.page.d;
    return table[pg];
  };

  floatx16 o[OT];
#pragma unroll
  for (int i = 0; i < OT; i++) o[i] = floatx16{};
  float mrun = -INFINITY, lrun = 0.0f;
  char *vrow = lds[wave] + klane * ROW + (HD == 128 ? 128 * lg : 0);
  const char *vread = lds[wave] + (4 * lg + ((lane & 15) >> 2)) * ROW + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);

  auto compute = [&](const Raw &kr, const Raw &vr, int tile) __attribute__((always_inline)) {
    const int k0 = tile * KT;
    const bool masked = k0 + KT - 1 > Pmin || k0 <= Pmax - win;
    // S^T
    floatx16 st[NS];
    {
      uint32_t x[17];
#pragma unroll
      for (int i = 0; i < 17; i++) x[i] = kr.w[i] ^ 0x80808080u;
      const half2v d0 = as_h2(__builtin_amdgcn_perm(kr.w[0], kr.w[0], 0x01000100u));
      const half2v d1 = as_h2(__builtin_amdgcn_perm(kr.w[8], kr.w[8], 0x03020302u));
      half8 f[8] = {chunk<0>(x, d0, d1), chunk<1>(x, d0, d1), chunk<2>(x, d0, d1), chunk<3>(x, d0, d1),
                    chunk<4>(x, d0, d1), chunk<5>(x, d0, d1), chunk<6>(x, d0, d1), chunk<7>(x, d0, d1)};
#pragma unroll
      for (int i = 0; i < NS; i++) st[i] = floatx16{};
      if constexpr (HD == 128) {
#pragma unroll
        for (int s = 0; s < QS; s++) st[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[s], qf[s], st[0], 0, 0, 0);
      } else {
#pragma unroll
        for (int s = 0; s < QS; s++) {
          typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
          u32x4 u = __builtin_bit_cast(u32x4, f[2 * s]), v = __builtin_bit_cast(u32x4, f[2 * s + 1]);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const auto w = __builtin_amdgcn_permlane32_swap(u[e], v[e], false, false);
            u[e] = w[0];
            v[e] = w[1];
          }
          st[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, u), qf[s], st[0], 0, 0, 0);
          st[NS - 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, v), qf[s], st[NS - 1], 0, 0, 0);
        }
      }
    }
    // V rows to LDS. A block whose scale is not finite makes every row that sees its key NaN;
    // in tiles where some rows do not, it is set to zero and the others are marked.
    half2v d0 = as_h2(__builtin_amdgcn_perm(vr.w[0], vr.w[0], 0x01000100u));
    half2v d1 = as_h2(__builtin_amdgcn_perm(vr.w[8], vr.w[8], 0x03020302u));
    uint64_t bad0 = 0, bad1 = 0;
    if (masked) {
      const bool b0 = (vr.w[0] & 0x7c00u) == 0x7c00u, b1 = (vr.w[8] & 0x7c000000u) == 0x7c000000u;
      bad0 = __ballot(b0);
      bad1 = __ballot(b1);
      if (b0) d0 = half2v{0, 0};
      if (b1) d1 = half2v{0, 0};
    }
    {
      uint32_t x[17];
#pragma unroll
      for (int i = 0; i < 17; i++) x[i] = vr.w[i] ^ 0x80808080u;
      half8 *dst = reinterpret_cast<half8 *>(vrow);
      dst[0] = chunk<0>(x, d0, d1);
      dst[1] = chunk<1>(x, d0, d1);
      dst[2] = chunk<2>(x, d0, d1);
      dst[3] = chunk<3>(x, d0, d1);
      dst[4] = chunk<4>(x, d0, d1);
      dst[5] = chunk<5>(x, d0, d1);
      dst[6] = chunk<6>(x, d0, d1);
      dst[7] = chunk<7>(x, d0, d1);
    }
    if (masked) {
#pragma unroll
      for (int i = 0; i < NS; i++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const int p = k0 + 32 * i + 8 * (e >> 2) + 4 * lg + (e & 3);
          st[i][e] = (p > P || p <= P - win) ? -INFINITY : st[i][e];
        }
    }
    // softmax
    float mt = -INFINITY;
#pragma unroll
    for (int i = 0; i < NS; i++)
#pragma unroll
      for (int e = 0; e < 16; e++) mt = fmaxf(mt, st[i][e]);
    mt = half_swap_max(mt) * c;
    const bool grow = mt > mrun + kLazy;
    const float alpha = grow && mrun != -INFINITY ? __builtin_amdgcn_exp2f(mrun - mt) : 1.0f;
    if (grow) mrun = mt;
    const float ms = mrun == -INFINITY ? 0.0f : mrun;  // no key seen yet: exp2(-inf) = 0
    half8 pf[2 * NS];
    const half2v one = {(_Float16)1.0f, (_Float16)1.0f};
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NS; i++)
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const half2v w = {(_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(st[i][e], c, -ms)),
                          (_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(st[i][e + 1], c, -ms))};
        sum = __builtin_amdgcn_fdot2(w, one, sum, false);  // the f16 weights the products use
        pf[2 * i + (e >> 3)][e & 7] = w[0];
        pf[2 * i + (e >> 3)][(e & 7) + 1] = w[1];
      }
    lrun = lrun * alpha + sum;
    if (__ballot(alpha != 1.0f)) {
#pragma unroll
      for (int i = 0; i < OT; i++) o[i] *= alpha;
    }
    // O^T += V^T P^T, 16 keys a step: registers 8 kk .. of S^T are keys 16 kk + {0-3, 8-11} + 4 lg
#pragma unroll
    for (int kk = 0; kk < KT / 16; kk++)
#pragma unroll
      for (int i = 0; i < OT; i++) {
        const char *src = vread + 16 * kk * ROW + 64 * i;
        o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(read_tr(src, src + 8 * ROW), pf[kk], o[i], 0, 0, 0);
      }
    if (masked && (bad0 | bad1)) {
      // keys of this tile that the row sees
      uint64_t sees = ~0ull;
      const int up = P - k0, dn = P - win < k0 ? 0 : P - win - k0 + 1;  // keys dn .. up
      sees = up < 0 ? 0 : up >= 63 ? sees : (2ull << up) - 1;
      sees = dn >= 64 ? 0 : sees & (~0ull << dn);
#pragma unroll
      for (int i = 0; i < OT; i++) {  // O^T tile i is block i of the head
        uint64_t b = (i & 1) ? bad1 : bad0;
        if constexpr (HD == 128) b = (uint32_t)(b >> (32 * (i >> 1)));
        const float x = (b & sees) ? __builtin_nanf("") : 0.0f;
#pragma unroll
        for (int e = 0; e < 16; e++) o[i][e] += x;
      }
    }
  };

  // key tiles tile0 + sw, + sub, ... of this wave
  {
    int tile = pc.tile0 + sw;
    const uint8_t *kb = a.k + col, *vb = a.vc + col;
    uint32_t in0, in1;
    int32_t pg0 = 0, pg1 = 0;
    Raw k0, v0, k1, v1;
    auto fetch = [&](Raw &k, Raw &v, int32_t pg, uint32_t in) __attribute__((always_inline)) {
      const size_t at = ((size_t)(uint32_t)pg * a.page.d + in) * row_bytes;
      k = load_raw(kb + at);
      v = load_raw(vb + at);
    };
    if (tile < pc.tile1) {
      pg0 = page_of(tile, &in0);
      pg1 = page_of(tile + sub, &in1);
      fetch(k0, v0, pg0, in0);
      for (;;) {
        // two tiles a turn, so that no register moves between the buffers
        pg0 = page_of(tile + 2 * sub, &in0);
        if (tile + sub < pc.tile1) fetch(k1, v1, pg1, in1);
        compute(k0, v0, tile);
        tile += sub;
        if (tile >= pc.tile1) break;
        pg1 = page_of(tile + 2 * sub, &in1);
        if (tile + sub < pc.tile1) fetch(k0, v0, pg0, in0);
        compute(k1, v1, tile);
        tile += sub;
        if (tile >= pc.tile1) break;
      }
    }
  }

  // ---- the waves of a head: joint max and sum, then O^T tile by tile ----
  lrun += __shfl_xor(lrun, 32, 64);  // lane halves hold different keys
  const int w0 = wave - sw;
  float M = mrun;
  if (sub > 1) {
    if (lg == 0) lml[wave][l32] = float2{mrun, lrun};
    __syncthreads();
    float L = 0.0f;
    for (int j = 0; j < sub; j++) M = fmaxf(M, lml[w0 + j][l32].x);
    const float Ms = M == -INFINITY ? 0.0f : M;
    for (int j = 0; j < sub; j++) L += lml[w0 + j][l32].y * __builtin_amdgcn_exp2f(lml[w0 + j][l32].x - Ms);
    const float mine = __builtin_amdgcn_exp2f(mrun - Ms);
    lrun = L;
    // O^T tile i is added up by wave i mod sub of the head, into its o[i]
#pragma unroll
    for (int i = 0; i < OT; i++) {
      float4 *dst = reinterpret_cast<float4 *>(lds[wave]) + lane;
#pragma unroll
      for (int g = 0; g < 4; g++)
        dst[64 * g] = float4{o[i][4 * g] * mine, o[i][4 * g + 1] * mine, o[i][4 * g + 2] * mine, o[i][4 * g + 3] * mine};
      __syncthreads();
      if (i % sub == sw) {
        floatx16 acc{};
        for (int j = 0; j < sub; j++) {
          const float4 *src = reinterpret_cast<const float4 *>(lds[w0 + j]) + lane;
#pragma unroll
          for (int g = 0; g < 4; g++) {
            const float4 x = src[64 * g];
            acc[4 * g] += x.x;
            acc[4 * g + 1] += x.y;
            acc[4 * g + 2] += x.z;
            acc[4 * g + 3] += x.w;
          }
        }
        o[i] = acc;
      }
      __syncthreads();
    }
  }

  if (pc.n_pieces == 1) {
    if (l32 >= live) return;
    const float inv = 1.0f / lrun;
    _Float16 *dst = a.out + ((size_t)(off + t) * a.n_head + h) * HD + 4 * lg;
#pragma unroll
    for (int i = 0; i < OT; i++)
      if (i % sub == sw) {
#pragma unroll
        for (int g = 0; g < 4; g++)
          *reinterpret_cast<half4 *>(dst + 32 * i + 8 * g) =
              half4{(_Float16)(o[i][4 * g] * inv), (_Float16)(o[i][4 * g + 1] * inv), (_Float16)(o[i][4 * g + 2] * inv),
                    (_Float16)(o[i][4 * g + 3] * inv)};
      }
    return;
  }

  if (l32 < live) {
    const size_t rr = (size_t)pc.rec + ((size_t)pc.piece * a.n_head_kv + kvh) * live + l32;
    if (sw == 0 && lg == 0) st_dev(a.join.ml + rr, float2{M, lrun});
#pragma unroll
    for (int i = 0; i < OT; i++)
      if (i % sub == sw) record_tile<HD>(a.join, rr, i, lg, o[i]);
  }
  if (!arrived_last(a.join, pc, blockIdx.y, &last_one)) return;
  join_pieces<HD, 512>(a.join, pc, blockIdx.y * heads, heads, live, a.n_head, a.n_head_kv, a.out + (size_t)off * a.n_head * HD);
}

}  // namespace

int32_t launch_cache_attention(const StepAttnArgs &c, const uint8_t *k_cache, const uint8_t *v_cache, hipStream_t s) {
  CacheAttn a{c.v, c.pieces, c.q, c.out, k_cache, v_cache, c.n_head, c.n_head_kv, fast_div((uint32_t)c.v.page_size),
              c.join};
  const dim3 grid(c.n_pieces, c.n_head_kv / cache_heads(c.n_head_kv));
  if (c.head_dim == 64) hipLaunchKernelGGL((cache_attn_kernel<64>), grid, dim3(512), 0, s, a);
  else hipLaunchKernelGGL((cache_attn_kernel<128>), grid, dim3(512), 0, s, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SULIMO_HIP_OK : hip_fail(e, "cache_attn_kernel launch");
}

}  // namespace sulimo
