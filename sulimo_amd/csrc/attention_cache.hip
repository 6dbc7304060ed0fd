// attention_cache.hip - attention of a step's short runs of rows over the paged Q8_0 cache.
//
// Query row t of sequence s is position P = start[s] + t and sees positions
// max(0, P - window + 1) .. P of its own sequence (window 0: all):
//   out = sum_p softmax_p(q . K_p / sqrt(d)) V_p,   K, V = code * f16(scale).
// The work is the cache's bytes, 34 per 32 values and read once for all query heads of a KV
// head and all rows of a tile; 4 d flops per (row, key) are few next to them.
//
// A wave takes one KV head and RT tiles of 16 query rows (rows past the sequence's are computed
// on and dropped) and runs over key tiles of 32 (head_dim 128) or 64 (64) positions:
//   - The tile's rows of the head come as 8-byte units, consecutive lanes along a row: lanes that
//     each took their own key's bytes read at 4.0 to 4.4 TB/s (every load touched 64 lines),
//     this order at 5.3 to 5.7. They go through the wave's LDS, from where a lane takes blocks
//     of keys as whole dwords. K of the next tile and V of this one are in flight while the
//     other is worked on.
//   - Codes become f16 exactly: byte ^ 0x80 under the exponent of 1024 is 1152 + code; minus
//     1152, times the block's scale. For K what that rounding drops is kept as a second f16
//     operand and the weights are split in the same way, for the result's sake: the roundings of
//     K, V, weights and result would each add 2e-4 of the result, in squares; without the
//     first and third a result is as near to the 64-bit one as with f16 keys in hand.
//   - S^T = K Q^T by v_mfma_f32_16x16x32_f16 with K from registers as A: lane (r, g) holds a block
//     of key r (a 64-wide head: block g mod 2 of key r + 16 (g / 2), and lane halves exchange
//     chunks). The contraction runs over a block's dimensions in the order in which they lie
//     in dwords: blocks of odd number start in the middle of one, so theirs is rotated by two
//     (positions 2 .. 31, 0, 1 hold dimensions 0 .. 29, 30, 31), and Q^T has the same.
//   - softmax: running max and sum per lane (a lane's scores belong to one row), the max moved
//     only when a tile exceeds it by 2^8, sums in f32.
//   - V goes back to LDS as f16 rows (the same order of dimensions, padded so that neither the
//     writes nor the reads meet in a bank) and comes out transposed by ds_read_tr16, 4 keys of
//     one dimension a lane: O^T += V^T P^T with P^T straight from the registers of S^T.
// Waves of a head add up through LDS; pieces of a row tile (several workgroups, few rows over
// a long cache) leave f32 records, and the workgroup that arrives last joins them in piece
// order, so the result does not depend on who that is.
#include <math.h>

#include <type_traits>

#include "step_attn.h"

namespace sulimo {
namespace {

typedef uint32_t u32x2a4 __attribute__((ext_vector_type(2), aligned(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct CacheAttn {
  SeqView v;
  const AttnPiece *pieces;
  const _Float16 *q;  // [rows][n_head][HD]
  _Float16 *out;
  const uint8_t *k, *vc;  // the cache
  int n_head, n_head_kv, heads;  // heads: KV heads of a workgroup
  FastDiv page;
  Join join;
};

// A tile of the head's rows on its way to LDS: kUnits 8-byte units, unit 64 j + lane in register
// j. A row of 136 bytes is 17 units, one of 68 is 8 and a last one that repeats a dword.
constexpr int kUnits = 9;
template <int HD>
__device__ __forceinline__ void unit_of(int j, int lane, int *row, int *dword) {
  if constexpr (HD == 128) {
    const int e = min(64 * j + lane, 32 * 17 - 1);
    *row = e / 17;
    *dword = 2 * (e - 17 * *row);
  } else {
    const int e = 64 * j + lane;
    *row = e / 9;
    *dword = min(2 * (e - 9 * *row), 15);
  }
}
struct Raw {
  u32x2a4 u[kUnits];
};

// One Q8_0 block of a lane as it lies in dwords 0 .. 8 from its pair's start (even blocks) or
// from the dword that ends the one before (odd): codes with their sign bits flipped.
struct Block {
  uint32_t x[9], first;  // first: the dword whose high half is position pair 0
  half2v d;
};
// sel: where the scale is in dword 0
__device__ __forceinline__ Block load_block(const uint32_t *p, bool odd, uint32_t sel) {
  Block b;
#pragma unroll
  for (int i = 0; i < 9; i++) b.x[i] = p[i];
  b.d = as_h2(__builtin_amdgcn_perm(b.x[0], b.x[0], sel));
#pragma unroll
  for (int i = 0; i < 9; i++) b.x[i] ^= 0x80808080u;
  b.first = odd ? b.x[8] : b.x[0];
  return b;
}
// Positions 8c .. 8c + 7 as f16(code * scale); lo receives what that rounding dropped, exactly.
template <int C, bool LO>
__device__ __forceinline__ half8 chunk(const Block &b, half8 *lo = nullptr) {
  const half2v off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
  half8 o;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const int pair = 4 * C + e, h = pair + 1;  // pair j >= 1 is halfword j + 1
    const uint32_t w = pair ? b.x[h >> 1] : b.first;
    const half2v c = as_h2(__builtin_amdgcn_perm(0x64646464u, w, !pair || (h & 1) ? 0x04030402u : 0x04010400u)) + off;
    const half2v v = c * b.d;
    o[2 * e] = v[0];
    o[2 * e + 1] = v[1];
    if constexpr (LO) {
      const half2v r = __builtin_elementwise_fma(c, b.d, -v);
      (*lo)[2 * e] = r[0];
      (*lo)[2 * e + 1] = r[1];
    }
  }
  return o;
}
template <bool LO>
__device__ __forceinline__ void chunks(const Block &b, half8 (&hi)[4], half8 (&lo)[4]) {
  hi[0] = chunk<0, LO>(b, &lo[0]);
  hi[1] = chunk<1, LO>(b, &lo[1]);
  hi[2] = chunk<2, LO>(b, &lo[2]);
  hi[3] = chunk<3, LO>(b, &lo[3]);
}

// max over the four lanes r, r + 16, r + 32, r + 48
__device__ __forceinline__ float quad_max(float v) {
  v = half_swap_max(v);
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}

// RT: tiles of 16 rows a wave. WHOLE: tiles end inside no page.
template <int HD, int RT, bool WHOLE>
__global__ __launch_bounds__(64 * kCacheWaves, 2) void cache_attn_kernel(CacheAttn a) {
  constexpr int KT = HD == 128 ? 32 : 64, MT = KT / 16;  // keys of a tile, S^T tiles of 16 keys
  constexpr int OT = HD / 16;                            // O^T tiles of 16 dimensions
  constexpr int QS = HD / 32;                            // contraction steps of S^T
  constexpr int RD = HD == 128 ? 34 : 19;                // dwords of a raw row in LDS: reads of 32 lanes meet in no bank
  constexpr int ROW = HD == 128 ? 288 : 144;             // LDS bytes of a V row
  constexpr int OROW = HD + 4;                           // floats of a row of sums in LDS
  constexpr bool QLDS = RT > 1;  // Q^T of two row tiles is read from LDS: in registers, loads in flight would spill
  constexpr int WT = KT * ROW + (QLDS ? RT * QS * 1024 : 0);
  constexpr int WB = WT > 16 * RT * OROW * 4 ? WT : 16 * RT * OROW * 4;  // LDS bytes of a wave
  static_assert(KT * ROW >= KT * RD * 4 + 512, "a wave's LDS also holds raw rows");
  __shared__ __attribute__((aligned(16))) char lds[kCacheWaves][WB];
  __shared__ float2 lml[kCacheWaves][16 * RT];
  __shared__ int last_one;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const AttnPiece pc = a.pieces[blockIdx.x];
  const int heads = a.heads;
  const int sub = kCacheWaves / heads;
  const int kvh = blockIdx.y * heads + wave / sub, sw = wave % sub;
  const int G = a.n_head / a.n_head_kv;
  const int off = a.v.off[pc.seq], n = a.v.off[pc.seq + 1] - off, start = a.v.start[pc.seq];
  const int live = min(16 * RT, n * G - pc.row0);
  const int Pmin = start + pc.row0 / G, Pmax = start + (pc.row0 + live - 1) / G;
  const int win = a.v.window ? a.v.window : INT_MAX;
  const float c = 1.4426950408889634f / sqrtf((float)HD);
  const int blk = HD == 128 ? (g >> 1) | (g & 1) << 1 : g & 1;  // the lane's block of a head
  const bool odd = blk & 1;

  // Q^T (B operand) in the lanes' order of dimensions
  char *mine = lds[wave];
  half8 qf[RT][QS];
  auto q_at = [&](int x, int s) __attribute__((always_inline)) {
    return reinterpret_cast<half8 *>(mine + KT * ROW + (x * QS + s) * 1024) + lane;
  };
  int P[RT];
#pragma unroll
  for (int x = 0; x < RT; x++) {
    const int r = pc.row0 + min(16 * x + r16, live - 1);  // dead rows repeat the last one
    const int t = r / G;
    P[x] = start + t;
    // the block's 16 dimension pairs, turned by one where positions are
    const u32x4 *q = reinterpret_cast<const u32x4 *>(a.q + ((size_t)(off + t) * a.n_head + kvh * G + r % G) * HD + 32 * blk);
    const u32x4 n0 = q[0], n1 = q[1], n2 = q[2], n3 = q[3];
    const uint32_t n[16] = {n0[0], n0[1], n0[2], n0[3], n1[0], n1[1], n1[2], n1[3],
                            n2[0], n2[1], n2[2], n2[3], n3[0], n3[1], n3[2], n3[3]};
#pragma unroll
    for (int s = 0; s < QS; s++) {
      u32x4 y;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        auto pair = [&](int j) { return odd ? n[(j + 15) & 15] : n[j]; };
        if constexpr (HD == 128) y[e] = pair(4 * s + e);
        else y[e] = g >> 1 ? pair(8 * s + 4 + e) : pair(8 * s + e);
      }
      qf[x][s] = __builtin_bit_cast(half8, y);
      if constexpr (QLDS) *q_at(x, s) = qf[x][s];
    }
  }

  const int32_t *table = a.v.pages + a.v.page_off[pc.seq];
  const uint32_t row_bytes = (uint32_t)a.n_head_kv * (HD / 32) * 34;
  const uint32_t col = (uint32_t)kvh * (HD / 32) * 34;
  // Where a tile lies: WHOLE, its first byte; else the cache row of each lane's key. Keys past
  // the last position stand for it.
  struct Place {
    size_t at;
    uint32_t slot;
  };
  auto place = [&](int tile) __attribute__((always_inline)) {
    Place w{};
    if constexpr (WHOLE) {
      const uint32_t p = (uint32_t)min(tile * KT, Pmax), pg = (uint32_t)((uint64_t)p * a.page.magic >> a.page.shift);
      const uint32_t slot = __builtin_amdgcn_readfirstlane((uint32_t)table[pg] * a.page.d + (p - pg * a.page.d));
      w.at = (size_t)slot * row_bytes + col;
    } else {
      const uint32_t p = (uint32_t)min(tile * KT + (lane & (KT - 1)), Pmax);
      const uint32_t pg = (uint32_t)((uint64_t)p * a.page.magic >> a.page.shift);
      w.slot = (uint32_t)table[pg] * a.page.d + (p - pg * a.page.d);
    }
    return w;
  };
  auto fetch = [&](const uint8_t *cache, const Place &w, Raw &x) __attribute__((always_inline)) {
    int lane = tid & 63;
    if constexpr (!WHOLE || RT > 1) asm volatile("" : "+v"(lane));  // the units' rows and offsets are not worth 18 registers
#pragma unroll
    for (int j = 0; j < kUnits; j++) {
      int row, dw;
      unit_of<HD>(j, lane, &row, &dw);
      if constexpr (WHOLE) {
        x.u[j] = *reinterpret_cast<const u32x2a4 *>((cache + w.at) + ((uint32_t)row * row_bytes + 4 * dw));
      } else {
        const size_t o = (size_t)(uint32_t)__shfl((int)w.slot, row, 64) * row_bytes + (col + 4 * dw);
        x.u[j] = *reinterpret_cast<const u32x2a4 *>(cache + o);
      }
    }
  };
  auto stage = [&](const Raw &x) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kUnits; j++) {
      if constexpr (HD == 128) {  // rows back to back: unit e at 8 e (the lanes past the last unit write behind it)
        reinterpret_cast<u32x2a4 *>(mine)[64 * j + lane] = x.u[j];
      } else {
        int row, dw;
        unit_of<HD>(j, lane, &row, &dw);
        *reinterpret_cast<u32x2a4 *>(reinterpret_cast<uint32_t *>(mine) + row * RD + dw) = x.u[j];
      }
    }
  };
  // the lane's two keys of a tile: key0, and key0 + step
  const int key0 = HD == 128 ? r16 : 16 * (g >> 1) + r16;
  constexpr int kStep = HD == 128 ? 16 : 32;
  const uint32_t *blk0 = reinterpret_cast<const uint32_t *>(mine) + key0 * RD + 17 * (blk >> 1) + 8 * (blk & 1);
  const uint32_t scale_sel = odd ? 0x03020302u : 0x01000100u;
  char *vrow = mine + key0 * ROW + 64 * blk;
  const char *vread = mine + (4 * g + (r16 >> 2)) * ROW + 8 * (r16 & 3);

  floatx4 o[RT][OT];
  float mrun[RT], lrun[RT];
#pragma unroll
  for (int x = 0; x < RT; x++) {
#pragma unroll
    for (int i = 0; i < OT; i++) o[x][i] = floatx4{};
    mrun[x] = -INFINITY;
    lrun[x] = 0.0f;
  }

  half8 pf[RT][KT / 32], pl[RT][KT / 32];  // the tile's weights, and what their rounding dropped
  // S^T of the K rows in LDS, and the weights
  auto scores = [&](int tile) __attribute__((always_inline)) {
    const int k0 = tile * KT;
    floatx4 st[RT][MT];
#pragma unroll
    for (int x = 0; x < RT; x++)
#pragma unroll
      for (int m = 0; m < MT; m++) st[x][m] = floatx4{};
    auto product = [&](half8 k, int s, int m) __attribute__((always_inline)) {
#pragma unroll
      for (int x = 0; x < RT; x++)
        st[x][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, QLDS ? *q_at(x, s) : qf[x][s], st[x][m], 0, 0, 0);
    };
#pragma unroll
    for (int u = 0; u < 2; u++) {
      half8 hi[4], lo[4];
      chunks<true>(load_block(blk0 + u * kStep * RD, odd, scale_sel), hi, lo);
      if constexpr (HD == 128) {
#pragma unroll
        for (int s = 0; s < QS; s++) {
          product(hi[s], s, u);
          product(lo[s], s, u);
        }
      } else {
        auto both = [&](half8 p, half8 q, int s) __attribute__((always_inline)) {
          u32x4 y = __builtin_bit_cast(u32x4, p), z = __builtin_bit_cast(u32x4, q);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const auto w = __builtin_amdgcn_permlane32_swap(y[e], z[e], false, false);
            y[e] = w[0];
            z[e] = w[1];
          }
          product(__builtin_bit_cast(half8, y), s, 2 * u);
          product(__builtin_bit_cast(half8, z), s, 2 * u + 1);
        };
#pragma unroll
        for (int s = 0; s < QS; s++) {
          both(hi[2 * s], hi[2 * s + 1], s);
          both(lo[2 * s], lo[2 * s + 1], s);
        }
      }
    }
    if (k0 + KT - 1 > Pmin || k0 <= Pmax - win) {
#pragma unroll
      for (int x = 0; x < RT; x++)
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int p = k0 + 16 * m + 4 * g + e;
            st[x][m][e] = (p > P[x] || p <= P[x] - win) ? -INFINITY : st[x][m][e];
          }
    }
#pragma unroll
    for (int x = 0; x < RT; x++) {
      float mt = -INFINITY;
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int e = 0; e < 4; e++) mt = fmaxf(mt, st[x][m][e]);
      mt = quad_max(mt) * c;
      const bool grow = mt > mrun[x] + kLazy;
      const float alpha = grow && mrun[x] != -INFINITY ? __builtin_amdgcn_exp2f(mrun[x] - mt) : 1.0f;
      if (grow) mrun[x] = mt;
      const float ms = mrun[x] == -INFINITY ? 0.0f : mrun[x];  // no key seen yet: exp2(-inf) = 0
      float sum = 0.0f;
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(st[x][m][e], c, -ms));
          const _Float16 h = (_Float16)w;
          pf[x][m >> 1][4 * (m & 1) + e] = h;
          pl[x][m >> 1][4 * (m & 1) + e] = (_Float16)(w - (float)h);
          sum += w;
        }
      lrun[x] = lrun[x] * alpha + sum;
      if (__ballot(alpha != 1.0f)) {
#pragma unroll
        for (int i = 0; i < OT; i++) o[x][i] *= alpha;
      }
    }
  };
  // O^T += V^T P^T of the raw V rows in LDS, which become f16 rows there. A block whose scale is
  // not finite makes every row that sees its key NaN; in tiles that some rows do not see as a
  // whole, it is set to zero and the others are marked.
  auto values = [&](int tile) __attribute__((always_inline)) {
    const int k0 = tile * KT;
    const bool masked = k0 + KT - 1 > Pmin || k0 <= Pmax - win;
    Block b0 = load_block(blk0, odd, scale_sel), b1 = load_block(blk0 + kStep * RD, odd, scale_sel);
    uint64_t bad0 = 0, bad1 = 0;
    if (masked) {
      auto off_scale = [](half2v d) { return (__builtin_bit_cast(uint32_t, d) & 0x7c00u) == 0x7c00u; };
      bad0 = __ballot(off_scale(b0.d));
      bad1 = __ballot(off_scale(b1.d));
      if (off_scale(b0.d)) b0.d = half2v{0, 0};
      if (off_scale(b1.d)) b1.d = half2v{0, 0};
    }
    half8 y[4], z[4], none[4];
    chunks<false>(b0, y, none);
    chunks<false>(b1, z, none);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      reinterpret_cast<half8 *>(vrow)[i] = y[i];
      reinterpret_cast<half8 *>(vrow + kStep * ROW)[i] = z[i];
    }
    // registers 4 m .. of S^T are keys 16 m + 4 g + {0-3}: a step takes m = 2 kk and 2 kk + 1
#pragma unroll
    for (int kk = 0; kk < KT / 32; kk++)
#pragma unroll
      for (int i = 0; i < OT; i++) {
        const char *src = vread + 32 * kk * ROW + 32 * i;
        const half8 vf = read_tr(src, src + 16 * ROW);
#pragma unroll
        for (int x = 0; x < RT; x++) {
          o[x][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[x][kk], o[x][i], 0, 0, 0);
          o[x][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[x][kk], o[x][i], 0, 0, 0);
        }
      }
    if (masked && (bad0 | bad1)) {
#pragma unroll
      for (int x = 0; x < RT; x++) {
        // keys of this tile that the row sees
        uint64_t sees = ~0ull;
        const int up = P[x] - k0, dn = P[x] - win < k0 ? 0 : P[x] - win - k0 + 1;  // keys dn .. up
        sees = up < 0 ? 0 : up >= 63 ? sees : (2ull << up) - 1;
        sees = dn >= 64 ? 0 : sees & (~0ull << dn);
#pragma unroll
        for (int i = 0; i < OT; i++) {  // block i / 2 of the head
          auto keys = [&](uint64_t bad, int at) { return (bad >> (16 * at)) & 0xffffull; };
          uint64_t b;
          constexpr int at[4] = {0, 2, 1, 3};  // the lanes of a block
          if constexpr (HD == 128) b = keys(bad0, at[i >> 1]) | keys(bad1, at[i >> 1]) << 16;
          else b = keys(bad0, i >> 1) | keys(bad0, 2 + (i >> 1)) << 16 | keys(bad1, i >> 1) << 32 | keys(bad1, 2 + (i >> 1)) << 48;
          const float nan = (b & sees) ? __builtin_nanf("") : 0.0f;
#pragma unroll
          for (int e = 0; e < 4; e++) o[x][i][e] += nan;
        }
      }
    }
  };

  // key tiles tile0 + sw, + sub, ... of this wave; the loads of a tile are issued as soon as the
  // registers of the one before are in LDS
  // (two row tiles leave registers for one of the two, so half a tile ahead)
  if (pc.tile0 + sw < pc.tile1) {
    Raw k, v;
    Place at = place(pc.tile0 + sw), next = place(pc.tile0 + sw + sub);
    fetch(a.k, at, k);
    if constexpr (RT == 1) fetch(a.vc, at, v);
    for (int tile = pc.tile0 + sw; tile < pc.tile1; tile += sub) {
      const bool more = tile + sub < pc.tile1;
      stage(k);
      if constexpr (RT > 1) fetch(a.vc, at, v);
      else if (more) fetch(a.k, next, k);
      scores(tile);
      stage(v);
      if (more) fetch(RT > 1 ? a.k : a.vc, next, RT > 1 ? k : v);
      at = next;
      next = place(tile + 2 * sub);
      values(tile);
    }
  }

  // ---- the waves of a head: sums of the live rows to LDS, [row][dimension] ----
  float *sums = reinterpret_cast<float *>(mine);
#pragma unroll
  for (int x = 0; x < RT; x++) {
    lrun[x] += __shfl_xor(lrun[x], 16, 64);  // lanes of a row hold different keys
    lrun[x] += __shfl_xor(lrun[x], 32, 64);
    if (16 * x + r16 >= live) continue;
    if (g == 0) lml[wave][16 * x + r16] = float2{mrun[x], lrun[x]};
#pragma unroll
    for (int i = 0; i < OT; i++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        // position pairs 2 g and 2 g + 1 (+ 8 for odd tiles) of block i / 2
        const int pair = (8 * (i & 1) + 2 * g + e + (i & 2 ? 15 : 0)) & 15;
        *reinterpret_cast<float2 *>(sums + (16 * x + r16) * OROW + 32 * (i >> 1) + 2 * pair) = float2{o[x][i][2 * e], o[x][i][2 * e + 1]};
      }
  }
  __syncthreads();
  // four dimensions of a row a thread
  const int w0 = wave - sw;
  auto add_up = [&](auto subs) __attribute__((always_inline)) {
    constexpr int SUB = decltype(subs)::value;
    for (int job = 64 * sw + lane; job < live * (HD / 4); job += 64 * SUB) {
      const int row = job / (HD / 4), d = 4 * (job % (HD / 4));
      float2 ml[SUB];
      floatx4 part[SUB];
#pragma unroll
      for (int j = 0; j < SUB; j++) {
        ml[j] = lml[w0 + j][row];
        part[j] = *reinterpret_cast<const floatx4 *>(reinterpret_cast<const float *>(lds[w0 + j]) + row * OROW + d);
      }
      float m = ml[0].x, l = 0.0f;
#pragma unroll
      for (int j = 1; j < SUB; j++) m = fmaxf(m, ml[j].x);
      const float ms = m == -INFINITY ? 0.0f : m;
      floatx4 acc{};
#pragma unroll
      for (int j = 0; j < SUB; j++) {
        const float f = __builtin_amdgcn_exp2f(ml[j].x - ms);
        l += ml[j].y * f;
        acc += part[j] * f;
      }
      if (pc.n_pieces == 1) {
        const int r = pc.row0 + row;
        const float inv = 1.0f / l;
        *reinterpret_cast<half4 *>(a.out + ((size_t)(off + r / G) * a.n_head + kvh * G + r % G) * HD + d) =
            half4{(_Float16)(acc[0] * inv), (_Float16)(acc[1] * inv), (_Float16)(acc[2] * inv), (_Float16)(acc[3] * inv)};
      } else {
        const size_t rr = (size_t)pc.rec + ((size_t)pc.piece * a.n_head_kv + kvh) * live + row;
        st_dev4(a.join.o + rr * HD + d, acc);
        if (d == 0) st_dev(a.join.ml + rr, float2{m, l});
      }
    }
  };
  if (sub == 8) add_up(std::integral_constant<int, 8>{});
  else if (sub == 4) add_up(std::integral_constant<int, 4>{});
  else if (sub == 2) add_up(std::integral_constant<int, 2>{});
  else add_up(std::integral_constant<int, 1>{});
  if (pc.n_pieces > 1 && arrived_last(a.join, pc, blockIdx.y, &last_one))
    join_pieces<HD, 64 * kCacheWaves>(a.join, pc, blockIdx.y * heads, heads, live, a.n_head, a.n_head_kv,
                                      a.out + (size_t)off * a.n_head * HD);
}

template <int HD, int RT>
void launch(const CacheAttn &a, dim3 grid, hipStream_t s) {
  if (a.page.d % (HD == 128 ? 32 : 64) == 0) hipLaunchKernelGGL((cache_attn_kernel<HD, RT, true>), grid, dim3(64 * kCacheWaves), 0, s, a);
  else hipLaunchKernelGGL((cache_attn_kernel<HD, RT, false>), grid, dim3(64 * kCacheWaves), 0, s, a);
}

}  // namespace

int32_t launch_cache_attention(const StepAttnArgs &c, int row_tiles, const uint8_t *k_cache, const uint8_t *v_cache, hipStream_t s) {
  const CacheAttn a{c.v, c.pieces, c.q, c.out, k_cache, v_cache, c.n_head, c.n_head_kv, c.heads,
                    fast_div((uint32_t)c.v.page_size), c.join};
  const dim3 grid(c.n_pieces, c.n_head_kv / c.heads);
  if (c.head_dim == 64 && row_tiles == 1) launch<64, 1>(a, grid, s);
  else if (c.head_dim == 64) launch<64, 2>(a, grid, s);
  else if (row_tiles == 1) launch<128, 1>(a, grid, s);
  else launch<128, 2>(a, grid, s);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SULIMO_HIP_OK : hip_fail(e, "cache_attn_kernel launch");
}

}  // namespace sulimo
