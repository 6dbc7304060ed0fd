// attention_rows.hip - causal grouped attention of many query rows over f16 keys and values.
//
// Whole prompts with their keys and values in hand, and the longer chunks of a step, whose part
// of the paged cache is read back first. Rows r = token * G + head of one KV head (G query heads
// share it), 128 of them (kRowTile) a workgroup of 4 waves, 32 a wave: tokens of all G heads
// together see nearly the same keys, so little of the causal corner is computed in vain. Key
// tiles of 64 (kRowKeys) stream into two LDS slots by buffer DMA, K one tile ahead of V:
//   S^T = K Q^T    v_mfma_f32_32x32x16_f16, K from LDS as A, Q^T in registers as B; a lane holds
//                  16 keys of one row, so the running max and sum are per lane;
//   O^T += V^T P^T V comes transposed out of its row-major tile by ds_read_tr16 as A, P^T is the
//                  registers of S^T.
// A step's 64 keys take each wave 1024 clocks of MFMA, about as many of softmax VALU and of LDS
// reads; the S MFMAs of a half tile and the PV MFMAs of the one before run under the softmax of
// the one between them. Both tiles are swizzled by 16-byte chunks where the DMA picks its
// source, so that neither the row reads of K nor the transposed reads of V meet in a bank.
//
// Measured: four prompts of 4096 tokens (24 heads over 8, 128 wide) 447 us, 923 TFLOP/s of the
// causal half, where a large f16 matrix product reaches 1205; eight of 560 to 2867 tokens 268 us.
// What bounds it: a 32-row wave reads 1 KiB of LDS for each MFMA, so at the full MFMA rate these
// reads alone would take all of the 128 bytes a clock; they, the DMA's writes and the softmax's
// VALU leave the MFMA units busy 45 % of the time. Waves of 64 rows read half as much, but need
// 485 registers and so stand alone on their SIMD: 542 us, the softmax's chains uncovered.
//
// EXACT, for keys read back from the Q8_0 cache: code * scale has up to 18 bits, so K and the
// weights come in two f16 parts each, and only values and results are rounded, as where few rows
// read the cache directly. One part each gave an rms error of 4.1e-4 of the result, two 2.9e-4
// (rounding the result alone: 2.1e-4), for twice the MFMAs, half again the LDS reads and 333
// registers, so that a workgroup of 128-wide heads has a CU alone: two chunks of 540 and 610 tokens
// behind 4200 and 4600 positions 115 and 178 us. Eight waves, each half of every key tile, spill
// their registers and take 20 us longer.
//
// Keys and values that are not finite: a masked score is replaced before the softmax, but a
// masked weight of 0 times such a value is not 0. A workgroup whose sums came out not finite
// therefore runs once more, slowly, with such values taken out of the tiles that the mask
// crosses and counted by MFMAs of their own for the rows that see them.
#include "step_attn.h"

namespace sulimo {
namespace {

typedef __attribute__((address_space(3))) void lds_void;
typedef __amdgpu_buffer_rsrc_t rsrc_t;
constexpr uint32_t kRsrcWord3 = 0x00020000u;

__device__ __forceinline__ void dma16(rsrc_t r, void *dst, uint32_t voff, uint32_t soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void *)dst, 16, (int)voff, (int)soff, 0, 0);
}
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | (0x7 << 4) | (0xF << 8));
}

struct RowAttn {
  StepAttnArgs s;
  const SeqKv *kv;
  const _Float16 *k, *k_rest, *v;
};

// Chunk c of V row `row` stands at chunk c ^ vswz(row): the 4 rows x 64 bytes that 32 lanes of a
// transposed read take are 8 different 32-byte segments of the banks.
template <int HD>
__device__ __forceinline__ int vswz(int row) {
  return HD == 128 ? 2 * (2 * (row & 3) + ((row >> 2) & 1)) : 2 * (2 * ((row >> 1) & 1) + ((row >> 2) & 1));
}

template <int HD, bool EXACT>
__global__ __launch_bounds__(256, EXACT && HD == 128 ? 1 : 2) void row_attn_kernel(RowAttn a) {
  constexpr int KS = HD / 16, OT = HD / 32, KCH = HD / 8;
  constexpr int ROWB = HD * 2, TILE = kRowKeys * ROWB;
  constexpr int RPI = 64 / KCH;             // rows per DMA instruction
  constexpr int NI = kRowKeys / RPI / 4;    // DMA instructions per wave and tile
  constexpr int REST = EXACT ? TILE : 16;
  constexpr int NK = EXACT ? 2 * NI : NI;   // of a K tile
  __shared__ __attribute__((aligned(16))) char ka[TILE], va[TILE], kb[TILE], vb[TILE], ra[REST], rb[REST];
  __shared__ int shared_flag;
  const int n_head_kv = a.s.n_head_kv, n_head = a.s.n_head, G = n_head / n_head_kv;
  const int kvh = blockIdx.x % n_head_kv;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l32 = lane & 31, lg = lane >> 5;
  const AttnPiece pc = a.s.pieces[blockIdx.x / n_head_kv];
  const SeqKv kv = a.kv[pc.seq];
  const int off = a.s.v.off[pc.seq], total = (a.s.v.off[pc.seq + 1] - off) * G, start = a.s.v.start[pc.seq];
  const int live = min(kRowTile, total - pc.row0);
  const int rw0 = 32 * wave;               // the wave's rows of the tile
  const bool wave_live = rw0 < live;
  const int wlive = wave_live ? min(32, live - rw0) : 1;
  const int rl = wave_live ? rw0 + min(l32, wlive - 1) : 0;  // dead rows repeat a live one
  const int r = pc.row0 + rl;
  const int t = r / G, h = kvh * G + r % G;
  const int P = start + t;
  const int Pmin = start + (pc.row0 + (wave_live ? rw0 : 0)) / G;
  const int Pmax = start + (pc.row0 + (wave_live ? rw0 + wlive - 1 : 0)) / G;
  const int win = a.s.v.window ? a.s.v.window : INT_MAX;
  const float c = 1.4426950408889634f / sqrtf((float)HD);

  half8 qf[KS];
  {
    const _Float16 *src = a.s.q + ((size_t)(off + t) * n_head + h) * HD + 8 * lg;
#pragma unroll
    for (int s = 0; s < KS; s++) qf[s] = *reinterpret_cast<const half8 *>(src + 16 * s);
  }

  // The sequence's rows of this KV head; rows past its end read as zero.
  const uint32_t stride = (uint32_t)n_head_kv * ROWB;
  const size_t base = ((size_t)kv.row0 * n_head_kv + kvh) * HD;
  const uint32_t bytes = (uint32_t)(kv.len - 1) * stride + ROWB;
  const rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(const_cast<_Float16 *>(a.k + base), (short)0, (int)bytes, (int)kRsrcWord3);
  const rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(const_cast<_Float16 *>(a.v + base), (short)0, (int)bytes, (int)kRsrcWord3);
  const rsrc_t rr = __builtin_amdgcn_make_buffer_rsrc(const_cast<_Float16 *>(EXACT ? a.k_rest + base : nullptr), (short)0,
                                                      EXACT ? (int)bytes : 0, (int)kRsrcWord3);
  uint32_t koff[NI], voff[NI];
#pragma unroll
  for (int i = 0; i < NI; i++) {
    const int row = RPI * (NI * wave + i) + lane / KCH, ch = lane % KCH;
    koff[i] = (uint32_t)row * stride + 16 * (ch ^ (row % KCH));
    voff[i] = (uint32_t)row * stride + 16 * (ch ^ vswz<HD>(row));
  }
  auto issue = [&](rsrc_t rs, const uint32_t (&o)[NI], char *dst, int tile) __attribute__((always_inline)) {
    // the tile's start goes into the lanes' offsets: the bounds check does not see the scalar one
    const uint32_t so = (uint32_t)(tile * kRowKeys - kv.lo) * stride;
#pragma unroll
    for (int i = 0; i < NI; i++) dma16(rs, dst + RPI * (NI * wave + i) * ROWB, o[i] + so, 0);
  };

  // K of a tile, and with EXACT what its rounding dropped
  struct KTile {
    char *k, *rest;
  };
  const KTile slot_a{ka, ra}, slot_b{kb, rb};
  auto issue_k = [&](const KTile &dst, int tile) __attribute__((always_inline)) {
    issue(rk, koff, dst.k, tile);
    if constexpr (EXACT) issue(rr, koff, dst.rest, tile);
  };
  // Weights of a half tile in f16, and with EXACT what that rounding dropped
  struct Weights {
    half8 p[2], rest[EXACT ? 2 : 1];
  };

  floatx16 o[OT];
  float mrun, lrun;
  auto reset = [&]() {
#pragma unroll
    for (int i = 0; i < OT; i++) o[i] = floatx16{};
    mrun = -INFINITY;
    lrun = 0.0f;
  };

  auto s_mfma = [&](const KTile &sk, int kt, int s, floatx16 &st) __attribute__((always_inline)) {
    const int row = 32 * kt + l32, at = row * ROWB + 16 * ((2 * s + lg) ^ (row % KCH));
    st = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const half8 *>(sk.k + at), qf[s], st, 0, 0, 0);
    if constexpr (EXACT)
      st = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const half8 *>(sk.rest + at), qf[s], st, 0, 0, 0);
  };
  // V^T fragment of dimensions 32 i .. and keys 32 kt + 16 j + {0-3, 8-11} + 4 lg
  const int vr = 4 * lg + ((lane & 15) >> 2), vc = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1), vb8 = 8 * (lane & 1);
  auto v_frag = [&](const char *sv, int kt, int j, int i) __attribute__((always_inline)) {
    // Rows 8 apart have the same swizzle. Constant parts stand on the tile and the lane's
    // part is added last: so the compiler sees which tile a read is in, and does not wait for the
    // DMA into the others.
    const int lane_at = vr * ROWB + 16 * ((4 * i + vc) ^ vswz<HD>(vr)) + vb8;
    const char *p = sv + (32 * kt + 16 * j) * ROWB, *q = p + 8 * ROWB;
    return read_tr(p + lane_at, q + lane_at);
  };
  auto add_values = [&](const half8 &vf, int j, int i, const Weights &w) __attribute__((always_inline)) {
    o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, w.p[j], o[i], 0, 0, 0);
    if constexpr (EXACT) o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, w.rest[j], o[i], 0, 0, 0);
  };
  auto pv_mfma = [&](const char *sv, int kt, int s, const Weights &w) __attribute__((always_inline)) {
    add_values(v_frag(sv, kt, s / OT, s % OT), s / OT, s % OT, w);
  };
  static_assert(2 * OT == KS, "a half tile's S and PV take equally many MFMAs");
  auto mask = [&](floatx16 &st, int p_reg0) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 16; e++) {
      const int p = p_reg0 + 8 * (e >> 2) + (e & 3);
      st[e] = (p > P || p <= P - win) ? -INFINITY : st[e];
    }
  };
  auto softmax = [&](const floatx16 &st, Weights &w) __attribute__((always_inline)) -> float {
    float mt = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; e++) mt = fmaxf(mt, st[e]);
    mt = half_swap_max(mt) * c;
    const bool grow = mt > mrun + kLazy;
    const float alpha = grow && mrun != -INFINITY ? __builtin_amdgcn_exp2f(mrun - mt) : 1.0f;
    if (grow) mrun = mt;
    const float ms = mrun == -INFINITY ? 0.0f : mrun;
    float sum = 0.0f;
    if constexpr (EXACT) {
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(st[e], c, -ms));
        const _Float16 hi = (_Float16)x;
        w.p[e >> 3][e & 7] = hi;
        w.rest[e >> 3][e & 7] = (_Float16)(x - (float)hi);
        sum += x;
      }
    } else {  // the sum of the weights as they are rounded: their common error cancels
#pragma unroll
      for (int e = 0; e < 16; e++) w.p[e >> 3][e & 7] = (_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(st[e], c, -ms));
      const half2v one = {(_Float16)1.0f, (_Float16)1.0f};
#pragma unroll
      for (int e = 0; e < 16; e += 2) sum = __builtin_amdgcn_fdot2(half2v{w.p[e >> 3][e & 7], w.p[e >> 3][(e & 7) + 1]}, one, sum, false);
    }
    lrun = lrun * alpha + sum;
    return alpha;
  };
  auto rescale = [&](float alpha) __attribute__((always_inline)) {
    if (__ballot(alpha != 1.0f)) {
#pragma unroll
      for (int i = 0; i < OT; i++) o[i] *= alpha;
    }
  };
  // The S^T MFMAs of half tile h+1 and the PV MFMAs of h-1 under the softmax of h.
  auto phase = [&](const KTile &sk, int kt, floatx16 &snext, const char *sv, int vt, const Weights &pp,
                   const floatx16 &scur, Weights &pc_) __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    snext = floatx16{};
#pragma unroll
    for (int s = 0; s < KS; s++) {
      s_mfma(sk, kt, s, snext);
      pv_mfma(sv, vt, s, pp);
    }
    const float alpha = softmax(scur, pc_);
    // LDS reads two pairs of steps ahead (1 of K, or 2, and 2 of V), the softmax's VALU between
    __builtin_amdgcn_sched_group_barrier(0x100, EXACT ? 8 : 6, 0);
#pragma unroll
    for (int k = 0; k < 2 * KS; k++) {
      if (EXACT) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
      if (k + 4 < 2 * KS) {
        if (EXACT || (k & 1)) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        else __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x002, EXACT ? 4 : 5, 0);  // VALU
    }
    if constexpr (EXACT)  // the compiler would move this phase's exponentials behind the next one's MFMAs
      asm volatile("" : "+v"(pc_.p[0]), "+v"(pc_.p[1]), "+v"(pc_.rest[0]), "+v"(pc_.rest[1]), "+v"(lrun));
    __builtin_amdgcn_sched_barrier(0);
    rescale(alpha);
  };

  const int tb = pc.tile0, steps = pc.tile1 - pc.tile0;
  auto visible = [&](int tile) {
    return tile < pc.tile1 && wave_live && tile * kRowKeys <= Pmax && tile * kRowKeys + kRowKeys - 1 > Pmin - win;
  };
  auto unmasked = [&](int tile) { return tile * kRowKeys + kRowKeys - 1 <= Pmin && tile * kRowKeys > Pmax - win; };

  auto fast = [&]() __attribute__((always_inline)) {
    floatx16 sa, sb;
    Weights pa, pb;
    auto first = [&](const KTile &sk, int tile) __attribute__((always_inline)) {  // S^T of both halves, P of the first
      sa = floatx16{};
      sb = floatx16{};
#pragma unroll
      for (int s = 0; s < KS; s++) s_mfma(sk, 0, s, sa);
#pragma unroll
      for (int s = 0; s < KS; s++) s_mfma(sk, 1, s, sb);
      if (!unmasked(tile)) mask(sa, tile * kRowKeys + 4 * lg);
      rescale(softmax(sa, pa));
    };
    auto last = [&](const char *sv, int tile) __attribute__((always_inline)) {  // PV of both halves
#pragma unroll
      for (int s = 0; s < KS; s++) pv_mfma(sv, 0, s, pa);
      if (!unmasked(tile)) mask(sb, tile * kRowKeys + 32 + 4 * lg);
      rescale(softmax(sb, pb));
#pragma unroll
      for (int s = 0; s < KS; s++) pv_mfma(sv, 1, s, pb);
    };
    auto both = [&](const KTile &sk, const char *sv, int tile) __attribute__((always_inline)) {
      const int p1 = tile * kRowKeys + 32 + 4 * lg;
      if (!unmasked(tile)) mask(sb, p1);
      phase(sk, 0, sa, sv, 0, pa, sb, pb);
      if (!unmasked(tile + 1)) mask(sa, p1 + 32);
      phase(sk, 1, sb, sv, 1, pb, sa, pa);
    };
    // At the start of step t the K tile of t + 1 and the V tile of t have landed, and every wave
    // is done with the slots that K of t + 2 and V of t + 1 go to.
    auto step = [&](const KTile &k_use, const KTile &k_next, char *v_use, char *v_next, int u) __attribute__((always_inline)) {
      __builtin_amdgcn_sched_barrier(0);
      wait_vmcnt<0>();
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      if (u + 2 < steps) issue_k(k_next, tb + u + 2);
      if (u + 1 < steps) issue(rv, voff, v_next, tb + u + 1);
      const int tile = tb + u;
      const bool more = u + 1 < steps && visible(tile + 1);
      if (visible(tile) && more) {
        both(k_use, v_use, tile);
      } else {
        if (visible(tile)) last(v_use, tile);
        if (more) first(k_use, tile + 1);
      }
    };
    issue_k(slot_a, tb);  // first: the wait below counts on all others being younger
    __builtin_amdgcn_sched_barrier(0);
    issue(rv, voff, va, tb);
    issue_k(slot_b, steps > 1 ? tb + 1 : tb);
    __builtin_amdgcn_sched_barrier(0);
    wait_vmcnt<NI + NK>();
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    if (visible(tb)) first(slot_a, tb);
    for (int u = 0; u < steps; u += 2) {
      step(slot_b, slot_a, va, vb, u);
      if (u + 1 < steps) step(slot_a, slot_b, vb, va, u + 1);
    }
    wait_vmcnt<0>();
    __syncthreads();
  };

  // The same tile by tile, values that are not finite taken out where the mask crosses.
  auto careful = [&]() {
    for (int u = 0; u < steps; u++) {
      const int tile = tb + u;
      issue_k(slot_a, tile);
      issue(rv, voff, va, tile);
      wait_vmcnt<0>();
      __syncthreads();
      if (visible(tile)) {
        const bool crossed = !unmasked(tile);
#pragma unroll 1
        for (int kt = 0; kt < 2; kt++) {
          floatx16 st{};
#pragma unroll
          for (int s = 0; s < KS; s++) s_mfma(slot_a, kt, s, st);
          const int p0 = tile * kRowKeys + 32 * kt + 4 * lg;
          if (crossed) mask(st, p0);
          Weights pp;
          half8 seen[2];
#pragma unroll
          for (int e = 0; e < 16; e++) {
            const int p = p0 + 8 * (e >> 2) + (e & 3);
            seen[e >> 3][e & 7] = (p > P || p <= P - win) ? (_Float16)0.0f : (_Float16)1.0f;
          }
          rescale(softmax(st, pp));
#pragma unroll
          for (int s = 0; s < KS; s++) {
            const int j = s / OT, i = s % OT;
            half8 vf = v_frag(va, kt, j, i);
            half8 up, dn, nn;
            bool odd = false;
#pragma unroll
            for (int e = 0; e < 8; e++) {
              const _Float16 value = vf[e];  // (a bit cast of the element itself reads element 0)
              const uint16_t b = __builtin_bit_cast(uint16_t, value);
              const bool x = crossed && (b & 0x7c00u) == 0x7c00u;
              odd |= x;
              up[e] = x && b == 0x7c00u ? (_Float16)1.0f : (_Float16)0.0f;
              dn[e] = x && b == 0xfc00u ? (_Float16)1.0f : (_Float16)0.0f;
              nn[e] = x && (b & 0x3ffu) ? (_Float16)1.0f : (_Float16)0.0f;
              vf[e] = x ? (_Float16)0.0f : vf[e];
            }
            add_values(vf, j, i, pp);
            if (__ballot(odd)) {
              const floatx16 u1 = __builtin_amdgcn_mfma_f32_32x32x16_f16(up, seen[j], floatx16{}, 0, 0, 0);
              const floatx16 d1 = __builtin_amdgcn_mfma_f32_32x32x16_f16(dn, seen[j], floatx16{}, 0, 0, 0);
              const floatx16 n1 = __builtin_amdgcn_mfma_f32_32x32x16_f16(nn, seen[j], floatx16{}, 0, 0, 0);
#pragma unroll
              for (int e = 0; e < 16; e++) {
                if (u1[e] > 0.0f) o[i][e] += INFINITY;
                if (d1[e] > 0.0f) o[i][e] -= INFINITY;
                if (n1[e] > 0.0f) o[i][e] = __builtin_nanf("");
              }
            }
          }
        }
      }
      __syncthreads();
    }
  };

  reset();
  fast();
  {
    float z = 0.0f;  // 0, or NaN if any sum is not finite
#pragma unroll
    for (int i = 0; i < OT; i++)
#pragma unroll
      for (int e = 0; e < 16; e++) z = __builtin_fmaf(o[i][e], 0.0f, z);
    if (tid == 0) shared_flag = 0;
    __syncthreads();
    if (wave_live && __ballot(z != 0.0f) && lane == 0) shared_flag = 1;
    __syncthreads();
    const bool again = shared_flag != 0;
    __syncthreads();
    if (again) {
      reset();
      careful();
    }
  }

  lrun += __shfl_xor(lrun, 32, 64);  // lane halves hold different keys
  const bool mine = wave_live && l32 < wlive;
  if (pc.n_pieces == 1) {
    if (mine) {
      const float inv = 1.0f / lrun;
      _Float16 *dst = a.s.out + ((size_t)(off + t) * n_head + h) * HD + 4 * lg;
#pragma unroll
      for (int i = 0; i < OT; i++)
#pragma unroll
        for (int g = 0; g < 4; g++)
          *reinterpret_cast<half4 *>(dst + 32 * i + 8 * g) =
              half4{(_Float16)(o[i][4 * g] * inv), (_Float16)(o[i][4 * g + 1] * inv), (_Float16)(o[i][4 * g + 2] * inv),
                    (_Float16)(o[i][4 * g + 3] * inv)};
    }
  } else {
    if (mine) {
      const size_t rr = (size_t)pc.rec + ((size_t)pc.piece * n_head_kv + kvh) * live + rl;
      if (lg == 0) st_dev(a.s.join.ml + rr, float2{mrun, lrun});
#pragma unroll
      for (int i = 0; i < OT; i++)
#pragma unroll
        for (int g = 0; g < 4; g++)
          st_dev4(a.s.join.o + rr * HD + 32 * i + 8 * g + 4 * lg, floatx4{o[i][4 * g], o[i][4 * g + 1], o[i][4 * g + 2], o[i][4 * g + 3]});
    }
    if (arrived_last(a.s.join, pc, kvh, &shared_flag))
      join_pieces<HD, 256>(a.s.join, pc, kvh, 1, live, n_head, n_head_kv, a.s.out + (size_t)off * n_head * HD);
  }
}

}  // namespace

int32_t launch_row_attention(const StepAttnArgs &c, const SeqKv *kv, const _Float16 *k, const _Float16 *k_rest,
                             const _Float16 *v, hipStream_t s) {
  RowAttn a{c, kv, k, k_rest, v};
  const dim3 grid((unsigned)c.n_pieces * c.n_head_kv), block(256);
  if (c.head_dim == 64 && k_rest) hipLaunchKernelGGL((row_attn_kernel<64, true>), grid, block, 0, s, a);
  else if (c.head_dim == 64) hipLaunchKernelGGL((row_attn_kernel<64, false>), grid, block, 0, s, a);
  else if (k_rest) hipLaunchKernelGGL((row_attn_kernel<128, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((row_attn_kernel<128, false>), grid, block, 0, s, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SULIMO_HIP_OK : hip_fail(e, "row_attn_kernel launch");
}

}  // namespace sulimo
