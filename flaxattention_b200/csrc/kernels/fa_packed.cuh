// Attention of prompts laid end to end, and of the newest tokens of many requests over a prefix that they share (FA_PREFIX), general kernel: any head dim
// that is a multiple of 16, fp16 / bf16 / fp32, any strides of 16 bytes.  (fa_fwd_tc.cuh has the one for 16-bit types and head dims up to 128.)
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(score_mod(scale q_i.k_j) - max) over the keys j of query i's request that are not behind it, not
//   further back than the window and kept by mask_mod;  lse_i = log sum_j p_ij + max.  Over a prefix: the sums and the maximum, for fa_merge_kernel.
//
// A CTA takes 64 rows (fa_packed_rows.cuh) in four warps of 16, and their keys in tiles of FA_BN, the next one on its way while one is computed.  16-bit types
// multiply with mma.sync and fp32 sums, fp32 with FMAs.
//
// Compile-time parameters (macros): FA_DTYPE, FA_D, FA_DV, FA_BN, FA_PREFIX.
#pragma once
#include "fa_packed_rows.cuh"

namespace fa_pk {

constexpr int DT = FA_DTYPE;
constexpr bool F32 = DT == FA_DT_F32, PREFIX = FA_PREFIX != 0;
constexpr int D = FA_D, DV = FA_DV, BN = FA_BN, BM = 64, NT = 128, ES = F32 ? 4 : 2;
constexpr int PQ = FaTile<D, ES>::PITCH, PV = FaTile<DV, ES>::PITCH, PP = FaTile<BN, 4>::PITCH;
constexpr int Q_BYTES = BM * PQ, K_BYTES = BN * PQ, V_BYTES = BN * PV, P_BYTES = F32 ? BM * PP : 0;
constexpr int SMEM_BYTES = Q_BYTES + 2 * K_BYTES + 2 * V_BYTES + P_BYTES;
static_assert(D % 16 == 0 && DV % 16 == 0 && BN % 16 == 0 && DV <= D, "tiles of multiples of 16, values no wider than keys");

}  // namespace fa_pk

extern "C" __global__ void __launch_bounds__(fa_pk::NT) fa_packed_kernel(const __grid_constant__ FaPackedParams p) {
  using namespace fa_pk;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ FaPlace found;
  FA_MOD_BUFS_INIT(p);
  fa_grid_wait();
  if (PREFIX) fa_grid_release();  // (the CTAs of the pages' kernel are there, waiting, when this one ends)
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, hk = PREFIX ? blockIdx.x % p.Hkv : blockIdx.x, G = p.Hq / p.Hkv;
  if (PREFIX) {
    if (tid == 0) found = {0, p.tokens, 0, p.keys, 0, (int)blockIdx.y * BM, 1};  // (grid: parts of the prefix and kv heads, items)
  } else {
    const long long item = (long long)blockIdx.z * gridDim.y + blockIdx.y;
    if (warp == 0) {
      const FaPlace at = fa_find_item<BM>(p, item);
      if (lane == 0) found = at;
    }
    if (hk == 0 && item == 0) fa_check_starts(p, tid, NT);
  }
  __syncthreads();
  const FaPlace place = found;
  if (!place.any || (PREFIX && place.first >= p.tokens * G)) return;
  const fa_u32 sQ = fa_smem_u32(smem), sK = sQ + Q_BYTES, sV = sK + 2 * K_BYTES;
  const char* qg = (const char*)p.q.ptr + (long long)hk * G * p.q.sh * ES;
  const char* kg = (const char*)p.k.ptr + (hk * p.k.sh + place.k0 * p.k.ss) * ES;
  const char* vg = (const char*)p.v.ptr + (hk * p.v.sh + place.k0 * p.v.ss) * ES;

  // ---- this thread's two rows, and the keys that any row of the CTA sees
  FaRow row[2];
  int from = 0x7fffffff, to = 0, last_from = 0, first_to = 0x7fffffff;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    row[h] = fa_row<PREFIX>(p, place, place.first + warp * 16 + h * 8 + (lane >> 2));
    if (row[h].from < row[h].to) {
      from = min(from, row[h].from);
      to = max(to, row[h].to);
    }
    if (row[h].at >= 0) {
      last_from = max(last_from, row[h].from);
      first_to = min(first_to, row[h].to);
    }
  }
  __shared__ int bounds[4][4];
  from = (int)__reduce_min_sync(0xffffffffu, (fa_u32)from);
  to = __reduce_max_sync(0xffffffffu, to);
  last_from = __reduce_max_sync(0xffffffffu, last_from);
  first_to = __reduce_min_sync(0xffffffffu, first_to);
  if (lane == 0) {
    bounds[warp][0] = from; bounds[warp][1] = to; bounds[warp][2] = last_from; bounds[warp][3] = first_to;
  }
  {
    constexpr int CPR = D * ES / 16;
    for (int i = tid; i < BM * CPR; i += NT) {
      const int r = i / CPR, c = i - r * CPR;
      const FaRow x = fa_row<PREFIX>(p, place, place.first + r);
      fa_cp_async16(sQ + r * PQ + c * 16, qg + (x.at >= 0 ? x.at * ES + c * 16 : 0), x.at >= 0 ? 16 : 0);
    }
    fa_cp_commit();
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    from = min(from, bounds[w][0]);
    to = max(to, bounds[w][1]);
    last_from = max(last_from, bounds[w][2]);
    first_to = min(first_to, bounds[w][3]);
  }
  int t0 = to > 0 ? from / BN : 0, t1 = (to + BN - 1) / BN;
  if (PREFIX) {  // this CTA's part of the tiles
    const int per = (t1 - t0 + p.splits - 1) / p.splits;
    t0 = min(t0 + (int)(blockIdx.x / p.Hkv) * per, t1);
    t1 = min(t0 + per, t1);
  }
  auto load_kv = [&](int stage, int n0) {
    fa_load_tile<D, ES, NT>(sK + stage * K_BYTES, kg + (long long)n0 * p.k.ss * ES, p.k.ss * ES, BN, place.nk - n0, tid);
    fa_load_tile<DV, ES, NT>(sV + stage * V_BYTES, vg + (long long)n0 * p.v.ss * ES, p.v.ss * ES, BN, place.nk - n0, tid);
  };

  float o[DV / 8][4], m[2] = {FA_NEG_INF, FA_NEG_INF}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int dj = 0; dj < DV / 8; ++dj) o[dj][0] = o[dj][1] = o[dj][2] = o[dj][3] = 0.f;
  if (t0 < t1) load_kv(0, t0 * BN);
  fa_cp_commit();
#if FA_DTYPE != FA_DT_F32
  fa_u32 qf[D / 16][4];
#endif
#pragma unroll 1
  for (int t = t0; t < t1; ++t) {
    const int stage = (t - t0) & 1, n0 = t * BN;
    if (t + 1 < t1) load_kv(stage ^ 1, n0 + BN);
    fa_cp_commit();
    fa_cp_wait<1>();
    __syncthreads();
    const fa_u32 sKc = sK + stage * K_BYTES;
    [[maybe_unused]] const fa_u32 sVc = sV + stage * V_BYTES;
    float s[BN / 8][4];
#pragma unroll
    for (int nj = 0; nj < BN / 8; ++nj) s[nj][0] = s[nj][1] = s[nj][2] = s[nj][3] = 0.f;
#if FA_DTYPE != FA_DT_F32
    if (t == t0) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
        fa_ldsm_x4(sQ + (warp * 16 + ((lane >> 3) & 1) * 8 + (lane & 7)) * PQ + (kk * 16 + (lane >> 4) * 8) * 2, qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3]);
    }
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
      for (int nj = 0; nj < BN / 16; ++nj) {
        fa_u32 r0, r1, r2, r3;
        fa_ldsm_x4(sKc + (nj * 16 + (lane >> 4) * 8 + (lane & 7)) * PQ + (kk * 16 + ((lane >> 3) & 1) * 8) * 2, r0, r1, r2, r3);
        fa_mma16816<DT>(s[2 * nj], qf[kk], r0, r1);
        fa_mma16816<DT>(s[2 * nj + 1], qf[kk], r2, r3);
      }
    }
#else
    {
      // (every thread has the scores of its places in an accumulator fragment)
      const unsigned char *Qa = smem + (warp * 16 + (lane >> 2)) * PQ, *Qb = Qa + 8 * PQ, *Kc = smem + Q_BYTES + stage * K_BYTES + (lane & 3) * 2 * PQ;
#pragma unroll 2
      for (int d4 = 0; d4 < D / 4; ++d4) {
        const float4 qa = *(const float4*)(Qa + d4 * 16), qb = *(const float4*)(Qb + d4 * 16);
#pragma unroll
        for (int nj = 0; nj < BN / 8; ++nj) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float4 k4 = *(const float4*)(Kc + (nj * 8 + e) * PQ + d4 * 16);
            s[nj][e] = fmaf(qa.x, k4.x, fmaf(qa.y, k4.y, fmaf(qa.z, k4.z, fmaf(qa.w, k4.w, s[nj][e]))));
            s[nj][2 + e] = fmaf(qb.x, k4.x, fmaf(qb.y, k4.y, fmaf(qb.z, k4.z, fmaf(qb.w, k4.w, s[nj][2 + e]))));
          }
        }
      }
    }
#endif
    // ---- softmax: does any row of the CTA have to look at the positions?
    const bool edge = n0 + BN > first_to || n0 < last_from;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      [[maybe_unused]] const int gb = row[h].b + p.b_off, gh = hk * G + row[h].head + p.h_off, qi = row[h].pos;
      float mx = FA_NEG_INF;
#pragma unroll
      for (int nj = 0; nj < BN / 8; ++nj) {
#if FA_HAS_SCORE_MOD && FA_SCORE_PAIRS
        {
          const int kv = n0 + nj * 8 + (lane & 3) * 2;
          fa_f2_unpack(fa_score_mod_pair(fa_mul2(fa_f2(s[nj][h * 2], s[nj][h * 2 + 1]), fa_both(p.scale)), gb, gh, qi, kv, kv + 1), s[nj][h * 2], s[nj][h * 2 + 1]);
        }
#endif
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int kv = n0 + nj * 8 + (lane & 3) * 2 + e;
#if FA_HAS_SCORE_MOD && FA_SCORE_PAIRS
          float x = s[nj][h * 2 + e];
#else
          float x = s[nj][h * 2 + e] * p.scale;
#endif
#if FA_HAS_SCORE_MOD && !FA_SCORE_PAIRS
          x = fa_score_mod(x, gb, gh, qi, kv);
#endif
          bool keep = !edge || (kv >= row[h].from && kv < row[h].to);
#if FA_HAS_MASK_MOD
          keep = keep && fa_mask_mod(gb, gh, qi, kv);
#endif
          x = keep ? x * FA_LOG2E : FA_NEG_INF;
          s[nj][h * 2 + e] = x;
          mx = fmaxf(mx, x);
        }
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float m_new = fmaxf(m[h], mx), m_use = m_new == FA_NEG_INF ? 0.f : m_new;
      const float corr = F32 ? exp2f(m[h] - m_use) : fa_ex2(m[h] - m_use);
      float sum = 0.f;
      m[h] = m_new;
#pragma unroll
      for (int nj = 0; nj < BN / 8; ++nj) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x = s[nj][h * 2 + e] - m_use, pv = F32 ? exp2f(x) : fa_ex2(x);
          s[nj][h * 2 + e] = pv;
          sum += pv;
        }
      }
      l[h] = l[h] * corr + sum;
#pragma unroll
      for (int dj = 0; dj < DV / 8; ++dj) {
        o[dj][h * 2] *= corr;
        o[dj][h * 2 + 1] *= corr;
      }
    }
    // ---- O += P V.  (16 bits: probabilities are rounded once, as in the forward kernel.)
#if FA_DTYPE != FA_DT_F32
#pragma unroll
    for (int kj = 0; kj < BN / 16; ++kj) {
      const fa_u32 a[4] = {fa_pack2<DT>(s[2 * kj][0], s[2 * kj][1]), fa_pack2<DT>(s[2 * kj][2], s[2 * kj][3]), fa_pack2<DT>(s[2 * kj + 1][0], s[2 * kj + 1][1]),
                           fa_pack2<DT>(s[2 * kj + 1][2], s[2 * kj + 1][3])};
#pragma unroll
      for (int dj = 0; dj < DV / 16; ++dj) {
        fa_u32 r0, r1, r2, r3;
        fa_ldsm_x4_t(sVc + (kj * 16 + ((lane >> 3) & 1) * 8 + (lane & 7)) * PV + (dj * 16 + (lane >> 4) * 8) * 2, r0, r1, r2, r3);
        fa_mma16816<DT>(o[2 * dj], a, r0, r1);
        fa_mma16816<DT>(o[2 * dj + 1], a, r2, r3);
      }
    }
#else
    {
      unsigned char *Pa = smem + Q_BYTES + 2 * K_BYTES + 2 * V_BYTES + (warp * 16 + (lane >> 2)) * PP, *Pb = Pa + 8 * PP;
      const unsigned char* Vc = smem + Q_BYTES + 2 * K_BYTES + stage * V_BYTES + (lane & 3) * 8;
#pragma unroll
      for (int nj = 0; nj < BN / 8; ++nj) {
        const int c = (nj * 8 + (lane & 3) * 2) * 4;
        *(float2*)(Pa + c) = make_float2(s[nj][0], s[nj][1]);
        *(float2*)(Pb + c) = make_float2(s[nj][2], s[nj][3]);
      }
      __syncwarp();
#pragma unroll 2
      for (int k = 0; k < BN; ++k) {
        const float pa = *(const float*)(Pa + k * 4), pb = *(const float*)(Pb + k * 4);
#pragma unroll
        for (int dj = 0; dj < DV / 8; ++dj) {
          const float2 vv = *(const float2*)(Vc + k * PV + dj * 32);
          o[dj][0] = fmaf(pa, vv.x, o[dj][0]);
          o[dj][1] = fmaf(pa, vv.y, o[dj][1]);
          o[dj][2] = fmaf(pb, vv.x, o[dj][2]);
          o[dj][3] = fmaf(pb, vv.y, o[dj][3]);
        }
      }
      __syncwarp();
    }
#endif
    __syncthreads();  // (before the tile behind the next goes there)
  }
  fa_cp_wait<0>();
  __syncthreads();

  // ---- the rows leave: 16-byte pieces over the query tile, or the sums as they are
  unsigned char* Os = smem;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    const int rl = warp * 16 + h * 8 + (lane >> 2);
    if (PREFIX) {
      if (row[h].at < 0) continue;
      const long long part = (long long)blockIdx.x * p.tokens * G + place.first + rl;
      if ((lane & 3) == 0) *(float2*)(p.part_ml + part * 2) = make_float2(m[h], l[h]);
#pragma unroll
      for (int dj = 0; dj < DV / 8; ++dj) *(float2*)(p.part_o + part * DV + dj * 8 + (lane & 3) * 2) = make_float2(o[dj][h * 2], o[dj][h * 2 + 1]);
      continue;
    }
    // (a row that has seen nothing is 0; one whose sum is no number stays so)
    const float inv = l[h] > 0.f ? 1.f / l[h] : l[h];
    if (p.lse != nullptr && (lane & 3) == 0 && row[h].at >= 0)
      p.lse[(long long)(hk * G + row[h].head) * p.tokens + place.q0 + row[h].token] = l[h] == 0.f ? FA_NEG_INF : (m[h] + log2f(l[h])) * FA_LN2;
#pragma unroll
    for (int dj = 0; dj < DV / 8; ++dj) {
      const int c = dj * 8 + (lane & 3) * 2;
      const float x0 = o[dj][h * 2] * inv, x1 = o[dj][h * 2 + 1] * inv;
      if (F32) *(float2*)(Os + rl * PV + c * 4) = make_float2(x0, x1);
      else *(fa_u32*)(Os + rl * PV + c * 2) = fa_pack2<DT>(x0, x1);
    }
  }
  if (PREFIX) return;
  __syncthreads();
  constexpr int CPR = DV * ES / 16;
  for (int i = tid; i < BM * CPR; i += NT) {
    const int r = i / CPR, c = i - r * CPR;
    const FaRow x = fa_row<PREFIX>(p, place, place.first + r);
    if (x.at >= 0) *(uint4*)((char*)p.o.ptr + fa_row_out(p, place, x, hk) * ES + c * 16) = *(const uint4*)(Os + r * PV + c * 16);
  }
}
