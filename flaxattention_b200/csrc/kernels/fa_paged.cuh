// Attention of the newest Sq tokens of each request over a key / value cache in pages.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(score_mod(scale q_i.k_j) - max)  over the keys j of the request that are
//   not behind query i, not further back than the window and kept by mask_mod;  lse_i = log sum_j p_ij + max.
//
// The keys of a request lie in pages of page_size tokens that a block table lists: key j is token j % page_size of page
// table[b][j / page_size].  Query i of the Sq is token len - Sq + i, which is also the index the mods see.
//
// The G query heads of a kv head share its K and V: their G * Sq rows (query-major, row r is head r % G of query r / G) are
// cut into row tiles of 16, 32 or 64.  Lengths are known on the device only and differ, so the work is cut there: a segment is
// the keys that a row tile of a kv head of a request has to see, in tiles of FA_WN keys; the tiles of all segments, one behind the
// other, are dealt out evenly to the CTAs ("workers") of a grid that is resident at once.  A worker keeps the running
// (max, sum, O) of one segment, over whose end its loads run on into the next.  A segment that lies in one worker's run is written out; of
// others the workers leave parts (O not divided, max, sum), which fa_paged_combine_kernel merges.
//
// CTA = FA_RG warps, each with 16 query rows; they share the tiles of K and V, which come by TMA (FA_TMA: pages that hold whole boxes of
// 8 keys and more, head dims of whole 128-byte columns) or in 16-byte cp.async pieces.
//
// Memory sets the pace: K and V are read once per kv head (and row tile).
//
// Compile-time parameters (macros): FA_DTYPE, FA_D, FA_DV, FA_RG (1, 2, 4), FA_WN (16, 32), FA_STAGES, FA_TMA.
#pragma once
#include "fa_sm100.cuh"

struct FaPagedLaunch {
  FaPagedParams p;
#if FA_TMA
  FaTensorMap tk, tv;  // 4-d maps (D, token in page, head, page), box 64 x p.box x 1 x 1, 128-byte swizzle
#endif
};

namespace fa_pg {

constexpr int DT = FA_DTYPE;
constexpr bool F32 = DT == FA_DT_F32;
constexpr int D = FA_D;
constexpr int DV = FA_DV;
constexpr int RG = FA_RG;
constexpr int NT = RG * 32;
constexpr int BM = RG * 16;
constexpr int WN = FA_WN;
constexpr int STAGES = FA_STAGES;
constexpr bool TMA = FA_TMA != 0;
constexpr int ES = F32 ? 4 : 2;
constexpr int PK = TMA ? D * ES : FaTile<D, ES>::PITCH;
constexpr int PV = TMA ? DV * ES : FaTile<DV, ES>::PITCH;
constexpr int ATOMS_K = D / 64, ATOMS_V = DV / 64;  // 128-byte column groups of a row (TMA)
constexpr int K_BYTES = WN * PK, V_BYTES = WN * PV;
constexpr int PIPE_BYTES = STAGES * (K_BYTES + V_BYTES);
constexpr int BAR_BYTES = TMA ? STAGES * 16 + 16 : 0;
// fp32: the query tile, and the probabilities of a tile
constexpr int PQ = FaTile<D, 4>::PITCH, PP = FaTile<WN, 4>::PITCH;
constexpr int Q_BYTES = F32 ? BM * (PQ + PP) : 0;
constexpr int SMEM_BYTES = PIPE_BYTES + Q_BYTES + BAR_BYTES + (TMA ? 1024 : 0);

static_assert(!TMA || (!F32 && D % 64 == 0 && DV % 64 == 0), "TMA: 16-bit types, whole column groups");
static_assert(WN == 16 || WN == 32, "tiles of 16 or 32 keys");

// A segment, and the tile of it that is next.
struct Seg {
  int item, hk, b;
  int first;  // first query of the row tile, and its position among the request's tokens
  int pos;
  int end;    // keys from here on are behind every row
  int tile, last;  // tiles of WN keys, first and one beyond the last
};
__device__ __forceinline__ void seg_open(const FaPagedParams& p, int item, Seg& s) {
  s.item = item;
  s.b = p.row_tiles == 1 ? item : item / p.row_tiles;
  const int rt = item - s.b * p.row_tiles, G = p.Hq / p.Hkv;
  const int len = min(max(p.lengths[s.b], 0), p.max_len);
  s.first = rt * BM / G;
  const int final = min(p.Sq, ((rt + 1) * BM - 1) / G + 1) - 1;  // its last query
  s.pos = len - p.Sq + s.first;
  s.end = max(len - p.Sq + final + 1, 0);
  s.tile = (p.window < 0 ? 0 : max(s.pos - p.window, 0)) / WN;
  s.last = max((s.end + WN - 1) / WN, s.tile + 1);  // (at least one: somebody has to write a row that sees nothing)
}
// tiles of item `item`'s segments
__device__ __forceinline__ int seg_tiles(const FaPagedParams& p, int item) {
  Seg s;
  seg_open(p, item, s);
  return s.last - s.tile;
}
__device__ __forceinline__ void seg_next(const FaPagedParams& p, Seg& s) {
  if (++s.tile < s.last) return;
  const bool wrap = s.hk + 1 == p.Hkv;
  s.hk = wrap ? 0 : s.hk + 1;
  if (wrap && s.item + 1 == p.B * p.row_tiles) return;  // (behind the last tile of all)
  seg_open(p, wrap ? s.item + 1 : s.item, s);
}

// Products over a tile as TMA leaves it: rows of 128 bytes, 16-byte chunk c of row r at c ^ (r & 7), one block of WN rows per
// 64 columns.
__device__ __forceinline__ void qk_swizzled(float (&acc)[WN / 8][4], const fa_u32 (&a)[D / 16][4], fa_u32 sB, int lane) {
  const fa_u32 x = ((lane >> 3) & 1) ^ (lane & 7);
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    const fa_u32 at = sB + (kk >> 2) * (WN * 128) + ((lane >> 4) * 8 + (lane & 7)) * 128 + (((kk & 3) * 2) ^ x) * 16;
#pragma unroll
    for (int nj = 0; nj < WN / 16; ++nj) {
      fa_u32 r0, r1, r2, r3;
      fa_ldsm_x4(at + nj * 2048, r0, r1, r2, r3);
      fa_mma16816<DT>(acc[2 * nj], a[kk], r0, r1);
      fa_mma16816<DT>(acc[2 * nj + 1], a[kk], r2, r3);
    }
  }
}
__device__ __forceinline__ void pv_swizzled(float (&out)[DV / 8][4], const float (&pacc)[WN / 8][4], fa_u32 sB, int lane) {
  const fa_u32 x = (lane >> 4) ^ (lane & 7);
#pragma unroll
  for (int kj = 0; kj < WN / 16; ++kj) {
    fa_u32 a[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float(&v)[4] = pacc[2 * kj + (i >> 1)];
      a[i] = fa_pack2<DT>(v[(i & 1) * 2], v[(i & 1) * 2 + 1]);
    }
    const fa_u32 row = sB + (kj * 16 + ((lane >> 3) & 1) * 8 + (lane & 7)) * 128;
#pragma unroll
    for (int dj = 0; dj < DV / 16; ++dj) {
      fa_u32 r0, r1, r2, r3;
      fa_ldsm_x4_t(row + (dj >> 2) * (WN * 128) + (((dj & 3) * 2) ^ x) * 16, r0, r1, r2, r3);
      fa_mma16816<DT>(out[2 * dj], a, r0, r1);
      fa_mma16816<DT>(out[2 * dj + 1], a, r2, r3);
    }
  }
}

// K and V of a tile on their way: where its keys are.  Every lane of every warp has the same but for its own key (TMA: box).
struct Load {
  bool any;     // there is a tile
  int hk;
  int page;     // this lane's, or -1: no such key, or no such page
  int row;      // token in it
  fa_u32 keep;  // keys of the tile that are there, bit by bit
};

// The rows of a tile in 16-byte pieces, those that are not there as zeros
template <int COLS, int PITCH>
__device__ __forceinline__ void load_pieces(const FaTensor& t, fa_u32 dst, const Load& n, int tid) {
  constexpr int CPR = COLS * ES / 16;
  const long long at = n.page >= 0 ? (n.page * t.sb + n.hk * t.sh + n.row * t.ss) * ES : -1;
#pragma unroll 4
  for (int i = tid; i < (WN * CPR + 31) / 32 * 32; i += NT) {  // (whole warps: the shuffle)
    const int r = i / CPR, c = i - r * CPR;
    const long long row = __shfl_sync(0xffffffffu, at, r & 31);
    if (i < WN * CPR) fa_cp_async16(dst + r * PITCH + c * 16, (const char*)t.ptr + (row >= 0 ? row + c * 16 : 0), row >= 0 ? 16 : 0);
  }
}

}  // namespace fa_pg

extern "C" __global__ void __launch_bounds__(fa_pg::NT) fa_paged_kernel(const __grid_constant__ FaPagedLaunch L) {
  using namespace fa_pg;
  const FaPagedParams& p = L.p;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  if (fa_dynamic_smem_size() < (fa_u32)SMEM_BYTES || blockDim.x != NT) {
    if (threadIdx.x == 0 && p.status != nullptr) atomicOr(p.status, FA_STATUS_BAD_LAUNCH);
    return;
  }
  unsigned char* const base = TMA ? smem_raw + ((1024u - (fa_smem_u32(smem_raw) & 1023u)) & 1023u) : smem_raw;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const fa_u32 sK = fa_smem_u32(base), sV = sK + STAGES * K_BYTES;
  [[maybe_unused]] unsigned char* const q_tile = base + PIPE_BYTES;
#if FA_TMA
  const fa_u32 bars = sK + PIPE_BYTES;  // K 0 .. STAGES - 1, V 0 .. STAGES - 1
  volatile int* abort_flag = (volatile int*)(base + PIPE_BYTES + STAGES * 16);
  if (tid == 0) {
    for (int i = 0; i < 2 * STAGES; ++i) fa_mbar_init(bars + i * 8, 1);
    fa_mbar_init_fence();
    *abort_flag = 0;
  }
#endif
  FA_MOD_BUFS_INIT(p);
  __syncthreads();
  fa_grid_wait();

  // ---- this worker's run of tiles --------------------------------------------------------
  const int G = p.Hq / p.Hkv, items = p.B * p.row_tiles;
  int total, t0, t1;
  Seg seg;
  {
    // every lane counts a run of items, then the lanes are added up
    const int per_lane = (items + 31) / 32, i0 = min(lane * per_lane, items), i1 = min(i0 + per_lane, items);
    int own = 0;
#pragma unroll 4
    for (int i = i0; i < i1; ++i) own += seg_tiles(p, i);
    int upto = own;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += v;
    }
    total = __shfl_sync(0xffffffffu, upto, 31) * p.Hkv;
    const int per = max(p.min_tiles, (total + p.workers - 1) / p.workers);
    if (blockIdx.x == 0 && warp == 0) {  // for the kernel that merges
      int at = upto - own;
      for (int i = i0; i < i1; ++i) {
        p.plan[i] = at;
        at += seg_tiles(p, i);
      }
      if (lane == 31) p.plan[items] = upto;
      // a length that the table has no room for
      bool beyond = false;
      for (int i = lane; i < p.B; i += 32) beyond |= p.lengths[i] > p.max_len || p.lengths[i] < 0;
      if (beyond && p.status != nullptr) atomicOr(p.status, FA_STATUS_BAD_PAGE);
    }
    t0 = (int)min((long long)blockIdx.x * per, (long long)total);
    t1 = min(t0 + per, total);
    if (t0 >= t1) return;
    const int from = __popc(__ballot_sync(0xffffffffu, (long long)upto * p.Hkv <= t0));  // the lane whose run has tile t0
    int item = __shfl_sync(0xffffffffu, i0, from), before = __shfl_sync(0xffffffffu, upto - own, from);
    seg_open(p, item, seg);
    while (t0 >= (before + seg.last - seg.tile) * p.Hkv) {
      before += seg.last - seg.tile;
      seg_open(p, ++item, seg);
    }
    const int n = seg.last - seg.tile, off = t0 - before * p.Hkv;
    seg.hk = off / n;
    seg.tile += off - seg.hk * n;
  }
  const int seg_first = seg.tile;  // where the first segment's part begins

  // ---- loads -----------------------------------------------------------------------------
  Seg ahead = seg;     // of the tile that is asked for next
  int to_load = t1 - t0;
  // looks the next tile's pages up
  auto look_up = [&](Load& n) {
    n.any = to_load > 0;
    n.page = -1;
    if (!n.any) return;
    const int key = ahead.tile * WN + lane * p.box;  // (box: 1 without TMA)
    const bool there = lane * p.box < WN && key < ahead.end;
    n.hk = ahead.hk;
    if (there) {
      const int slot = key / p.page_size;
      n.row = key - slot * p.page_size;
      n.page = p.table[ahead.b * p.table_stride + slot];
    }
    // (the number of keys that are there goes along; pages that are none are taken out when the entry has come)
    const int left = ahead.end - ahead.tile * WN;
    n.keep = left >= WN ? (WN == 32 ? 0xffffffffu : (1u << WN) - 1u) : left > 0 ? (1u << left) - 1u : 0u;
    --to_load;
    seg_next(p, ahead);
  };
  // takes keys out whose page is none
  auto settle = [&](Load& n) {
    const bool there = lane * p.box < WN && (n.keep >> (lane * p.box)) & 1u;
    const bool bad = there && (n.page < 0 || n.page >= p.num_pages);
    if (bad) n.page = -1;
    fa_u32 out = __ballot_sync(0xffffffffu, bad);
    if (out != 0) {
      if (lane == 0 && p.status != nullptr) atomicOr(p.status, FA_STATUS_BAD_PAGE);
      for (; out != 0; out &= out - 1) {
        const int first = (__ffs(out) - 1) * p.box;
        n.keep &= ~((p.box >= 32 ? 0xffffffffu : (1u << p.box) - 1u) << first);
      }
    }
  };
#if FA_TMA
  auto load = [&](const FaTensorMap* map, fa_u32 dst, fa_u32 bar, int atoms, const Load& n) {
    if (warp != 0) return;
    const fa_u32 boxes = __ballot_sync(0xffffffffu, n.page >= 0);
    if (lane == 0) fa_mbar_expect_tx(bar, __popc(boxes) * p.box * 128 * atoms);
    __syncwarp();
    if (n.page >= 0) {
      for (int a = 0; a < atoms; ++a)
        fa_tma_load_4d(dst + a * (WN * 128) + lane * p.box * 128, map, bar, a * 64, n.row, n.hk, n.page);
    }
  };
  auto load_k = [&](int stage, const Load& n) { load(&L.tk, sK + stage * K_BYTES, bars + stage * 8, ATOMS_K, n); };
  auto load_v = [&](int stage, const Load& n) { load(&L.tv, sV + stage * V_BYTES, bars + (STAGES + stage) * 8, ATOMS_V, n); };
#else
  auto load_k = [&](int stage, const Load& n) { load_pieces<D, PK>(p.k, sK + stage * K_BYTES, n, tid); };
  auto load_v = [&](int stage, const Load& n) { load_pieces<DV, PV>(p.v, sV + stage * V_BYTES, n, tid); };
#endif

  fa_u32 keep[STAGES];
#pragma unroll
  for (int st = 0; st < STAGES; ++st) {
    Load n;
    look_up(n);
    keep[st] = 0;
    if (n.any) {
      settle(n);
      keep[st] = n.keep;
      load_k(st, n);
    }
    fa_cp_commit();
    if (n.any) load_v(st, n);
    fa_cp_commit();
  }
  Load next;  // the tile STAGES ahead of the one that is computed
  look_up(next);

  // ---- the tiles -------------------------------------------------------------------------
  float o[DV / 8][4], m_run[2], l_run[2];
  int qpos[2], qidx[2], head[2];  // of this thread's two rows: position (-1: no row), query, head
  fa_u32 qf[F32 ? 1 : D / 16][4];
  const float sc2 = p.scale * FA_LOG2E;
  bool open = false, failed = false;
  [[maybe_unused]] bool k_again = false;  // K of the tile STAGES ahead has been asked for, V not yet
  int cur = 0;
  [[maybe_unused]] fa_u32 phase = 0;
  bool first_part = true;  // of this worker

  [[maybe_unused]] int t_now = t0;
  for (int t = t0; t < t1; ++t) {
    t_now = t;
    if (!open) {
      open = true;
      const int rt = seg.item - seg.b * p.row_tiles;
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int row = rt * BM + warp * 16 + hh * 8 + (lane >> 2);
        const int i = row / G;
        qidx[hh] = i;
        head[hh] = seg.hk * G + row - i * G;
        qpos[hh] = i < p.Sq ? seg.pos - seg.first + i : -1;
        m_run[hh] = FA_NEG_INF;
        l_run[hh] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < DV / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
      const char* qb = (const char*)p.q.ptr + seg.b * p.q.sb * ES;
      if (F32) {
        __syncthreads();  // (the tile before has been read)
        for (int i = tid; i < BM * (D / 4); i += NT) {
          const int r = i / (D / 4), c = i - r * (D / 4), row = rt * BM + r, qi = row / G;
          const float* src = (const float*)(qb + (qi * p.q.ss + (long long)(seg.hk * G + row - qi * G) * p.q.sh) * ES) + c * 4;
          *(float4*)(q_tile + r * PQ + c * 16) = qi < p.Sq ? *(const float4*)src : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        __syncthreads();
      } else {
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const bool row = qidx[hh] < p.Sq;
          const fa_u32* src = (const fa_u32*)(qb + (qidx[hh] * p.q.ss + head[hh] * p.q.sh) * ES) + (lane & 3);
#pragma unroll
          for (int kk = 0; kk < (F32 ? 1 : D / 16); ++kk) {
            qf[kk][hh] = row ? src[kk * 8] : 0u;
            qf[kk][2 + hh] = row ? src[kk * 8 + 4] : 0u;
          }
        }
      }
    }
    // ---- scores
#if FA_TMA
    failed = !fa_mbar_wait_all(bars + cur * 8, phase, abort_flag);
#else
    fa_cp_wait<2 * STAGES - 1>();
    if (RG == 1) __syncwarp();
    else __syncthreads();
#endif
    float s[WN / 8][4];
#pragma unroll
    for (int j = 0; j < WN / 8; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
    if (F32) fa_simt_nt<D, WN>(s, q_tile, PQ, warp * 16, base + cur * K_BYTES, PK, lane);
#if FA_TMA
    else qk_swizzled(s, qf, sK + cur * K_BYTES, lane);
#else
    else fa_mma_nt<DT, F32 ? 16 : D, WN>(s, qf, sK + cur * K_BYTES, PK, lane);
#endif
    // K's buffer is free
    if (RG == 1) __syncwarp();
    else failed = __syncthreads_or(failed) != 0;
    if (failed) break;
    if (next.any) {
      settle(next);
      load_k(cur, next);
      k_again = true;
    }
    fa_cp_commit();

    const int n0 = seg.tile * WN, kv0 = n0 + (lane & 3) * 2;
    const fa_u32 kept = keep[0];
    // does any row of the tile have to look at the positions?
    const bool edge = n0 + WN - 1 > seg.pos || (p.window >= 0 && n0 < seg.end - 1 - p.window) || kept != (WN == 32 ? 0xffffffffu : (1u << WN) - 1u);
    const int gb = seg.b + p.b_off;
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const int qp = max(qpos[hh], 0), gh = head[hh] + p.h_off;
#pragma unroll
      for (int j = 0; j < WN / 8; ++j) {
        const int kv = kv0 + j * 8;
        float x0 = s[j][hh * 2], x1 = s[j][hh * 2 + 1];
#if FA_HAS_SCORE_MOD && defined(FA_SCORE_AFFINE)
        x0 = fmaf(x0, fa_score_mul(0.f, gb, gh, qp, kv) * sc2, fa_score_add2(0.f, gb, gh, qp, kv));
        x1 = fmaf(x1, fa_score_mul(0.f, gb, gh, qp, kv + 1) * sc2, fa_score_add2(0.f, gb, gh, qp, kv + 1));
#elif FA_HAS_SCORE_MOD
        x0 = fa_score_mod(x0 * p.scale, gb, gh, qp, kv) * FA_LOG2E;
        x1 = fa_score_mod(x1 * p.scale, gb, gh, qp, kv + 1) * FA_LOG2E;
#else
        x0 *= sc2;
        x1 *= sc2;
#endif
        s[j][hh * 2] = x0;
        s[j][hh * 2 + 1] = x1;
      }
      if (edge || FA_HAS_MASK_MOD) {
#pragma unroll
        for (int j = 0; j < WN / 8; ++j) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int kv = kv0 + j * 8 + e;
            bool see = kv <= qpos[hh] && (p.window < 0 || qpos[hh] - kv <= p.window) && ((kept >> (kv - n0)) & 1u);
#if FA_HAS_MASK_MOD
            see = see && fa_mask_mod(gb, gh, qp, kv);
#endif
            if (!see) s[j][hh * 2 + e] = FA_NEG_INF;
          }
        }
      }
      float mx = FA_NEG_INF;
#pragma unroll
      for (int j = 0; j < WN / 8; ++j) mx = fa_max3(mx, s[j][hh * 2], s[j][hh * 2 + 1]);
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float m_new = fmaxf(m_run[hh], mx);
      const float m_use = (m_new == FA_NEG_INF) ? 0.f : m_new;
      const float corr = fa_ex2(m_run[hh] - m_use);
      m_run[hh] = m_new;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < WN / 8; ++j) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float pv = fa_ex2(s[j][hh * 2 + e] - m_use);
          s[j][hh * 2 + e] = pv;
          sum += pv;
        }
      }
      l_run[hh] = l_run[hh] * corr + sum;
      if (__any_sync(0xffffffffu, corr != 1.f)) {
#pragma unroll
        for (int j = 0; j < DV / 8; ++j) {
          o[j][hh * 2] *= corr;
          o[j][hh * 2 + 1] *= corr;
        }
      }
    }
    // ---- values
#if FA_TMA
    failed = !fa_mbar_wait_all(bars + (STAGES + cur) * 8, phase, abort_flag);
    // Rows of keys that are not there hold whatever was in the page or the buffer, perhaps no number: 0, since a weight of 0
    // does not take that out of the product.  (Each warp for itself; all write the same.)
    if (kept != (WN == 32 ? 0xffffffffu : (1u << WN) - 1u)) {
      for (int i = lane; i < WN * ATOMS_V * 8; i += 32) {
        const int r = (i >> 3) % WN;
        if (!((kept >> r) & 1u)) *(uint4*)(base + STAGES * K_BYTES + cur * V_BYTES + i * 16) = make_uint4(0, 0, 0, 0);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // (before TMA writes the buffer again)
      __syncwarp();
    }
#else
    fa_cp_wait<2 * STAGES - 1>();
    if (RG == 1) __syncwarp();
    else __syncthreads();
#endif
    if (F32) fa_simt_nn<WN, DV>(o, s, q_tile + BM * PQ, PP, warp * 16, base + STAGES * K_BYTES + cur * V_BYTES, PV, lane);
#if FA_TMA
    else pv_swizzled(o, s, sV + cur * V_BYTES, lane);
#else
    else fa_mma_nn<DT, WN, DV>(o, s, sV + cur * V_BYTES, PV, lane);
#endif
    if (RG == 1) __syncwarp();
    else failed = __syncthreads_or(failed) != 0;
    if (failed) break;
    if (next.any) load_v(cur, next);
    fa_cp_commit();
    k_again = false;
#pragma unroll
    for (int i = 0; i + 1 < STAGES; ++i) keep[i] = keep[i + 1];
    keep[STAGES - 1] = next.any ? next.keep : 0u;
    look_up(next);
    if (++cur == STAGES) {
      cur = 0;
      phase ^= 1u;
    }

    // ---- the end of the segment, or of this worker's part of it
    const bool ends = seg.tile + 1 == seg.last;
    if (ends || t + 1 == t1) {
      open = false;
      const int rt = seg.item - seg.b * p.row_tiles;
      // whole: the part begins where the segment does
      int begin = 0;
      {
        Seg x;
        seg_open(p, seg.item, x);
        begin = x.tile;
      }
      const bool whole = ends && (!first_part || seg_first == begin);
      const int slot = (int)blockIdx.x * 2 + (first_part ? 0 : 1);
      first_part = false;
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        float l = l_run[hh];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const int r = warp * 16 + hh * 8 + (lane >> 2);
        if (rt * BM + r >= G * p.Sq) continue;
        if (whole) {
          const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
          char* og = (char*)p.o.ptr + (seg.b * p.o.sb + head[hh] * p.o.sh + qidx[hh] * p.o.ss) * ES;
#pragma unroll
          for (int j = 0; j < DV / 8; ++j) {
            const int c = j * 8 + (lane & 3) * 2;
            if (F32) *(float2*)(og + c * 4) = make_float2(o[j][hh * 2] * inv, o[j][hh * 2 + 1] * inv);
            else *(fa_u32*)(og + c * 2) = fa_pack2<DT>(o[j][hh * 2] * inv, o[j][hh * 2 + 1] * inv);
          }
          if ((lane & 3) == 0 && p.lse != nullptr)
            p.lse[((long long)seg.b * p.Hq + head[hh]) * p.Sq + qidx[hh]] = l == 0.f ? FA_NEG_INF : (m_run[hh] + log2f(l)) * FA_LN2;
        } else {
          float* po = p.part_o + ((long long)slot * BM + r) * DV;
#pragma unroll
          for (int j = 0; j < DV / 8; ++j) *(float2*)(po + j * 8 + (lane & 3) * 2) = make_float2(o[j][hh * 2], o[j][hh * 2 + 1]);
          if ((lane & 3) == 0) *(float2*)(p.part_ml + ((long long)slot * BM + r) * 2) = make_float2(m_run[hh], l);
        }
      }
    }
    seg_next(p, seg);
  }
  fa_grid_release();
  fa_cp_wait<0>();
#if FA_TMA
  if (failed) {
    // The copies in flight have to land before the shared memory goes to another CTA (with a limit of its own: the flag is up).
    // Buffers from `cur` on hold the tiles up to the end of the ring, those before it the next round's.
    if (tid == 0) {
      const fa_u64 start = fa_globaltimer();
      for (int i = 0; i < 2 * STAGES; ++i) {
        const int st = i < STAGES ? i : i - STAGES, ahead_by = st >= cur ? st - cur : st - cur + STAGES;
        const bool again = i == cur && k_again;
        if (t_now + ahead_by + (again ? STAGES : 0) >= t1) continue;  // (nothing was asked for)
        while (!fa_mbar_try(bars + i * 8, phase ^ (st < cur || again ? 1u : 0u)) && fa_globaltimer() - start <= FA_WAIT_LIMIT_NS / 4) {
        }
      }
    }
    if (lane == 0 && p.status != nullptr) atomicOr(p.status, FA_STATUS_WAIT_TIMEOUT);
  }
#endif
}
