// Attention of the newest Sq tokens of each request over a key / value cache in pages.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(score_mod(scale q_i.k_j) - max)  over the keys j of the request that are
//   not behind query i, not further back than the window and kept by mask_mod;  lse_i = log sum_j p_ij + max.
//
// The keys of a request lie in pages of page_size tokens that a block table lists: key j is token j % page_size of page
// table[b][j / page_size].  Query i of the Sq is token len - Sq + i, which is also the index the mods see.
//
// The G query heads of a kv head share its K and V: their G * Sq rows (query-major, row r is head r % G of query r / G) are
// cut into row tiles of 16, 32 or 64.  A segment is the keys that a row tile of a kv head of a request has to see, in tiles of FA_WN
// keys.  Memory sets the pace: K and V are read once per segment.
//
// Who takes which tiles:
//   * Lengths are known on the device only and differ, so the work is cut there: the tiles of all segments, one behind the other, are
//     dealt out evenly to the CTAs ("workers") of a grid that is resident at once.  A worker keeps the running (max, sum, O) of one
//     segment, over whose end its loads run on into the next.  A segment that lies in one worker's run is written out; of others the
//     workers leave parts (O not divided, max, sum), which fa_paged_combine_kernel merges.
//   * FA_SHORT, for tables that have room for a few tiles only: a CTA per segment, whose warps take every FA_NW-th tile and merge
//     in shared memory; one launch, and no sums over the lengths in front.
//
// The warps of a worker (FA_RG; FA_SHORT: each on its own) have 16 query rows each and share the tiles of K and V, which come by TMA
// (FA_TMA: pages that hold whole boxes of 8 keys and more, head dims of whole 128-byte columns) or in 16-byte cp.async pieces.
// Three ways to multiply:
//   * FA_FEW, up to 8 rows, which is what one new token has: S' = K Q' and O' = V' P', so that keys and columns fill the 16 rows of an
//     mma.sync and the queries its 8 columns: half the instructions of the next way, of which the queries would fill half.
//   * 16-bit, more rows: S = Q K', O = P V, 16 rows per warp.
//   * fp32: on the FMA pipes, in fp32 throughout; a lane has a key (and a part of the head dim) for the scores, columns for the values.
//
// Compile-time parameters (macros): FA_DTYPE, FA_D, FA_DV, FA_RG (1, 2, 4), FA_WN (keys of a tile: 32; fp32: 32, 16, 8), FA_STAGES, FA_TMA,
// FA_FEW, FA_FR (fp32: rows of a warp), FA_NW (FA_SHORT: warps of a CTA).
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
constexpr bool FEW = FA_FEW != 0;
constexpr bool SHORT = FA_NW > 0;
constexpr bool TMA = FA_TMA != 0;
constexpr int D = FA_D;
constexpr int DV = FA_DV;
constexpr int RG = FA_RG;
constexpr int NW = SHORT ? FA_NW : RG;  // warps of the CTA
constexpr int NT = NW * 32;
constexpr int BM = RG * 16;             // rows of a row tile
constexpr int WN = FA_WN;
constexpr int STAGES = FA_STAGES;
constexpr int ES = F32 ? 4 : 2;
constexpr int PK = TMA ? D * ES : FaTile<D, ES>::PITCH;
constexpr int PV = TMA ? DV * ES : FaTile<DV, ES>::PITCH;
constexpr int ATOMS_K = D / 64, ATOMS_V = DV / 64;  // 128-byte column groups of a row (TMA)
constexpr int K_BYTES = WN * PK, V_BYTES = WN * PV;
constexpr int PIPE_BYTES = STAGES * (K_BYTES + V_BYTES);  // of a worker
constexpr int WORKERS = SHORT ? NW : 1;                   // of a CTA
constexpr int FR = FA_FR;
// fp32: the query rows, and per warp the probabilities of a tile
constexpr int PQ = D * 4, QROWS = RG == 1 ? FR : BM;
constexpr int Q_BYTES = F32 ? QROWS * PQ + NW * FR * WN * 4 : 0;
constexpr int BAR_BYTES = TMA ? WORKERS * STAGES * 16 + 16 : 0;
constexpr int SMEM_BYTES = WORKERS * PIPE_BYTES + Q_BYTES + BAR_BYTES + (TMA ? 1024 : 0);
constexpr fa_u32 ALL = WN == 32 ? 0xffffffffu : (1u << (WN & 31)) - 1u;  // every key of a tile
// rows that the warps of a CTA merge (SHORT), in a warp's own part of the buffers
constexpr int MROWS = F32 ? FR : (FEW ? 8 : 16), MPITCH = DV + 4;

static_assert(!TMA || (!F32 && D % 64 == 0 && DV % 64 == 0), "TMA: 16-bit types, whole column groups");
static_assert(F32 || WN == 32, "tiles of 32 keys");
static_assert(!FEW || (RG == 1 && !F32), "few rows: one warp, 16-bit types");
static_assert(!SHORT || RG == 1, "a CTA per segment: up to 16 rows");
static_assert(MROWS * MPITCH * 4 <= PIPE_BYTES, "the merge of the warps fits into their buffers");

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
  if (SHORT) {
    s.tile += NW;
    return;
  }
  if (++s.tile < s.last) return;
  const bool wrap = s.hk + 1 == p.Hkv;
  s.hk = wrap ? 0 : s.hk + 1;
  if (wrap && s.item + 1 == p.B * p.row_tiles) return;  // (behind the last tile of all)
  seg_open(p, wrap ? s.item + 1 : s.item, s);
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
  constexpr int CPR = COLS * ES / 16, NL = SHORT ? 32 : NT;  // (NL threads share a tile)
  const long long at = n.page >= 0 ? (n.page * t.sb + n.hk * t.sh + n.row * t.ss) * ES : -1;
#pragma unroll 4
  for (int i = tid; i < (WN * CPR + 31) / 32 * 32; i += NL) {  // (whole warps: the shuffle)
    const int r = i / CPR, c = i - r * CPR;
    const long long row = __shfl_sync(0xffffffffu, at, r & 31);
    if (i < WN * CPR) fa_cp_async16(dst + r * PITCH + c * 16, (const char*)t.ptr + (row >= 0 ? row + c * 16 : 0), row >= 0 ? 16 : 0);
  }
}

// The address of 16-byte chunk c of row r in a tile: rows with a pad behind, or as TMA leaves them, 64 columns of all rows one behind
// the other, chunk c of 8 at c ^ (r & 7).
template <int PITCH>
__device__ __forceinline__ fa_u32 chunk_at(fa_u32 tile, int r, int c) {
  return TMA ? tile + (c >> 3) * (WN * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4) : tile + r * PITCH + c * 16;
}
__device__ __forceinline__ fa_u32 transposed(fa_u32 x) {  // an 8 x 8 matrix of 16-bit values, a row over four lanes
  fa_u32 r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// ---- the rows of a warp: scores, softmax and values of a tile --------------------------------
// HR rows per thread with NS scores each: row(h) is row h's number in the row tile, key(j) the j-th key's in the tile.
#if FA_DTYPE == FA_DT_F32
constexpr int HR = FR, NS = 1, PARTS = 32 / WN, NC = (DV + 31) / 32;
struct Rows {
  float s[HR], o[HR][NC], m[HR], l[HR];
  float* probs;  // [FR][WN]
  const float* q;
  int lane, first_row;
  __device__ __forceinline__ float& score(int h, int) { return s[h]; }
  __device__ __forceinline__ int key(int) const { return lane % WN; }
  __device__ __forceinline__ int row(int h) const { return first_row + h; }
  __device__ __forceinline__ bool idle(int h, int rows) const { return first_row + h >= rows; }
  template <class F>
  static __device__ __forceinline__ float over_keys(float v, F f) {
#pragma unroll
    for (int off = WN / 2; off > 0; off >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, off));
    return v;
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int h = 0; h < HR; ++h)
#pragma unroll
      for (int i = 0; i < NC; ++i) o[h][i] = 0.f;
  }
  __device__ __forceinline__ void rescale(int h, float c) {
#pragma unroll
    for (int i = 0; i < NC; ++i) o[h][i] *= c;
  }
  __device__ __forceinline__ void scores(const unsigned char* tile, fa_u32, int rows) {
    const unsigned char* k = tile + (lane % WN) * PK + (lane / WN) * (D / PARTS * 4);
    const float* qp = q + (lane / WN) * (D / PARTS);
#pragma unroll
    for (int h = 0; h < HR; ++h) s[h] = 0.f;
#pragma unroll 4
    for (int c = 0; c < D / PARTS / 4; ++c) {
      const float4 x = *(const float4*)(k + c * 16);
#pragma unroll
      for (int h = 0; h < HR; ++h) {
        if (HR > 4 && idle(h, rows)) break;
        const float4 y = *(const float4*)(qp + h * D + c * 4);
        s[h] = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, s[h]))));
      }
    }
#pragma unroll
    for (int h = 0; h < HR; ++h)
#pragma unroll
      for (int off = WN; off < 32; off <<= 1) s[h] += __shfl_xor_sync(0xffffffffu, s[h], off);
  }
  __device__ __forceinline__ void values(const unsigned char* tile, fa_u32, int rows) {
    __syncwarp();
#pragma unroll
    for (int h = 0; h < HR; ++h)
      if (lane < WN) probs[h * WN + lane] = s[h];
    __syncwarp();
#pragma unroll 2
    for (int j = 0; j < WN; j += 4) {
      float v[4][NC];
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < NC; ++i) v[e][i] = lane + 32 * i < DV ? *(const float*)(tile + (j + e) * PV + (lane + 32 * i) * 4) : 0.f;
#pragma unroll
      for (int h = 0; h < HR; ++h) {
        if (HR > 4 && idle(h, rows)) break;
        const float4 x = *(const float4*)(probs + h * WN + j);
#pragma unroll
        for (int i = 0; i < NC; ++i) o[h][i] = fmaf(x.x, v[0][i], fmaf(x.y, v[1][i], fmaf(x.z, v[2][i], fmaf(x.w, v[3][i], o[h][i]))));
      }
    }
  }
  // f(h, column, value) for every value of this thread
  template <class F>
  __device__ __forceinline__ void each(F f) {
#pragma unroll
    for (int h = 0; h < HR; ++h)
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (lane + 32 * i < DV) f(h, lane + 32 * i, o[h][i]);
  }
  __device__ __forceinline__ bool speaks() const { return lane == 0; }  // writes a row's max and sum
};
#elif FA_FEW
constexpr int HR = 2, NS = WN / 8;
struct Rows {
  float s[WN / 16][4], o[DV / 16][4], m[2], l[2];
  fa_u32 qf[D / 16][2];
  int lane;
  __device__ __forceinline__ float& score(int h, int j) { return s[j >> 1][(j & 1) * 2 + h]; }
  __device__ __forceinline__ int key(int j) const { return (lane >> 2) + j * 8; }
  __device__ __forceinline__ int row(int h) const { return (lane & 3) * 2 + h; }
  __device__ __forceinline__ bool idle(int h, int rows) const { return h >= rows; }
  template <class F>
  static __device__ __forceinline__ float over_keys(float v, F f) {
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, off));
    return v;
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < DV / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  }
  __device__ __forceinline__ void rescale(int h, float c) {
#pragma unroll
    for (int i = 0; i < DV / 16; ++i) {
      o[i][h] *= c;
      o[i][2 + h] *= c;
    }
  }
  __device__ __forceinline__ void scores(const unsigned char*, fa_u32 tile, int) {
#pragma unroll
    for (int i = 0; i < WN / 16; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
      for (int i = 0; i < WN / 16; ++i) {
        fa_u32 a[4];
        fa_ldsm_x4(chunk_at<PK>(tile, i * 16 + (lane & 15), kk * 2 + (lane >> 4)), a[0], a[1], a[2], a[3]);
        fa_mma16816<DT>(s[i], a, qf[kk][0], qf[kk][1]);
      }
    }
  }
  // The probabilities go in as two parts, rounded and what the rounding left: with one, bf16 results were 2.3e-3 off in place of the 1.7e-3
  // that rounding the output takes (D 128, 16384 keys).
  __device__ __forceinline__ void values(const unsigned char*, fa_u32 tile, int) {
#pragma unroll
    for (int kj = 0; kj < WN / 16; ++kj) {
      float r[4];
      fa_rest2<DT>(s[kj][0], s[kj][1], r[0], r[1]);
      fa_rest2<DT>(s[kj][2], s[kj][3], r[2], r[3]);
      const fa_u32 b0 = transposed(fa_pack2<DT>(s[kj][0], s[kj][1])), b1 = transposed(fa_pack2<DT>(s[kj][2], s[kj][3]));
      const fa_u32 c0 = transposed(fa_pack2<DT>(r[0], r[1])), c1 = transposed(fa_pack2<DT>(r[2], r[3]));
#pragma unroll
      for (int i = 0; i < DV / 16; ++i) {
        fa_u32 a[4];
        fa_ldsm_x4_t(chunk_at<PV>(tile, kj * 16 + (lane >> 4) * 8 + (lane & 7), i * 2 + ((lane >> 3) & 1)), a[0], a[1], a[2], a[3]);
        fa_mma16816<DT>(o[i], a, b0, b1);
        fa_mma16816<DT>(o[i], a, c0, c1);
      }
    }
  }
  template <class F>
  __device__ __forceinline__ void each(F f) {
#pragma unroll
    for (int i = 0; i < DV / 16; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) f(e & 1, i * 16 + (lane >> 2) + (e >> 1) * 8, o[i][e]);
  }
  __device__ __forceinline__ bool speaks() const { return lane < 4; }
};
#else
constexpr int HR = 2, NS = WN / 4;
struct Rows {
  float s[WN / 8][4], o[DV / 8][4], m[2], l[2];
  fa_u32 qf[D / 16][4];
  int lane, first_row;
  __device__ __forceinline__ float& score(int h, int j) { return s[j >> 1][h * 2 + (j & 1)]; }
  __device__ __forceinline__ int key(int j) const { return (lane & 3) * 2 + (j >> 1) * 8 + (j & 1); }
  __device__ __forceinline__ int row(int h) const { return first_row + h * 8 + (lane >> 2); }
  __device__ __forceinline__ bool idle(int h, int rows) const { return first_row + h * 8 >= rows; }
  template <class F>
  static __device__ __forceinline__ float over_keys(float v, F f) {
    v = f(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return f(v, __shfl_xor_sync(0xffffffffu, v, 2));
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < DV / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  }
  __device__ __forceinline__ void rescale(int h, float c) {
#pragma unroll
    for (int j = 0; j < DV / 8; ++j) {
      o[j][h * 2] *= c;
      o[j][h * 2 + 1] *= c;
    }
  }
  __device__ __forceinline__ void scores(const unsigned char*, fa_u32 tile, int rows) {
#pragma unroll
    for (int j = 0; j < WN / 8; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
    if (RG > 1 && first_row >= rows) return;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
      for (int nj = 0; nj < WN / 16; ++nj) {
        fa_u32 r0, r1, r2, r3;
        fa_ldsm_x4(chunk_at<PK>(tile, nj * 16 + (lane >> 4) * 8 + (lane & 7), kk * 2 + ((lane >> 3) & 1)), r0, r1, r2, r3);
        fa_mma16816<DT>(s[2 * nj], qf[kk], r0, r1);
        fa_mma16816<DT>(s[2 * nj + 1], qf[kk], r2, r3);
      }
    }
  }
  __device__ __forceinline__ void values(const unsigned char*, fa_u32 tile, int rows) {
    if (RG > 1 && first_row >= rows) return;
#pragma unroll
    for (int kj = 0; kj < WN / 16; ++kj) {
      fa_u32 a[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float(&v)[4] = s[2 * kj + (i >> 1)];
        a[i] = fa_pack2<DT>(v[(i & 1) * 2], v[(i & 1) * 2 + 1]);
      }
#pragma unroll
      for (int dj = 0; dj < DV / 16; ++dj) {
        fa_u32 r0, r1, r2, r3;
        fa_ldsm_x4_t(chunk_at<PV>(tile, kj * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), dj * 2 + (lane >> 4)), r0, r1, r2, r3);
        fa_mma16816<DT>(o[2 * dj], a, r0, r1);
        fa_mma16816<DT>(o[2 * dj + 1], a, r2, r3);
      }
    }
  }
  template <class F>
  __device__ __forceinline__ void each(F f) {
#pragma unroll
    for (int j = 0; j < DV / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) f(e >> 1, j * 8 + (lane & 3) * 2 + (e & 1), o[j][e]);
  }
  __device__ __forceinline__ bool speaks() const { return (lane & 3) == 0; }
};
#endif

struct Max {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Sum {
  __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};

// two values of an output row beside each other
__device__ __forceinline__ void put2(char* row, int c, float x, float y) {
  if (F32) *(float2*)(row + c * 4) = make_float2(x, y);
  else *(fa_u32*)(row + c * 2) = fa_pack2<DT>(x, y);
}
// 1 / sum; 0 of a row that has seen nothing, no number of a sum that is none
__device__ __forceinline__ float inverse(float l) { return l > 0.f ? 1.f / l : l; }
__device__ __forceinline__ float log_sum(float m, float l) { return l == 0.f ? FA_NEG_INF : (m + log2f(l)) * FA_LN2; }

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
  // this worker's buffers: K, V
  unsigned char* const bufs = base + (SHORT ? warp * PIPE_BYTES : 0);
  const fa_u32 sK = fa_smem_u32(bufs), sV = sK + STAGES * K_BYTES;
  [[maybe_unused]] unsigned char* const q_tile = base + WORKERS * PIPE_BYTES;
  const int row0 = SHORT ? 0 : warp * 16;  // first row of this warp
#if FA_TMA
  const fa_u32 all_bars = fa_smem_u32(base) + WORKERS * PIPE_BYTES;
  const fa_u32 bars = all_bars + (SHORT ? warp * STAGES * 16 : 0);  // K 0 .. STAGES - 1, V 0 .. STAGES - 1
  volatile int* abort_flag = (volatile int*)(base + WORKERS * (PIPE_BYTES + STAGES * 16));
  if (tid == 0) {
    for (int i = 0; i < WORKERS * 2 * STAGES; ++i) fa_mbar_init(all_bars + i * 8, 1);
    fa_mbar_init_fence();
    *abort_flag = 0;
  }
#endif
  FA_MOD_BUFS_INIT(p);
  __syncthreads();
  fa_grid_wait();

  // ---- this worker's run of tiles --------------------------------------------------------
  const int G = p.Hq / p.Hkv, items = p.B * p.row_tiles;
  int t0, t1;
  Seg seg;
  if (SHORT) {
    seg.hk = blockIdx.x % p.Hkv;
    seg_open(p, blockIdx.x / p.Hkv, seg);
    t0 = 0;
    t1 = max(seg.last - seg.tile - warp + NW - 1, 0) / NW;
    seg.tile += warp;
    if (tid == 0 && seg.hk == 0 && (p.lengths[seg.b] > p.max_len || p.lengths[seg.b] < 0) && p.status != nullptr) atomicOr(p.status, FA_STATUS_BAD_PAGE);
  } else {
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
    const int total = __shfl_sync(0xffffffffu, upto, 31) * p.Hkv;
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
  [[maybe_unused]] const int seg_first = seg.tile;  // where the first segment's part begins

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
      const int slot = p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size;
      n.row = key - slot * p.page_size;
      n.page = p.table[ahead.b * p.table_stride + slot];
    }
    // (the keys that are there go along; those whose page is none are taken out when the entry has come)
    const int left = ahead.end - ahead.tile * WN;
    n.keep = left >= WN ? ALL : left > 0 ? (1u << left) - 1u : 0u;
    --to_load;
    seg_next(p, ahead);
  };
  // takes keys out whose page is none
  auto settle = [&](Load& n) {
    const bool there = lane * p.box < WN && ((n.keep >> (lane * p.box)) & 1u);
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
    if (!SHORT && warp != 0) return;
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
  const int loader = SHORT ? lane : tid;
  auto load_k = [&](int stage, const Load& n) { load_pieces<D, PK>(p.k, sK + stage * K_BYTES, n, loader); };
  auto load_v = [&](int stage, const Load& n) { load_pieces<DV, PV>(p.v, sV + stage * V_BYTES, n, loader); };
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
  Load next, after;  // the tile STAGES ahead of the one that is computed, and the one behind it
  look_up(next);

  // ---- the tiles -------------------------------------------------------------------------
  Rows R;
  R.lane = lane;
#if FA_DTYPE == FA_DT_F32
  R.first_row = row0;
  R.q = (const float*)q_tile + row0 * D;
  R.probs = (float*)(q_tile + QROWS * PQ) + warp * FR * WN;
#elif !FA_FEW
  R.first_row = row0;
#endif
  int qpos[HR], head[HR];  // of this thread's rows: position (-1: no row), query head
  const float sc2 = p.scale * FA_LOG2E;
  bool open = false, failed = false;
  [[maybe_unused]] bool k_again = false;  // K of the tile STAGES ahead has been asked for, V not yet
  int cur = 0, rows = 0;                  // buffer of this tile; rows of the row tile
  [[maybe_unused]] fa_u32 phase = 0;
  bool first_part = true;  // of this worker
  // (a warp of a CTA with a segment of its own has to take part in its end even if it has no tile)
  auto begin_rows = [&]() {
    const int rt = seg.item - seg.b * p.row_tiles;
    rows = min(G * p.Sq - rt * BM, BM);
    const char* qb = (const char*)p.q.ptr + seg.b * p.q.sb * ES;
#pragma unroll
    for (int h = 0; h < HR; ++h) {
      const int row = rt * BM + R.row(h), i = row / G;
      head[h] = seg.hk * G + row - i * G;
      qpos[h] = i < p.Sq ? seg.pos - seg.first + i : -1;
      R.m[h] = FA_NEG_INF;
      R.l[h] = 0.f;
    }
    R.clear();
#if FA_DTYPE == FA_DT_F32
    if (RG == 1 && !SHORT) __syncwarp();
    else __syncthreads();  // (the tile before has been read)
    for (int i = tid; i < QROWS * (D / 4); i += NT) {
      const int r = i / (D / 4), c = i - r * (D / 4), row = rt * BM + r, qi = row / G;
      const float* src = (const float*)(qb + (qi * p.q.ss + (long long)(seg.hk * G + row - qi * G) * p.q.sh) * ES) + c * 4;
      *(float4*)(q_tile + r * PQ + c * 16) = qi < p.Sq ? *(const float4*)src : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if (RG == 1 && !SHORT) __syncwarp();
    else __syncthreads();
#else
    constexpr int NR = FEW ? 1 : 2;  // fragments of rows g and, where there are as many, g + 8
#pragma unroll
    for (int hh = 0; hh < NR; ++hh) {
      const int row = rt * BM + row0 + hh * 8 + (lane >> 2), i = row / G;
      const fa_u32* src = (const fa_u32*)(qb + (i * p.q.ss + (long long)(seg.hk * G + row - i * G) * p.q.sh) * ES) + (lane & 3);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        R.qf[kk][hh] = i < p.Sq ? src[kk * 8] : 0u;
        R.qf[kk][NR + hh] = i < p.Sq ? src[kk * 8 + 4] : 0u;
      }
    }
#endif
  };
  if (SHORT) begin_rows();

  [[maybe_unused]] int t_now = t0;
  for (int t = t0; t < t1; ++t) {
    t_now = t;
    if (!SHORT && !open) {
      open = true;
      begin_rows();
    }
    // ---- scores
#if FA_TMA
    failed = !fa_mbar_wait_all(bars + cur * 8, phase, abort_flag);
#else
    fa_cp_wait<2 * STAGES - 1>();
    if (RG == 1) __syncwarp();
    else __syncthreads();
#endif
    R.scores(bufs + cur * K_BYTES, sK + cur * K_BYTES, rows);
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
    look_up(after);

    const int n0 = seg.tile * WN;
    const fa_u32 kept = keep[0];
    // does any row of the tile have to look at the positions?
    const bool edge = n0 + WN - 1 > seg.pos || (p.window >= 0 && n0 < seg.end - 1 - p.window) || kept != ALL;
    const int gb = seg.b + p.b_off;
#pragma unroll
    for (int h = 0; h < HR; ++h) {
      if (R.idle(h, rows)) {  // (the rows of all lanes)
#pragma unroll
        for (int j = 0; j < NS; ++j) R.score(h, j) = 0.f;
        continue;
      }
      [[maybe_unused]] const int qp = max(qpos[h], 0), gh = head[h] + p.h_off;
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        [[maybe_unused]] const int kv = n0 + R.key(j);
        float x = R.score(h, j);
#if FA_HAS_SCORE_MOD && defined(FA_SCORE_AFFINE)
        x = fmaf(x, fa_score_mul(0.f, gb, gh, qp, kv) * sc2, fa_score_add2(0.f, gb, gh, qp, kv));
#elif FA_HAS_SCORE_MOD
        x = fa_score_mod(x * p.scale, gb, gh, qp, kv) * FA_LOG2E;
#else
        x *= sc2;
#endif
        R.score(h, j) = x;
      }
      if (edge || FA_HAS_MASK_MOD) {
#pragma unroll
        for (int j = 0; j < NS; ++j) {
          const int kv = n0 + R.key(j);
          bool see = kv <= qpos[h] && (p.window < 0 || qpos[h] - kv <= p.window) && ((kept >> R.key(j)) & 1u);
#if FA_HAS_MASK_MOD
          see = see && fa_mask_mod(gb, gh, qp, kv);
#endif
          if (!see) R.score(h, j) = FA_NEG_INF;
        }
      }
      float mx = FA_NEG_INF;
#pragma unroll
      for (int j = 0; j < NS; ++j) mx = fmaxf(mx, R.score(h, j));
      mx = Rows::over_keys(mx, Max());
      const float m_new = fmaxf(R.m[h], mx);
      const float m_use = (m_new == FA_NEG_INF) ? 0.f : m_new;
      const float corr = fa_ex2(R.m[h] - m_use);
      R.m[h] = m_new;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        const float e = fa_ex2(R.score(h, j) - m_use);
        R.score(h, j) = e;
        sum += e;
      }
      R.l[h] = R.l[h] * corr + sum;
      // (after the first tiles the maximum seldom moves)
      if (__any_sync(0xffffffffu, corr != 1.f)) R.rescale(h, corr);
    }
    // ---- values
#if FA_TMA
    failed = !fa_mbar_wait_all(bars + (STAGES + cur) * 8, phase, abort_flag);
    // Rows of keys that are not there hold whatever was in the page or the buffer, perhaps no number: 0, since a weight of 0
    // does not take that out of the product.  (Each warp for itself; all write the same.)
    if (kept != ALL) {
      for (int i = lane; i < WN * ATOMS_V * 8; i += 32) {
        const int r = (i >> 3) % WN;
        if (!((kept >> r) & 1u)) *(uint4*)(bufs + STAGES * K_BYTES + cur * V_BYTES + i * 16) = make_uint4(0, 0, 0, 0);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // (before TMA writes the buffer again)
      __syncwarp();
    }
#else
    fa_cp_wait<2 * STAGES - 1>();
    if (RG == 1) __syncwarp();
    else __syncthreads();
#endif
    R.values(bufs + STAGES * K_BYTES + cur * V_BYTES, sV + cur * V_BYTES, rows);
    if (RG == 1) __syncwarp();
    else failed = __syncthreads_or(failed) != 0;
    if (failed) break;
    if (next.any) load_v(cur, next);
    fa_cp_commit();
    k_again = false;
#pragma unroll
    for (int i = 0; i + 1 < STAGES; ++i) keep[i] = keep[i + 1];
    keep[STAGES - 1] = next.any ? next.keep : 0u;
    next = after;
    if (++cur == STAGES) {
      cur = 0;
      phase ^= 1u;
    }

    // ---- the end of the segment, or of this worker's part of it
    const bool ends = seg.tile + 1 == seg.last;
    if (!SHORT && (ends || t + 1 == t1)) {
      open = false;
      const int rt = seg.item - seg.b * p.row_tiles;
      // whole: the part begins where the segment does
      Seg x;
      seg_open(p, seg.item, x);
      const bool whole = ends && (!first_part || seg_first == x.tile);
      const int slot = (int)blockIdx.x * 2 + (first_part ? 0 : 1);
      first_part = false;
      float l[HR];
#pragma unroll
      for (int h = 0; h < HR; ++h) l[h] = F32 ? Rows::over_keys(R.l[h], Sum()) : Rows::over_keys(R.l[h], Sum());
      if (whole) {
        char* out[HR];
#pragma unroll
        for (int h = 0; h < HR; ++h) {
          const int row = rt * BM + R.row(h), i = row / G;
          out[h] = R.row(h) < rows ? (char*)p.o.ptr + (seg.b * p.o.sb + head[h] * p.o.sh + i * p.o.ss) * ES : nullptr;
          if (out[h] != nullptr && R.speaks() && p.lse != nullptr) p.lse[((long long)seg.b * p.Hq + head[h]) * p.Sq + i] = log_sum(R.m[h], l[h]);
          l[h] = inverse(l[h]);
        }
#if FA_DTYPE != FA_DT_F32 && FA_FEW
        // (transposed back: lane / 4 is the row then, and a lane has two columns beside each other)
        const int r = lane >> 2, i = (rt * BM + r) / G, hd = seg.hk * G + rt * BM + r - i * G;
        char* og = (char*)p.o.ptr + (seg.b * p.o.sb + hd * p.o.sh + i * p.o.ss) * ES;
#pragma unroll
        for (int c = 0; c < DV / 8; ++c) {
          const fa_u32 v = transposed(fa_pack2<DT>(R.o[c >> 1][(c & 1) * 2] * l[0], R.o[c >> 1][(c & 1) * 2 + 1] * l[1]));
          if (r < rows) *(fa_u32*)(og + (c * 8 + (lane & 3) * 2) * 2) = v;
        }
#elif FA_DTYPE == FA_DT_F32
        R.each([&](int h, int c, float v) {
          if (out[h] != nullptr) *(float*)(out[h] + c * 4) = v * l[h];
        });
#else
#pragma unroll
        for (int j = 0; j < DV / 8; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (out[h] != nullptr) put2(out[h], j * 8 + (lane & 3) * 2, R.o[j][h * 2] * l[h], R.o[j][h * 2 + 1] * l[h]);
#endif
      } else {
        R.each([&](int h, int c, float v) {
          if (R.row(h) < rows) p.part_o[((long long)slot * BM + R.row(h)) * DV + c] = v;
        });
#pragma unroll
        for (int h = 0; h < HR; ++h)
          if (R.row(h) < rows && R.speaks()) *(float2*)(p.part_ml + ((long long)slot * BM + R.row(h)) * 2) = make_float2(R.m[h], l[h]);
      }
    }
    seg_next(p, seg);
  }
  fa_grid_release();
  fa_cp_wait<0>();
#if FA_TMA
  if (failed) {
    // The copies in flight have to land before the shared memory goes to another CTA or is used again (with a limit of its own: the flag
    // is up).  Buffers from `cur` on hold the tiles up to the end of the ring, those before it the next round's.
    if (SHORT ? lane == 0 : tid == 0) {
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
    __syncwarp();
  }
#endif
  if (SHORT) {
    // ---- merge the warps: each leaves its rows in its own buffers, [MROWS][O | max, sum]
    float* const mine = (float*)bufs;
    __syncwarp();
    R.each([&](int h, int c, float v) { mine[R.row(h) * MPITCH + c] = v; });
#pragma unroll
    for (int h = 0; h < HR; ++h) {
      const float l = Rows::over_keys(R.l[h], Sum());
      if (R.speaks()) *(float2*)(mine + R.row(h) * MPITCH + DV) = make_float2(R.m[h], l);
    }
    __syncthreads();
    for (int i = tid; i < rows * (DV / 2); i += NT) {
      const int r = i / (DV / 2), c = (i - r * (DV / 2)) * 2, qi = r / G, h = seg.hk * G + r - qi * G;
      float m = FA_NEG_INF;
#pragma unroll
      for (int w = 0; w < NW; ++w) m = fmaxf(m, ((const float*)(base + w * PIPE_BYTES))[r * MPITCH + DV]);
      const float m_use = m == FA_NEG_INF ? 0.f : m;
      float x = 0.f, y = 0.f, l = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float* part = (const float*)(base + w * PIPE_BYTES) + r * MPITCH;
        const float2 ml = *(const float2*)(part + DV), v = *(const float2*)(part + c);
        const float f = ml.y == 0.f ? 0.f : exp2f(ml.x - m_use);  // (a warp that has seen nothing counts for nothing)
        l += f * ml.y;
        x += f * v.x;
        y += f * v.y;
      }
      const float inv = inverse(l);
      put2((char*)p.o.ptr + (seg.b * p.o.sb + h * p.o.sh + qi * p.o.ss) * ES, c, x * inv, y * inv);
      if (c == 0 && p.lse != nullptr) p.lse[((long long)seg.b * p.Hq + h) * p.Sq + qi] = log_sum(m_use, l);
    }
  }
}
