// Attention of the newest Sq tokens of each request over a key / value cache in pages.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(score_mod(scale q_i.k_j) - max)  over the keys j of the request that are
//   not behind query i, not further back than the window and kept by mask_mod;  lse_i = log sum_j p_ij + max.
//
// The keys of a request lie in pages of page_size tokens that a block table lists: key j is token j % page_size of page
// table[b][j / page_size].  Query i of the Sq is token len - Sq + i, which is also the index the mods see.
//
// The G query heads of a kv head share its K and V: their G * Sq rows (query-major, row r is head r % G of query r / G) are
// cut into row tiles of 8, 16, 24, 32 or 64.  A segment is the keys that a row tile of a kv head of a request has to see, in tiles of FA_WN
// keys.  Memory sets the pace: K and V are read once per segment.
//
// Who takes which tiles:
//   * Lengths are known on the device only and differ, so the work is cut there: the tiles of all segments, one behind the other, are
//     dealt out evenly to the CTAs ("workers") of a grid that is resident at once.  A worker goes through the segments of its run; its key
//     groups take every FA_CG-th tile, each with a running (max, sum, O) of its own, and merge through shared memory where a segment
//     ends, while the loads of the next are on their way.  A segment that lies in one worker's run is written out; of others the workers leave
//     parts (O not divided, max, sum), which fa_paged_combine_kernel merges.
//   * FA_SHORT: a CTA per segment; one launch, no parts and no sums over the lengths in front.  For tables with room for a few tiles, and for
//     many segments of middling length, where the SMs take the next segment when they have done one (the host's rule has both sides' times).
//
// Measured (us on the GPU, bf16, up to 8 rows; of the bytes of K and V): 32 requests of 1640 to 16384 keys in pages of 64, 32 / 8 heads, D 128, 1.21 GB,
// 182, 6.7 TB/s; one of 131072, 0.54 GB, 84 and 4 for the merge, 6.1 TB/s: DRAM, and 5.5 in front of the first product (the launch, the lengths,
// the table, the first tiles) and behind the last.  64 requests of 16 keys 6.3: that chain alone.  20 rows under a capped score, 16 x 4 segments of 4097 keys (floor 20.6), 43: the chains of products
// and exponentials of 8 warps per SM, more than which 255 registers a thread do not allow.
//
// CTA = FA_CG key groups of FA_RG warps with 16 query rows each.  The warps of a key group share its tiles of K and V, which come by TMA
// (FA_TMA: pages that hold whole boxes of 8 keys and more, head dims of whole 128-byte columns) or in 16-byte cp.async pieces.  That the groups
// of a CTA read beside each other counts (B32 H8 D64, 16384 keys in pages of 64: 6.6 TB/s; with a run for each warp 6.1 to 6.2).
// Three ways to multiply:
//   * FA_FEW groups of 8 rows, by one warp: S' = K Q' and O' = V' P', so that keys and columns fill the 16 rows of an mma.sync and the
//     queries its 8 columns.  For up to 8 rows, which is what one new token has, half the instructions of the next way, of which the
//     queries would fill half; for 17 to 24, three quarters, and no second warp to wait for.
//   * 16-bit, other rows: S = Q K', O = P V, 16 rows per warp.
//   * fp32: on the FMA pipes, in fp32 throughout; a lane has a key, or from 8 rows on four keys of eight rows, and a part of the head dim for the
//     scores, columns for the values.
//
// Compile-time parameters (macros): FA_DTYPE, FA_D, FA_DV, FA_RG (1, 2, 4), FA_WN (keys of a tile: 32 or 16; fp32: 32, 16, 8), FA_SLOTS, FA_TMA,
// FA_FEW (0: the other way), FA_FR (fp32: rows of a warp), FA_CG, FA_SHORT.
#pragma once
#include "fa_sm100.cuh"

struct FaPagedLaunch {
  FaPagedParams p;
#if FA_TMA
  FaTensorMap tk, tv;  // 4-d maps (D, token in page, head, page), box 128 bytes x p.box x 1 x 1, 128-byte swizzle
#endif
};

namespace fa_pg {

constexpr int DT = FA_DTYPE;
constexpr bool F32 = DT == FA_DT_F32;
constexpr bool FEW = FA_FEW != 0;
constexpr bool SHORT = FA_SHORT != 0;
constexpr bool TMA = FA_TMA != 0;
constexpr int D = FA_D;
constexpr int DV = FA_DV;
constexpr int RG = FA_RG;
constexpr int CG = FA_CG;
constexpr int NW = CG * RG;  // warps of the CTA
constexpr int NT = NW * 32;
constexpr int NQ = FA_FEW;               // groups of 8 rows
constexpr int BM = FEW ? NQ * 8 : RG * 16;  // rows of a row tile
constexpr int WN = FA_WN;
constexpr int SLOTS = FA_SLOTS;
constexpr int ES = F32 ? 4 : 2;
constexpr int PK = TMA ? D * ES : FaTile<D, ES>::PITCH;
constexpr int PV = TMA ? DV * ES : FaTile<DV, ES>::PITCH;
constexpr int ATOMS_K = D * ES / 128, ATOMS_V = DV * ES / 128;  // 128-byte column groups of a row (TMA)
// A key group's buffers are a ring of slots that take a tile of K or of V: K, V, K of the next, ..; what was in a slot has been used up, and the
// tile half a ring ahead is asked for.  Two slots and as many warps per SM as fit, so that one's products run under the
// others' softmax: a warp alone takes 1.5 us per tile (D 128, up to 8 rows), and fewer warps with more slots are slower (the host's rule).
constexpr int SLOT_BYTES = WN * (PK > PV ? PK : PV);
constexpr int PIPE_BYTES = SLOTS * SLOT_BYTES;  // of a key group
constexpr bool ODD = SLOTS % 2 != 0;
constexpr int AHEAD = (SLOTS + 1) / 2;  // tiles that are known before the first is computed
constexpr int FR = FA_FR;
// fp32: the query rows, and per warp the probabilities of a tile
constexpr int PQ = D * 4, QROWS = RG == 1 ? FR : BM;
constexpr int Q_BYTES = F32 ? QROWS * PQ + NW * FR * WN * 4 : 0;
// where the key groups merge: 32 columns of their rows at a time, and the rows' max and sum
constexpr int MROWS = F32 && RG == 1 ? FR : BM, MPITCH = 36;
constexpr int MERGE_BYTES = CG > 1 ? CG * MROWS * (MPITCH + 2) * 4 : 0;
constexpr int BAR_BYTES = TMA ? CG * SLOTS * 8 + 16 : 0;
constexpr int SMEM_BYTES = CG * PIPE_BYTES + Q_BYTES + MERGE_BYTES + BAR_BYTES + (TMA ? 1024 : 0);
constexpr float RISE = 8.f;  // (log2 units) what scores may rise before a row's maximum is looked for again
constexpr fa_u32 ALL = WN == 32 ? 0xffffffffu : (1u << (WN & 31)) - 1u;  // every key of a tile
static_assert(!TMA || (D * ES % 128 == 0 && DV * ES % 128 == 0), "TMA: whole column groups");
static_assert(F32 || WN == 32 || WN == 16, "tiles of 16 or 32 keys");
static_assert(!FEW || (RG == 1 && !F32), "few rows: one warp, 16-bit types");

__device__ __forceinline__ int divided(int n, const FaDiv& d) { return d.shift < 0 ? n : (int)(__umulhi((fa_u32)n, d.mul) >> d.shift); }

// A segment, and the tile of it that is next.
struct Seg {
  int item, hk, b;
  int first;  // first query of the row tile, and its position among the request's tokens
  int pos;
  int begin, end;  // keys in front of begin are out of every row's window, those from end on are behind every row
  int tile, last;  // tiles of WN keys, first and one beyond the last
  const int* pages;  // row of the block table
};
__device__ __forceinline__ void seg_open(const FaPagedParams& p, int item, Seg& s) {
  s.item = item;
  s.b = divided(item, p.by_tiles);
  s.pages = p.table + s.b * p.table_stride;
  const int rt = item - s.b * p.row_tiles;
  const int len = min(max(p.lengths[s.b], 0), p.max_len);
  s.first = divided(rt * BM, p.by_group);
  const int final = min(p.Sq, divided((rt + 1) * BM - 1, p.by_group) + 1) - 1;  // its last query
  s.pos = len - p.Sq + s.first;
  s.end = max(len - p.Sq + final + 1, 0);
  s.begin = p.window < 0 ? 0 : max(s.pos - p.window, 0);
  s.tile = s.begin / WN;
  s.last = max((s.end + WN - 1) / WN, s.tile + 1);  // (at least one: somebody has to write a row that sees nothing)
}
// tiles of item `item`'s segments
__device__ __forceinline__ int seg_tiles(const FaPagedParams& p, int item) {
  Seg s;
  seg_open(p, item, s);
  return s.last - s.tile;
}
// n tiles on, over the ends of segments
__device__ __forceinline__ void seg_advance(const FaPagedParams& p, Seg& s, int n) {
  s.tile += n;
#pragma unroll 1
  while (!SHORT && s.tile >= s.last) {
    const int over = s.tile - s.last;
    if (++s.hk == p.Hkv) {
      s.hk = 0;
      if (s.item + 1 == p.B * p.row_tiles) return;  // (behind the last tile of all)
      seg_open(p, s.item + 1, s);
    } else {
      s.tile = s.begin / WN;
    }
    s.tile += over;
  }
}

// K and V of a tile on their way: where its keys are.  Every lane of every warp has the same but for its own key (TMA: box).
struct Load {
  bool any;     // there is a tile
  bool looked;  // this lane has a page to look at
  int hk;
  int page;     // this lane's, or -1: no such key, or no such page
  int row;      // token in it
  fa_u32 keep;  // keys of the tile that are there, bit by bit
  fa_u32 boxes; // lanes with a page
};

// The rows of a tile in 16-byte pieces, those that are not there as zeros
template <int COLS, int PITCH>
__device__ __forceinline__ void load_pieces(const FaTensor& t, fa_u32 dst, const Load& n, int tid) {
  constexpr int CPR = COLS * ES / 16, NL = RG * 32;  // (the threads of a key group)
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
  static __device__ __forceinline__ void over_keys(float (&v)[HR], F f) {
#pragma unroll
    for (int off = WN / 2; off > 0; off >>= 1)
#pragma unroll
      for (int h = 0; h < HR; ++h) v[h] = f(v[h], __shfl_xor_sync(0xffffffffu, v[h], off));
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
  // Eight rows and more: what a lane reads of shared memory sets the pace (16 bytes of each lane take four cycles, also where lanes read the same), so a lane
  // takes eight rows and four keys at a time, 12 reads for 64 two-value products where one key takes 17 for 32, of 1 in 128 / WN pieces of the
  // head dim; then the lanes of a key swap and add what they have.  (64 segments of 4096 keys, D 128, one key / four: 8 rows 99 / 66 us, 16 rows 171 / 117,
  // 28 rows 319 / 221; D 64, 8 rows 58 / 41; D 256, 16 rows 383 / 268.)  Not unrolled: twice is slower at D 256, 268 / 297, and the same elsewhere.
  __device__ __forceinline__ void scores_by_four(const unsigned char* tile, int rows) {
    constexpr int B4 = WN / 4, P = 32 / B4;
    const int p0 = lane / B4, r = lane % B4;
    // (the pieces of the lanes that are served together lie in different banks)
    const int p = P == 4 ? p0 : P == 8 ? (p0 & 1) * 4 + (p0 >> 1) : (p0 & 3) * 2 + ((p0 >> 2) & 1) + (p0 & 8);
#pragma unroll
    for (int h0 = 0; h0 < HR; h0 += 8) {
      fa_u64 acc[8][4];
#pragma unroll
      for (int h = 0; h < 8; ++h) acc[h][0] = acc[h][1] = acc[h][2] = acc[h][3] = 0ull;
      if (!idle(h0, rows)) {
        const bool all = !idle(h0 + 4, rows);
#pragma unroll 1
        for (int c = p; c < D / 4; c += P) {
          ulonglong2 x[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) x[k] = *(const ulonglong2*)(tile + chunk_at<PK>(0, r + k * B4, c));
#pragma unroll
          for (int h = 0; h < 8; ++h) {
            if (h == 4 && !all) break;
            const ulonglong2 y = *(const ulonglong2*)(q + (h0 + h) * D + c * 4);
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[h][k] = fa_fma2(x[k].y, y.y, fa_fma2(x[k].x, y.x, acc[h][k]));
          }
        }
        __syncwarp();
      }
      const bool upper = (lane & (WN / 2)) != 0, odd = (lane & B4) != 0;
#pragma unroll
      for (int h = 0; h < 8; ++h) {
        float t[4], u[2];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float e, o2;
          fa_f2_unpack(acc[h][k], e, o2);
          t[k] = e + o2;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) u[k] = (upper ? t[k + 2] : t[k]) + __shfl_xor_sync(0xffffffffu, upper ? t[k] : t[k + 2], WN / 2);
        s[h0 + h] = (odd ? u[1] : u[0]) + __shfl_xor_sync(0xffffffffu, odd ? u[0] : u[1], B4);
#pragma unroll
        for (int off = WN; off < 32; off <<= 1) s[h0 + h] += __shfl_xor_sync(0xffffffffu, s[h0 + h], off);
      }
    }
  }
  __device__ __forceinline__ void scores(const unsigned char* tile, fa_u32, int rows) {
    if constexpr (HR >= 8) {
      scores_by_four(tile, rows);
      return;
    }
    // (four sums for a product, two to an instruction: a chain of D / PARTS additions would be waited for)
    const float* qp = q + (lane / WN) * (D / PARTS);
    const int r = lane % WN, c0 = (lane / WN) * (D / PARTS / 4);
    fa_u64 acc[HR][2];
#pragma unroll
    for (int h = 0; h < HR; ++h) acc[h][0] = acc[h][1] = 0ull;
#pragma unroll 4
    for (int c = 0; c < D / PARTS / 4; ++c) {
      const ulonglong2 x = *(const ulonglong2*)(tile + chunk_at<PK>(0, r, c0 + c));
#pragma unroll
      for (int h = 0; h < HR; ++h) {
        if (HR > 4 && idle(h, rows)) break;
        const ulonglong2 y = *(const ulonglong2*)(qp + h * D + c * 4);
        acc[h][0] = fa_fma2(x.x, y.x, acc[h][0]);
        acc[h][1] = fa_fma2(x.y, y.y, acc[h][1]);
      }
    }
#pragma unroll
    for (int h = 0; h < HR; ++h) {
      float x0, x1, x2, x3;
      fa_f2_unpack(acc[h][0], x0, x1);
      fa_f2_unpack(acc[h][1], x2, x3);
      s[h] = (x0 + x1) + (x2 + x3);
    }
#pragma unroll
    for (int off = WN; off < 32; off <<= 1)
#pragma unroll
      for (int h = 0; h < HR; ++h) s[h] += __shfl_xor_sync(0xffffffffu, s[h], off);
  }
  __device__ __forceinline__ void values(const unsigned char* tile, fa_u32, int rows) {
    __syncwarp();
#pragma unroll
    for (int h = 0; h < HR; ++h)
      if (lane < WN) probs[h * WN + lane] = s[h];
    __syncwarp();
    // (few rows: even and odd keys apart, two to an instruction)
    constexpr bool APART = HR * NC <= 16;
    fa_u64 acc[APART ? HR : 1][APART ? NC : 1];
    if (APART) {
#pragma unroll
      for (int h = 0; h < (APART ? HR : 1); ++h)
#pragma unroll
        for (int i = 0; i < (APART ? NC : 1); ++i) acc[h][i] = 0ull;
    }
#pragma unroll 2
    for (int j = 0; j < WN; j += 4) {
      float v[4][NC];
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          const int c = lane + 32 * i;
          v[e][i] = c < DV ? *(const float*)(tile + chunk_at<PV>(0, j + e, c >> 2) + (c & 3) * 4) : 0.f;
        }
#pragma unroll
      for (int h = 0; h < HR; ++h) {
        if (HR > 4 && idle(h, rows)) break;
        if constexpr (APART) {
          const ulonglong2 x = *(const ulonglong2*)(probs + h * WN + j);
#pragma unroll
          for (int i = 0; i < NC; ++i) acc[h][i] = fa_fma2(x.y, fa_f2(v[2][i], v[3][i]), fa_fma2(x.x, fa_f2(v[0][i], v[1][i]), acc[h][i]));
        } else {
          const float4 x = *(const float4*)(probs + h * WN + j);
#pragma unroll
          for (int i = 0; i < NC; ++i) o[h][i] = fmaf(x.x, v[0][i], fmaf(x.y, v[1][i], fmaf(x.z, v[2][i], fmaf(x.w, v[3][i], o[h][i]))));
        }
      }
    }
    if constexpr (APART) {
#pragma unroll
      for (int h = 0; h < HR; ++h)
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          float x, y;
          fa_f2_unpack(acc[h][i], x, y);
          o[h][i] += x + y;
        }
    }
  }
  // f(h, column, value) for every value of this thread in columns 32 i ..
  template <class F>
  __device__ __forceinline__ void each(int i, F f) {
#pragma unroll
    for (int h = 0; h < HR; ++h)
      if (lane + 32 * i < DV) f(h, lane + 32 * i, o[h][i]);
  }
  __device__ __forceinline__ bool speaks() const { return lane == 0; }  // writes a row's max and sum
};
#elif FA_FEW
constexpr int HR = 2 * NQ, NS = WN / 8;
struct Rows {
  float s[WN / 16][NQ][4], o[DV / 16][NQ][4], m[HR], l[HR];
  fa_u32 qf[D / 16][NQ][2];
  int lane;
  __device__ __forceinline__ float& score(int h, int j) { return s[j >> 1][h >> 1][(j & 1) * 2 + (h & 1)]; }
  __device__ __forceinline__ int key(int j) const { return (lane >> 2) + j * 8; }
  __device__ __forceinline__ int row(int h) const { return (h >> 1) * 8 + (lane & 3) * 2 + (h & 1); }
  __device__ __forceinline__ bool idle(int h, int rows) const { return (h >> 1) * 8 + (h & 1) >= rows; }
  template <class F>
  static __device__ __forceinline__ void over_keys(float (&v)[HR], F f) {
#pragma unroll
    for (int off = 4; off < 32; off <<= 1)
#pragma unroll
      for (int h = 0; h < HR; ++h) v[h] = f(v[h], __shfl_xor_sync(0xffffffffu, v[h], off));
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < DV / 16; ++i)
#pragma unroll
      for (int q = 0; q < NQ; ++q) o[i][q][0] = o[i][q][1] = o[i][q][2] = o[i][q][3] = 0.f;
  }
  __device__ __forceinline__ void rescale(int h, float c) {
#pragma unroll
    for (int i = 0; i < DV / 16; ++i) {
      o[i][h >> 1][h & 1] *= c;
      o[i][h >> 1][2 + (h & 1)] *= c;
    }
  }
  __device__ __forceinline__ void scores(const unsigned char*, fa_u32 tile, int) {
#pragma unroll
    for (int i = 0; i < WN / 16; ++i)
#pragma unroll
      for (int q = 0; q < NQ; ++q) s[i][q][0] = s[i][q][1] = s[i][q][2] = s[i][q][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
      for (int i = 0; i < WN / 16; ++i) {
        fa_u32 a[4];
        fa_ldsm_x4(chunk_at<PK>(tile, i * 16 + (lane & 15), kk * 2 + (lane >> 4)), a[0], a[1], a[2], a[3]);
#pragma unroll
        for (int q = 0; q < NQ; ++q) fa_mma16816<DT>(s[i][q], a, qf[kk][q][0], qf[kk][q][1]);
      }
    }
  }
  // Up to 8 rows the probabilities go in as two parts, rounded and what the rounding left: with one, bf16 results were 2.3e-3 off in place of the
  // 1.7e-3 that rounding the output takes (D 128, 16384 keys).  With 17 to 24 rows the products would cost time: 8 % at D 64, 10 % at D 128 over calls of 100 to
  // 131072 keys (20 rows, 32 x 8 segments of 8192, D 128: 179 us, 203 in two parts), for an error of 2.1e-4 in place of 2.9e-4 (fp16).
  __device__ __forceinline__ void values(const unsigned char*, fa_u32 tile, int) {
    constexpr bool TWO = NQ == 1;
#pragma unroll
    for (int kj = 0; kj < WN / 16; ++kj) {
      fa_u32 b[NQ][2], rest[2];
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int e = 0; e < 2; ++e) b[q][e] = transposed(fa_pack2<DT>(s[kj][q][2 * e], s[kj][q][2 * e + 1]));
      if (TWO) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float r0, r1;
          fa_rest2<DT>(s[kj][0][2 * e], s[kj][0][2 * e + 1], r0, r1);
          rest[e] = transposed(fa_pack2<DT>(r0, r1));
        }
      }
#pragma unroll
      for (int i = 0; i < DV / 16; ++i) {
        fa_u32 a[4];
        fa_ldsm_x4_t(chunk_at<PV>(tile, kj * 16 + (lane >> 4) * 8 + (lane & 7), i * 2 + ((lane >> 3) & 1)), a[0], a[1], a[2], a[3]);
#pragma unroll
        for (int q = 0; q < NQ; ++q) fa_mma16816<DT>(o[i][q], a, b[q][0], b[q][1]);
        if (TWO) fa_mma16816<DT>(o[i][0], a, rest[0], rest[1]);
      }
    }
  }
  template <class F>
  __device__ __forceinline__ void each(int b, F f) {
#pragma unroll
    for (int i = 2 * b; i < 2 * b + 2 && i < DV / 16; ++i)
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) f(2 * q + (e & 1), i * 16 + (lane >> 2) + (e >> 1) * 8, o[i][q][e]);
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
  static __device__ __forceinline__ void over_keys(float (&v)[HR], F f) {
#pragma unroll
    for (int off = 1; off < 4; off <<= 1)
#pragma unroll
      for (int h = 0; h < HR; ++h) v[h] = f(v[h], __shfl_xor_sync(0xffffffffu, v[h], off));
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
  // Probabilities in two parts up to 16 rows, as the decode kernel has them (9 to 16: 3 % of the time at D 64 to 256 on average, 6 at D 32, 11 at most; 16 rows,
  // 32 x 8 segments of 8192 keys, D 128 177 / 180 us, one request of 131072, D 64 52.5 / 53.2); not with more, where they would cost 4 to 9 % (28 rows,
  // 32 x 8 segments of 8192, D 128: 217 / 242) and one part is what the forward kernel has.
  __device__ __forceinline__ void values(const unsigned char*, fa_u32 tile, int rows) {
    constexpr bool TWO = RG == 1;
    if (RG > 1 && first_row >= rows) return;
#pragma unroll
    for (int kj = 0; kj < WN / 16; ++kj) {
      fa_u32 a[4], rest[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float(&v)[4] = s[2 * kj + (i >> 1)];
        a[i] = fa_pack2<DT>(v[(i & 1) * 2], v[(i & 1) * 2 + 1]);
        if (TWO) {
          float x, y;
          fa_rest2<DT>(v[(i & 1) * 2], v[(i & 1) * 2 + 1], x, y);
          rest[i] = fa_pack2<DT>(x, y);
        }
      }
#pragma unroll
      for (int dj = 0; dj < DV / 16; ++dj) {
        fa_u32 r0, r1, r2, r3;
        fa_ldsm_x4_t(chunk_at<PV>(tile, kj * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), dj * 2 + (lane >> 4)), r0, r1, r2, r3);
        fa_mma16816<DT>(o[2 * dj], a, r0, r1);
        fa_mma16816<DT>(o[2 * dj + 1], a, r2, r3);
        if (TWO) {
          fa_mma16816<DT>(o[2 * dj], rest, r0, r1);
          fa_mma16816<DT>(o[2 * dj + 1], rest, r2, r3);
        }
      }
    }
  }
  template <class F>
  __device__ __forceinline__ void each(int b, F f) {
#pragma unroll
    for (int j = 4 * b; j < 4 * b + 4 && j < DV / 8; ++j)
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

// a value of an output row
__device__ __forceinline__ void put1(char* row, int c, float x) {
  if (F32) *(float*)(row + c * 4) = x;
  else *(fa_u16*)(row + c * 2) = (fa_u16)fa_pack2<DT>(x, 0.f);
}
// two beside each other
__device__ __forceinline__ void put2(char* row, int c, float x, float y) {
  if (F32) *(float2*)(row + c * 4) = make_float2(x, y);
  else *(fa_u32*)(row + c * 2) = fa_pack2<DT>(x, y);
}
// 1 / sum; 0 of a row that has seen nothing, no number of a sum that is none
__device__ __forceinline__ float inverse(float l) { return l > 0.f ? 1.f / l : l; }
__device__ __forceinline__ float log_sum(float m, float l) { return l == 0.f ? FA_NEG_INF : (m + log2f(l)) * FA_LN2; }

// The warps of a key group wait for one another; true where any of their threads says so.
__device__ __forceinline__ bool group_sync(int cg, bool v) {
  if (RG == 1) {
    __syncwarp();
    return v;
  }
  if (CG == 1) return __syncthreads_or(v) != 0;
  int r;
  asm volatile(
      "{\n\t.reg .pred a, b;\n\t"
      "setp.ne.s32 a, %1, 0;\n\t"
      "barrier.cta.red.or.pred b, %2, %3, a;\n\t"
      "selp.s32 %0, 1, 0, b;\n\t}"
      : "=r"(r) : "r"((int)v), "r"(cg + 1), "n"(RG * 32) : "memory");
  return r != 0;
}

}  // namespace fa_pg

extern "C" __global__ void __launch_bounds__(fa_pg::NT, FA_CTAS) fa_paged_kernel(const __grid_constant__ FaPagedLaunch L) {
  using namespace fa_pg;
  const FaPagedParams& p = L.p;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  if (fa_dynamic_smem_size() < (fa_u32)SMEM_BYTES || blockDim.x != NT) {
    if (threadIdx.x == 0 && p.status != nullptr) atomicOr(p.status, FA_STATUS_BAD_LAUNCH);
    return;
  }
  unsigned char* const base = TMA ? smem_raw + ((1024u - (fa_smem_u32(smem_raw) & 1023u)) & 1023u) : smem_raw;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rg = warp % RG, cg = warp / RG;
  // [rings of the key groups | fp32: queries, probabilities | merge | barriers]
  unsigned char* const bufs = base + cg * PIPE_BYTES;
  const fa_u32 ring = fa_smem_u32(bufs);
  [[maybe_unused]] unsigned char* const q_tile = base + CG * PIPE_BYTES;
  [[maybe_unused]] float* const merge = (float*)(base + CG * PIPE_BYTES + Q_BYTES);  // [CG][MROWS][MPITCH]
  [[maybe_unused]] float2* const merge_ml = (float2*)(merge + CG * MROWS * MPITCH);  // [MROWS][CG]
  const int row0 = rg * 16;  // first row of this warp
#if FA_TMA
  const fa_u32 all_bars = fa_smem_u32(base) + CG * PIPE_BYTES + Q_BYTES + MERGE_BYTES;
  const fa_u32 bars = all_bars + cg * SLOTS * 8;  // one per slot
  volatile int* abort_flag = (volatile int*)(base + CG * (PIPE_BYTES + SLOTS * 8) + Q_BYTES + MERGE_BYTES);
  if (tid == 0) {
    for (int i = 0; i < CG * SLOTS; ++i) fa_mbar_init(all_bars + i * 8, 1);
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
    t1 = seg.last - seg.tile;
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
    const int per = (total + p.workers - 1) / p.workers;
    if (blockIdx.x == 0 && warp == 0) {  // for the kernel that merges
      int at = upto - own;
#pragma unroll 1
      for (int i = i0; i < i1; ++i) {
        p.plan[i] = at;
        at += seg_tiles(p, i);
      }
      if (lane == 31) p.plan[items] = upto;
      // a length that the table has no room for
      bool beyond = false;
#pragma unroll 1
      for (int i = lane; i < p.B; i += 32) beyond |= p.lengths[i] > p.max_len || p.lengths[i] < 0;
      if (beyond && p.status != nullptr) atomicOr(p.status, FA_STATUS_BAD_PAGE);
    }
    t0 = (int)min((long long)blockIdx.x * per, (long long)total);
    t1 = min(t0 + per, total);
    if (t0 >= t1) return;
    const int from = __popc(__ballot_sync(0xffffffffu, (long long)upto * p.Hkv <= t0));  // the lane whose run has tile t0
    int item = __shfl_sync(0xffffffffu, i0, from), before = __shfl_sync(0xffffffffu, upto - own, from);
    seg_open(p, item, seg);
#pragma unroll 1
    while (t0 >= (before + seg.last - seg.tile) * p.Hkv) {
      before += seg.last - seg.tile;
      seg_open(p, ++item, seg);
    }
    const int n = seg.last - seg.tile, off = t0 - before * p.Hkv;
    seg.hk = off / n;
    seg.tile += off - seg.hk * n;
  }

  // ---- loads -----------------------------------------------------------------------------
  Seg ahead = seg;  // of the tile that is asked for next: every CG-th of the run
  int to_load = max(t1 - t0 - cg + CG - 1, 0) / CG;
  if (to_load > 0) seg_advance(p, ahead, cg);
  // looks the next tile's pages up
  auto look_up = [&](Load& n) {
    n.any = to_load > 0;
    n.page = -1;
    n.looked = false;
    if (!n.any) return;
    const int key = ahead.tile * WN + lane * p.box;  // (box: 1 without TMA)
    const bool there = lane * p.box < WN && key < ahead.end && key + p.box > ahead.begin;  // (pages out of the window may be gone)
    n.hk = ahead.hk;
    n.looked = there;
    if (there) {
      const int slot = divided(key, p.by_page);
      n.row = key - slot * p.page_size;
      n.page = ahead.pages[slot];
    }
    // (the keys that are there go along; those whose page is none are taken out when the entry has come)
    const int left = ahead.end - ahead.tile * WN;
    n.keep = left >= WN ? ALL : left > 0 ? (1u << left) - 1u : 0u;
    const int gone = ahead.begin - ahead.tile * WN;  // (below WN)
    if (gone > 0) n.keep &= ALL << gone;
    if (--to_load > 0) seg_advance(p, ahead, CG);
  };
  // takes keys out whose page is none
  auto settle = [&](Load& n) {
    const bool bad = n.looked && (n.page < 0 || n.page >= p.num_pages);
    if (bad) n.page = -1;
    n.boxes = __ballot_sync(0xffffffffu, n.page >= 0);
    fa_u32 out = __ballot_sync(0xffffffffu, bad);
    if (out != 0) {
      if (lane == 0 && p.status != nullptr) atomicOr(p.status, FA_STATUS_BAD_PAGE);
#pragma unroll 1
      for (; out != 0; out &= out - 1) {
        const int first = (__ffs(out) - 1) * p.box;
        n.keep &= ~((p.box >= 32 ? 0xffffffffu : (1u << p.box) - 1u) << first);
      }
    }
  };
#if FA_TMA
  auto load = [&](const FaTensorMap* map, fa_u32 dst, fa_u32 bar, int atoms, const Load& n) {
    if (rg != 0) return;
    if (lane == 0) fa_mbar_expect_tx(bar, __popc(n.boxes) * p.box * 128 * atoms);
    __syncwarp();
    if (n.page >= 0) {
      for (int a = 0; a < atoms; ++a)
        fa_tma_load_4d(dst + a * (WN * 128) + lane * p.box * 128, map, bar, a * (128 / ES), n.row, n.hk, n.page);
    }
  };
  auto load_k = [&](int slot, const Load& n) { load(&L.tk, ring + slot * SLOT_BYTES, bars + slot * 8, ATOMS_K, n); };
  auto load_v = [&](int slot, const Load& n) { load(&L.tv, ring + slot * SLOT_BYTES, bars + slot * 8, ATOMS_V, n); };
#else
  const int loader = rg * 32 + lane;
  auto load_k = [&](int slot, const Load& n) { load_pieces<D, PK>(p.k, ring + slot * SLOT_BYTES, n, loader); };
  auto load_v = [&](int slot, const Load& n) { load_pieces<DV, PV>(p.v, ring + slot * SLOT_BYTES, n, loader); };
#endif

  fa_u32 keep[AHEAD];
  Load pending, next, after;  // the tile whose V is asked for next, the one whose K is, and the one behind that
  pending.any = next.any = after.any = false;
  int asked = 0;  // slots asked for
#pragma unroll 1
  for (int st = 0;; ++st) {  // (not unrolled: its instructions come from memory before the first tile does)
    look_up(next);
    if (st == AHEAD) break;
#pragma unroll
    for (int i = 0; i + 1 < AHEAD; ++i) keep[i] = keep[i + 1];
    keep[AHEAD - 1] = 0;
    if (next.any) {
      settle(next);
      keep[AHEAD - 1] = next.keep;
      load_k(2 * st, next);
    }
    fa_cp_commit();
    if (2 * st + 1 < SLOTS) {
      if (next.any) load_v(2 * st + 1, next);
      fa_cp_commit();
    }
    asked += next.any ? (2 * st + 1 < SLOTS ? 2 : 1) : 0;
    pending = next;
  }

  // ---- the segments ----------------------------------------------------------------------
  Rows R;
  R.lane = lane;
#if FA_DTYPE == FA_DT_F32
  R.first_row = row0;
  R.q = (const float*)q_tile + row0 * D;
  R.probs = (float*)(q_tile + QROWS * PQ) + warp * FR * WN;
#elif !FA_FEW
  R.first_row = row0;
#endif
  const float sc2 = p.scale * FA_LOG2E;
  bool failed = false;
  int slot = 0;  // that is used next
  [[maybe_unused]] fa_u32 phase = 0;
  [[maybe_unused]] int n_used = 0;  // slots
  // a slot's tile has come: its number; then it is used up, and the next is looked at
  auto arrived = [&]() {
#if FA_TMA
    failed = !fa_mbar_wait_all(bars + slot * 8, phase, abort_flag);
#else
    fa_cp_wait<SLOTS - 1>();
    group_sync(cg, false);
#endif
    return slot;
  };
  auto used = [&]() {
    failed = group_sync(cg, failed);
    if (++slot == SLOTS) {
      slot = 0;
      phase ^= 1u;
    }
    ++n_used;
  };

  if (SHORT) fa_grid_release();
#if FA_DTYPE != FA_DT_F32
  // the queries of a segment: rows g, g + 8, .. of the row tile, g = lane / 4
  auto load_q = [&]() {
    const int rt = seg.item - seg.b * p.row_tiles;
    const char* qb = (const char*)p.q.ptr + seg.b * p.q.sb * ES;
#pragma unroll
    for (int q = 0; q < (FEW ? NQ : 2); ++q) {
      const int row = rt * BM + row0 + q * 8 + (lane >> 2), i = divided(row, p.by_group);
      const fa_u32* src = (const fa_u32*)(qb + (i * p.q.ss + (long long)(seg.hk * G + row - i * G) * p.q.sh) * ES) + (lane & 3);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const fa_u32 lo = i < p.Sq ? src[kk * 8] : 0u, hi = i < p.Sq ? src[kk * 8 + 4] : 0u;
#if FA_FEW
        R.qf[kk][q][0] = lo;
        R.qf[kk][q][1] = hi;
#else
        R.qf[kk][q] = lo;
        R.qf[kk][2 + q] = hi;
#endif
      }
    }
  };
  load_q();
#endif

#pragma unroll 1
  for (int t = t0; t < t1;) {
    // this worker's part of the segment: tiles seg.tile .. part_end - 1
    const int part_end = min(seg.last, seg.tile + (t1 - t)), rt = seg.item - seg.b * p.row_tiles;
    const int rows = min(G * p.Sq - rt * BM, BM);
    int qpos[HR], head[HR];  // of this thread's rows: position (-1: no row), query head
#pragma unroll
    for (int h = 0; h < HR; ++h) {
      const int row = rt * BM + R.row(h), i = divided(row, p.by_group);
      head[h] = seg.hk * G + row - i * G;
      qpos[h] = i < p.Sq ? seg.pos - seg.first + i : -1;
      R.m[h] = FA_NEG_INF;
      R.l[h] = 0.f;
    }
    R.clear();
#if FA_DTYPE == FA_DT_F32
    const char* qb = (const char*)p.q.ptr + seg.b * p.q.sb * ES;
    __syncthreads();  // (the rows of the segment before have been read)
    for (int i = tid; i < QROWS * (D / 4); i += NT) {
      const int r = i / (D / 4), c = i - r * (D / 4), row = rt * BM + r, qi = divided(row, p.by_group);
      const float* src = (const float*)(qb + (qi * p.q.ss + (long long)(seg.hk * G + row - qi * G) * p.q.sh) * ES) + c * 4;
      *(float4*)(q_tile + r * PQ + c * 16) = qi < p.Sq ? *(const float4*)src : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __syncthreads();
#endif

    // ---- the tiles of this key group (a group whose wait has run out leaves them out, but takes part in the merges)
#pragma unroll 1
    for (int tile = seg.tile + (CG - (t - t0) % CG + cg) % CG; tile < part_end && !failed; tile += CG) {
      // (its pages were looked up a tile ago; here, so that nothing waits for them when a slot is free)
      if (next.any) settle(next);
      int at = arrived();
      R.scores(bufs + at * SLOT_BYTES, ring + at * SLOT_BYTES, rows);
      used();
      if (failed) break;
      // the slot takes what is SLOTS behind: V of the tile whose K is on its way (odd rings), or K of the next
      if (ODD) {
        if (pending.any) load_v(at, pending);
        asked += pending.any;
      } else {
        if (next.any) load_k(at, next);
        asked += next.any;
      }
      fa_cp_commit();
      look_up(after);

      const int n0 = tile * WN;
      const fa_u32 kept = keep[0];
      // does any row of the tile have to look at the positions?
      const bool edge = n0 + WN - 1 > seg.pos || (p.window >= 0 && n0 < seg.end - 1 - p.window) || kept != ALL;
      const int gb = seg.b + p.b_off;
      // Scores are taken relative to a maximum that need not be the present one: as long as none is more than 2^RISE times what a row's
      // maximum was when it was last looked for, probabilities stay in range, and one vote takes the place of the lanes' search for it (and of
      // the correction of O), which a warp would wait for in every tile.
      float top[HR];
      bool rises = false;
#pragma unroll
      for (int h = 0; h < HR; ++h) {
        top[h] = FA_NEG_INF;
        if (R.idle(h, rows)) continue;  // (the rows of all lanes)
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
#pragma unroll
        for (int j = 0; j < NS; ++j) top[h] = fmaxf(top[h], R.score(h, j));
        rises |= top[h] > R.m[h] + RISE;
      }
      if (__any_sync(0xffffffffu, rises)) {
        Rows::over_keys(top, Max());
#pragma unroll
        for (int h = 0; h < HR; ++h) {
          const float m_new = fmaxf(R.m[h], top[h]);
          const float corr = fa_ex2(R.m[h] - (m_new == FA_NEG_INF ? 0.f : m_new));
          R.m[h] = m_new;
          R.l[h] *= corr;
          R.rescale(h, corr);
        }
      }
#pragma unroll
      for (int h = 0; h < HR; ++h) {
        if (R.idle(h, rows)) {
#pragma unroll
          for (int j = 0; j < NS; ++j) R.score(h, j) = 0.f;
          continue;
        }
        const float m = R.m[h] == FA_NEG_INF ? 0.f : R.m[h];
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < NS; ++j) {
          const float e = fa_ex2(R.score(h, j) - m);
          R.score(h, j) = e;
          sum += e;
        }
        R.l[h] += sum;
      }

      at = arrived();
#if FA_TMA
      // Rows of keys that are not there hold whatever was in the page or the buffer, perhaps no number: 0, since a weight of 0
      // does not take that out of the product.  (Each warp for itself; all write the same.)
      if (kept != ALL) {
        for (int i = lane; i < WN * ATOMS_V * 8; i += 32) {
          const int r = (i >> 3) % WN;
          if (!((kept >> r) & 1u)) *(uint4*)(bufs + at * SLOT_BYTES + i * 16) = make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // (before TMA writes the buffer again)
        __syncwarp();
      }
#endif
      R.values(bufs + at * SLOT_BYTES, ring + at * SLOT_BYTES, rows);
      used();
      if (failed) break;
      if (ODD) {
        if (next.any) load_k(at, next);
        asked += next.any;
        pending = next;
      } else {
        if (next.any) load_v(at, next);
        asked += next.any;
      }
      fa_cp_commit();
#pragma unroll
      for (int i = 0; i + 1 < AHEAD; ++i) keep[i] = keep[i + 1];
      keep[AHEAD - 1] = next.any ? next.keep : 0u;
      next = after;
    }

    // ---- the end of the segment, or of this worker's part of it: written out if the part is the segment
    const bool whole = SHORT || (seg.tile == seg.begin / WN && part_end == seg.last);
    const int part = (int)blockIdx.x * 2 + (t == t0 ? 0 : 1), b = seg.b, hk = seg.hk;
    t += part_end - seg.tile;
    if (t < t1) {
      seg_advance(p, seg, part_end - seg.tile);
#if FA_DTYPE != FA_DT_F32
      load_q();  // (on their way during the merge)
#endif
    }
    float* const part_o = p.part_o + (long long)part * BM * DV;
    float* const part_ml = p.part_ml + (long long)part * BM * 2;
    Rows::over_keys(R.l, Sum());
    if (CG > 1) {
#pragma unroll
      for (int h = 0; h < HR; ++h)
        if (R.speaks()) merge_ml[R.row(h) * CG + cg] = make_float2(R.m[h], R.l[h]);
#pragma unroll 1
      for (int blk = 0; blk < (DV + 31) / 32; ++blk) {
        if (blk > 0) __syncthreads();  // (the columns before have been read)
#pragma unroll
        for (int b = 0; b < (DV + 31) / 32; ++b)
          if (b == blk) R.each(b, [&](int h, int c, float v) { merge[(cg * MROWS + R.row(h)) * MPITCH + c - b * 32] = v; });
        __syncthreads();
        if (blk == 0) {
          // what a group's values of a row count for, once for all columns; the groups of a row are lanes beside each other
          for (int i = tid; i < (rows * CG + 31) / 32 * 32; i += NT) {
            const bool in = i < rows * CG;
            const int r = i / CG;
            const float2 ml = in ? merge_ml[i] : make_float2(FA_NEG_INF, 0.f);
            float m = ml.x;
#pragma unroll
            for (int off = 1; off < CG; off <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
            const float m_use = m == FA_NEG_INF ? 0.f : m;
            float f = ml.y == 0.f ? 0.f : exp2f(ml.x - m_use);  // (a group that has seen nothing counts for nothing)
            float l = f * ml.y;
#pragma unroll
            for (int off = 1; off < CG; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
            if (!in) continue;
            if (whole) {
              f *= inverse(l);
              if (i % CG == 0 && p.lse != nullptr) {
                const int qi = divided(rt * BM + r, p.by_group), hd = hk * G + rt * BM + r - qi * G;
                p.lse[((long long)b * p.Hq + hd) * p.Sq + qi] = log_sum(m_use, l);
              }
            } else if (i % CG == 0) {
              *(float2*)(part_ml + r * 2) = make_float2(m, l);
            }
            merge_ml[i].x = f;
          }
          __syncthreads();
        }
        constexpr int PAIRS = DV < 32 ? DV / 2 : 16;
#pragma unroll 1
        for (int i = tid; i < rows * PAIRS; i += NT) {
          const int r = i / PAIRS, c = (i - r * PAIRS) * 2;
          if (blk * 32 + c >= DV) continue;
          float x = 0.f, y = 0.f;
#pragma unroll
          for (int g = 0; g < CG; ++g) {
            const float2 v = *(const float2*)(merge + (g * MROWS + r) * MPITCH + c);
            const float f = merge_ml[r * CG + g].x;
            x += f * v.x;
            y += f * v.y;
          }
          if (whole) {
            const int qi = divided(rt * BM + r, p.by_group), hd = hk * G + rt * BM + r - qi * G;
            put2((char*)p.o.ptr + (b * p.o.sb + hd * p.o.sh + qi * p.o.ss) * ES, blk * 32 + c, x, y);
          } else {
            *(float2*)(part_o + r * DV + blk * 32 + c) = make_float2(x, y);
          }
        }
      }
      __syncthreads();  // (before the next segment's sums)
    } else {
      char* out[HR];
      float inv[HR];
#pragma unroll
      for (int h = 0; h < HR; ++h) {
        const int i = divided(rt * BM + R.row(h), p.by_group);
        out[h] = (char*)p.o.ptr + (b * p.o.sb + head[h] * p.o.sh + i * p.o.ss) * ES;
        inv[h] = inverse(R.l[h]);
        if (R.row(h) >= rows || !R.speaks()) continue;
        if (!whole) *(float2*)(part_ml + R.row(h) * 2) = make_float2(R.m[h], R.l[h]);
        else if (p.lse != nullptr) p.lse[((long long)b * p.Hq + head[h]) * p.Sq + i] = log_sum(R.m[h], R.l[h]);
      }
#pragma unroll
      for (int blk = 0; blk < (DV + 31) / 32; ++blk)
        R.each(blk, [&](int h, int c, float v) {
          if (R.row(h) >= rows) return;
          if (whole) put1(out[h], c, v * inv[h]);
          else part_o[R.row(h) * DV + c] = v;
        });
    }
  }
  if (!SHORT) fa_grid_release();
  fa_cp_wait<0>();
#if FA_TMA
  if (failed) {
    // The copies in flight have to land before the shared memory goes to another CTA (with a limit of its own: the flag is up).
    if (rg == 0 && lane == 0) {
      const fa_u64 start = fa_globaltimer();
#pragma unroll 1
      for (int i = n_used; i < asked; ++i) {
        while (!fa_mbar_try(bars + (i % SLOTS) * 8, (i / SLOTS) & 1) && fa_globaltimer() - start <= FA_WAIT_LIMIT_NS / 4) {
        }
      }
    }
    if (lane == 0 && p.status != nullptr) atomicOr(p.status, FA_STATUS_WAIT_TIMEOUT);
  }
#endif
}
