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
// Pages in 8 bits (FA_KV8): whole numbers w and a scale per key and kv head, k = ks w, v = vs w'.  The scales go where they cost least, on the scores
// and on the probabilities,  s_ij = scale ks_j (q_i . w_j),  o_i = sum_j (p_ij vs_j) w'_j / sum_j p_ij,  and the whole numbers become 16-bit values, exactly,
// in the registers that the products take them from: the way for few rows, in which a thread reads 16 bytes of a key, or its columns of
// four keys, and has the operands of four products.
//
// Compile-time parameters (macros): FA_DTYPE, FA_D, FA_DV, FA_RG (1, 2, 4), FA_WN (keys of a tile: 32 or 16; fp32: 32, 16, 8), FA_SLOTS, FA_TMA,
// FA_FEW (0: the other way), FA_FR (fp32: rows of a warp), FA_CG, FA_SHORT, FA_KV8, FA_AFTER (the keys lie behind a prefix, over which
// another kernel goes: results in float32 with their sums, for fa_merge_kernel).
#pragma once
#include "fa_sm100.cuh"

struct FaPagedLaunch {
  FaPagedParams p;
#if FA_TMA
  FaTensorMap tk, tv;  // 4-d maps (D, token in page, head, page), box 128 bytes x p.box x 1 x 1, 128-byte swizzle (FA_KV8 and D <= 64: of 64 bytes)
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
constexpr bool KV8 = FA_KV8 != 0;
constexpr bool AFTER = FA_AFTER != 0;
constexpr int EO = F32 || AFTER ? 4 : 2;  // bytes of a result
constexpr int EK = KV8 ? 1 : ES;  // bytes of a cached value
// Rows in 8 bits are column groups of 128 bytes, or one of 64, whole ones also where the head dim is not: what lies behind it is some whole number or
// other and is multiplied with zeros, or in columns that nobody writes out.  Tiles lie as TMA leaves them however they come.
constexpr int GROUP = KV8 && D <= 64 ? 64 : 128;
constexpr int PK = KV8 ? (D + GROUP - 1) / GROUP * GROUP : TMA ? D * ES : FaTile<D, ES>::PITCH;
constexpr int PV = KV8 ? (DV + GROUP - 1) / GROUP * GROUP : TMA ? DV * ES : FaTile<DV, ES>::PITCH;
constexpr int ATOMS_K = (KV8 ? PK : D * ES) / GROUP, ATOMS_V = (KV8 ? PV : DV * ES) / GROUP;  // column groups of a row (TMA)
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
static_assert(!TMA || KV8 || (D * ES % 128 == 0 && DV * ES % 128 == 0), "TMA: whole column groups");
static_assert(F32 || WN == 32 || WN == 16, "tiles of 16 or 32 keys");
static_assert(!FEW || (RG == 1 && !F32), "few rows: one warp, 16-bit types");
static_assert(!KV8 || (FEW && WN == 32), "8 bits: few rows, a key per lane");

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
#if FA_KV8
  float ks, vs; // scales of this lane's key; 0: it is not there
#endif
};

// The address of 16-byte chunk c of row r in a tile: rows with a pad behind, or as TMA leaves them, 64 columns of all rows one behind
// the other, chunk c of 8 at c ^ (r & 7).  (Of 64-byte rows chunk c of 4 at c ^ (r / 2 & 3).)
template <int PITCH>
__device__ __forceinline__ fa_u32 chunk_at(fa_u32 tile, int r, int c) {
  if (KV8 && GROUP == 64) return tile + r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
  return TMA || KV8 ? tile + (c >> 3) * (WN * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4) : tile + r * PITCH + c * 16;
}

// The rows of a tile in 16-byte pieces, those that are not there as zeros
template <int COLS, int PITCH>
__device__ __forceinline__ void load_pieces(const FaTensor& t, fa_u32 dst, const Load& n, int tid) {
  constexpr int CPR = COLS * EK / 16, NL = RG * 32;  // (the threads of a key group)
  const long long at = n.page >= 0 ? (n.page * t.sb + n.hk * t.sh + n.row * t.ss) * EK : -1;
#pragma unroll 4
  for (int i = tid; i < (WN * CPR + 31) / 32 * 32; i += NL) {  // (whole warps: the shuffle)
    const int r = i / CPR, c = i - r * CPR;
    const long long row = __shfl_sync(0xffffffffu, at, r & 31);
    if (i < WN * CPR) fa_cp_async16(KV8 ? chunk_at<PITCH>(dst, r, c) : dst + r * PITCH + c * 16, (const char*)t.ptr + (row >= 0 ? row + c * 16 : 0), row >= 0 ? 16 : 0);
  }
}

__device__ __forceinline__ fa_u32 transposed(fa_u32 x) {  // an 8 x 8 matrix of 16-bit values, a row over four lanes
  fa_u32 r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

struct Max {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Sum {
  __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};

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
#elif FA_KV8
constexpr int HR = 2 * NQ, NS = WN / 8;
constexpr int BLOCKS = (D + 63) / 64;  // of 64 columns of K, four products each
constexpr int VB = PV / 8;             // columns of V of a thread, beside each other
// Which of eight keys is row g of a product.  Lanes that are served together then read different banks: 16 bytes of the keys of two rows g beside each other
// (K), and two threads' columns of the keys of every other row (V).
__device__ __forceinline__ int key_of(int g) { return GROUP == 128 ? (g & 1 ? (g - 1) ^ 5 : g) : g ^ ((g >> 1) & 1); }
// Probabilities times the scales of their values.  A scale that is no number or infinite is the rows' that see its key: 0 times it, of a row that does not, is 0.  Which
// those are the scores say in front of the softmax; there is one vote per tile for this and for rows whose maximum rises.
template <class R>
__device__ __forceinline__ void find_unseen(R& r) {
  r.unseen = 0;
#pragma unroll
  for (int j = 0; j < NS; ++j)
#pragma unroll
    for (int h = 0; h < HR; ++h) r.unseen |= r.score(h, j) == FA_NEG_INF ? 1u << (HR * j + h) : 0u;
}
template <class R>
__device__ __forceinline__ void clear_unseen(R& r) {
#pragma unroll
  for (int j = 0; j < NS; ++j)
#pragma unroll
    for (int h = 0; h < HR; ++h)
      if ((r.unseen >> (HR * j + h)) & 1u) r.score(h, j) = 0.f;
}
#if FA_FEW == 1
// Whole numbers with whole numbers: products of 8 bits, summed in 32 (m16n8k32), which take K as it lies in the tile and V with its bytes exchanged
// (12 instructions for 16 values of K and of V together, where their way to 16 bits takes 68).
//   Scores: a row of queries is 2^(e - 22) times whole numbers of 23 bits (2^(e - 1) <= max|q| < 2^e), which are three digits of 8 bits, -128 to 127, so a score is
//   three sums, exact, and one rounding to fp32.  What 16-bit queries lose is below 2^-23 of the row's largest.
//   Values: of a tile, probabilities times scales are whole numbers of 16 bits, in two digits, of 1 / 32639 of the largest of the row's 32: 2^-16 of that is what one is off by
//   at most.  (A single rounding to fp16 is off by more than the three-fold of that, by the rms of a tile, and to bf16 by the 25-fold; with a third digit a tile
//   would take 9 % more instructions.)
__device__ __forceinline__ fa_u32 bytes_of(fa_u32 a, fa_u32 b, fa_u32 which) {
  fa_u32 r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(which));
  return r;
}
__device__ __forceinline__ void imma(int (&c)[4], const fa_u32 (&a)[4], fa_u32 b0, fa_u32 b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
constexpr int MAGIC = 0x4b400000;  // the bits of 1.5 * 2^23: with n added, below 2^22 in size, those of that number plus n
__device__ __forceinline__ float from_magic(int c) { return __int_as_float(c) - 12582912.f; }
// the three digits of four whole numbers, a register each
__device__ __forceinline__ void digits(const int (&x)[4], fa_u32 (&d)[3]) {
  int y[4], z[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[i] = (x[i] + 128) >> 8;  // (what is left above the low digit)
    z[i] = (y[i] + 128) >> 8;
  }
  d[0] = bytes_of(bytes_of(x[0], x[1], 0x0040u), bytes_of(x[2], x[3], 0x0040u), 0x5410u);
  d[1] = bytes_of(bytes_of(y[0], y[1], 0x0040u), bytes_of(y[2], y[3], 0x0040u), 0x5410u);
  d[2] = bytes_of(bytes_of(z[0], z[1], 0x0040u), bytes_of(z[2], z[3], 0x0040u), 0x5410u);
}
struct Rows {
  float s[WN / 16][1][4], o[VB / 2][1][4], m[HR], l[HR];
  fa_u32 qf[BLOCKS * 2][3][2]; // digits of 16 values of each 64 of query g = lane / 4
  float qs[HR];                // 2^(e - 22) of this lane's rows
  float ks, vs;                // scales of this lane's key of the tile
  fa_u32 unseen;               // scores of the tile that a value's scale must not come to, bit HR j + h
  int lane;
  __device__ __forceinline__ float& score(int h, int j) { return s[j >> 1][0][(j & 1) * 2 + h]; }
  __device__ __forceinline__ int key(int j) const { return key_of(lane >> 2) + j * 8; }
  __device__ __forceinline__ int row(int h) const { return (lane & 3) * 2 + h; }
  __device__ __forceinline__ bool idle(int h, int rows) const { return h >= rows; }
  template <class F>
  static __device__ __forceinline__ void over_keys(float (&v)[HR], F f) {
#pragma unroll
    for (int off = 4; off < 32; off <<= 1)
#pragma unroll
      for (int h = 0; h < HR; ++h) v[h] = f(v[h], __shfl_xor_sync(0xffffffffu, v[h], off));
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < VB / 2; ++i) o[i][0][0] = o[i][0][1] = o[i][0][2] = o[i][0][3] = 0.f;
  }
  __device__ __forceinline__ void rescale(int h, float c) {
#pragma unroll
    for (int i = 0; i < VB / 2; ++i) {
      o[i][0][h] *= c;
      o[i][0][2 + h] *= c;
    }
  }
  __device__ __forceinline__ void take_queries(const fa_u32 (&raw)[BLOCKS * 8]) {  // 16 values of each 64, as they were loaded
    fa_u32 most = 0;  // (sizes as bits: infinities and no numbers are the largest)
#pragma unroll
    for (int i = 0; i < BLOCKS * 8; ++i) most = max(most, max(raw[i] & 0x7fffu, (raw[i] >> 16) & 0x7fffu));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    most = __float_as_uint(fa_to_float<DT>((fa_u16)most));
    // (below 2^-100 a row has fewer bits, and no score that shows)
    const int e = max((int)(most >> 23) - 126, -100);
    const float up = __uint_as_float((fa_u32)(22 - e + 127) << 23);
    const float down = most >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : __uint_as_float((fa_u32)(e - 22 + 127) << 23);
#pragma unroll
    for (int h = 0; h < HR; ++h) qs[h] = __shfl_sync(0xffffffffu, down, ((lane & 3) * 2 + h) * 4);
#pragma unroll
    for (int i = 0; i < BLOCKS * 4; ++i) {
      int n[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) n[k] = __float2int_rn(fa_to_float<DT>((fa_u16)(raw[2 * i + (k >> 1)] >> (16 * (k & 1)))) * up);
      fa_u32 d[3];
      digits(n, d);
#pragma unroll
      for (int k = 0; k < 3; ++k) qf[i >> 1][k][i & 1] = d[k];
    }
  }
  // S' = K Q'.  A product's 32 columns are bytes 8 i .. 8 i + 7 of the 16 that each of four threads has of a key (of 64 columns in all); the queries'
  // digits lie in their registers in the same order.
  __device__ __forceinline__ void scores(const unsigned char* bytes, fa_u32, int) {
#pragma unroll
    for (int i = 0; i < WN / 16; ++i) {
      int c[3][4];
#pragma unroll
      for (int k = 0; k < 3; ++k) c[k][0] = c[k][1] = c[k][2] = c[k][3] = MAGIC;
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        const uint4 x = *(const uint4*)(bytes + chunk_at<PK>(0, i * 16 + key_of(lane >> 2), b * 4 + (lane & 3)));
        const uint4 y = *(const uint4*)(bytes + chunk_at<PK>(0, i * 16 + 8 + key_of(lane >> 2), b * 4 + (lane & 3)));
        const fa_u32 a0[4] = {x.x, y.x, x.y, y.y}, a1[4] = {x.z, y.z, x.w, y.w};
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          imma(c[k], a0, qf[b * 2][k][0], qf[b * 2][k][1]);
          imma(c[k], a1, qf[b * 2 + 1][k][0], qf[b * 2 + 1][k][1]);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][0][e] = fmaf(fmaf(from_magic(c[2][e]), 256.f, from_magic(c[1][e])), 256.f, from_magic(c[0][e]));
    }
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const float f = __shfl_sync(0xffffffffu, ks, key(j));
#pragma unroll
      for (int h = 0; h < HR; ++h) score(h, j) *= f * qs[h];
    }
  }
  // O' = V' P'
  __device__ __forceinline__ void values(const unsigned char* bytes, fa_u32, int) {
    float top[HR] = {0.f, 0.f};
    fa_u32 nan = 0;
    const auto look = [&]() {
#pragma unroll
      for (int j = 0; j < NS; ++j) {
#pragma unroll
        for (int h = 0; h < HR; ++h) {
          top[h] = fmaxf(top[h], fabsf(score(h, j)));
          nan |= !(fabsf(score(h, j)) <= 3.4e38f) ? 1u << h : 0u;
        }
      }
    };
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const float f = __shfl_sync(0xffffffffu, vs, key(j));
#pragma unroll
      for (int h = 0; h < HR; ++h) score(h, j) *= f;
    }
    look();
    const bool no_number = __any_sync(0xffffffffu, nan != 0);
    if (no_number) {
      clear_unseen(*this);
      top[0] = top[1] = 0.f;
      nan = 0;
      look();
    }
    over_keys(top, Max());
    float step[HR];
#pragma unroll
    for (int h = 0; h < HR; ++h) {
      // (a largest value below 2^-100 counts as 2^-100, whose reciprocal is a number)
      const float t = fmaxf(top[h], 7.9e-31f), up = 32639.f / t;
      step[h] = t * (1.f / 32639.f);
#pragma unroll
      for (int j = 0; j < NS; ++j) score(h, j) = fmaf(score(h, j), up, 12582912.f);  // (the whole number in the low 16 bits)
    }
    if (no_number) {  // of a row with no number in it, nothing is one
#pragma unroll
      for (int h = 0; h < HR; ++h) {
        fa_u32 any = nan >> h & 1u;
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) any |= __shfl_xor_sync(0xffffffffu, any, off);
        if (any) step[h] = __uint_as_float(0x7fffffffu);
      }
    }
    // Of every 8 keys the numbers of two rows in a register become those of two keys of row g = lane / 4; the low digit is taken out of the high one
    // (which is one more where the low one is negative) before.
    fa_u32 r[NS], b[2][2];
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const fa_u32 x = bytes_of(__float_as_uint(score(0, j)), __float_as_uint(score(1, j)), 0x5410u);
      fa_u32 y;
      asm("add.u16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"((x & 0x00800080u) << 1));
      r[j] = transposed(y);
    }
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {  // digit d of the keys of rows 16 hf + 2 t, 2 t + 1, 2 t + 8 and 2 t + 9
      b[0][hf] = bytes_of(r[2 * hf], r[2 * hf + 1], 0x6420u);
      b[1][hf] = bytes_of(r[2 * hf], r[2 * hf + 1], 0x7531u);
    }
    // columns VB g .. VB g + VB - 1 of those keys
    const int g = lane >> 2, t = lane & 3, k0 = key_of(2 * t), k1 = key_of(2 * t + 1);
#pragma unroll
    for (int c = 0; c < VB; c += 8) {
      fa_u32 w[8][2];  // (16 bytes at once would take registers that the tiles on their way need)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint2 x = *(const uint2*)(bytes + chunk_at<PV>(0, (k & 1 ? k1 : k0) + (k >> 1) * 8, (g * VB + c) >> 4) + ((VB < 16 ? g : c >> 3) & 1) * 8);
        w[k][0] = x.x;
        w[k][1] = x.y;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // four columns of four keys: columns and keys change places
        fa_u32 col[2][4];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const fa_u32 lo0 = bytes_of(w[4 * hf][i], w[4 * hf + 1][i], 0x5140u), hi0 = bytes_of(w[4 * hf][i], w[4 * hf + 1][i], 0x7362u);
          const fa_u32 lo1 = bytes_of(w[4 * hf + 2][i], w[4 * hf + 3][i], 0x5140u), hi1 = bytes_of(w[4 * hf + 2][i], w[4 * hf + 3][i], 0x7362u);
          col[hf][0] = bytes_of(lo0, lo1, 0x5410u);
          col[hf][1] = bytes_of(lo0, lo1, 0x7632u);
          col[hf][2] = bytes_of(hi0, hi1, 0x5410u);
          col[hf][3] = bytes_of(hi0, hi1, 0x7632u);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const fa_u32 a[4] = {col[0][2 * u], col[0][2 * u + 1], col[1][2 * u], col[1][2 * u + 1]};
          int acc[4] = {0, 0, 0, 0};
          imma(acc, a, b[1][0], b[1][1]);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] *= 256;
          imma(acc, a, b[0][0], b[0][1]);
          float(&out)[4] = o[c / 2 + i * 2 + u][0];
#pragma unroll
          for (int e = 0; e < 4; ++e) out[e] = fmaf((float)acc[e], step[e & 1], out[e]);
        }
      }
    }
  }
  template <class F>
  __device__ __forceinline__ void each(int b, F f) {
    if ((lane >> 2) * VB / 32 != b) return;
#pragma unroll
    for (int i = 0; i < VB / 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = (lane >> 2) * VB + 2 * i + (e >> 1);
        if (PV == DV || c < DV) f(e & 1, c, o[i][0][e]);
      }
  }
  __device__ __forceinline__ bool speaks() const { return lane < 4; }
};
#else
// Four whole numbers as 16-bit values, two to a register.  fp16: in the low byte of 1024, made positive by 128.  bf16 has 8 bits: 128 plus the low seven of
// the number, minus 128, or 256 of a negative one, whose sign is the bit that tells the two apart.
template <int TO>
__device__ __forceinline__ fa_u32 whole2(fa_u32 w, fa_u32 which) {  // which: 0x4140, bytes 0 and 1; 0x4342, 2 and 3 (fp16: of w ^ 0x80808080)
  fa_u32 r;
  if (TO == FA_DT_F16) {
    asm("{\n\t.reg .b32 x;\n\tprmt.b32 x, %1, 0x64646464, %2;\n\tsub.rn.f16x2 %0, x, %3;\n\t}" : "=r"(r) : "r"(w), "r"(which), "r"(0x64806480u));
  } else {
    asm("{\n\t.reg .b32 x, y;\n\tprmt.b32 x, %1, 0x43434343, %2;\n\tand.b32 y, x, 0xff80ff80;\n\tand.b32 x, x, 0xff7fff7f;\n\tsub.rn.bf16x2 %0, x, y;\n\t}"
        : "=r"(r) : "r"(w), "r"(which));
  }
  return r;
}
template <int TO>
__device__ __forceinline__ fa_u32 biased(fa_u32 w) { return TO == FA_DT_F16 ? w ^ 0x80808080u : w; }
__device__ __forceinline__ fa_u32 bytes_of(fa_u32 a, fa_u32 b, fa_u32 which) {
  fa_u32 r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(which));
  return r;
}
struct Rows {
  float s[WN / 16][NQ][4], o[VB / 2][NQ][4], m[HR], l[HR];
  fa_u32 qf[BLOCKS * 4][NQ][2];
  float ks, vs;  // scales of this lane's key of the tile
  fa_u32 unseen; // scores of the tile that a value's scale must not come to, bit HR j + h
  int lane;
  __device__ __forceinline__ float& score(int h, int j) { return s[j >> 1][h >> 1][(j & 1) * 2 + (h & 1)]; }
  __device__ __forceinline__ int key(int j) const { return key_of(lane >> 2) + j * 8; }
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
    for (int i = 0; i < VB / 2; ++i)
#pragma unroll
      for (int q = 0; q < NQ; ++q) o[i][q][0] = o[i][q][1] = o[i][q][2] = o[i][q][3] = 0.f;
  }
  __device__ __forceinline__ void rescale(int h, float c) {
#pragma unroll
    for (int i = 0; i < VB / 2; ++i) {
      o[i][h >> 1][h & 1] *= c;
      o[i][h >> 1][2 + (h & 1)] *= c;
    }
  }
  // S' = K Q'.  A product's 16 columns are bytes 4 i .. 4 i + 3 of the 16 that each of four threads has of a key (of 64 columns in all); the queries lie
  // in their registers in the same order.
  __device__ __forceinline__ void scores(const unsigned char* bytes, fa_u32, int) {
#pragma unroll
    for (int i = 0; i < WN / 16; ++i) {
#pragma unroll
      for (int q = 0; q < NQ; ++q) s[i][q][0] = s[i][q][1] = s[i][q][2] = s[i][q][3] = 0.f;
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        const uint4 x = *(const uint4*)(bytes + chunk_at<PK>(0, i * 16 + key_of(lane >> 2), b * 4 + (lane & 3)));
        const uint4 y = *(const uint4*)(bytes + chunk_at<PK>(0, i * 16 + 8 + key_of(lane >> 2), b * 4 + (lane & 3)));
        const fa_u32 xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const fa_u32 u = biased<DT>(xs[k]), v = biased<DT>(ys[k]);
          const fa_u32 a[4] = {whole2<DT>(u, 0x4140u), whole2<DT>(v, 0x4140u), whole2<DT>(u, 0x4342u), whole2<DT>(v, 0x4342u)};
#pragma unroll
          for (int q = 0; q < NQ; ++q) fa_mma16816<DT>(s[i][q], a, qf[b * 4 + k][q][0], qf[b * 4 + k][q][1]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const float f = __shfl_sync(0xffffffffu, ks, key(j));
#pragma unroll
      for (int h = 0; h < HR; ++h) score(h, j) *= f;
    }
  }
  // O' = V' P'.  Probabilities times scales may have any size, so they go in as bf16, in two parts, rounded and what the rounding left: 16 bits of them.
  __device__ __forceinline__ void values(const unsigned char* bytes, fa_u32, int) {
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const float f = __shfl_sync(0xffffffffu, vs, key(j));
#pragma unroll
      for (int h = 0; h < HR; ++h) score(h, j) *= f;
    }
    if (unseen != 0) clear_unseen(*this);
#pragma unroll
    for (int kj = 0; kj < WN / 16; ++kj) {
      fa_u32 b[NQ][2], rest[NQ][2];
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p0 = s[kj][q][2 * e], p1 = s[kj][q][2 * e + 1];
          float r0, r1;
          b[q][e] = transposed(fa_pack2<FA_DT_BF16>(p0, p1));
          fa_rest2<FA_DT_BF16>(p0, p1, r0, r1);
          rest[q][e] = transposed(fa_pack2<FA_DT_BF16>(r0, r1));
        }
      // columns VB g .. VB g + VB - 1 of the keys of rows 2 t, 2 t + 1, 2 t + 8 and 2 t + 9 (g = lane / 4, t = lane % 4), eight at a time
      const int g = lane >> 2, t = lane & 3, k0 = kj * 16 + key_of(2 * t), k1 = kj * 16 + key_of(2 * t + 1);
#pragma unroll
      for (int c = 0; c < VB; c += VB < 16 ? 8 : 16) {
        fa_u32 w[4][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = (k & 1 ? k1 : k0) + (k >> 1) * 8;
          if (VB < 16) {
            const uint2 x = *(const uint2*)(bytes + chunk_at<PV>(0, r, g >> 1) + (g & 1) * 8);
            w[k][0] = x.x; w[k][1] = x.y; w[k][2] = w[k][3] = 0u;
          } else {
            const uint4 x = *(const uint4*)(bytes + chunk_at<PV>(0, r, g * (VB / 16) + c / 16));
            w[k][0] = x.x; w[k][1] = x.y; w[k][2] = x.z; w[k][3] = x.w;
          }
        }
#pragma unroll
        for (int i = 0; i < (VB < 16 ? 2 : 4); ++i) {
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {  // two columns at a time: rows g and g + 8 of a product
            const fa_u32 x = bytes_of(w[0][i], w[1][i], hf ? 0x7362u : 0x5140u), y = bytes_of(w[2][i], w[3][i], hf ? 0x7362u : 0x5140u);
            const fa_u32 a[4] = {whole2<FA_DT_BF16>(x, 0x4140u), whole2<FA_DT_BF16>(x, 0x4342u), whole2<FA_DT_BF16>(y, 0x4140u), whole2<FA_DT_BF16>(y, 0x4342u)};
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
              fa_mma16816<FA_DT_BF16>(o[c / 2 + i * 2 + hf][q], a, b[q][0], b[q][1]);
              fa_mma16816<FA_DT_BF16>(o[c / 2 + i * 2 + hf][q], a, rest[q][0], rest[q][1]);
            }
          }
        }
      }
    }
  }
  template <class F>
  __device__ __forceinline__ void each(int b, F f) {
    if ((lane >> 2) * VB / 32 != b) return;
#pragma unroll
    for (int i = 0; i < VB / 2; ++i)
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = (lane >> 2) * VB + 2 * i + (e >> 1);
          if (PV == DV || c < DV) f(2 * q + (e & 1), c, o[i][q][e]);
        }
  }
  __device__ __forceinline__ bool speaks() const { return lane < 4; }
};
#endif
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

// a value of an output row
__device__ __forceinline__ void put1(char* row, int c, float x) {
  if (EO == 4) *(float*)(row + c * 4) = x;
  else *(fa_u16*)(row + c * 2) = (fa_u16)fa_pack2<DT>(x, 0.f);
}
// two beside each other
__device__ __forceinline__ void put2(char* row, int c, float x, float y) {
  if (EO == 4) *(float2*)(row + c * 4) = make_float2(x, y);
  else *(fa_u32*)(row + c * 2) = fa_pack2<DT>(x, y);
}
// 1 / sum; 0 of a row that has seen nothing, no number of a sum that is none
__device__ __forceinline__ float inverse(float l) { return l > 0.f ? 1.f / l : l; }
__device__ __forceinline__ float log_sum(float m, float l) { return l == 0.f ? FA_NEG_INF : (m + log2f(l)) * FA_LN2; }
// what is left of a whole row's maximum and sum
__device__ __forceinline__ void put_sums(const FaPagedParams& p, long long row, float m, float l) {
  if (AFTER) *(float2*)(p.out_ml + row * 2) = make_float2(m, l);
  else if (p.lse != nullptr) p.lse[row] = log_sum(m, l);
}

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
  // (Also behind a prefix, whose kernel is in front and whose results are not needed here: lengths, tables and pages are written by kernels in front of that one, and
  // only this wait says that they can be seen.)
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
#if FA_KV8
    const int box = divided(lane, p.by_box), page = __shfl_sync(0xffffffffu, n.page, box), row = __shfl_sync(0xffffffffu, n.row, box) + lane - box * p.box;
    const bool in = page >= 0 && ((n.keep >> lane) & 1u);
    n.ks = in ? ((const float*)p.k_scales.ptr)[page * p.k_scales.sb + n.hk * p.k_scales.sh + row * p.k_scales.ss] : 0.f;
    n.vs = in ? ((const float*)p.v_scales.ptr)[page * p.v_scales.sb + n.hk * p.v_scales.sh + row * p.v_scales.ss] : 0.f;
#endif
  };
#if FA_TMA
  auto load = [&](const FaTensorMap* map, fa_u32 dst, fa_u32 bar, int atoms, const Load& n) {
    if (rg != 0) return;
    if (lane == 0) fa_mbar_expect_tx(bar, __popc(n.boxes) * p.box * GROUP * atoms);
    __syncwarp();
    if (n.page >= 0) {
      for (int a = 0; a < atoms; ++a)
        fa_tma_load_4d(dst + a * (WN * GROUP) + lane * p.box * GROUP, map, bar, a * (GROUP / EK), n.row, n.hk, n.page);
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
#if FA_KV8
  float scales_k[AHEAD], scales_v[AHEAD];
  auto push_scales = [&](const Load& n) {
#pragma unroll
    for (int i = 0; i + 1 < AHEAD; ++i) {
      scales_k[i] = scales_k[i + 1];
      scales_v[i] = scales_v[i + 1];
    }
    scales_k[AHEAD - 1] = n.any ? n.ks : 0.f;
    scales_v[AHEAD - 1] = n.any ? n.vs : 0.f;
  };
#endif
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
#if FA_KV8
    push_scales(next);
#endif
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
      const fa_u32* src = (const fa_u32*)(qb + (i * p.q.ss + (long long)(seg.hk * G + row - i * G) * p.q.sh) * ES) + (KV8 ? 0 : (lane & 3));
#if FA_KV8
      // (columns 16 t .. of each 64, t = lane % 4, as K's)
#if FA_FEW == 1
      fa_u32 raw[BLOCKS * 8];
#endif
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        const int c = b * 64 + (lane & 3) * 16;
        uint4 x = make_uint4(0u, 0u, 0u, 0u), y = x;
        if (i < p.Sq && (D % 64 == 0 || c < D)) {
          x = *(const uint4*)(src + c / 2);
          y = *(const uint4*)(src + c / 2 + 4);
        }
#if FA_FEW == 1
        raw[b * 8] = x.x; raw[b * 8 + 1] = x.y; raw[b * 8 + 2] = x.z; raw[b * 8 + 3] = x.w;
        raw[b * 8 + 4] = y.x; raw[b * 8 + 5] = y.y; raw[b * 8 + 6] = y.z; raw[b * 8 + 7] = y.w;
#else
        R.qf[b * 4][q][0] = x.x; R.qf[b * 4][q][1] = x.y;
        R.qf[b * 4 + 1][q][0] = x.z; R.qf[b * 4 + 1][q][1] = x.w;
        R.qf[b * 4 + 2][q][0] = y.x; R.qf[b * 4 + 2][q][1] = y.y;
        R.qf[b * 4 + 3][q][0] = y.z; R.qf[b * 4 + 3][q][1] = y.w;
#endif
      }
#if FA_FEW == 1
      R.take_queries(raw);
#endif
      continue;
#endif
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
#if FA_KV8
      R.ks = scales_k[0];
      R.vs = scales_v[0];
#endif
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
        [[maybe_unused]] const int qp = max(qpos[h], 0) + (AFTER ? p.after : 0), gh = head[h] + p.h_off;
#pragma unroll
        for (int j = 0; j < NS; ++j) {
          [[maybe_unused]] const int kv = n0 + R.key(j) + (AFTER ? p.after : 0);
          float x = R.score(h, j);
#if FA_HAS_SCORE_MOD && FA_SCORE_PAIRS
          static_assert(NS % 2 == 0, "keys of a thread come in pairs");
          if (j % 2 == 0) {
            float y = R.score(h, j + 1);
            fa_f2_unpack(fa_mul2(fa_score_mod_pair(fa_mul2(fa_f2(x, y), fa_both(p.scale)), gb, gh, qp, kv, n0 + R.key(j + 1) + (AFTER ? p.after : 0)), fa_both(FA_LOG2E)), x, y);
            R.score(h, j + 1) = y;
          }
#elif FA_HAS_SCORE_MOD && defined(FA_SCORE_AFFINE)
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
            see = see && fa_mask_mod(gb, gh, qp, kv + (AFTER ? p.after : 0));
#endif
            if (!see) R.score(h, j) = FA_NEG_INF;
          }
        }
#pragma unroll
        for (int j = 0; j < NS; ++j) top[h] = fmaxf(top[h], R.score(h, j));
        rises |= top[h] > R.m[h] + RISE;
      }
#if FA_KV8
      R.unseen = 0;
      const bool strange = !(fabsf(R.vs) <= 3.4e38f);
      if (__any_sync(0xffffffffu, rises || strange)) {
        if (__any_sync(0xffffffffu, strange)) find_unseen(R);
        rises = __any_sync(0xffffffffu, rises);
      }
      if (rises) {
#else
      if (__any_sync(0xffffffffu, rises)) {
#endif
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
      if (!KV8 && kept != ALL) {  // (whole numbers are numbers, and their scale is 0)
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
#if FA_KV8
      push_scales(next);
#endif
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
              if (i % CG == 0) {
                const int qi = divided(rt * BM + r, p.by_group), hd = hk * G + rt * BM + r - qi * G;
                put_sums(p, ((long long)b * p.Hq + hd) * p.Sq + qi, m_use, l);
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
            put2((char*)p.o.ptr + (b * p.o.sb + hd * p.o.sh + qi * p.o.ss) * EO, blk * 32 + c, x, y);
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
        out[h] = (char*)p.o.ptr + (b * p.o.sb + head[h] * p.o.sh + i * p.o.ss) * EO;
        inv[h] = inverse(R.l[h]);
        if (R.row(h) >= rows || !R.speaks()) continue;
        if (!whole) *(float2*)(part_ml + R.row(h) * 2) = make_float2(R.m[h], R.l[h]);
        else put_sums(p, ((long long)b * p.Hq + head[h]) * p.Sq + i, R.m[h] == FA_NEG_INF ? 0.f : R.m[h], R.l[h]);
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
