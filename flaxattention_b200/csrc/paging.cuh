// Pages of a key / value cache: places for the new tokens of a batch of requests (fa_page_step) and attention over
// the pages (fa_paged; its kernel is kernels/fa_paged.cuh).  Part of flaxattn.cu.
namespace {

// ---- block tables, slots and positions of new tokens --------------------------------------
// Request b has len[b] tokens in its pages and gets n[b] more.  It keeps its ceil(len / P) pages and takes as many free ones
// as the new length needs; the free list is gone through in the order of the requests.  The new tokens, request after
// request, are numbered through: token t of the step is token len + (t - start) of its request.
//
// One launch: every block runs over all requests, 1024 at a time, adds up their tokens and pages and fills what lies in its own range
// of tokens, and in its own range of new pages.  The prefix sums that a block needs are its own, so that
// no block waits for another.  What bounds it is the chain launch - lengths - sums - pages - slots: 4.2 us for 64 tokens of 64 requests, 6.9 for 524288
// tokens of 512 requests, of which the 16 bytes written per token take 1.3.  (With a search and a load per token one behind the other, and the new pages
// filled by the blocks whose tokens have the same numbers, 11.3.)
constexpr int kStepThreads = 256, kStepItems = 4, kStepChunk = kStepThreads * kStepItems;

struct FaStepParams {
  const int *len, *count, *free_pages, *taken_in;
  int* table;
  long long table_stride, num_free, tokens;
  int B, width, page, per_block, pages_per_block;  // what a block fills: tokens, and table entries of new pages
  int *out_len, *positions, *requests, *starts, *taken_out;
  long long* slots;
};

// Where the things (tokens, pages) that a block fills lie among those of the requests of a chunk: `from[k]` is the first one of request k,
// relative to the block's first.
struct FaStepRange {
  int from[kStepChunk];
  int lo, hi;  // the requests that hold the block's first and last
  static __device__ __forceinline__ int clamp(long long v) { return (int)max(min(v, 0x7fffffffll), -0x7fffffffll); }
  // the requests whose ranges hold x[..]: the last that begin at or in front of them.  Looked for together, in as many steps as the block's
  // range of requests takes: one at a time, each would wait for its own.
  template <int N>
  __device__ __forceinline__ void find(const int (&x)[N], int (&k)[N]) const {
    int c[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      k[i] = lo;
      c[i] = hi + 1;
    }
    for (int left = hi - lo; left > 0; left >>= 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int m = (k[i] + c[i]) >> 1;
        if (from[m] <= x[i]) k[i] = m;
        else c[i] = m;
      }
    }
  }
};

__global__ void __launch_bounds__(kStepThreads) fa_page_step_kernel(const __grid_constant__ FaStepParams P) {
  grid_wait();
  __shared__ FaStepRange tok, pag;
  __shared__ int len[kStepChunk];
  __shared__ long long warp_sum[2][kStepThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long lo = (long long)blockIdx.x * P.per_block, hi = min(lo + P.per_block, P.tokens);
  const long long page_lo = (long long)blockIdx.x * P.pages_per_block;
  const bool first = blockIdx.x == 0, last = blockIdx.x == gridDim.x - 1;
  const long long taken = P.taken_in != nullptr ? max(*P.taken_in, 0) : 0;
  long long tokens = 0, pages = 0;  // of the chunks in front
  for (int b0 = 0; b0 < P.B; b0 += kStepChunk) {
    int l[kStepItems], n[kStepItems], g[kStepItems];
    long long own_t = 0, own_p = 0;
#pragma unroll
    for (int i = 0; i < kStepItems; ++i) {
      const int b = b0 + tid * kStepItems + i;
      l[i] = b < P.B ? max(P.len[b], 0) : 0;
      n[i] = b < P.B ? min(max(P.count[b], 0), 0x7fffffff - l[i]) : 0;
      g[i] = (int)(((unsigned)l[i] + n[i] + P.page - 1u) / P.page - ((unsigned)l[i] + P.page - 1u) / P.page);
      own_t += n[i];
      own_p += g[i];
    }
    long long sum_t = own_t, sum_p = own_p;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long a = __shfl_up_sync(0xffffffffu, sum_t, off), c = __shfl_up_sync(0xffffffffu, sum_p, off);
      if (lane >= off) {
        sum_t += a;
        sum_p += c;
      }
    }
    __syncthreads();  // (the chunk in front has been read)
    if (lane == 31) {
      warp_sum[0][warp] = sum_t;
      warp_sum[1][warp] = sum_p;
    }
    __syncthreads();
    long long at_t = tokens + sum_t - own_t, at_p = pages + sum_p - own_p;
    const long long tokens0 = tokens, pages0 = pages;
#pragma unroll
    for (int w = 0; w < kStepThreads / 32; ++w) {
      if (w < warp) {
        at_t += warp_sum[0][w];
        at_p += warp_sum[1][w];
      }
      tokens += warp_sum[0][w];
      pages += warp_sum[1][w];
    }
    // what this block fills of the chunk's, relative to its range (in 64 bits up to there: the requests may ask for more than 2^31 tokens in all)
    const auto within = [](long long v, long long n) { return (int)max(min(v, n), 0ll); };
    const int t_lo = within(tokens0 - lo, hi - lo), t_hi = within(tokens - lo, hi - lo);
    const int p_lo = within(pages0 - page_lo, P.pages_per_block), p_hi = within(pages - page_lo, P.pages_per_block);
#pragma unroll
    for (int i = 0; i < kStepItems; ++i) {
      const int k = tid * kStepItems + i, b = b0 + k;
      const long long ta = at_t - lo, tb = ta + n[i], pa = at_p - page_lo, pb = pa + g[i];
      tok.from[k] = FaStepRange::clamp(ta);
      pag.from[k] = FaStepRange::clamp(pa);
      len[k] = l[i];
      if (t_lo < t_hi && ta <= t_lo && t_lo < tb) tok.lo = k;
      if (t_lo < t_hi && ta < t_hi && t_hi <= tb) tok.hi = k;
      if (p_lo < p_hi && pa <= p_lo && p_lo < pb) pag.lo = k;
      if (p_lo < p_hi && pa < p_hi && p_hi <= pb) pag.hi = k;
      if (first && b < P.B) {
        P.out_len[b] = l[i] + n[i];
        P.starts[b] = (int)min(at_t, 0x7fffffffll);
      }
      at_t += n[i];
      at_p += g[i];
    }
    __syncthreads();
    const auto had_of = [&](int k) { return (int)(((unsigned)len[k] + P.page - 1u) / P.page); };
    const auto fresh = [&](long long nth) {  // the nth new page
      const long long at = taken + nth;
      return at < P.num_free ? max(P.free_pages[at], -1) : -1;
    };
    constexpr int U = 4;
    for (int t0 = t_lo + tid; t0 < t_hi; t0 += U * kStepThreads) {
      int t[U], k[U], pos[U], col[U], page[U];
#pragma unroll
      for (int i = 0; i < U; ++i) t[i] = min(t0 + i * kStepThreads, t_hi - 1);
      tok.find(t, k);
#pragma unroll
      for (int i = 0; i < U; ++i) {
        pos[i] = len[k[i]] + (t[i] - tok.from[k[i]]);
        col[i] = pos[i] / P.page;
        // (one load whichever list the page is in, and nothing waits for it before the others are on their way)
        const int had = had_of(k[i]);
        const long long nth = taken + page_lo + pag.from[k[i]] + (col[i] - had);
        const int* from = col[i] < had ? P.table + (b0 + k[i]) * P.table_stride + col[i] : P.free_pages + nth;
        page[i] = -1;
        if (col[i] < P.width && (col[i] < had || nth < P.num_free)) page[i] = *from;
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (t0 + i * kStepThreads >= t_hi) continue;
        P.positions[lo + t[i]] = pos[i];
        P.requests[lo + t[i]] = b0 + k[i];
        P.slots[lo + t[i]] = page[i] < 0 ? -1ll : (long long)page[i] * P.page + (pos[i] - col[i] * P.page);
      }
    }
    for (int q0 = p_lo + tid; q0 < p_hi; q0 += kStepThreads) {
      const int q[1] = {q0};
      int k[1];
      pag.find(q, k);
      const int c = had_of(k[0]) + (q0 - pag.from[k[0]]);
      if (c < P.width) P.table[(long long)(b0 + k[0]) * P.table_stride + c] = fresh(page_lo + q0);
    }
    if (last && pages - page_lo > P.pages_per_block) {  // more new pages than the call has tokens for: request by request
      for (int k = warp; k < kStepChunk && b0 + k < P.B; k += kStepThreads / 32) {
        // (a request that begins 2^31 pages on has its place clamped: its number of pages is counted again, and the list has come to its end there)
        const long long had = had_of(k), need = ((long long)len[k] + min(max(P.count[b0 + k], 0), 0x7fffffff - len[k]) + P.page - 1) / P.page;
        const long long from = pag.from[k], end = min(need, (long long)P.width);
        for (long long c = had + max(P.pages_per_block - from, 0ll) + lane; c < end; c += 32)
          P.table[(b0 + k) * P.table_stride + c] = fresh(page_lo + from + c - had);
      }
    }
  }
  if (first && tid == 0) {
    P.starts[P.B] = (int)min(tokens, 0x7fffffffll);
    *P.taken_out = (int)min(taken + pages, 0x7fffffffll);
  }
  for (long long t = max(lo, tokens) + tid; t < hi; t += kStepThreads) {  // no tokens
    P.positions[t] = 0;
    P.requests[t] = -1;
    P.slots[t] = -1;
  }
}

// ---- attention: the parts of segments that several workers share ---------------------------
// WARPS warps per query row, which take the row's parts in turn: eight where a row may have many (one request of 131072 keys, 444 workers, 32 rows: 4.4 us,
// a chain of plan, parts and sums), else one (3.4).
template <int DT, int WARPS>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : WARPS * 32) fa_paged_combine_kernel(const __grid_constant__ FaPagedParams p, int BM, int Dv, int n_rows) {
  grid_wait();
  constexpr int U = 4;
  __shared__ float4 sums[WARPS == 1 ? 1 : WARPS][64];
  __shared__ float2 totals[WARPS];
  const int lane = threadIdx.x & 31, warp = WARPS == 1 ? 0 : threadIdx.x >> 5;
  const int row = WARPS == 1 ? blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= n_rows) return;
  // row: request, kv head, row among the G * Sq of the head
  const int G = p.Hq / p.Hkv, per_head = G * p.Sq;
  const int bh = row / per_head, r = row - bh * per_head, b = bh / p.Hkv, hk = bh - b * p.Hkv;
  const int rt = r / BM, item = b * p.row_tiles + rt, items = p.B * p.row_tiles;
  const int before = p.plan[item], n = p.plan[item + 1] - before, total = p.plan[items] * p.Hkv;
  const int per = (total + p.workers - 1) / p.workers;
  const int begin = before * p.Hkv + hk * n, c0 = begin / per, c1 = (begin + n - 1) / per;
  if (c0 == c1) return;  // (one worker's: written by it)
  const int q = r / G, h = hk * G + r - q * G;
  // part of worker c: its first part, but for the first worker's, which begins inside the run
  const auto at = [&](int c) { return ((long long)c * 2 + (c == c0 && begin != c0 * per ? 1 : 0)) * BM + (r - rt * BM); };
  const bool second = lane * 4 + 128 < Dv, active = lane * 4 < Dv;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f), acc2 = acc;
  float m = -INFINITY, l = 0.f;
  const auto scale = [&](float f) {
    l *= f;
    acc.x *= f; acc.y *= f; acc.z *= f; acc.w *= f;
    acc2.x *= f; acc2.y *= f; acc2.z *= f; acc2.w *= f;
  };
  const auto add = [&](float f, float sum, const float4& x, const float4& y) {
    l += f * sum;
    acc.x += f * x.x; acc.y += f * x.y; acc.z += f * x.z; acc.w += f * x.w;
    acc2.x += f * y.x; acc2.y += f * y.y; acc2.z += f * y.z; acc2.w += f * y.w;
  };
  // (a part that has seen nothing counts for nothing; one whose sum is no number stays so)
  const auto weight = [](float2 ml, float top) { return ml.y == 0.f ? 0.f : exp2f(ml.x - (top == -INFINITY ? 0.f : top)); };
  for (int c = c0 + warp; c <= c1; c += WARPS * U) {
    float2 ml[U];
    float4 x[U], y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {  // (all of them on their way at once)
      const bool in = c + u * WARPS <= c1;
      const long long a = in ? at(c + u * WARPS) : 0;
      ml[u] = in ? *(const float2*)(p.part_ml + a * 2) : make_float2(-INFINITY, 0.f);
      x[u] = in && active ? *(const float4*)(p.part_o + a * Dv + lane * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
      y[u] = in && second ? *(const float4*)(p.part_o + a * Dv + lane * 4 + 128) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float top = m;
#pragma unroll
    for (int u = 0; u < U; ++u) top = fmaxf(top, ml[u].x);
    scale(weight(make_float2(m, l), top));
    m = top;
#pragma unroll
    for (int u = 0; u < U; ++u) add(weight(ml[u], top), ml[u].y, x[u], y[u]);
  }
  if (WARPS > 1) {
    sums[WARPS == 1 ? 0 : warp][lane] = acc;
    sums[WARPS == 1 ? 0 : warp][lane + 32] = acc2;
    if (lane == 0) totals[warp] = make_float2(m, l);
    __syncthreads();
    if (warp != 0) return;
    float top = m;
#pragma unroll
    for (int w = 1; w < WARPS; ++w) top = fmaxf(top, totals[w].x);
    scale(weight(make_float2(m, l), top));
    m = top;
#pragma unroll
    for (int w = 1; w < WARPS; ++w) add(weight(totals[w], top), totals[w].y, sums[WARPS == 1 ? 0 : w][lane], sums[WARPS == 1 ? 0 : w][lane + 32]);
  }
  const float m_use = m == -INFINITY ? 0.f : m;
  const float inv = l > 0.f ? 1.f / l : l;  // (0 and no number stay)
  char* og = (char*)p.o.ptr + ((long long)b * p.o.sb + (long long)h * p.o.sh + (long long)q * p.o.ss) * (DT == FA_F32 ? 4 : 2);
  const auto put = [&](int col, const float4& v) {
    const float f[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
#pragma unroll
    for (int i = 0; i < 4; ++i) rot_put<DT>(og, col + i, f[i]);
  };
  if (active) put(lane * 4, acc);
  if (second) put(lane * 4 + 128, acc2);
  if (lane == 0 && p.lse != nullptr)
    p.lse[((long long)b * p.Hq + h) * p.Sq + q] = l == 0.f ? -INFINITY : (m_use + log2f(l)) * 0.6931471805599453f;
}

// ---- host --------------------------------------------------------------------------------
struct FaPagedLaunchHost {
  FaPagedParams p;
  FaTensorMapHost tk, tv;
};
struct PagedCfg {
  int RG, CG, BM, WN, slots, smem, per_sm, box, few, fr;
  bool tma, one_each;  // one_each: a CTA per segment (FA_SHORT)
};
int gcd(int a, int b) { return b == 0 ? a : gcd(b, a % b); }
FaDiv divide_by(int d) {
  FaDiv r{0, -1};
  while (d > 1 && (d - 1) >> (r.shift + 1) != 0) ++r.shift;  // 2^shift < d <= 2^(shift + 1)
  if (d > 1) r.mul = (unsigned)((1ull << (32 + r.shift)) / (unsigned)d + 1);
  return r;
}

// Tiles, buffers and CTAs per SM (the map of fa_paged.cuh).
//   * Rows: a warp takes 16; of 16-bit types up to 8, and 17 to 24 where the registers allow it, in the way made for few (`few` groups of 8);
//     fp32 rounds up to a power of two.  17 to 24 rows, three groups in a warp against two warps of 16 (us, 20 rows, D 64 and D 128): 32 x 8 segments of
//     8192 keys 103 / 166 and 182 / 211, one request of 131072 61 / 88 and 99 / 111, 64 x 8 segments of 400 26 / 35 and 34 / 44, 8 x 8 of 100 6.1 / 9.0 and 8.0 / 10.2.  Two warps
//     are faster where a table has room for far more than there is, so that segments are cut, and a worker's run is a few tiles (8 x 8 segments of 500 in tables of 16384
//     17.5 / 11.0 and 16.4 / 14.6, 64 x 8 of 400 38 / 35 and 48 / 44); lengths are not known here.  All of 17 to 24 rows, lengths and mods timed: 12 % faster on average.
//   * Keys of a tile: 32; fewer for wide heads, so that a tile of K or V stays at 8 KB and an SM has room for as many of them.
//   * CTAs of four warps, as many per SM as hold two slots (a tile of K and one of V) for each key group, up to four: that many warps hide each
//     other's waits, and more slots for fewer do not (us, two CTAs with three or more slots / three or four with two: 32 requests of up to 16384 keys D 128
//     191 / 182, one of 131072 88 / 84, 300 of up to 700 D 64 78 / 58, D 96 105 / 87, fp32 D 64 103 / 99).  Two where registers are short: more than 8
//     rows of wide heads (D 128, 12 rows 37 / 41), two and four row groups.
//   * A CTA per segment, one launch and no parts, instead of cut segments:
//     - no more segments than SMs, and tables with room for four tiles per key group: as many groups as fit, four slots each.  (us on the GPU, cut / a
//       CTA each: 64 segments of 32 tiles, D 64, eight groups 12.1 / 8.7; D 128, four groups, 8 tiles 9.3 / 7.0, 16 10.2 / 9.8, 32 14.6 / 15.5.)
//     - more segments, and tables with room for 64 tiles (32 while they would not fill the SMs one and a half times): four groups.  The SMs take a
//       segment when they have done one, while a cut run ends and begins inside segments.  (1024 segments of up to 64 tiles, D 128 108 / 95, 512 of 16, D 64
//       30 / 9.4, 256 of 4 13 / 4.4; of up to 256 tiles 98 / 114: the longest is waited for.)
void pick_paged(const fa_paged_params* p, PagedCfg& c) {
  const long long rows = (long long)(p->Hq / p->Hkv) * p->Sq;
  const bool f32 = p->dtype == FA_F32;
  const int es = esize(p->dtype);
  c.few = f32 ? 0 : rows <= 8 ? 1 : rows > 16 && rows <= 24 && p->D <= 128 ? 3 : 0;
  c.RG = rows <= 16 || c.few > 0 ? 1 : rows <= 32 ? 2 : 4;
  c.BM = c.few > 0 ? c.few * 8 : c.RG * 16;
  c.WN = !f32 ? (p->D <= 128 ? 32 : 16) : p->D <= 64 ? 32 : p->D <= 128 ? 16 : 8;
  c.fr = 0;
  if (f32)
    for (c.fr = 1; c.fr < std::min<long long>(rows, 16);) c.fr *= 2;
  c.box = gcd(p->page_size, c.WN);
  c.tma = p->D * es % 128 == 0 && p->Dv * es % 128 == 0 && c.box >= 8 && p->num_pages > 0 && !(p->flags & FA_FLAG_GENERAL_KERNELS);
  if (!c.tma) c.box = 1;
  const int slot = c.WN * (c.tma ? p->D * es : pitch(p->D, es));  // (K's: the value dim is no larger)
  const int mrows = f32 && c.RG == 1 ? c.fr : c.BM;
  const auto smem = [&](int slots) {
    const int q = f32 ? (c.RG == 1 ? c.fr : c.RG * 16) * p->D * 4 + c.CG * c.RG * c.fr * c.WN * 4 : 0;
    return c.CG * slots * slot + q + (c.CG > 1 ? c.CG * mrows * 38 * 4 : 0) + (c.tma ? c.CG * slots * 8 + 16 + 1024 : 0);
  };
  long long keys = (long long)p->table_width * p->page_size;
  if (p->window >= 0) keys = std::min<long long>(keys, (long long)p->window + p->Sq + c.WN);
  const long long segments = (long long)p->B * p->Hkv, sms = device_sm_count();
  const int most = c.RG > 1 || (f32 ? c.fr > 8 : c.few != 1 && p->D > 64) ? 2 : c.few == 1 || f32 ? 4 : 3;  // CTAs of an SM
  // as many as there is room for with `slots`
  const auto fit = [&](int slots) {
    for (c.per_sm = most; c.per_sm > 1 && smem(slots) > 227 * 1024 / c.per_sm - 1024;) --c.per_sm;
  };
  c.one_each = true;
  if (c.RG == 1 && segments <= sms) {
    c.per_sm = 1;
    c.slots = 4;
    for (c.CG = 8; c.CG >= 4; c.CG /= 2) {
      c.smem = smem(c.slots);
      if (c.smem <= kMaxSmem && keys <= 4LL * c.CG * c.WN) return;
    }
  }
  c.CG = 4 / c.RG;
  c.slots = 2;
  fit(c.slots);
  c.smem = smem(c.slots);
  if (c.RG == 1 && segments > sms && keys <= (2 * segments > 3 * sms ? 64LL : 32LL) * c.WN) return;
  c.one_each = false;
  const int room = std::min(227 * 1024 / c.per_sm - 1024, kMaxSmem);
  while (c.slots < 8 && smem(c.slots + 1) <= room) ++c.slots;
  c.smem = smem(c.slots);
}
int paged_row_tiles(const fa_paged_params* p, const PagedCfg& c) {
  return (int)(((long long)(p->Hq / p->Hkv) * p->Sq + c.BM - 1) / c.BM);
}
int paged_workers(const PagedCfg& c) { return c.per_sm * device_sm_count(); }

// (16-bit types: quotients and tanh of scores without branches, fa_score_math.cuh)
int get_paged_kernel(fa_module* m, const fa_paged_params* p, const PagedCfg& c, Kernel** k) {
  return get_kernel(m, kernel_key(kIdPaged, {{p->dtype, 2}, {p->D, 9}, {p->Dv, 9}, {c.RG, 3}, {c.WN, 6}, {c.slots, 4}, {c.tma ? 1 : 0, 1}, {c.few, 2}, {c.fr, 5}, {c.CG, 4}, {c.one_each ? 1 : 0, 1}, {c.per_sm, 3}}), "fa_paged.cuh",
                    [&] { return std::string(p->dtype == FA_F32 ? "" : "#include \"fa_score_math.cuh\"\n") +
                                defs({{"FA_DTYPE", p->dtype}, {"FA_D", p->D}, {"FA_DV", p->Dv}, {"FA_RG", c.RG}, {"FA_WN", c.WN},
                                       {"FA_SLOTS", c.slots}, {"FA_TMA", c.tma ? 1 : 0}, {"FA_FEW", c.few}, {"FA_FR", c.fr}, {"FA_CG", c.CG}, {"FA_SHORT", c.one_each ? 1 : 0}, {"FA_CTAS", c.per_sm}}); },
                    "fa_paged_kernel", c.smem, k);
}

int paged_check(fa_module* m, const fa_paged_params* p, PagedCfg& c) {
  if (!m) return fail(FA_EINVAL, "module is null");
  if (!p) return fail(FA_EINVAL, "params is null");
  if (p->dtype < FA_F16 || p->dtype > FA_F32) return fail(FA_EINVAL, "unknown dtype");
  if (p->B <= 0 || p->Hq <= 0 || p->Hkv <= 0 || p->Sq <= 0) return fail(FA_EINVAL, "B, Hq, Hkv and Sq must be positive");
  if (p->Hq % p->Hkv) return fail(FA_EINVAL, "Hq must be a multiple of Hkv");
  if (p->D <= 0 || p->D % 16 || p->Dv <= 0 || p->Dv % 16) return fail(FA_EUNSUPPORTED, "head dims must be positive multiples of 16");
  if (p->Dv > p->D) return fail(FA_EINVAL, "value head dim must not exceed the query/key head dim");
  if (p->D > 256) return fail(FA_EUNSUPPORTED, "head dim above 256 is not supported");
  if (p->Sq > 1 << 20) return fail(FA_EUNSUPPORTED, "Sq must not exceed 2^20");
  if (p->page_size <= 0 || p->num_pages < 0 || p->table_width < 0) return fail(FA_EINVAL, "page_size must be positive, num_pages and table_width not negative");
  if (p->num_pages > 0x7fffffffll) return fail(FA_EUNSUPPORTED, "num_pages must stay below 2^31");
  if (!p->lengths) return fail(FA_EINVAL, "lengths is null");
  if (p->table_width > 0 && !p->block_table) return fail(FA_EINVAL, "block_table is null");
  const int es = esize(p->dtype);
  if (int rc = check_tensor(p->q, "q", es)) return rc;
  if (int rc = check_tensor(p->o, "o", es)) return rc;
  if (int rc = check_tensor(p->k_pages, "k_pages", es, p->num_pages > 0)) return rc;
  if (int rc = check_tensor(p->v_pages, "v_pages", es, p->num_pages > 0)) return rc;
  pick_paged(p, c);
  if ((long long)p->B * p->Hq * p->Sq > 0x7fffffffll - 1024) return fail(FA_EUNSUPPORTED, "B * Hq * Sq must stay below 2^31");
  const long long longest = std::min<long long>((long long)p->table_width * p->page_size, 0x7fffffffll);
  if ((double)p->B * paged_row_tiles(p, c) * p->Hkv * (double)(longest / c.WN + 2) > 2e9) return fail(FA_EUNSUPPORTED, "more than 2e9 tiles of keys");
  return FA_OK;
}

size_t paged_up(size_t n) { return (n + 255) / 256 * 256; }
size_t paged_bytes(const fa_paged_params* p, const PagedCfg& c) {
  if (c.one_each) return 0;
  const size_t rows = 2 * (size_t)paged_workers(c) * c.BM;
  return paged_up(rows * p->Dv * 4) + paged_up(rows * 8) + paged_up(((size_t)p->B * paged_row_tiles(p, c) + 1) * 4);
}

}  // namespace

extern "C" {

int fa_page_step(const int32_t* lengths, const int32_t* new_tokens, int B, int32_t* block_table, int64_t block_table_stride, int table_width,
                 const int32_t* free_pages, int64_t num_free, const int32_t* taken, int page_size, int64_t num_tokens,
                 int32_t* out_lengths, int32_t* positions, int64_t* slots, int32_t* requests, int32_t* starts, int32_t* out_taken, void* stream) {
  if (B < 0 || table_width < 0 || num_free < 0 || num_tokens < 0 || page_size <= 0)
    return fail(FA_EINVAL, "B, table_width, num_free and num_tokens must not be negative, page_size must be positive");
  if (B > 0 && (!lengths || !new_tokens || !out_lengths)) return fail(FA_EINVAL, "lengths, new_tokens or out_lengths is null");
  if (!starts || !out_taken) return fail(FA_EINVAL, "starts or out_taken is null");
  if (num_tokens > 0 && (!positions || !slots || !requests)) return fail(FA_EINVAL, "positions, slots or requests is null");
  if ((B > 0 && table_width > 0 && !block_table) || (num_free > 0 && !free_pages)) return fail(FA_EINVAL, "block_table or free_pages is null");
  if (num_tokens > 0x7fffffffll) return fail(FA_EUNSUPPORTED, "num_tokens must stay below 2^31");
  prof_reset();
  FaStepParams k{};
  k.len = lengths; k.count = new_tokens; k.free_pages = free_pages; k.taken_in = taken;
  k.table = block_table; k.table_stride = block_table_stride; k.tokens = num_tokens;
  k.num_free = std::min<int64_t>(num_free, 0x7fffffffll);  // (no more pages have a number)
  k.B = B; k.width = table_width; k.page = page_size;
  k.out_len = out_lengths; k.positions = positions; k.requests = requests; k.starts = starts; k.taken_out = out_taken;
  k.slots = (long long*)slots;
  // Two blocks per SM at most, since each goes over all requests.
  k.per_block = (int)std::max<long long>(4 * kStepThreads, (num_tokens / (2 * device_sm_count()) + kStepThreads) / kStepThreads * kStepThreads);
  const unsigned blocks = (unsigned)std::max<long long>(1, (num_tokens + k.per_block - 1) / k.per_block);
  k.pages_per_block = (int)((num_tokens / page_size + B) / blocks + 1);  // (n tokens more take ceil(n / page_size) pages more at most)
  return launch_here("fa_page_step_kernel", fa_page_step_kernel, dim3(blocks), dim3(kStepThreads), stream, k);
}

size_t fa_paged_workspace_bytes(const fa_paged_params* p) {
  if (!p || p->Hkv <= 0 || p->Hq <= 0 || p->Sq <= 0 || p->D <= 0 || p->Dv <= 0 || p->page_size <= 0 || p->B <= 0) return 0;
  PagedCfg c;
  pick_paged(p, c);
  size_t most = paged_bytes(p, c);
  if (c.tma) {  // (what runs where no tensor map takes the strides)
    fa_paged_params q = *p;
    q.flags |= FA_FLAG_GENERAL_KERNELS;
    pick_paged(&q, c);
    most = std::max(most, paged_bytes(&q, c));
  }
  return most;
}

int fa_paged_prepare(fa_module* m, const fa_paged_params* p) {
  if (!m || !p) return fail(FA_EINVAL, "module or params is null");
  if (p->dtype < FA_F16 || p->dtype > FA_F32 || p->Hkv <= 0 || p->Hq <= 0 || p->Hq % p->Hkv || p->Sq <= 0 || p->page_size <= 0 || p->D <= 0 || p->D > 256 ||
      p->D % 16 || p->Dv <= 0 || p->Dv > p->D || p->Dv % 16)
    return fail(FA_EINVAL, "type, heads, head dims or sizes that fa_paged does not take");
  PagedCfg c;
  pick_paged(p, c);
  Kernel* kernel = nullptr;
  return get_paged_kernel(m, p, c, &kernel);
}

int fa_paged(fa_module* m, const fa_paged_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  PagedCfg c;
  if (int rc = paged_check(m, p, c)) return rc;
  if ((uintptr_t)workspace & 15) return fail(FA_EINVAL, "workspace must be 16-byte aligned");
  prof_reset();
  FaPagedLaunchHost L;
  memset(&L, 0, sizeof L);
  FaPagedParams& k = L.p;
  fill_buffers(m, k.mod_buf);
  k.q = cvt(p->q); k.k = cvt(p->k_pages); k.v = cvt(p->v_pages); k.o = cvt(p->o);
  k.lse = p->lse; k.table = p->block_table; k.table_stride = p->block_table_stride; k.lengths = p->lengths; k.status = p->status;
  k.B = p->B; k.Hq = p->Hq; k.Hkv = p->Hkv; k.Sq = p->Sq;
  k.num_pages = (int)p->num_pages; k.page_size = p->page_size;
  k.by_page = divide_by(p->page_size);
  k.by_group = divide_by(p->Hq / p->Hkv);
  k.max_len = (int)std::min<long long>((long long)p->table_width * p->page_size, 0x7fffffffll - 64);
  k.window = p->window < 0 ? -1 : std::min(p->window, 1 << 30);
  k.b_off = p->b_offset; k.h_off = p->h_offset; k.scale = p->scale;
  if (c.tma) {
    // (strides that no tensor map takes: 16-byte pieces)
    if (make_map(&L.tk, p->dtype, p->k_pages, p->D, p->page_size, p->Hkv, (int)p->num_pages, c.box) != FA_OK ||
        make_map(&L.tv, p->dtype, p->v_pages, p->Dv, p->page_size, p->Hkv, (int)p->num_pages, c.box) != FA_OK) {
      fa_paged_params q = *p;
      q.flags |= FA_FLAG_GENERAL_KERNELS;
      pick_paged(&q, c);
    }
  }
  const size_t need = paged_bytes(p, c);
  if (need && (!workspace || workspace_bytes < need)) return fail(FA_EWORKSPACE, "paged attention workspace too small");
  k.row_tiles = paged_row_tiles(p, c);
  k.by_tiles = divide_by(k.row_tiles);
  k.workers = paged_workers(c);
  const size_t rows = 2 * (size_t)k.workers * c.BM;
  k.part_o = (float*)workspace;
  k.part_ml = (float*)((char*)workspace + paged_up(rows * p->Dv * 4));
  k.plan = (int*)((char*)k.part_ml + paged_up(rows * 8));
  k.box = c.box;
  Kernel* kernel = nullptr;
  if (int rc = get_paged_kernel(m, p, c, &kernel)) return rc;
  const dim3 block((unsigned)(c.CG * c.RG * 32));
  if (c.one_each) return launch(kernel, dim3((unsigned)((long long)p->B * k.row_tiles * p->Hkv)), block, &L, stream);
  if (int rc = launch(kernel, dim3((unsigned)k.workers), block, &L, stream)) return rc;
  // Few segments for the workers: many parts each, and eight warps add up a row's.
  const long long segments = (long long)p->B * k.row_tiles * p->Hkv;
  const int n_rows = p->B * p->Hq * p->Sq;
  const bool wide = k.workers / segments >= 16;
  return rot_dispatch(p->dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    return wide ? launch_here("fa_paged_combine_kernel", fa_paged_combine_kernel<DT, 8>, dim3((unsigned)n_rows), dim3(256), stream, k, c.BM, p->Dv, n_rows)
                : launch_here("fa_paged_combine_kernel", fa_paged_combine_kernel<DT, 1>, dim3((unsigned)((n_rows + 3) / 4)), dim3(128), stream, k, c.BM, p->Dv, n_rows);
  });
}

}  // extern "C"
