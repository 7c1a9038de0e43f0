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

// ---- tokens out of their pages ---------------------------------------------------------------
//   row t of key and value = token t - starts[b] of request b: w scale of pages in 8 bits, rounded once, or a copy.
//
// A block takes a run of tokens: it finds their requests and pages (the requests that end in front of the first are counted by all threads, the
// others are walked through from there), then goes through their rows, a group of lanes to a row and 16 bytes of it to a lane, four rows of a lane on their way at a
// time.  Rows of tokens beside each other, which lie one behind the other in a page, are in groups beside each other.
constexpr int kReadThreads = 256, kReadTokens = 64, kReadEight = 3;  // (kReadEight: the type of pages in 8 bits, beside FA_F16, FA_BF16 and FA_F32)

struct FaReadKernelParams {
  FaRotTensor pages[2], out[2];  // byte strides
  const float* scales[2];        // element strides of page, head and token in a page
  long long scale_sp[2], scale_sh[2], scale_ss[2];
  const int *table, *starts;
  long long table_stride;
  int B, Hkv, D[2], width, num_pages, page_size, tokens;
  int token_shift, lane_shift;   // log2 of a block's tokens, of the lanes that share a row
  int* status;
};

// Four values of 8 bits: in the low byte of 2^23, which is subtracted with the 128 that makes them positive.
__device__ __forceinline__ void read_four(unsigned w, F2 scale, F2* f) {
  w ^= 0x80808080u;
  const auto at = [&](int i) { return __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 | i)); };
  const F2 one = f2(1.f, 1.f), bias = f2(-8388736.f, -8388736.f);
  f[0] = fma(f2(at(0), at(1)), one, bias) * scale;
  f[1] = fma(f2(at(2), at(3)), one, bias) * scale;
}

// PIECES: 16 bytes of the pages at a time; else value by value.  Four blocks per SM; with the registers for three, 45000 tokens in 8 bits (8 heads, D 128) take 4 us more.  (72000
// tokens: bf16 102 us, 5.8 TB/s, in 8 bits 94.)
template <int IN, int OUT, bool PIECES>
__global__ void __launch_bounds__(kReadThreads, 4) fa_read_pages_kernel(const __grid_constant__ FaReadKernelParams P) {
  grid_wait();
  constexpr bool EIGHT = IN == kReadEight;
  constexpr int ES = OUT == FA_F32 ? 4 : 2, EI = EIGHT ? 1 : ES, V = PIECES ? 16 / EI : 1, U = 4;
  __shared__ long long from_of[kReadTokens], scale_of[kReadTokens];  // where a token's row of head 0 is; below 0: it has none
  const int kind = blockIdx.y;  // keys or values
  const int t0 = blockIdx.x << P.token_shift, n = min(1 << P.token_shift, P.tokens - t0), tid = threadIdx.x;
  int before = 0;
  if (blockIdx.x == 0 && kind == 0 && P.status != nullptr) {  // starts that decrease
#pragma unroll 1
    for (int b = tid; b < P.B; b += kReadThreads)
      if (P.starts[b] > P.starts[b + 1]) atomicOr(P.status, FA_STATUS_BAD_START);
  }
  for (int b0 = 0; b0 < P.B; b0 += kReadThreads) before += __syncthreads_count(b0 + tid < P.B && P.starts[min(b0 + tid, P.B - 1) + 1] <= t0);
  if (tid < n) {
    const int t = t0 + tid;
    int b = before;
    while (b < P.B && P.starts[b + 1] <= t) ++b;
    long long page = -1;
    int row = 0;
    if (b < P.B && P.starts[b] <= t) {
      const int j = (int)min((long long)t - P.starts[b], (long long)INT_MAX), slot = j / P.page_size;
      row = j - slot * P.page_size;
      if (slot < P.width) page = P.table[b * P.table_stride + slot];
      if (page < 0 || page >= P.num_pages) {
        page = -1;
        if (P.status != nullptr) atomicOr(P.status, FA_STATUS_BAD_PAGE);
      }
    }
    from_of[tid] = page < 0 ? -1 : page * P.pages[kind].sb + row * P.pages[kind].ss;
    if (EIGHT) scale_of[tid] = page < 0 ? 0 : page * P.scale_sp[kind] + row * P.scale_ss[kind];
  }
  __syncthreads();
  const int groups = kReadThreads >> P.lane_shift, lane = tid & ((1 << P.lane_shift) - 1), rows = P.Hkv << P.token_shift, D = P.D[kind];
  const FaRotTensor src = P.pages[kind], dst = P.out[kind];
  const float* const scales = P.scales[kind];
  const long long scale_sh = P.scale_sh[kind];
#pragma unroll 1
  for (int r0 = tid >> P.lane_shift; r0 < rows; r0 += U * groups) {
#pragma unroll 1
    for (int c = lane;; c += 1 << P.lane_shift) {
      if (c * V >= D) break;
      uint4 raw[U];
      float scale[U];
      char* to[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {  // (all of them on their way at once)
        const int r = r0 + u * groups, t = r & ((1 << P.token_shift) - 1), h = r >> P.token_shift;
        to[u] = nullptr;
        raw[u] = make_uint4(0, 0, 0, 0);
        scale[u] = 0.f;
        if (r >= rows || t >= n) continue;
        to[u] = dst.ptr + h * dst.sh + (t0 + t) * dst.ss + c * V * ES;
        const long long at = from_of[t];
        if (at < 0) continue;
        const char* from = src.ptr + at + h * src.sh + c * V * EI;
        if (EIGHT) scale[u] = scales[scale_of[t] + h * scale_sh];
        if (PIECES) raw[u] = __ldcs((const uint4*)from);
        else raw[u].x = EI == 1 ? (unsigned)*(const unsigned char*)from : EI == 2 ? (unsigned)*(const unsigned short*)from : *(const unsigned*)from;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (to[u] == nullptr) continue;
        if constexpr (!EIGHT) {
          if (PIECES) *(uint4*)to[u] = raw[u];
          else if (ES == 2) *(unsigned short*)to[u] = (unsigned short)raw[u].x;
          else *(unsigned*)to[u] = raw[u].x;
        } else {
          const F2 s = f2(scale[u], scale[u]);
          F2 f[8];
          read_four(raw[u].x, s, f);
          if (!PIECES) {
            float x, y;
            f2_get(f[0], x, y);
            rot_put<OUT>(to[u], 0, x);
          } else {
            read_four(raw[u].y, s, f + 2);
            read_four(raw[u].z, s, f + 4);
            read_four(raw[u].w, s, f + 6);
#pragma unroll
            for (int w = 0; w < ES; ++w) {
              F2 g[kRotPairs<OUT>];
#pragma unroll
              for (int k = 0; k < kRotPairs<OUT>; ++k) g[k] = f[w * kRotPairs<OUT> + k];
              __stcs((uint4*)(to[u] + w * 16), rot_pack<OUT>(g));
            }
          }
        }
      }
    }
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
  if (p.out_ml != nullptr) {  // (behind a prefix: fa_merge_kernel goes on from here)
    float* const to = (float*)p.o.ptr + (long long)b * p.o.sb + (long long)h * p.o.sh + (long long)q * p.o.ss;
    if (active) *(float4*)(to + lane * 4) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    if (second) *(float4*)(to + lane * 4 + 128) = make_float4(acc2.x * inv, acc2.y * inv, acc2.z * inv, acc2.w * inv);
    if (lane == 0) *(float2*)(p.out_ml + (((long long)b * p.Hq + h) * p.Sq + q) * 2) = make_float2(m_use, l);
    return;
  }
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
  bool eight, after;   // pages in 8 bits (FA_KV8), keys behind a prefix (FA_AFTER)
};
int gcd(int a, int b) { return b == 0 ? a : gcd(b, a % b); }

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
//   * 8 bits: three CTAs, and two for more than 8 rows, with two slots: the whole numbers' way to 16 bits takes registers, and with four CTAs (128 registers a
//     thread) they spill.  (us, four / three / two CTAs: 32 requests of up to 16384 keys D 128 171 / 147 / 168, 20 rows over 16 x 4 segments of 4097 140 / 95 / 57;
//     with more slots 257 / 150 / 171 and 140 / 99 / 60.)
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
  c.eight = p->k_scales.ptr != nullptr;
  c.after = p->prefix_length > 0;
  c.few = c.eight ? (rows <= 8 || p->D > 128 ? 1 : rows <= 16 ? 2 : 3) : f32 ? 0 : rows <= 8 ? 1 : rows > 16 && rows <= 24 && p->D <= 128 ? 3 : 0;
  c.RG = rows <= 16 || c.few > 0 ? 1 : rows <= 32 ? 2 : 4;
  c.BM = c.few > 0 ? c.few * 8 : c.RG * 16;
  c.WN = c.eight ? 32 : !f32 ? (p->D <= 128 ? 32 : 16) : p->D <= 64 ? 32 : p->D <= 128 ? 16 : 8;
  c.fr = 0;
  if (f32)
    for (c.fr = 1; c.fr < std::min<long long>(rows, 16);) c.fr *= 2;
  c.box = gcd(p->page_size, c.WN);
  c.tma = (c.eight || (p->D * es % 128 == 0 && p->Dv * es % 128 == 0)) && c.box >= 8 && p->num_pages > 0 && !(p->flags & FA_FLAG_GENERAL_KERNELS);
  if (!c.tma) c.box = 1;
  const int group = p->D <= 64 ? 64 : 128;  // (8 bits: whole column groups)
  const int slot = c.WN * (c.eight ? (p->D + group - 1) / group * group : c.tma ? p->D * es : pitch(p->D, es));  // (K's: the value dim is no larger)
  const int mrows = f32 && c.RG == 1 ? c.fr : c.BM;
  const auto smem = [&](int slots) {
    const int q = f32 ? (c.RG == 1 ? c.fr : c.RG * 16) * p->D * 4 + c.CG * c.RG * c.fr * c.WN * 4 : 0;
    return c.CG * slots * slot + q + (c.CG > 1 ? c.CG * mrows * 38 * 4 : 0) + (c.tma ? c.CG * slots * 8 + 16 + 1024 : 0);
  };
  long long keys = (long long)p->table_width * p->page_size;
  if (p->window >= 0) keys = std::min<long long>(keys, (long long)p->window + p->Sq + c.WN);
  const long long segments = (long long)p->B * p->Hkv, sms = device_sm_count();
  const int most = c.eight ? (c.few > 1 || p->D > 128 ? 2 : p->D > 64 ? 3 : 4) : c.RG > 1 || (f32 ? c.fr > 8 : c.few != 1 && p->D > 64) ? 2 : c.few == 1 || f32 ? 4 : 3;  // CTAs of an SM
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
  while (c.slots < (c.eight ? 2 : 8) && smem(c.slots + 1) <= room) ++c.slots;
  c.smem = smem(c.slots);
}
int paged_row_tiles(const fa_paged_params* p, const PagedCfg& c) {
  return (int)(((long long)(p->Hq / p->Hkv) * p->Sq + c.BM - 1) / c.BM);
}
int paged_workers(const PagedCfg& c) { return c.per_sm * device_sm_count(); }

// (16-bit types: quotients and tanh of scores without branches, fa_score_math.cuh)
int get_paged_kernel(fa_module* m, const fa_paged_params* p, const PagedCfg& c, Kernel** k) {
  return get_kernel(m, kernel_key(kIdPaged, {{p->dtype, 2}, {p->D, 9}, {p->Dv, 9}, {c.RG, 3}, {c.WN, 6}, {c.slots, 4}, {c.tma ? 1 : 0, 1}, {c.few, 2}, {c.fr, 5}, {c.CG, 4}, {c.one_each ? 1 : 0, 1}, {c.per_sm, 3}, {c.eight ? 1 : 0, 1}, {c.after ? 1 : 0, 1}}), "fa_paged.cuh",
                    [&] { return std::string(p->dtype == FA_F32 ? "" : c.eight ? "#define FA_PAIRS 1\n#include \"fa_score_math.cuh\"\n" : "#include \"fa_score_math.cuh\"\n") +
                                defs({{"FA_DTYPE", p->dtype}, {"FA_D", p->D}, {"FA_DV", p->Dv}, {"FA_RG", c.RG}, {"FA_WN", c.WN},
                                       {"FA_SLOTS", c.slots}, {"FA_TMA", c.tma ? 1 : 0}, {"FA_FEW", c.few}, {"FA_FR", c.fr}, {"FA_CG", c.CG}, {"FA_SHORT", c.one_each ? 1 : 0}, {"FA_CTAS", c.per_sm}, {"FA_KV8", c.eight ? 1 : 0}, {"FA_AFTER", c.after ? 1 : 0}}); },
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
  const bool eight = p->k_scales.ptr || p->v_scales.ptr;
  if (eight && !(p->k_scales.ptr && p->v_scales.ptr)) return fail(FA_EINVAL, "scales of keys and of values, or none");
  if (eight && p->dtype == FA_F32) return fail(FA_EUNSUPPORTED, "pages in 8 bits take queries of 16 bits");
  if (p->prefix_length < 0) return fail(FA_EINVAL, "prefix_length must not be negative");
  if (p->prefix_length > 0) {
    if (int rc = check_tensor(p->k_prefix, "k_prefix", es)) return rc;
    if (int rc = check_tensor(p->v_prefix, "v_prefix", es)) return rc;
    if (p->prefix_length > 1 << 23) return fail(FA_EUNSUPPORTED, "a prefix of more than 2^23 tokens");
  }
  if (int rc = check_tensor(p->k_pages, "k_pages", eight ? 1 : es, p->num_pages > 0)) return rc;
  if (int rc = check_tensor(p->v_pages, "v_pages", eight ? 1 : es, p->num_pages > 0)) return rc;
  pick_paged(p, c);
  if ((long long)p->B * p->Hq * p->Sq > 0x7fffffffll - 1024) return fail(FA_EUNSUPPORTED, "B * Hq * Sq must stay below 2^31");
  const long long longest = std::min<long long>((long long)p->table_width * p->page_size, 0x7fffffffll);
  if ((double)p->B * paged_row_tiles(p, c) * p->Hkv * (double)(longest / c.WN + 2) > 2e9) return fail(FA_EUNSUPPORTED, "more than 2e9 tiles of keys");
  return FA_OK;
}

size_t paged_up(size_t n) { return (n + 255) / 256 * 256; }
// what the pages' part of a call needs
size_t paged_own_bytes(const fa_paged_params* p, const PagedCfg& c) {
  if (c.one_each) return 0;
  const size_t rows = 2 * (size_t)paged_workers(c) * c.BM;
  return paged_up(rows * p->Dv * 4) + paged_up(rows * 8) + paged_up(((size_t)p->B * paged_row_tiles(p, c) + 1) * 4);
}
// Behind a prefix: the sums of its parts and of the pages, too
size_t paged_bytes(const fa_paged_params* p, const PagedCfg& c) {
  if (!c.after) return paged_own_bytes(p, c);
  const size_t rows = (size_t)p->B * p->Hq * p->Sq;
  return paged_own_bytes(p, c) + (size_t)(prefix_parts(p) + 1) * (paged_up(rows * p->Dv * 4) + paged_up(rows * 8));
}

// the kernels over the pages; `rows`: of the parts in the workspace
int launch_paged(fa_module* m, const fa_paged_params* p, const PagedCfg& c, FaPagedLaunchHost& L, void* workspace, size_t rows, void* stream) {
  FaPagedParams& k = L.p;
  k.part_o = (float*)workspace;
  k.part_ml = (float*)((char*)workspace + paged_up(rows * p->Dv * 4));
  k.plan = (int*)((char*)k.part_ml + paged_up(rows * 8));
  k.box = c.box;
  k.by_box = divide_by(c.box);
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

int fa_read_pages(const fa_read_params* p, void* stream) {
  if (!p) return fail(FA_EINVAL, "params is null");
  if (p->dtype < FA_F16 || p->dtype > FA_F32) return fail(FA_EINVAL, "unknown dtype");
  if (p->B < 0 || p->Hkv < 0 || p->D <= 0 || p->Dv <= 0 || p->num_tokens < 0) return fail(FA_EINVAL, "B, Hkv and num_tokens must not be negative, head dims must be positive");
  if (p->D > 256 || p->Dv > 256) return fail(FA_EUNSUPPORTED, "head dims from 1 to 256");
  if (p->Hkv > 65535) return fail(FA_EUNSUPPORTED, "Hkv must not exceed 65535");
  if (p->num_tokens > 0x7fffffffll - 256 || p->num_pages > 0x7fffffffll) return fail(FA_EUNSUPPORTED, "num_tokens and num_pages must stay below 2^31");
  if (p->page_size <= 0 || p->num_pages < 0 || p->table_width < 0) return fail(FA_EINVAL, "page_size must be positive, num_pages and table_width not negative");
  const bool eight = p->k_scales.ptr || p->v_scales.ptr;
  if (eight && !(p->k_scales.ptr && p->v_scales.ptr)) return fail(FA_EINVAL, "scales of keys and of values, or none");
  prof_reset();
  if (p->num_tokens == 0 || p->Hkv == 0) return FA_OK;
  if (!p->k.ptr || !p->v.ptr || (p->num_pages > 0 && (!p->k_pages.ptr || !p->v_pages.ptr))) return fail(FA_EINVAL, "a tensor is null");
  if (p->B > 0 && (!p->starts || (p->table_width > 0 && !p->block_table))) return fail(FA_EINVAL, "starts or block_table is null");
  FaReadKernelParams k;
  memset(&k, 0, sizeof k);
  const int es = esize(p->dtype), ei = eight ? 1 : es;
  const fa_tensor *from[2] = {&p->k_pages, &p->v_pages}, *to[2] = {&p->k, &p->v}, *scales[2] = {&p->k_scales, &p->v_scales};
  const int v = 16 / ei;
  bool pieces = p->D % v == 0 && p->Dv % v == 0;
  for (int i = 0; i < 2; ++i) {
    k.pages[i] = rot_tensor(*from[i], ei);
    k.out[i] = rot_tensor(*to[i], es);
    k.out[i].sb = 0;
    k.scales[i] = (const float*)scales[i]->ptr;
    k.scale_sp[i] = scales[i]->stride_b; k.scale_sh[i] = scales[i]->stride_h; k.scale_ss[i] = scales[i]->stride_s;
    pieces = pieces && rot_aligned(k.pages[i]) && rot_aligned(k.out[i]);
  }
  k.D[0] = p->D; k.D[1] = p->Dv;
  k.table = p->block_table; k.table_stride = p->block_table_stride; k.width = p->table_width;
  k.starts = p->starts; k.B = p->B; k.Hkv = p->Hkv;
  k.num_pages = (int)p->num_pages; k.page_size = p->page_size; k.tokens = (int)p->num_tokens;
  k.status = p->status;
  // As many tokens of a block as leave four blocks per SM: the search for the requests is paid once for them.
  while (1 << k.token_shift < kReadTokens && (p->num_tokens >> (k.token_shift + 1)) >= 3LL * device_sm_count()) ++k.token_shift;
  while (1 << k.lane_shift < 32 && (pieces ? v : 1) << k.lane_shift < std::max(p->D, p->Dv)) ++k.lane_shift;
  const dim3 grid((unsigned)((p->num_tokens + (1ll << k.token_shift) - 1) >> k.token_shift), 2);
  return rot_dispatch(p->dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    void (*const fns[2][2])(FaReadKernelParams) = {{fa_read_pages_kernel<DT, DT, false>, fa_read_pages_kernel<DT, DT, true>},
                                                   {fa_read_pages_kernel<kReadEight, DT, false>, fa_read_pages_kernel<kReadEight, DT, true>}};
    return launch_here("fa_read_pages_kernel", fns[eight][pieces], grid, dim3(kReadThreads), stream, k);
  });
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
  if (c.eight && p->dtype == FA_F32) return fail(FA_EUNSUPPORTED, "pages in 8 bits take queries of 16 bits");
  if (p->prefix_length > 0)
    if (int rc = get_prefix_kernel(m, p, prefix_rows(p), &kernel)) return rc;
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
  k.k_scales = cvt(p->k_scales); k.v_scales = cvt(p->v_scales);
  if (c.tma) {
    // (strides that no tensor map takes: 16-byte pieces)
    const int type = c.eight ? kMapInt8 : p->dtype, group = c.eight && p->D <= 64 ? 64 : 128;
    if (make_map(&L.tk, type, p->k_pages, p->D, p->page_size, p->Hkv, (int)p->num_pages, c.box, group) != FA_OK ||
        make_map(&L.tv, type, p->v_pages, p->Dv, p->page_size, p->Hkv, (int)p->num_pages, c.box, group) != FA_OK) {
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
  if (c.after) {
    // the prefix first: its kernel has the most to do, and the CTAs of the pages' get ready while it ends
    char* at = (char*)workspace;
    const size_t all = (size_t)p->B * p->Hq * p->Sq, parts = (size_t)prefix_parts(p);
    const auto take = [&](size_t n) {
      char* r = at;
      at += paged_up(n);
      return (float*)r;
    };
    float *const po = take(parts * all * p->Dv * 4), *const pml = take(parts * all * 8), *const own = take(all * p->Dv * 4);
    k.out_ml = take(all * 8);
    k.after = p->prefix_length;
    k.o = FaTensor{own, (long long)p->Hq * p->Sq * p->Dv, (long long)p->Sq * p->Dv, p->Dv};
    workspace = at;
    if (int rc = launch_prefix(m, p, po, pml, stream)) return rc;
    if (int rc = launch_paged(m, p, c, L, workspace, rows, stream)) return rc;
    return launch_merge(p->dtype, FaMergeParams{po, pml, own, k.out_ml, cvt(p->o), p->lse, p->B, p->Hq, p->Hkv, p->Sq, p->Dv, (int)parts}, stream);
  }
  return launch_paged(m, p, c, L, workspace, rows, stream);
}

}  // extern "C"
