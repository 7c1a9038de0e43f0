// The rows of attention over requests of different lengths that lie end to end, and of the newest tokens of many requests over a prefix that
// they share.  The G query heads of a kv head share its keys, so rows are (token, head of the group), row r is head r % G of token r / G, and a
// kernel takes them in items of R rows.
//
//   prompts  An item's rows are of one request.  Lengths are known on the device only; every CTA looks its item up.  Up to 256 requests, items
//            with the most keys in front: in the order of their place in the request, the last first, over all requests.  Of more, request by
//            request, a third of the items nobody's: a look at all requests for each item takes longer (16 tokens each, 32 / 8 heads, D 128, bf16:
//            by level 256 requests 67 us, 512 193, 1024 614; by request 81, 161, 329).  Rows that belong to no request, in front of the first and
//            behind the last, have items too, and see nothing.
//   prefix   The rows of all requests, one behind the other.
#pragma once
#include "fa_common.cuh"

// What an item works on
struct FaPlace {
  int q0, n;    // first token of the request among all queries, how many it has
  int k0, nk;   // the same of its keys
  int b;        // request
  int first;    // first row of the item among the request's
  int any;      // 0: there is no such item
};

__device__ __forceinline__ int fa_divided(int n, const FaDiv& d) { return d.shift < 0 ? n : (int)(__umulhi((fa_u32)n, d.mul) >> d.shift); }

// begin and end of request s, whatever stands in the starts
__device__ __forceinline__ void fa_range(const int* starts, int s, int most, int& begin, int& end) {
  begin = min(max(starts[s], 0), most);
  end = min(max(starts[s + 1], begin), most);
}

// the rows of no request in front of the first and behind the last, from their item `item` on
template <int R>
__device__ __forceinline__ FaPlace fa_no_request(const FaPackedParams& p, bool behind, int front, int back, long long item) {
  FaPlace r = {0, 0, 0, 0, 0, 0, 0};
  r.q0 = behind ? back : 0;
  r.n = behind ? p.tokens - back : front;
  const long long first = item * R;
  r.first = (int)min(max(first, 0ll), (long long)0x7fffffff);
  r.any = first >= 0 && first < (long long)r.n * (p.Hq / p.Hkv);  // (below 0: of broken starts)
  return r;
}
__device__ __forceinline__ FaPlace fa_request(const FaPackedParams& p, int b, int first) {
  FaPlace r = {0, 0, 0, 0, b, first, 1};
  int end;
  fa_range(p.starts, b, p.tokens, r.q0, end);
  r.n = end - r.q0;
  fa_range(p.key_starts, b, p.keys, r.k0, end);
  r.nk = end - r.k0;
  return r;
}

// Up to 256 requests, by the 32 lanes of a warp together.  The items of level l are those with l others of their request in front of
// them; total(l) of all have level l or more, so the level of an item is found by halving, and its request by counting those that
// reach it.
template <int R>
__device__ __forceinline__ FaPlace fa_find_by_level(const FaPackedParams& p, long long item) {
  constexpr int KEEP = 8;
  const int lane = threadIdx.x & 31, G = p.Hq / p.Hkv;
  int kept[KEEP], most = 0;
#pragma unroll
  for (int i = 0; i < KEEP; ++i) {
    kept[i] = 0;
    if (i * 32 + lane < p.B) {
      int begin, end;
      fa_range(p.starts, i * 32 + lane, p.tokens, begin, end);
      kept[i] = (int)(((long long)(end - begin) * G + R - 1) / R);
    }
    most = max(most, kept[i]);
  }
  most = __reduce_max_sync(0xffffffffu, most);
  const auto total = [&](int level) {
    long long sum = 0;
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      if (i * 32 < p.B) sum += max(kept[i] - level, 0);
    // (of broken starts the sum may need more than 32 bits)
    const fa_u32 lo = __reduce_add_sync(0xffffffffu, (fa_u32)sum & 0xffffffu), hi = __reduce_add_sync(0xffffffffu, (fa_u32)(sum >> 24));
    return (long long)lo + ((long long)hi << 24);
  };
  const long long all = total(0);
  if (item >= all) {
    const int front = p.B > 0 ? min(max(p.starts[0], 0), p.tokens) : 0, back = p.B > 0 ? min(max(p.starts[p.B], 0), p.tokens) : 0;
    const long long items_front = ((long long)front * G + R - 1) / R, left = item - all;
    const bool behind = left >= items_front;
    return fa_no_request<R>(p, behind, front, back, behind ? left - items_front : left);
  }
  int lo = 0, hi = most - 1;  // the last level l with total(l) > item
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (total(mid) > item) lo = mid;
    else hi = mid - 1;
  }
  int rank = (int)(item - total(lo + 1)), b = 0;
  bool found = false;
#pragma unroll
  for (int i = 0; i < KEEP; ++i) {
    const fa_u32 reach = __ballot_sync(0xffffffffu, kept[i] > lo);
    const int n = __popc(reach);
    const fa_u32 mine = __ballot_sync(0xffffffffu, ((reach >> lane) & 1u) && __popc(reach & ((1u << lane) - 1u)) == rank);
    if (!found && rank < n) {
      b = i * 32 + __ffs(mine) - 1;
      found = true;
    }
    if (!found) rank -= n;
  }
  return fa_request(p, b, lo * R);
}

// More requests.  Request s, which begins at row x of all, has the item numbers from x / R + s + 1 on up to the next request's: as many as it
// needs, or one more, which is nobody's.  The request whose numbers an item has is found by looking at 32 of them at a time.
template <int R>
__device__ __forceinline__ FaPlace fa_find_by_request(const FaPackedParams& p, long long item) {
  const int lane = threadIdx.x & 31, G = p.Hq / p.Hkv;
  const auto row = [&](int s) { return min(max(p.starts[s], 0), p.tokens); };
  const auto number = [&](int s) { return (long long)row(s) * G / R + s + 1; };
  int lo = -1, hi = p.B + 1;  // number(lo) <= item < number(hi); -1: in front of all requests, B: behind
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step;
    const int upto = __popc(__ballot_sync(0xffffffffu, at < hi && number(min(at, p.B)) <= item));  // (never decreasing)
    lo += upto * step;
    hi = min(hi, lo + step);
  }
  if (lo < 0 || lo >= p.B) return fa_no_request<R>(p, lo >= 0, row(0), row(p.B), lo < 0 ? item : item - number(p.B));
  const long long first = (item - number(lo)) * R;
  FaPlace r = fa_request(p, lo, (int)min(max(first, 0ll), (long long)0x7fffffff));
  r.any = first >= 0 && first < (long long)r.n * G;
  return r;
}
template <int R>
__device__ __forceinline__ FaPlace fa_find_item(const FaPackedParams& p, long long item) {
  return p.B <= 256 ? fa_find_by_level<R>(p, item) : fa_find_by_request<R>(p, item);
}

// starts that decrease, or lie where there are no tokens: said once, by the threads of one CTA.  (Of such that decrease requests overlap, and may have more items than the grid
// has CTAs: nothing is read or written out of range, but rows may be left out.  Finding that out in every CTA would take a look at all starts.)
__device__ __forceinline__ void fa_check_starts(const FaPackedParams& p, int tid, int threads) {
  bool bad = false;
  for (int s = tid; s < p.B; s += threads)
    bad |= p.starts[s] < 0 || p.starts[s] > p.starts[s + 1] || p.starts[s + 1] > p.tokens || p.key_starts[s] < 0 || p.key_starts[s] > p.key_starts[s + 1] || p.key_starts[s + 1] > p.keys;
  if (bad && p.status != nullptr) atomicOr(p.status, FA_STATUS_BAD_START);
}

// A row of an item
struct FaRow {
  long long at;  // its query, in elements from head 0 of the kv head's group on; -1: there is no such row
  int head;      // of the group
  int token;     // of the request (prompts), or among all (prefix)
  int b, pos;    // request; position in it
  int from, to;  // the keys that it sees
};
template <bool PREFIX>
__device__ __forceinline__ FaRow fa_row(const FaPackedParams& p, const FaPlace& place, int row) {
  FaRow r;
  const int t = fa_divided(row, p.by_group);
  r.token = t;
  r.head = row - t * (p.Hq / p.Hkv);
  r.from = 0;
  if (PREFIX) {
    const bool in = t < p.tokens;
    r.b = in ? fa_divided(t, p.by_sq) : 0;
    const int i = t - r.b * p.Sq, own = in ? min(p.lengths[r.b], 0x3fffffff) - p.Sq + i : -1;
    r.pos = p.keys + max(own, 0);
    r.to = own >= 0 ? p.keys : 0;  // (a query in front of the request's first token sees nothing)
    r.at = in ? r.b * p.q.sb + i * p.q.ss + r.head * p.q.sh : -1;
  } else {
    const bool in = t < place.n;
    r.b = place.b;
    const int pos = place.nk - place.n + t;
    r.pos = max(pos, 0);
    r.to = in ? max(min(pos + 1, place.nk), 0) : 0;
    r.at = in ? (long long)(place.q0 + t) * p.q.ss + r.head * p.q.sh : -1;
  }
  if (p.window >= 0) r.from = max(r.pos - p.window, 0);
  return r;
}
// where the output row goes, in elements (prompts)
__device__ __forceinline__ long long fa_row_out(const FaPackedParams& p, const FaPlace& place, const FaRow& r, int hk) {
  return (long long)(place.q0 + r.token) * p.o.ss + (long long)(hk * (p.Hq / p.Hkv) + r.head) * p.o.sh;
}
