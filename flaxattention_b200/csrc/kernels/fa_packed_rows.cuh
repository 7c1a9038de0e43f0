// The rows of attention over requests of different lengths that lie end to end, and of the newest tokens of many requests over a prefix that
// they share.  The G query heads of a kv head share its keys, so rows are (token, head of the group), row r is head r % G of token r / G, and a
// kernel takes them in items of R rows.
//
//   prompts  An item's rows are of one request.  Lengths are known on the device only; every CTA looks its item up.  Items with the most keys
//            in front: in the order of their place in the request, the last first, over all requests.  Behind the requests' items come those of
//            the rows that belong to none, in front of the first request and behind the last, which see nothing.
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

// Item `item` of items of R rows, by the 32 lanes of a warp together.  The items of level l are those with l others of their request in front of
// them; total(l) of all have level l or more, so the level of an item is found by halving, and its request by counting those that
// reach it.  (The counts of the first 256 requests stay in registers.)
template <int R>
__device__ __forceinline__ FaPlace fa_find_item(const FaPackedParams& p, long long item) {
  constexpr int KEEP = 8;
  const int lane = threadIdx.x & 31, G = p.Hq / p.Hkv;
  const auto items_of = [&](int s) {
    if (s >= p.B) return 0;
    int begin, end;
    fa_range(p.starts, s, p.tokens, begin, end);
    return (int)(((long long)(end - begin) * G + R - 1) / R);
  };
  int kept[KEEP], most = 0;
#pragma unroll
  for (int i = 0; i < KEEP; ++i) {
    kept[i] = i * 32 < p.B ? items_of(i * 32 + lane) : 0;
    most = max(most, kept[i]);
  }
#pragma unroll 1
  for (int s = KEEP * 32; s < p.B; s += 32) most = max(most, items_of(s + lane));
  most = __reduce_max_sync(0xffffffffu, most);
  const auto total = [&](int level) {
    long long sum = 0;
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      if (i * 32 < p.B) sum += max(kept[i] - level, 0);
#pragma unroll 1
    for (int s = KEEP * 32; s < p.B; s += 32) sum += max(items_of(s + lane) - level, 0);
    // (of broken starts the sum may need more than 32 bits)
    const fa_u32 lo = __reduce_add_sync(0xffffffffu, (fa_u32)sum & 0xffffffu), hi = __reduce_add_sync(0xffffffffu, (fa_u32)(sum >> 24));
    return (long long)lo + ((long long)hi << 24);
  };
  FaPlace r = {0, 0, 0, 0, 0, 0, 0};
  const long long all = total(0);
  if (item >= all) {
    // rows of no request
    long long left = item - all;
    const int front = p.B > 0 ? min(max(p.starts[0], 0), p.tokens) : 0, back = p.B > 0 ? min(max(p.starts[p.B], 0), p.tokens) : 0;
    const long long items_front = ((long long)front * G + R - 1) / R;
    const bool behind = left >= items_front;
    if (behind) left -= items_front;
    r.q0 = behind ? back : 0;
    r.n = behind ? p.tokens - back : front;
    r.first = (int)min(left * R, (long long)0x7fffffff);
    r.any = left * R < (long long)r.n * G;
    return r;
  }
  int lo = 0, hi = most - 1;  // the last level l with total(l) > item
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (total(mid) > item) lo = mid;
    else hi = mid - 1;
  }
  int rank = (int)(item - total(lo + 1));
  r.any = 1;
  r.first = lo * R;
  const auto find = [&](int s0, int count) {  // whether the request is among the 32 from s0 on
    const fa_u32 reach = __ballot_sync(0xffffffffu, count > lo);
    const int n = __popc(reach);
    if (rank >= n) {
      rank -= n;
      return false;
    }
    const fa_u32 below = reach & ((1u << lane) - 1u);
    r.b = s0 + __ffs(__ballot_sync(0xffffffffu, ((reach >> lane) & 1u) && __popc(below) == rank)) - 1;
    return true;
  };
  bool found = false;
#pragma unroll
  for (int i = 0; i < KEEP; ++i)
    if (!found && i * 32 < p.B) found = find(i * 32, kept[i]);
#pragma unroll 1
  for (int s = KEEP * 32; s < p.B && !found; s += 32) found = find(s, items_of(s + lane));
  int end;
  fa_range(p.starts, r.b, p.tokens, r.q0, end);
  r.n = end - r.q0;
  fa_range(p.key_starts, r.b, p.keys, r.k0, end);
  r.nk = end - r.k0;
  return r;
}

// starts that decrease, or lie where there are no tokens: said once, by the threads of one CTA
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
