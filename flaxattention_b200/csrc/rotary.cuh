// Rotary positions of queries and keys, with an optional RMS norm per head in the same pass (fa_rotary,
// fa_rotary_bwd), and the same for new tokens whose keys and values go into the pages of a cache
// (fa_rotary_append).  Part of flaxattn.cu.
//
//   y = x * rsqrt(mean(x^2) + eps) * w                    (with weights)
//   (a, b) -> (a cos - b sin, b cos + a sin)              pairs of the first R values of y: i and i + R / 2, or
//                                                         neighbours; the others stay as they are
// and backward, with g the gradient behind the rotation turned back by the same angles (the transposed map) and
// u = x * rsqrt(..):   dw = sum over rows of g u,   dx = rsqrt(..) (g w - u mean(g w u)).
//
// All sums are in fp32, and a result is rounded once, when it is written.  Memory sets the pace: every value is read
// and written once, with a few operations in between.
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotStages = 3;  // rows of a thread's ring in the backward
constexpr int kRotHeads = 16;  // most heads that a thread goes through

struct FaRotTensor {
  char* ptr;
  long long sb, sh, ss;  // byte strides of batch, head and token (pages: of page, head and token in a page)
};
struct FaRotParams {
  FaRotTensor x[3], y[3];  // q, k, v: where they come from and go (backward: dy of q and k, and dx)
  FaRotTensor in[2];       // backward: q and k
  const void* w[2];        // norm weights or null
  float* dw[2];            // backward: partial sums [parts, D] or null
  const float* table;      // [table_len] rows of cos[R / 2] | sin[R / 2]
  long long table_stride, table_len;
  const void* pos;         // null: the token's number in its sequence
  long long pos_sb, pos_ss;
  const long long* slots;  // null: y[1] and y[2] are tensors like y[0]
  long long slot_sb, slot_ss, num_slots;
  int page_size;
  int pos64, w_f32, interleaved;
  int tokens, S, heads[3], D, Dv, R;
  int groups[3], per_group;  // groups of heads of each tensor, heads of a group
  int lane_shift;            // log2 of the lanes that share a row
  float eps, sign;           // sign of sin: -1 turns back
  int* status;
  float* scales[2];          // of keys and values in 8 bits, element strides of page, head and token in a page
  long long scale_sp[2], scale_sh[2], scale_ss[2];
};

template <int DT>
__device__ __forceinline__ float rot_get(const void* p, long long i) {
  if (DT == FA_F32) return ((const float*)p)[i];
  if (DT == FA_F16) return __half2float(((const __half*)p)[i]);
  return __bfloat162float(((const __nv_bfloat16*)p)[i]);
}
template <int DT>
__device__ __forceinline__ void rot_put(void* p, long long i, float v) {
  if (DT == FA_F32) ((float*)p)[i] = v;
  else if (DT == FA_F16) ((__half*)p)[i] = __float2half_rn(v);
  else ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v);
}
template <int DT>
constexpr int kRotVec = DT == FA_F32 ? 4 : 8;  // values of 16 bytes
// Two fp32 values in a register pair: products and sums of both in one instruction
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float x, float y) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void f2_get(F2 a, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a.v)); }
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 swapped(F2 a) {
  float x, y;
  f2_get(a, x, y);
  return f2(y, x);
}
__device__ __forceinline__ float both(F2 a) {
  float x, y;
  f2_get(a, x, y);
  return x + y;
}
template <int DT>
constexpr int kRotPairs = kRotVec<DT> / 2;
template <int DT>
__device__ __forceinline__ void rot_unpack(const uint4& u, F2 (&f)[kRotPairs<DT>]) {
  const unsigned v[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == FA_F32) {
      if (i & 1) f[i / 2] = f2(__uint_as_float(v[i - 1]), __uint_as_float(v[i]));
    } else if constexpr (DT == FA_F16) {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&v[i]));
      f[i] = f2(t.x, t.y);
    } else {
      f[i] = f2(__uint_as_float(v[i] << 16), __uint_as_float(v[i] & 0xffff0000u));
    }
  }
}
template <int DT>
__device__ __forceinline__ uint4 rot_pack(const F2 (&f)[kRotPairs<DT>]) {
  unsigned v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x, y;
    if constexpr (DT == FA_F32) {
      f2_get(f[i / 2], x, y);
      v[i] = __float_as_uint(i & 1 ? y : x);
    } else if constexpr (DT == FA_F16) {
      f2_get(f[i], x, y);
      const __half2 t = __floats2half2_rn(x, y);
      v[i] = *reinterpret_cast<const unsigned*>(&t);
    } else {
      f2_get(f[i], x, y);
      const __nv_bfloat162 t = __floats2bfloat162_rn(x, y);
      v[i] = *reinterpret_cast<const unsigned*>(&t);
    }
  }
  return make_uint4(v[0], v[1], v[2], v[3]);
}
template <int DT>
__device__ __forceinline__ void rot_weights(const FaRotParams& P, int kind, int chunk, bool have, float (&w)[kRotVec<DT>]) {
  constexpr int V = kRotVec<DT>;
#pragma unroll
  for (int i = 0; i < V; ++i)
    w[i] = !have ? 0.f : P.w_f32 ? ((const float*)P.w[kind])[chunk * V + i] : rot_get<DT>(P.w[kind], chunk * V + i);
}

// row of the table for token s of sequence b; -1 (and the status bit) for a position that it does not reach
__device__ __forceinline__ long long rot_position(const FaRotParams& P, int b, int s) {
  long long pos = s;
  if (P.pos != nullptr) {
    const long long at = b * P.pos_sb + s * P.pos_ss;
    pos = P.pos64 ? ((const long long*)P.pos)[at] : ((const int*)P.pos)[at];
  }
  if (pos >= 0 && pos < P.table_len) return pos;
  if (P.status != nullptr) atomicOr(P.status, FA_STATUS_BAD_POSITION);
  return -1;
}
// byte offset of token (b, s) in the destination; -1: it has none (keys and values of a slot below 0 or, with the
// status bit, beyond the pages); scale_at: where its scale is
__device__ __forceinline__ long long rot_destination(const FaRotParams& P, int kind, int b, int s, long long* scale_at = nullptr) {
  const FaRotTensor& y = P.y[kind];
  if (P.slots == nullptr || kind == 0) return b * y.sb + s * y.ss;
  const long long slot = P.slots[b * P.slot_sb + s * P.slot_ss];
  if (slot < 0) return -1;
  if (slot >= P.num_slots) {
    if (P.status != nullptr) atomicOr(P.status, FA_STATUS_BAD_SLOT);
    return -1;
  }
  long long page, at;
  if (P.num_slots <= 0x7fffffffll) {
    page = (unsigned)slot / (unsigned)P.page_size;
    at = (unsigned)slot % (unsigned)P.page_size;
  } else {
    page = slot / P.page_size;
    at = slot % P.page_size;
  }
  if (scale_at != nullptr) *scale_at = page * P.scale_sp[kind - 1] + at * P.scale_ss[kind - 1];
  return page * y.sb + at * y.ss;
}

// This thread's place in the grid: a lane of the `1 << lane_shift` that share a row, a token, a tensor and its heads.
struct RotPlace {
  int lane, token, kind, h0, h1;
  __device__ __forceinline__ RotPlace(const FaRotParams& P) {
    lane = threadIdx.x & ((1 << P.lane_shift) - 1);
    token = (int)(blockIdx.x * (kRotThreads >> P.lane_shift) + (threadIdx.x >> P.lane_shift));
    int group = blockIdx.y;
    kind = 0;
    while (kind < 2 && group >= P.groups[kind]) group -= P.groups[kind++];
    h0 = group * P.per_group;
    h1 = min(h0 + P.per_group, P.heads[kind]);
  }
};
template <class T>
__device__ __forceinline__ T rot_sum(T v) {  // over a warp
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// cos and sin of the pairs `lane * V ..` of a token
template <int V>
__device__ __forceinline__ void rot_angles(const FaRotParams& P, long long pos, int lane, bool turns, float (&c)[V], float (&s)[V]) {
#pragma unroll
  for (int i = 0; i < V; i += 4) {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    if (turns && pos >= 0) {
      const float* row = P.table + pos * P.table_stride + lane * V + i;
      a = *(const float4*)row;
      b = *(const float4*)(row + P.R / 2);
    }
    c[i] = a.x; c[i + 1] = a.y; c[i + 2] = a.z; c[i + 3] = a.w;
    s[i] = P.sign * b.x; s[i + 1] = P.sign * b.y; s[i + 2] = P.sign * b.z; s[i + 3] = P.sign * b.w;
  }
}
// How a lane finds the other value of a pair.
//   kHalves         pairs i and i + R / 2, R / 2 whole pieces: a lane has both pieces
//   kNeighbours     neighbouring values, R whole pairs of pieces: they are in the piece
//   kNeighboursAny  neighbouring values, any even R
//   kAny            pairs i and i + R / 2, any even R: the pieces of a row lie side by side in the lanes, and the other values come
//                   through shared memory.  B4 H32/8 S2048 D128 bf16 with norms, R 20: forward and backward 86 and 88 us (value by value 219 and 633), R 128 28 and 45.
enum RotMode { kHalves, kNeighbours, kNeighboursAny, kAny };

// The rotation of a lane's two pieces a and b as a' = a p + (b or a with its neighbours exchanged) q, and b' with its own p and q: the
// factors, with the weights of the values that they multiply (1: none).  A lane whose values stay has the weights and 0.
template <int V>
struct RotFactors {
  F2 pa[V / 2], qa[V / 2], pb[V / 2], qb[V / 2];
};
template <int V, RotMode MODE>
__device__ __forceinline__ void rot_factors(RotFactors<V>& f, bool turns, const float (&c)[V], const float (&s)[V], const float (&wa)[V], const float (&wb)[V]) {
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    const int x = 2 * i, y = 2 * i + 1;
    if (MODE == kNeighbours) {  // pairs i of piece a, V / 2 + i of piece b
      const float ca = turns ? c[i] : 1.f, cb = turns ? c[V / 2 + i] : 1.f, sa = turns ? s[i] : 0.f, sb = turns ? s[V / 2 + i] : 0.f;
      f.pa[i] = f2(wa[x] * ca, wa[y] * ca);
      f.qa[i] = f2(-wa[y] * sa, wa[x] * sa);
      f.pb[i] = f2(wb[x] * cb, wb[y] * cb);
      f.qb[i] = f2(-wb[y] * sb, wb[x] * sb);
    } else {
      const float cx = turns ? c[x] : 1.f, cy = turns ? c[y] : 1.f, sx = turns ? s[x] : 0.f, sy = turns ? s[y] : 0.f;
      f.pa[i] = f2(wa[x] * cx, wa[y] * cy);
      f.qa[i] = f2(-wb[x] * sx, -wb[y] * sy);
      f.pb[i] = f2(wb[x] * cx, wb[y] * cy);
      f.qb[i] = f2(wa[x] * sx, wa[y] * sy);
    }
  }
}
template <int V, RotMode MODE>
__device__ __forceinline__ void rot_turn(F2 (&a)[V / 2], F2 (&b)[V / 2], const RotFactors<V>& f) {
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    const F2 u = a[i], v = b[i];
    a[i] = fma(MODE == kHalves ? v : swapped(u), f.qa[i], u * f.pa[i]);
    b[i] = fma(MODE == kHalves ? u : swapped(v), f.qb[i], v * f.pb[i]);
  }
}
// any R: value e of a row, its pair's number, the other value's place and whether e is the pair's first
struct RotPair {
  int pair, other;
  bool first;
  __device__ __forceinline__ RotPair(const FaRotParams& P, bool halves, int e) {
    const int half = P.R / 2;
    first = halves ? e < half : (e & 1) == 0;
    pair = !halves ? e >> 1 : first ? e : e - half;
    other = !halves ? e ^ 1 : first ? e + half : e - half;
  }
};
// Factors for values V * chunk .. (no such chunk: it holds zeros)
template <int DT>
__device__ __forceinline__ void rot_factors_any(const FaRotParams& P, bool halves, long long pos, int kind, int chunk, bool have, bool weighted, F2 (&p)[kRotPairs<DT>],
                                                F2 (&q)[kRotPairs<DT>]) {
  constexpr int V = kRotVec<DT>;
  const auto weight = [&](int i) { return !weighted ? 1.f : P.w_f32 ? ((const float*)P.w[kind])[i] : rot_get<DT>(P.w[kind], i); };
  float f[V], g[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = chunk * V + i;
    f[i] = have ? weight(e) : 0.f;
    g[i] = 0.f;
    if (have && e < P.R) {
      const RotPair t(P, halves, e);
      const float c = pos < 0 ? 0.f : P.table[pos * P.table_stride + t.pair], s = pos < 0 ? 0.f : P.sign * P.table[pos * P.table_stride + P.R / 2 + t.pair];
      f[i] *= c;
      g[i] = weight(t.other) * (t.first ? -s : s);
    }
  }
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    p[i] = f2(f[2 * i], f[2 * i + 1]);
    q[i] = f2(g[2 * i], g[2 * i + 1]);
  }
}
// kAny: the other values of those of a chunk; 0 for values that stay.  The row's even and odd pieces lie in two planes, a piece per lane from
// `lane0` on.
template <int DT>
__device__ __forceinline__ void rot_others(const FaRotParams& P, const uint4* planes, int plane, int lane0, int chunk, F2 (&y)[kRotPairs<DT>]) {
  constexpr int V = kRotVec<DT>;
  const int half = P.R / 2;
  const auto place = [&](int o) { return planes + ((o / V) & 1) * plane + lane0 + o / V / 2; };
  if ((half & 1) == 0) {  // two others lie beside each other
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const int e = chunk * V + 2 * i, o = e < half ? e + half : e - half;
      y[i] = f2(0.f, 0.f);
      if (e < P.R) {
        if constexpr (DT == FA_F32) {
          const float2 t = ((const float2*)place(o))[(o % V) / 2];
          y[i] = f2(t.x, t.y);
        } else {
          const unsigned t = ((const unsigned*)place(o))[(o % V) / 2];
          if constexpr (DT == FA_F16) {
            const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&t));
            y[i] = f2(u.x, u.y);
          } else {
            y[i] = f2(__uint_as_float(t << 16), __uint_as_float(t & 0xffff0000u));
          }
        }
      }
    }
    return;
  }
  float f[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = chunk * V + i, o = e < half ? e + half : e - half;
    f[i] = e < P.R ? rot_get<DT>(place(o), o % V) : 0.f;
  }
#pragma unroll
  for (int i = 0; i < V / 2; ++i) y[i] = f2(f[2 * i], f[2 * i + 1]);
}
// any R, without a norm: the values of a piece that stay as they came (a NaN loses its payload on the way through fp32)
template <int DT>
__device__ __forceinline__ uint4 rot_keep(const FaRotParams& P, int chunk, uint4 to, const uint4& from) {
  constexpr int V = kRotVec<DT>;
  const int stays = P.R - chunk * V;  // from here on
  if (0 >= stays) to.x = from.x;
  if (V / 4 >= stays) to.y = from.y;
  if (V / 2 >= stays) to.z = from.z;
  if (3 * V / 4 >= stays) to.w = from.w;
  return to;
}
// kNeighboursAny: the pairs of a piece, those that turn
template <int V>
__device__ __forceinline__ void rot_turn_any(const FaRotParams& P, int chunk, F2 (&a)[V / 2], const F2 (&p)[V / 2], const F2 (&q)[V / 2]) {
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    const F2 u = a[i];
    a[i] = u * p[i];
    if (chunk * V + 2 * i < P.R) a[i] = fma(swapped(u), q[i], a[i]);  // (0 times what stays may be no number)
  }
}

// the sums of N values over the lanes of a row each
template <int N>
__device__ __forceinline__ void rot_sums(float (&v)[N], int lane_shift) {
  for (int off = 1 << lane_shift >> 1; off > 0; off >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], off);
  }
}

// ---- rows in 8 bits ------------------------------------------------------------------------
//   scale = max|y| / 127,  w = y / scale rounded to the nearest whole number, ties to the even one,
// both as fp32 divides, so that w is what the two formulas say to the last bit of y.  A row of zeros has the scale 0; of a row with an infinity or
// no number in it the scale is no number, which its values then are too when they are read.
__device__ __forceinline__ unsigned rot_size(unsigned most, F2 v) {  // (as bits: no number is the largest)
  float x, y;
  f2_get(v, x, y);
  return max(most, max(__float_as_uint(x) & 0x7fffffffu, __float_as_uint(y) & 0x7fffffffu));
}
// Quotients as an fp32 division rounds them: the product with the reciprocal, itself rounded to nearest, and once more with what that left (Markstein's theorem on the
// last step of a quotient), three instructions for two values.  Where nothing underflows: below 2^-100 by a division.
constexpr float kRotTiny = 7.9e-31f;
__device__ __forceinline__ float rot_scale(unsigned most) {
  if (most >= 0x7f800000u) return __uint_as_float(0x7fffffffu);
  const float a = __uint_as_float(most);
  if (a < kRotTiny) return a / 127.f;
  const float q = a * (1.f / 127.f);
  return fmaf(fmaf(-127.f, q, a), 1.f / 127.f, q);
}
__device__ __forceinline__ int rot_whole(float y, float scale) { return scale > 0.f ? (int)fminf(fmaxf(rintf(y / scale), -127.f), 127.f) : 0; }
// A lane's two pieces.  A quotient added to 1.5 * 2^23 has the whole number in its low byte.  (By divisions of what is near a tie only, which a warp has in every
// tenth row, 8000 tokens took 64 us, 40 without any; an IEEE division is some 30 instructions.)
template <int N>
__device__ __forceinline__ void rot_eight(F2 (&x)[N], F2 (&y)[N], float scale, uint2& to_x, uint2& to_y) {
  static_assert(N == 4, "eight values of each piece");
  if (scale < kRotTiny && scale > 0.f) {  // the same quotients 2^100 higher up; one of subnormals may be beyond 127
    constexpr float kUp = 1.2676506e30f;
    scale *= kUp;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float a, b;
      f2_get(x[i], a, b);
      x[i] = f2(fminf(fmaxf(a * kUp, -127.f * scale), 127.f * scale), fminf(fmaxf(b * kUp, -127.f * scale), 127.f * scale));
      f2_get(y[i], a, b);
      y[i] = f2(fminf(fmaxf(a * kUp, -127.f * scale), 127.f * scale), fminf(fmaxf(b * kUp, -127.f * scale), 127.f * scale));
    }
  }
  const float inverse = __frcp_rn(scale);
  const F2 r = f2(inverse, inverse), minus = f2(-scale, -scale), one = f2(1.f, 1.f), magic = f2(12582912.f, 12582912.f);
  unsigned w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v[4];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const F2 a = i < 2 ? x[2 * i + k] : y[2 * i - 4 + k], q = a * r;
      f2_get(fma(fma(fma(q, minus, a), r, q), one, magic), v[2 * k], v[2 * k + 1]);
    }
    w[i] = __byte_perm(__byte_perm(__float_as_uint(v[0]), __float_as_uint(v[1]), 0x0040), __byte_perm(__float_as_uint(v[2]), __float_as_uint(v[3]), 0x0040), 0x5410);
    if (!(scale > 0.f)) w[i] = 0u;
  }
  to_x = make_uint2(w[0], w[1]);
  to_y = make_uint2(w[2], w[3]);
}
// Two 16-byte pieces of a row per lane: the two that hold its pairs.  A thread keeps the angles of its token, times the weights, in
// registers for all heads of its group, and the lanes of a warp beside each other are tokens beside each other.  Four rows are computed
// while the next four are on their way.
//
// B4 H32/8 S4096 D128 bf16 with norms: 55 us for 335 MB, 6.1 TB/s.  In single values, with an angle and a weight multiplied per value and each group
// of rows asked for when the one before was written, it was bound by the instructions' issue: 79 us; 65 with two values per instruction
// and the weights in the angles.  Two rows at a time 61, more blocks per SM (fewer registers) 85 and more.
// 16384 tokens appended to pages (H32/8 D128 bf16): 70 us for 411 MB, 5.8 TB/s: the values only change place, and keys and values are written
// in runs of a row (256 bytes).  One token of 32 requests: 3.9 us, the launch, the slot and the row one behind the other.
// Q8: keys and values are written in 8 bits, and their scales.
template <int DT, RotMode MODE, bool Q8 = false>
__global__ void __launch_bounds__(kRotThreads, 2) fa_rotary_kernel(const __grid_constant__ FaRotParams P) {
  grid_wait();
  constexpr int V = kRotVec<DT>, N = V / 2, U = 4;
  __shared__ uint4 planes[MODE == kAny ? kRotThreads / 32 : 1][64];  // kAny: the pieces of a warp's rows, even ones and odd ones
  const RotPlace at(P);
  const bool live = at.token < P.tokens;
  const int b = live ? at.token / P.S : 0, s = live ? at.token - b * P.S : 0;
  const int kind = at.kind, chunks = (kind == 2 ? P.Dv : P.D) / V, pairs = kind == 2 ? 0 : P.R / (2 * V);
  const bool turns = MODE >= kNeighboursAny ? kind < 2 && 2 * at.lane * V < P.R : at.lane < pairs;
  const int ca = MODE == kHalves ? (turns ? at.lane : 2 * pairs + 2 * (at.lane - pairs)) : 2 * at.lane;
  const int cb = MODE == kHalves && turns ? at.lane + pairs : ca + 1;
  const bool eight = Q8 && kind > 0;
  [[maybe_unused]] long long scale_at = 0;
  const long long to = live ? rot_destination(P, kind, b, s, eight ? &scale_at : nullptr) : -1;
  const bool have_a = live && to >= 0 && ca < chunks, have_b = live && to >= 0 && cb < chunks;
  const bool norm = kind < 2 && P.w[kind < 2 ? kind : 0] != nullptr;
  // (the first rows are asked for before the angles, which come over the positions)
  const char* src = P.x[kind].ptr + b * P.x[kind].sb + s * P.x[kind].ss;
  uint4 na[U], nb[U];
  const auto load = [&](int h) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const char* row = src + (h + u) * P.x[kind].sh;
      const bool in = h + u < at.h1;
      na[u] = in && have_a ? *(const uint4*)(row + ca * 16) : make_uint4(0, 0, 0, 0);
      nb[u] = in && have_b ? *(const uint4*)(row + cb * 16) : make_uint4(0, 0, 0, 0);
    }
  };
  load(at.h0);
  RotFactors<V> f;
  if constexpr (MODE >= kNeighboursAny) {
    const long long pos = turns && live ? rot_position(P, b, s) : -1;
    rot_factors_any<DT>(P, MODE == kAny, pos, kind, ca, ca < chunks, norm, f.pa, f.qa);
    rot_factors_any<DT>(P, MODE == kAny, pos, kind, cb, cb < chunks, norm, f.pb, f.qb);
  } else {
    float c[V], sn[V], wa[V], wb[V];
    rot_angles<V>(P, turns && live ? rot_position(P, b, s) : -1, at.lane, turns, c, sn);
#pragma unroll
    for (int i = 0; i < V; ++i) wa[i] = wb[i] = 1.f;
    if (norm) {
      rot_weights<DT>(P, kind, ca, ca < chunks, wa);
      rot_weights<DT>(P, kind, cb, cb < chunks, wb);
    }
    rot_factors<V, MODE>(f, turns, c, sn, wa, wb);
  }
  char* dst = P.y[kind].ptr + to;
  const float per_value = 1.f / P.D;
  if constexpr (Q8) {
    if (eight) {
      // Two rows at a time, side by side, with nothing that branches between them: the shuffles of one are waited for under the other's.
      for (int h = at.h0; h < at.h1; h += 2) {
        uint4 ra[2], rb[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          ra[u] = na[u];
          rb[u] = nb[u];
          na[u] = na[u + 2];
          nb[u] = nb[u + 2];
        }
        if (((h - at.h0) & 2) && h + 2 < at.h1) load(h + 2);
        F2 x[2][N], y[2][N];
        float ss[2] = {0.f, 0.f};
        unsigned most[2] = {0u, 0u};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          rot_unpack<DT>(ra[u], x[u]);
          rot_unpack<DT>(rb[u], y[u]);
          if (norm) {
            F2 sum = x[u][0] * x[u][0];
#pragma unroll
            for (int i = 0; i < N; ++i) {
              if (i > 0) sum = fma(x[u][i], x[u][i], sum);
              sum = fma(y[u][i], y[u][i], sum);
            }
            ss[u] = both(sum);
          }
        }
        if (norm) rot_sums(ss, P.lane_shift);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float r = norm ? rsqrtf(ss[u] * per_value + P.eps) : 1.f;
          const F2 rr = f2(r, r);
          if (norm) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
              x[u][i] = x[u][i] * rr;
              y[u][i] = y[u][i] * rr;
            }
          }
          if (kind == 2) {  // (as they are)
          } else if constexpr (MODE == kAny) {
            F2 ox[N], oy[N];
            uint4* const mine = planes[threadIdx.x >> 5];
            __syncwarp();  // (the row before has been read)
            mine[threadIdx.x & 31] = ra[u];
            mine[32 + (threadIdx.x & 31)] = rb[u];
            __syncwarp();
            if (turns) {
              const int lane0 = (threadIdx.x & 31) - at.lane;
              rot_others<DT>(P, mine, 32, lane0, ca, ox);
              rot_others<DT>(P, mine, 32, lane0, cb, oy);
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
              x[u][i] = x[u][i] * f.pa[i];
              y[u][i] = y[u][i] * f.pb[i];
              if (!turns) continue;
              x[u][i] = fma(ox[i] * rr, f.qa[i], x[u][i]);
              y[u][i] = fma(oy[i] * rr, f.qb[i], y[u][i]);
            }
          } else if constexpr (MODE == kNeighboursAny) {
            rot_turn_any<V>(P, ca, x[u], f.pa, f.qa);
            rot_turn_any<V>(P, cb, y[u], f.pb, f.qb);
          } else {
            rot_turn<V, MODE>(x[u], y[u], f);
          }
#pragma unroll
          for (int i = 0; i < N; ++i) most[u] = rot_size(rot_size(most[u], x[u][i]), y[u][i]);
        }
        for (int off = 1 << P.lane_shift >> 1; off > 0; off >>= 1) {
#pragma unroll
          for (int u = 0; u < 2; ++u) most[u] = max(most[u], __shfl_xor_sync(0xffffffffu, most[u], off));
        }
        float scale[2];
        uint2 wa[2], wb[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          scale[u] = rot_scale(most[u]);
          rot_eight(x[u], y[u], scale[u], wa[u], wb[u]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if (h + u >= at.h1) break;
          char* row = dst + (h + u) * P.y[kind].sh;
          if (have_a) *(uint2*)(row + ca * 8) = wa[u];
          if (have_b) *(uint2*)(row + cb * 8) = wb[u];
          if (to >= 0 && at.lane == 0) P.scales[kind - 1][scale_at + (h + u) * P.scale_sh[kind - 1]] = scale[u];
        }
      }
      return;
    }
  }
  for (int h = at.h0; h < at.h1; h += U) {
    uint4 ra[U], rb[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      ra[u] = na[u];
      rb[u] = nb[u];
    }
    if (h + U < at.h1) load(h + U);  // (on their way while these are computed)
    float ss[U];
    if (norm) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        F2 x[N], y[N];
        rot_unpack<DT>(ra[u], x);
        rot_unpack<DT>(rb[u], y);
        F2 sum = x[0] * x[0];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (i > 0) sum = fma(x[i], x[i], sum);
          sum = fma(y[i], y[i], sum);
        }
        ss[u] = both(sum);
      }
      rot_sums(ss, P.lane_shift);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (h + u >= at.h1) break;
      F2 ox[N], oy[N];
      if constexpr (MODE == kAny) {
        uint4* const mine = planes[threadIdx.x >> 5];
        __syncwarp();  // (the row before has been read)
        mine[threadIdx.x & 31] = ra[u];
        mine[32 + (threadIdx.x & 31)] = rb[u];
        __syncwarp();
        const int lane0 = (threadIdx.x & 31) - at.lane;
        if (turns) {
          rot_others<DT>(P, mine, 32, lane0, ca, ox);
          rot_others<DT>(P, mine, 32, lane0, cb, oy);
        }
      }
      if (norm || turns) {
        F2 x[N], y[N];
        rot_unpack<DT>(ra[u], x);
        rot_unpack<DT>(rb[u], y);
        const float r = norm ? rsqrtf(ss[u] * per_value + P.eps) : 1.f;
        if (norm) {
          const F2 rr = f2(r, r);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            x[i] = x[i] * rr;
            y[i] = y[i] * rr;
          }
        }
        if constexpr (MODE == kAny) {
          const F2 rr = f2(r, r);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            x[i] = x[i] * f.pa[i];
            y[i] = y[i] * f.pb[i];
            if (!turns) continue;
            x[i] = fma(ox[i] * rr, f.qa[i], x[i]);
            y[i] = fma(oy[i] * rr, f.qb[i], y[i]);
          }
        } else if constexpr (MODE == kNeighboursAny) {
          rot_turn_any<V>(P, ca, x, f.pa, f.qa);
          rot_turn_any<V>(P, cb, y, f.pb, f.qb);
        } else {
          rot_turn<V, MODE>(x, y, f);
        }
        const uint4 pa = rot_pack<DT>(x), pb = rot_pack<DT>(y);
        ra[u] = MODE >= kNeighboursAny && !norm ? rot_keep<DT>(P, ca, pa, ra[u]) : pa;
        rb[u] = MODE >= kNeighboursAny && !norm ? rot_keep<DT>(P, cb, pb, rb[u]) : pb;
      }
      char* row = dst + (h + u) * P.y[kind].sh;
      if (have_a) *(uint4*)(row + ca * 16) = ra[u];
      if (have_b) *(uint4*)(row + cb * 16) = rb[u];
    }
  }
}

__device__ __forceinline__ void rot_copy16(void* shared, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(shared)), "l"(from) : "memory");
}

// The backward with norm weights: blocks go through the tokens in steps of the grid and keep the sums for dw in
// registers; what a block has goes to one row of partial sums, which fa_rotary_dw_kernel adds up in order.
//
// B4 H32/8 S4096 D128 bf16: 82 us for the 503 MB that have to move, 6.1 TB/s.  What it took: two values per instruction
// (fma.rn.f32x2), 157 us to 107, and rows on their way through shared memory instead of one row ahead in registers, which has
// twice as many bytes in flight, 107 to 83.
template <int DT, RotMode MODE>
__global__ void __launch_bounds__(kRotThreads, 2) fa_rotary_bwd_kernel(const __grid_constant__ FaRotParams P) {
  grid_wait();
  constexpr int V = kRotVec<DT>, N = V / 2;
  __shared__ float sums[kRotThreads / 32][256];
  const RotPlace at(P);
  const int kind = at.kind, chunks = P.D / V, pairs = P.R / (2 * V);
  const bool turns = MODE >= kNeighboursAny ? 2 * at.lane * V < P.R : at.lane < pairs;
  const int ca = MODE == kHalves ? (turns ? at.lane : 2 * pairs + 2 * (at.lane - pairs)) : 2 * at.lane;
  const int cb = MODE == kHalves && turns ? at.lane + pairs : ca + 1;
  const bool norm = P.w[kind] != nullptr;
  F2 wa[N], wb[N], da[N], db[N];
  {
    float x[V], y[V];
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = y[i] = 0.f;
    if (norm) {
      rot_weights<DT>(P, kind, ca, ca < chunks, x);
      rot_weights<DT>(P, kind, cb, cb < chunks, y);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      wa[i] = f2(x[2 * i], x[2 * i + 1]);
      wb[i] = f2(y[2 * i], y[2 * i + 1]);
      da[i] = db[i] = f2(0.f, 0.f);
    }
  }
  const float per_value = 1.f / P.D;
  const int block_tokens = kRotThreads >> P.lane_shift, step = gridDim.x * block_tokens, heads = at.h1 - at.h0;
  // Rows come through shared memory, kRotStages - 1 of them on their way: every thread has 16-byte places of its own for its pieces of dy
  // and x (no barriers).  The rows of a thread are those of its heads of its first token, then of its next, ..; every thread goes round as
  // often as the first of its block, since the shuffles are the warp's.
  extern __shared__ uint4 ring[];  // [kRotStages][4][kRotThreads]
  const int t_first = blockIdx.x * block_tokens, rounds = t_first < P.tokens ? (P.tokens - 1 - t_first) / step + 1 : 0, rows = rounds * heads;
  int next = 0, next_h = at.h0, next_t = t_first + (threadIdx.x >> P.lane_shift);  // the row that is asked for next
  const char *next_g = nullptr, *next_x = nullptr;
  const auto ask = [&]() {
    if (next < rows && next_t < P.tokens) {
      if (next_h == at.h0) {
        const int b = next_t / P.S, s = next_t - b * P.S;
        next_g = P.x[kind].ptr + b * P.x[kind].sb + s * P.x[kind].ss + at.h0 * P.x[kind].sh;
        if (norm) next_x = P.in[kind].ptr + b * P.in[kind].sb + s * P.in[kind].ss + at.h0 * P.in[kind].sh;
      }
      uint4* place = ring + (next % kRotStages) * 4 * kRotThreads + threadIdx.x;
      if (ca < chunks) rot_copy16(place, next_g + ca * 16);
      if (cb < chunks) rot_copy16(place + kRotThreads, next_g + cb * 16);
      if (norm && ca < chunks) rot_copy16(place + 2 * kRotThreads, next_x + ca * 16);
      if (norm && cb < chunks) rot_copy16(place + 3 * kRotThreads, next_x + cb * 16);
      next_g += P.x[kind].sh;
      if (norm) next_x += P.in[kind].sh;
    }
    ++next;
    if (++next_h == at.h1) {
      next_h = at.h0;
      next_t += step;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kRotStages - 1; ++i) ask();
  int row = 0;
  for (int round = 0; round < rounds; ++round) {
    const int t = t_first + round * step + (threadIdx.x >> P.lane_shift);
    const bool live = t < P.tokens, have_a = live && ca < chunks, have_b = live && cb < chunks;
    const int b = live ? t / P.S : 0, s = live ? t - b * P.S : 0;
    RotFactors<V> f;
    if constexpr (MODE >= kNeighboursAny) {
      const long long pos = turns && live ? rot_position(P, b, s) : -1;
      rot_factors_any<DT>(P, MODE == kAny, pos, kind, ca, ca < chunks, false, f.pa, f.qa);
      rot_factors_any<DT>(P, MODE == kAny, pos, kind, cb, cb < chunks, false, f.pb, f.qb);
    } else {
      float c[V], sn[V], one[V];
#pragma unroll
      for (int i = 0; i < V; ++i) one[i] = 1.f;
      rot_angles<V>(P, turns && live ? rot_position(P, b, s) : -1, at.lane, turns, c, sn);
      rot_factors<V, MODE>(f, turns, c, sn, one, one);
    }
    char* ds = P.y[kind].ptr + b * P.y[kind].sb + s * P.y[kind].ss + at.h0 * P.y[kind].sh;
    for (int h = 0; h < heads; ++h, ++row) {
      ask();
      asm volatile("cp.async.wait_group %0;" ::"n"(kRotStages - 1) : "memory");
      const uint4* place = ring + (row % kRotStages) * 4 * kRotThreads + threadIdx.x;
      const uint4 zero = make_uint4(0, 0, 0, 0);
      F2 a[N], d[N], u[N], v[N];
      rot_unpack<DT>(have_a ? place[0] : zero, a);
      rot_unpack<DT>(have_b ? place[kRotThreads] : zero, d);
      if constexpr (MODE == kAny) {
        __syncwarp();  // (the other lanes' pieces)
        if (turns && live) {
          F2 oa[N], od[N];
          const int lane0 = threadIdx.x - at.lane;
          rot_others<DT>(P, place - threadIdx.x, kRotThreads, lane0, ca, oa);
          rot_others<DT>(P, place - threadIdx.x, kRotThreads, lane0, cb, od);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            a[i] = fma(oa[i], f.qa[i], a[i] * f.pa[i]);
            d[i] = fma(od[i], f.qb[i], d[i] * f.pb[i]);
          }
        }
        __syncwarp();  // (before the place takes another row)
      } else if constexpr (MODE == kNeighboursAny) {
        if (turns) {
          rot_turn_any<V>(P, ca, a, f.pa, f.qa);
          rot_turn_any<V>(P, cb, d, f.pb, f.qb);
        }
      } else {
        if (turns) rot_turn<V, MODE>(a, d, f);
      }
      if (norm) {
        rot_unpack<DT>(have_a ? place[2 * kRotThreads] : zero, u);
        rot_unpack<DT>(have_b ? place[3 * kRotThreads] : zero, v);
        F2 ss = u[0] * u[0], gx = f2(0.f, 0.f), tu[N], tv[N];  // g w
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (i > 0) ss = fma(u[i], u[i], ss);
          ss = fma(v[i], v[i], ss);
          tu[i] = a[i] * wa[i];
          tv[i] = d[i] * wb[i];
          gx = fma(tu[i], u[i], gx);
          gx = fma(tv[i], v[i], gx);
        }
        float sum[2] = {both(ss), both(gx)};
        rot_sums(sum, P.lane_shift);
        // (beyond the last token: 0, since an eps of 0 would leave no number in dw)
        const float r = live ? rsqrtf(sum[0] * per_value + P.eps) : 0.f, m = -(sum[1] * r * per_value);
        const F2 rr = f2(r, r), mm = f2(m, m);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          u[i] = u[i] * rr;  // x rsqrt(..)
          v[i] = v[i] * rr;
          da[i] = fma(a[i], u[i], da[i]);
          db[i] = fma(d[i], v[i], db[i]);
          a[i] = fma(u[i], mm, tu[i]) * rr;
          d[i] = fma(v[i], mm, tv[i]) * rr;
        }
      }
      if (have_a) *(uint4*)(ds + ca * 16) = rot_pack<DT>(a);
      if (have_b) *(uint4*)(ds + cb * 16) = rot_pack<DT>(d);
      ds += P.y[kind].sh;
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (P.dw[kind] == nullptr) return;
  // rows of a warp, then warps of the block
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float v[4];
    f2_get(da[i], v[0], v[1]);
    f2_get(db[i], v[2], v[3]);
    for (int off = 1 << P.lane_shift; off < 32; off <<= 1) {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], off);
    }
    if ((threadIdx.x & 31) == at.lane) {
      if (ca < chunks) *(float2*)&sums[threadIdx.x >> 5][ca * V + 2 * i] = make_float2(v[0], v[1]);
      if (cb < chunks) *(float2*)&sums[threadIdx.x >> 5][cb * V + 2 * i] = make_float2(v[2], v[3]);
    }
  }
  __syncthreads();
  const long long part = (long long)blockIdx.x * P.groups[kind] + at.h0 / P.per_group;
  for (int i = threadIdx.x; i < P.D; i += kRotThreads) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < kRotThreads / 32; ++k) v += sums[k][i];
    P.dw[kind][part * P.D + i] = v;
  }
}

// What no 16-byte pieces fit (head dims, strides, addresses): a warp per row, value by value.  Backward (BACK): the same with dy, as above.
template <int DT, bool BACK, bool Q8 = false>
__global__ void __launch_bounds__(kRotThreads) fa_rotary_any_kernel(const __grid_constant__ FaRotParams P) {
  grid_wait();
  __shared__ float sums[BACK ? kRotThreads / 32 : 1][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, kind = blockIdx.y;
  const int D = kind == 2 ? P.Dv : P.D, half = kind == 2 ? 0 : P.R / 2, H = P.heads[kind];
  const bool norm = kind < 2 && P.w[kind < 2 ? kind : 0] != nullptr;
  if (BACK) {
    for (int i = lane; i < D; i += 32) sums[warp][i] = 0.f;
    __syncwarp();
  }
  const auto weight = [&](int i) { return P.w_f32 ? ((const float*)P.w[kind])[i] : rot_get<DT>(P.w[kind], i); };
  const long long rows = (long long)P.tokens * H;
  for (long long row = (long long)blockIdx.x * (kRotThreads / 32) + warp; row < rows; row += (long long)gridDim.x * (kRotThreads / 32)) {
    const int t = (int)(row / H), h = (int)(row - (long long)t * H), b = t / P.S, s = t - b * P.S;
    [[maybe_unused]] long long scale_at = 0;
    const long long to = rot_destination(P, kind, b, s, Q8 && kind > 0 ? &scale_at : nullptr);
    if (to < 0) continue;
    const char* x = P.x[kind].ptr + b * P.x[kind].sb + s * P.x[kind].ss + h * P.x[kind].sh;
    char* y = P.y[kind].ptr + to + h * P.y[kind].sh;
    const long long pos = half > 0 ? rot_position(P, b, s) : -1;
    const float* angles = P.table + (pos < 0 ? 0 : pos) * P.table_stride;
    const char* in = BACK && norm ? P.in[kind].ptr + b * P.in[kind].sb + s * P.in[kind].ss + h * P.in[kind].sh : x;
    // (backward: in 64 bits, since with few values in a row the terms of dx nearly cancel)
    using Real = std::conditional_t<BACK, double, float>;
    Real r = 1, m = 0;
    if (norm) {
      Real ss = 0;
      for (int i = lane; i < D; i += 32) {
        const Real v = rot_get<DT>(in, i);
        ss += v * v;
      }
      ss = rot_sum(ss) / D + P.eps;
      if constexpr (BACK) r = rsqrt(ss);
      else r = rsqrtf(ss);
    }
    // pairs, then the values that stay: `first` and `second` of a unit (second < 0: there is none)
    const auto unit = [&](int k, int& i, int& j, float& c, float& sn) {
      const bool turns = k < half;
      i = turns ? (P.interleaved ? 2 * k : k) : 2 * half + (k - half);
      j = turns ? (P.interleaved ? 2 * k + 1 : k + half) : -1;
      c = !turns ? 1.f : pos < 0 ? 0.f : angles[k];
      sn = !turns || pos < 0 ? 0.f : P.sign * angles[half + k];
    };
    const int units = D - half;
    if (BACK && norm) {
      for (int k = lane; k < units; k += 32) {
        int i, j;
        float c, sn;
        unit(k, i, j, c, sn);
        const float a = rot_get<DT>(x, i), d = j >= 0 ? rot_get<DT>(x, j) : 0.f;
        m += ((Real)a * c - (Real)d * sn) * weight(i) * rot_get<DT>(in, i);
        if (j >= 0) m += ((Real)d * c + (Real)a * sn) * weight(j) * rot_get<DT>(in, j);
      }
      m = rot_sum(m) * r / D;
    }
    if constexpr (Q8) {
      if (kind > 0) {
        float v[8][2];
        unsigned most = 0;
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const int k = lane + 32 * n;
          v[n][0] = v[n][1] = 0.f;
          if (k >= units) continue;
          int i, j;
          float c, sn;
          unit(k, i, j, c, sn);
          float a = rot_get<DT>(x, i), d = j >= 0 ? rot_get<DT>(x, j) : 0.f;
          if (norm) {
            a *= r * weight(i);
            if (j >= 0) d *= r * weight(j);
          }
          v[n][0] = j >= 0 ? a * c - d * sn : a;
          v[n][1] = j >= 0 ? d * c + a * sn : 0.f;
          most = rot_size(most, f2(v[n][0], v[n][1]));
        }
        most = __reduce_max_sync(0xffffffffu, most);
        const float scale = rot_scale(most);
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const int k = lane + 32 * n;
          if (k >= units) continue;
          int i, j;
          float c, sn;
          unit(k, i, j, c, sn);
          y[i] = (char)rot_whole(v[n][0], scale);
          if (j >= 0) y[j] = (char)rot_whole(v[n][1], scale);
        }
        if (lane == 0) P.scales[kind - 1][scale_at + h * P.scale_sh[kind - 1]] = scale;
        continue;
      }
    }
    for (int k = lane; k < units; k += 32) {
      int i, j;
      float c, sn;
      unit(k, i, j, c, sn);
      if (j < 0 && !norm) {  // (as it is)
        if (DT == FA_F32) ((unsigned*)y)[i] = ((const unsigned*)x)[i];
        else ((unsigned short*)y)[i] = ((const unsigned short*)x)[i];
        continue;
      }
      float a = rot_get<DT>(x, i), d = j >= 0 ? rot_get<DT>(x, j) : 0.f;
      if (!BACK && norm) {
        a *= r * weight(i);
        if (j >= 0) d *= r * weight(j);
      }
      Real p = (Real)a * c - (Real)d * sn, q = (Real)d * c + (Real)a * sn;
      if (BACK && norm) {
        const Real u = rot_get<DT>(in, i) * r, v = j >= 0 ? rot_get<DT>(in, j) * r : 0;
        sums[warp][i] += (float)(p * u);
        if (j >= 0) sums[warp][j] += (float)(q * v);
        p = r * (p * weight(i) - u * m);
        if (j >= 0) q = r * (q * weight(j) - v * m);
      }
      rot_put<DT>(y, i, (float)p);
      if (j >= 0) rot_put<DT>(y, j, (float)q);
    }
  }
  if (!BACK || P.dw[kind < 2 ? kind : 0] == nullptr) return;
  __syncthreads();
  for (int i = threadIdx.x; i < D; i += kRotThreads) {
    float v = 0.f;
    for (int k = 0; k < kRotThreads / 32; ++k) v += sums[BACK ? k : 0][i];
    P.dw[kind][(long long)blockIdx.x * D + i] = v;
  }
}

// dw from the partial sums of the blocks: 8 columns per block, 128 rows of threads, always in the same order.  (32 columns and 32 rows, 8 blocks
// at D 128: 6.0 us for 472 + 118 parts.)
struct FaRotDw {
  const float* part[2];
  void* dw[2];
  int parts[2];
  int D;
};
template <int DT>
__global__ void __launch_bounds__(1024) fa_rotary_dw_kernel(const __grid_constant__ FaRotDw P) {
  grid_wait();
  __shared__ float sums[32][8];
  const int col = blockIdx.x * 8 + (threadIdx.x & 7), slice = threadIdx.x >> 3, kind = blockIdx.y;
  if (P.dw[kind] == nullptr) return;
  float v = 0.f;
  if (col < P.D) {
#pragma unroll 4
    for (int i = slice; i < P.parts[kind]; i += 128) v += P.part[kind][(long long)i * P.D + col];
  }
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  v += __shfl_xor_sync(0xffffffffu, v, 16);
  if ((threadIdx.x & 31) < 8) sums[threadIdx.x >> 5][threadIdx.x & 7] = v;
  __syncthreads();
  if (threadIdx.x >= 8 || col >= P.D) return;
  v = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) v += sums[i][threadIdx.x];
  rot_put<DT>(P.dw[kind], col, v);
}

// ---- host --------------------------------------------------------------------------------
FaRotTensor rot_tensor(const fa_tensor& t, int es) { return {(char*)t.ptr, t.stride_b * es, t.stride_h * es, t.stride_s * es}; }
bool rot_aligned(const FaRotTensor& t, int to = 16) { return (((uintptr_t)t.ptr | (uintptr_t)t.sb | (uintptr_t)t.sh | (uintptr_t)t.ss) & (to - 1)) == 0; }

int rot_check(const fa_rotary_params* p) {
  if (!p) return fail(FA_EINVAL, "params is null");
  if (p->dtype < FA_F16 || p->dtype > FA_F32) return fail(FA_EINVAL, "unknown dtype");
  if (p->weight_dtype != p->dtype && p->weight_dtype != FA_F32) return fail(FA_EINVAL, "norm weights have the type of the tensors or fp32");
  if (p->B < 0 || p->S < 0 || p->Hq < 0 || p->Hkv < 0) return fail(FA_EINVAL, "B, S, Hq and Hkv must not be negative");
  if ((long long)p->B * p->S > 0x7fffffffll - 256) return fail(FA_EUNSUPPORTED, "B * S must stay below 2^31");
  if ((long long)p->Hq + 2LL * p->Hkv > 65535) return fail(FA_EUNSUPPORTED, "Hq + 2 Hkv must not exceed 65535");
  if (p->D <= 0 || p->D > 256) return fail(FA_EUNSUPPORTED, "head dims from 1 to 256");
  if (p->rotary_dim < 0 || p->rotary_dim > p->D || p->rotary_dim % 2) return fail(FA_EINVAL, "rotary_dim must be even and at most the head dim");
  if (p->rotary_dim > 0 && !p->table) return fail(FA_EINVAL, "the table is null");
  if (p->table && (p->table_length <= 0 || p->table_stride < p->rotary_dim)) return fail(FA_EINVAL, "the table needs rows of at least rotary_dim values");
  if (p->positions && p->position_bits != 32 && p->position_bits != 64) return fail(FA_EINVAL, "positions of 32 or 64 bits");
  if (!(p->eps >= 0.f)) return fail(FA_EINVAL, "eps must not be negative");
  return FA_OK;
}

// Everything but the tensors; `heads`: of q, k and v (0: not there)
void rot_fill(const fa_rotary_params* p, int hq, int hk, int hv, FaRotParams& k) {
  memset(&k, 0, sizeof k);
  k.w[0] = p->q_weight;
  k.w[1] = p->k_weight;
  k.table = p->table; k.table_stride = p->table_stride; k.table_len = p->table_length;
  k.pos = p->positions; k.pos64 = p->position_bits == 64;
  k.pos_sb = p->position_stride_b; k.pos_ss = p->position_stride_s;
  k.w_f32 = p->weight_dtype == FA_F32;
  k.interleaved = p->interleaved != 0;
  k.tokens = p->B * p->S; k.S = p->S;
  k.heads[0] = hq; k.heads[1] = hk; k.heads[2] = hv;
  k.D = p->D; k.Dv = p->Dv; k.R = p->rotary_dim;
  k.eps = p->eps; k.sign = 1.f;
  k.status = p->status;
}
// Whether all rows can be taken in 16-byte pieces, two per lane; fills the lanes of a row.
bool rot_by_pieces(const FaRotParams& k, int dtype, int* lane_shift) {
  const int v = dtype == FA_F32 ? 4 : 8;
  if (k.D % v || k.Dv % v || k.Dv > k.D) return false;
  for (int i = 0; i < 3; ++i)
    if (k.heads[i] > 0 && !(rot_aligned(k.x[i]) && rot_aligned(k.y[i], i > 0 && k.scales[0] != nullptr ? 8 : 16) && (i == 2 || k.in[i].ptr == nullptr || rot_aligned(k.in[i])))) return false;
  int shift = 0;
  while ((1 << shift) < (k.D + 2 * v - 1) / (2 * v)) ++shift;
  *lane_shift = shift;
  return shift <= 5;
}
// (angles are read 16 bytes at a time, but for any R)
RotMode rot_mode(const FaRotParams& k, int dtype) {
  const bool whole = k.R % (dtype == FA_F32 ? 8 : 16) == 0 && (k.R == 0 || ((uintptr_t)k.table % 16 == 0 && k.table_stride % 4 == 0));
  return k.interleaved ? (whole ? kNeighbours : kNeighboursAny) : whole ? kHalves : kAny;
}
// Heads that a thread goes through.  Up to 16, so that the angles are read seldom (B4 H32/8 S4096 D128 bf16 with norms, us, 4 / 8 / 16 heads: forward
// 68 / 56 / 55; 16384 tokens appended 81 / 72 / 70); fewer while the grid would leave SMs with less than four blocks.
void rot_groups(FaRotParams& k, long long token_blocks) {
  int per = kRotHeads;
  const auto blocks = [&](int n) {
    long long g = 0;
    for (int i = 0; i < 3; ++i) g += (k.heads[i] + n - 1) / n;
    return g * token_blocks;
  };
  while (per > 1 && blocks(per) < 4LL * device_sm_count()) per /= 2;
  k.per_group = per;
  for (int i = 0; i < 3; ++i) k.groups[i] = (k.heads[i] + per - 1) / per;
}

template <class F>
int rot_dispatch(int dtype, F&& f) {
  if (dtype == FA_F16) return f(std::integral_constant<int, FA_F16>{});
  if (dtype == FA_BF16) return f(std::integral_constant<int, FA_BF16>{});
  return f(std::integral_constant<int, FA_F32>{});
}

// Leave for more than 48 KB of dynamic shared memory, asked for once per kernel and device
int allow_smem(const void* fn, int smem) {
  static std::mutex mu;
  static std::map<const void*, unsigned long long> known;
  int dev = 0;
  FA_CUDA_CHECK(cudaGetDevice(&dev));
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0ull;
  std::lock_guard<std::mutex> lk(mu);
  unsigned long long& have = known[fn];
  if (bit != 0 && (have & bit)) return FA_OK;
  FA_CUDA_CHECK(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  have |= bit;
  return FA_OK;
}

// x -> y of the tensors that `k` describes
int rot_launch(FaRotParams& k, int dtype, void* stream) {
  const int heads = k.heads[0] + k.heads[1] + k.heads[2];
  if (k.tokens == 0 || heads == 0) return FA_OK;
  if (rot_by_pieces(k, dtype, &k.lane_shift)) {
    const long long token_blocks = ((long long)k.tokens + (kRotThreads >> k.lane_shift) - 1) / (kRotThreads >> k.lane_shift);
    rot_groups(k, token_blocks);
    const dim3 grid((unsigned)token_blocks, (unsigned)(k.groups[0] + k.groups[1] + k.groups[2]));
    return rot_dispatch(dtype, [&](auto dt) {
      constexpr int DT = decltype(dt)::value;
      if constexpr (DT != FA_F32) {
        void (*const eight[])(FaRotParams) = {fa_rotary_kernel<DT, kHalves, true>, fa_rotary_kernel<DT, kNeighbours, true>, fa_rotary_kernel<DT, kNeighboursAny, true>, fa_rotary_kernel<DT, kAny, true>};
        if (k.scales[0]) return launch_here("fa_rotary_kernel", eight[rot_mode(k, dtype)], grid, dim3(kRotThreads), stream, k);
      }
      void (*const of_mode[])(FaRotParams) = {fa_rotary_kernel<DT, kHalves>, fa_rotary_kernel<DT, kNeighbours>, fa_rotary_kernel<DT, kNeighboursAny>, fa_rotary_kernel<DT, kAny>};
      return launch_here("fa_rotary_kernel", of_mode[rot_mode(k, dtype)], grid, dim3(kRotThreads), stream, k);
    });
  }
  const long long rows = (long long)k.tokens * std::max(k.heads[0], std::max(k.heads[1], k.heads[2]));
  const dim3 grid((unsigned)std::min<long long>((rows + kRotThreads / 32 - 1) / (kRotThreads / 32), 1 << 20), k.heads[2] > 0 ? 3 : 2);
  return rot_dispatch(dtype, [&](auto dt) {
    if constexpr (decltype(dt)::value != FA_F32) {
      if (k.scales[0]) return launch_here("fa_rotary_any_kernel", fa_rotary_any_kernel<decltype(dt)::value, false, true>, grid, dim3(kRotThreads), stream, k);
    }
    return launch_here("fa_rotary_any_kernel", fa_rotary_any_kernel<decltype(dt)::value, false>, grid, dim3(kRotThreads), stream, k);
  });
}

// Blocks along the tokens of the backward with norm weights: about four per SM in all, two of which it holds at once.
unsigned rot_bwd_blocks(const FaRotParams& k, long long token_blocks) {
  return (unsigned)std::min<long long>(token_blocks, std::max(1, 4 * device_sm_count() / (k.groups[0] + k.groups[1])));
}
// no more partial sums than that of a tensor, whichever kernel runs
long long rot_bwd_parts(int heads) { return 4LL * device_sm_count() + heads; }

}  // namespace

extern "C" {

int fa_rotary(const fa_rotary_params* p, void* stream) {
  if (int rc = rot_check(p)) return rc;
  prof_reset();
  FaRotParams k;
  rot_fill(p, p->Hq, p->Hkv, 0, k);
  const int es = esize(p->dtype);
  const fa_tensor* from[2] = {&p->q, &p->k};
  const fa_tensor* to[2] = {&p->q_out, &p->k_out};
  for (int i = 0; i < 2; ++i) {
    if (k.heads[i] > 0 && k.tokens > 0 && (!from[i]->ptr || !to[i]->ptr)) return fail(FA_EINVAL, "a tensor is null");
    k.x[i] = rot_tensor(*from[i], es);
    k.y[i] = rot_tensor(*to[i], es);
  }
  return rot_launch(k, p->dtype, stream);
}

size_t fa_rotary_bwd_workspace_bytes(const fa_rotary_params* p) {
  if (!p || !(p->q_weight || p->k_weight) || p->Hq < 0 || p->Hkv < 0 || p->D <= 0) return 0;
  return (size_t)(rot_bwd_parts(p->Hq) + rot_bwd_parts(p->Hkv)) * p->D * sizeof(float);
}

int fa_rotary_bwd(const fa_rotary_params* p, const fa_tensor* dq_out, const fa_tensor* dk_out, const fa_tensor* dq, const fa_tensor* dk,
                  void* dq_weight, void* dk_weight, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = rot_check(p)) return rc;
  if (!dq_out || !dk_out || !dq || !dk) return fail(FA_EINVAL, "a gradient is null");
  if ((dq_weight && !p->q_weight) || (dk_weight && !p->k_weight)) return fail(FA_EINVAL, "a gradient of weights that are not there");
  prof_reset();
  FaRotParams k;
  rot_fill(p, p->Hq, p->Hkv, 0, k);
  const int es = esize(p->dtype);
  const fa_tensor *from[2] = {dq_out, dk_out}, *to[2] = {dq, dk}, *in[2] = {&p->q, &p->k};
  void* dw[2] = {dq_weight, dk_weight};
  for (int i = 0; i < 2; ++i) {
    if (k.heads[i] > 0 && k.tokens > 0 && (!from[i]->ptr || !to[i]->ptr || (k.w[i] && !in[i]->ptr))) return fail(FA_EINVAL, "a tensor is null");
    k.x[i] = rot_tensor(*from[i], es);
    k.y[i] = rot_tensor(*to[i], es);
    if (k.w[i]) k.in[i] = rot_tensor(*in[i], es);
  }
  k.sign = -1.f;
  // (no norm: nothing but the rotation, which needs no inputs)
  if (!k.w[0] && !k.w[1]) return rot_launch(k, p->dtype, stream);
  const size_t need = fa_rotary_bwd_workspace_bytes(p);
  if (!workspace || workspace_bytes < need) return fail(FA_EWORKSPACE, "rotary backward workspace too small");
  if ((uintptr_t)workspace & 15) return fail(FA_EINVAL, "workspace must be 16-byte aligned");
  FaRotDw sum;
  memset(&sum, 0, sizeof sum);
  sum.D = p->D;
  float* part[2] = {(float*)workspace, (float*)workspace + rot_bwd_parts(p->Hq) * p->D};
  for (int i = 0; i < 2; ++i) {
    k.dw[i] = dw[i] ? part[i] : nullptr;
    sum.part[i] = part[i];
    sum.dw[i] = dw[i];
  }
  if (k.tokens > 0 && k.heads[0] + k.heads[1] > 0) {
    int rc;
    if (rot_by_pieces(k, p->dtype, &k.lane_shift)) {
      const long long token_blocks = ((long long)k.tokens + (kRotThreads >> k.lane_shift) - 1) / (kRotThreads >> k.lane_shift);
      rot_groups(k, token_blocks);
      const unsigned blocks = rot_bwd_blocks(k, token_blocks);
      for (int i = 0; i < 2; ++i) sum.parts[i] = (int)blocks * k.groups[i];
      rc = rot_dispatch(p->dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        void (*const of_mode[])(FaRotParams) = {fa_rotary_bwd_kernel<DT, kHalves>, fa_rotary_bwd_kernel<DT, kNeighbours>, fa_rotary_bwd_kernel<DT, kNeighboursAny>,
                                                fa_rotary_bwd_kernel<DT, kAny>};
        const auto fn = of_mode[rot_mode(k, DT)];
        constexpr int smem = kRotStages * 4 * kRotThreads * 16;
        if (int e = allow_smem((const void*)fn, smem)) return e;
        return launch_here_smem("fa_rotary_bwd_kernel", fn, dim3(blocks, (unsigned)(k.groups[0] + k.groups[1])), dim3(kRotThreads), smem, stream, k);
      });
    } else {
      const long long rows = (long long)k.tokens * std::max(k.heads[0], k.heads[1]);
      const unsigned blocks = (unsigned)std::min<long long>((rows + kRotThreads / 32 - 1) / (kRotThreads / 32), 2LL * device_sm_count());
      sum.parts[0] = sum.parts[1] = (int)blocks;
      rc = rot_dispatch(p->dtype, [&](auto dt) {
        return launch_here("fa_rotary_any_kernel", fa_rotary_any_kernel<decltype(dt)::value, true>, dim3(blocks, 2), dim3(kRotThreads), stream, k);
      });
    }
    if (rc) return rc;
  }
  if (!dw[0] && !dw[1]) return FA_OK;
  return rot_dispatch(p->weight_dtype, [&](auto dt) {
    return launch_here("fa_rotary_dw_kernel", fa_rotary_dw_kernel<decltype(dt)::value>, dim3((unsigned)((p->D + 7) / 8), 2), dim3(1024), stream, sum);
  });
}

int fa_rotary_append(const fa_rotary_params* p, void* stream) {
  if (int rc = rot_check(p)) return rc;
  if (p->Hkv > 0 && (p->Dv <= 0 || p->Dv > 256)) return fail(FA_EUNSUPPORTED, "head dims from 1 to 256");
  if (p->page_size <= 0 || p->num_pages < 0) return fail(FA_EINVAL, "page_size must be positive, num_pages not negative");
  if (p->num_pages > (1ll << 62) / p->page_size) return fail(FA_EINVAL, "too many pages");
  prof_reset();
  FaRotParams k;
  rot_fill(p, p->q.ptr ? p->Hq : 0, p->Hkv, p->Hkv, k);
  if (k.tokens == 0) return FA_OK;
  if (k.heads[1] > 0 && (!p->k.ptr || !p->v.ptr || !p->slots)) return fail(FA_EINVAL, "a tensor is null");
  if (k.heads[1] > 0 && p->num_pages > 0 && (!p->k_pages.ptr || !p->v_pages.ptr)) return fail(FA_EINVAL, "a tensor is null");
  if (k.heads[0] > 0 && !p->q_out.ptr) return fail(FA_EINVAL, "a tensor is null");
  const bool eight = p->k_scales.ptr || p->v_scales.ptr;
  if (eight && p->dtype == FA_F32) return fail(FA_EUNSUPPORTED, "pages in 8 bits take 16-bit tensors");
  if (eight && !(p->k_scales.ptr && p->v_scales.ptr)) return fail(FA_EINVAL, "scales of keys and of values, or none");
  const int es = esize(p->dtype);
  const fa_tensor *from[3] = {&p->q, &p->k, &p->v}, *to[3] = {&p->q_out, &p->k_pages, &p->v_pages}, *scales[2] = {&p->k_scales, &p->v_scales};
  for (int i = 0; i < 3; ++i) {
    k.x[i] = rot_tensor(*from[i], es);
    k.y[i] = rot_tensor(*to[i], eight && i > 0 ? 1 : es);
  }
  for (int i = 0; i < 2; ++i) {
    k.scales[i] = (float*)scales[i]->ptr;
    k.scale_sp[i] = scales[i]->stride_b; k.scale_sh[i] = scales[i]->stride_h; k.scale_ss[i] = scales[i]->stride_s;
  }
  k.slots = (const long long*)p->slots;
  k.slot_sb = p->slot_stride_b; k.slot_ss = p->slot_stride_s;
  k.page_size = p->page_size;
  k.num_slots = p->num_pages * p->page_size;
  return rot_launch(k, p->dtype, stream);
}

}  // extern "C"
