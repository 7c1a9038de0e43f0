// Attention of prompts laid end to end (fa_prompt) and over a prefix that requests share (the first of the two parts of fa_paged with one; the other is the
// pages', and fa_merge_kernel joins them).  Kernels: kernels/fa_packed.cuh.  Part of flaxattn.cu.
namespace {

FaDiv divide_by(int d) {
  FaDiv r{0, -1};
  while (d > 1 && (d - 1) >> (r.shift + 1) != 0) ++r.shift;  // 2^shift < d <= 2^(shift + 1)
  if (d > 1) r.mul = (unsigned)((1ull << (32 + r.shift)) / (unsigned)d + 1);
  return r;
}

// Shapes and types of either call, as the kernels have them
struct PackedShape {
  int dtype, Hq, Hkv, D, Dv, flags;
  float scale;
};

// (16-bit types: quotients and tanh of scores without branches, two at a time)
std::string packed_math(const PackedShape& s) { return s.dtype == FA_F32 ? "" : "#define FA_PAIRS 1\n#include \"fa_score_math.cuh\"\n"; }

// ---- general kernel: tiles of fa_packed.cuh ---------------------------------------------------
// Keys of a tile: as many as leave room for two CTAs on an SM.
int packed_bn(int dtype, int D) { return dtype == FA_F32 ? (D <= 64 ? 64 : D <= 128 ? 32 : 16) : D <= 128 ? 64 : 32; }
int get_packed_kernel(fa_module* m, const PackedShape& s, bool prefix, Kernel** k) {
  const int BN = packed_bn(s.dtype, s.D), es = esize(s.dtype);
  // (the map of fa_packed.cuh)
  const int smem = 64 * pitch(s.D, es) + 2 * BN * (pitch(s.D, es) + pitch(s.Dv, es)) + (s.dtype == FA_F32 ? 64 * pitch(BN, 4) : 0);
  return get_kernel(m, kernel_key(kIdPacked, {{s.dtype, 2}, {s.D, 9}, {s.Dv, 9}, {BN, 9}, {prefix ? 1 : 0, 1}}), "fa_packed.cuh",
                    [&] { return packed_math(s) + defs({{"FA_DTYPE", s.dtype}, {"FA_D", s.D}, {"FA_DV", s.Dv}, {"FA_BN", BN}, {"FA_PREFIX", prefix ? 1 : 0}}); },
                    "fa_packed_kernel", smem, k);
}

// ---- tcgen05 kernel: fa_fwd_tc.cuh with FA_TC_PACKED --------------------------------------------
struct FaTcPackedHost {
  FaPackedParams p;
  FaTensorMapHost tk, tv;
};
bool packed_tc_takes(const PackedShape& s, long long keys) {
  return s.dtype != FA_F32 && s.D <= 128 && s.scale > 0.f && keys > 0 && keys <= 1 << 23 && !(s.flags & FA_FLAG_GENERAL_KERNELS);
}
// variant: 1 prompts, 2 over a prefix, 3 prompts in parts
int get_packed_tc_kernel(fa_module* m, const PackedShape& s, int variant, int nq, Kernel** k) {
  // (must match the shared-memory map of fa_fwd_tc.cuh)
  const int D = s.D <= 64 ? 64 : 128, atoms = D / 64, nstage = D == 64 ? nq + 1 : nq;
  const int smem = nq * atoms * 16384 + 2 * nstage * atoms * 16384 + (1 + 4 * nstage + 14) * 8 + 16 + (256 + 4) * 4 + 2 * 256 + (256 / 32) * 4 + 1024;
  return get_kernel(m, kernel_key(kIdPackedTc, {{s.dtype, 2}, {D, 9}, {nq, 2}, {variant, 2}}), "fa_fwd_tc.cuh",
                    [&] { return packed_math(s) + defs({{"FA_DTYPE", s.dtype}, {"FA_D", D}, {"FA_ROUND_SCORES", 0}, {"FA_TC_DECODE", 0}, {"FA_TC_NQ", nq}, {"FA_TC_PACKED", variant}}); },
                    "fa_packed_tc_kernel", smem, k);
}
// keys and values as [tokens, heads]; false: strides that no tensor map takes
bool packed_maps(const PackedShape& s, const fa_tensor& k, const fa_tensor& v, int keys, FaTcPackedHost& L) {
  return make_map(&L.tk, s.dtype, k, s.D, keys, s.Hkv, 1) == FA_OK && make_map(&L.tv, s.dtype, v, s.Dv, keys, s.Hkv, 1) == FA_OK;
}

// items of `rows` rows for `n` rows of B requests, dealt over the y and z dimension of a grid (and those of rows of no request, in front and behind)
dim3 packed_grid(int heads, long long n, int rows, int B) {
  const long long items = n / rows + B + 2, y = std::min<long long>(items, 32768);
  return dim3((unsigned)heads, (unsigned)y, (unsigned)((items + y - 1) / y));
}

// ---- parts -------------------------------------------------------------------------------------
// The parts of a row (not divided, with their maximum in log2 units and sum) and, behind a prefix, what the pages of its request gave (divided,
// with the same), joined:  o = sum_k 2^(m_k - m) o_k / sum_k 2^(m_k - m) l_k.  A warp per row.
size_t merge_up(size_t n) { return (n + 255) / 256 * 256; }
struct FaMergeParams {
  const float *part_o, *part_ml;  // [parts, Hkv, tokens * G, ..]
  const float *own_o, *own_ml;    // [B, Hq, Sq, ..] or null
  FaTensor o;
  float* lse;
  int B, Hq, Hkv, Sq, Dv, parts;
};
template <int DT>
__global__ void __launch_bounds__(128) fa_merge_kernel(const __grid_constant__ FaMergeParams p) {
  grid_wait();
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5), n_rows = (long long)p.B * p.Hq * p.Sq;
  if (row >= n_rows) return;
  const int q = (int)(row % p.Sq), bh = (int)(row / p.Sq), h = bh % p.Hq, b = bh / p.Hq;
  const int G = p.Hq / p.Hkv, hk = h / G;
  const long long at = (long long)hk * p.B * p.Sq * G + ((long long)b * p.Sq + q) * G + (h - hk * G);
  const bool active = lane * 4 < p.Dv, second = lane * 4 + 128 < p.Dv;
  const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
  // Lane k has the weights of parts k and k + 32 (there are 64 at most), so that all rows of values can be on their way at once; the first eight are before the
  // weights are known.
  const float2 own = p.own_ml != nullptr ? *(const float2*)(p.own_ml + row * 2) : make_float2(-INFINITY, 0.f);
  float2 ml[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) ml[i] = lane + 32 * i < p.parts ? *(const float2*)(p.part_ml + ((lane + 32 * i) * n_rows + at) * 2) : make_float2(-INFINITY, 0.f);
  const bool has = p.own_o != nullptr;
  float4 x = has && active ? *(const float4*)(p.own_o + row * p.Dv + lane * 4) : zero, y = has && second ? *(const float4*)(p.own_o + row * p.Dv + lane * 4 + 128) : zero;
  constexpr int AHEAD = 8;
  const float* from = p.part_o + at * p.Dv + lane * 4;
  const long long step = n_rows * p.Dv;
  float4 u[AHEAD], v[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    u[k] = active && k < p.parts ? *(const float4*)(from + k * step) : zero;
    v[k] = second && k < p.parts ? *(const float4*)(from + k * step + 128) : zero;
  }
  // (a part that has seen nothing counts for nothing; one whose sum is no number stays so)
  float m = fmaxf(own.y == 0.f ? -INFINITY : own.x, fmaxf(ml[0].x, ml[1].x));
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  const float top = m == -INFINITY ? 0.f : m;
  const auto weight = [&](const float2& v) { return v.y == 0.f ? 0.f : exp2f(v.x - top); };
  const float w_own = weight(own) * own.y, w[2] = {weight(ml[0]), weight(ml[1])};  // (the pages' rows are divided already)
  const float l = w_own + rot_sum(w[0] * ml[0].y + w[1] * ml[1].y);
  const auto scale = [&](float f) {
    x.x *= f; x.y *= f; x.z *= f; x.w *= f;
    y.x *= f; y.y *= f; y.z *= f; y.w *= f;
  };
  scale(w_own);
  const auto add = [&](float f, const float4& u, const float4& v) {
    x.x += f * u.x; x.y += f * u.y; x.z += f * u.z; x.w += f * u.w;
    y.x += f * v.x; y.y += f * v.y; y.z += f * v.z; y.w += f * v.w;
  };
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) add(__shfl_sync(0xffffffffu, w[0], k), u[k], v[k]);  // (where there is no part, 0 times 0)
#pragma unroll 8
  for (int k = AHEAD; k < p.parts; ++k) {
    const float f = __shfl_sync(0xffffffffu, k < 32 ? w[0] : w[1], k & 31);
    add(f, active ? *(const float4*)(from + k * step) : zero, second ? *(const float4*)(from + k * step + 128) : zero);
  }
  scale(l > 0.f ? 1.f / l : l);  // (0 and no number stay)
  char* to = (char*)p.o.ptr + ((long long)b * p.o.sb + (long long)h * p.o.sh + (long long)q * p.o.ss) * (DT == FA_F32 ? 4 : 2);
  const auto put = [&](int c, const float4& t) {
    rot_put<DT>(to, c, t.x);
    rot_put<DT>(to, c + 1, t.y);
    rot_put<DT>(to, c + 2, t.z);
    rot_put<DT>(to, c + 3, t.w);
  };
  if (active) put(lane * 4, x);
  if (second) put(lane * 4 + 128, y);
  if (lane == 0 && p.lse != nullptr) p.lse[row] = l == 0.f ? -INFINITY : (top + log2f(l)) * 0.6931471805599453f;
}

PackedShape shape_of(const fa_paged_params* p) { return {p->dtype, p->Hq, p->Hkv, p->D, p->Dv, p->flags, p->scale}; }
// Rows of an item: 128, one query tile of the tcgen05 kernel; 64, the general kernel, also for short prefixes of few rows, since its CTAs begin sooner (us on the GPU of the whole
// call, general / tcgen05, one to eight requests behind 500 tokens, 8 heads, D 64 10.9 / 12.8, D 128 14.1 / 17.1; behind 1000 12.1 / 13.1 and 15.4 / 17.5; behind 2000 14.7 / 13.5 and 18.3 / 17.4).
int prefix_rows(const fa_paged_params* p) {
  const bool few = p->prefix_length <= 1024 && (long long)p->B * p->Sq * (p->Hq / p->Hkv) <= 64;
  return few || !packed_tc_takes(shape_of(p), p->prefix_length) ? 64 : 128;
}
// Parts that the prefix is cut into, of two tiles of 128 keys at least, or one of the general kernel's (us on the GPU, parts of one / two / four tiles:
// 8 requests with 200 tokens of their own behind 500, 8 heads, D 64, general kernel, 11.0 / 12.6; 16 with 300 behind 2000, 32 / 8 heads, D 128,
// tcgen05 kernel, 21.0 / 20.4 / 23.3).  As many as make a CTA for each SM: every part has to be written and read
// again (64 requests with 1000 tokens of their own behind 8192, 32 / 8 heads, D 128, pages alone 30: half a CTA per SM 67, one 58, two 61).  Two where the rows
// alone make half a CTA per SM or more, whose tiles then are what takes the time (500 requests: one part 90, two 83).
long long prefix_tiles(const fa_paged_params* p) {
  const int R = prefix_rows(p);
  return std::max(1ll, p->Hkv * (((long long)p->B * p->Sq * (p->Hq / p->Hkv) + R - 1) / R));
}
int prefix_parts(const fa_paged_params* p) {
  const int least = prefix_rows(p) == 64 ? packed_bn(p->dtype, p->D) : 2 * 128;
  const long long ctas = prefix_tiles(p), sms = device_sm_count();
  const int shares = (p->prefix_length + least - 1) / least;
  return (int)std::max<long long>(1, std::min<long long>(std::min(shares, 64), (2 * ctas > sms ? 2 : 1) * sms / ctas));
}
void prefix_fill(fa_module* m, const fa_paged_params* p, float* part_o, float* part_ml, FaPackedParams& k) {
  memset(&k, 0, sizeof k);
  fill_buffers(m, k.mod_buf);
  k.q = cvt(p->q); k.k = cvt(p->k_prefix); k.v = cvt(p->v_prefix);
  k.part_o = part_o; k.part_ml = part_ml; k.lengths = p->lengths; k.status = p->status;
  k.B = p->B; k.Hq = p->Hq; k.Hkv = p->Hkv; k.Sq = p->Sq; k.D = p->D; k.Dv = p->Dv;
  k.tokens = p->B * p->Sq; k.keys = p->prefix_length;
  k.window = p->window < 0 ? -1 : std::min(p->window, 1 << 30);
  k.b_off = p->b_offset; k.h_off = p->h_offset; k.splits = prefix_parts(p);
  k.by_group = divide_by(p->Hq / p->Hkv); k.by_sq = divide_by(p->Sq);
  k.scale = p->scale;
}
int get_prefix_kernel(fa_module* m, const fa_paged_params* p, int rows, Kernel** k) {
  return rows == 64 ? get_packed_kernel(m, shape_of(p), true, k) : get_packed_tc_kernel(m, shape_of(p), 2, 1, k);
}
int launch_prefix(fa_module* m, const fa_paged_params* p, float* part_o, float* part_ml, void* stream) {
  FaTcPackedHost L;
  prefix_fill(m, p, part_o, part_ml, L.p);
  Kernel* kernel = nullptr;
  int R = prefix_rows(p);
  if (R != 64 && !packed_maps(shape_of(p), p->k_prefix, p->v_prefix, p->prefix_length, L)) R = 64;
  if (int rc = get_prefix_kernel(m, p, R, &kernel)) return rc;
  const long long items = ((long long)p->B * p->Sq * (p->Hq / p->Hkv) + R - 1) / R;
  if (items > 65535) return fail(FA_EUNSUPPORTED, "too many rows for a prefix");
  return launch(kernel, dim3((unsigned)p->Hkv * L.p.splits, (unsigned)items), dim3(R == 64 ? 128 : 256), &L, stream);
}
int launch_merge(int dtype, const FaMergeParams& k, void* stream) {
  const unsigned blocks = (unsigned)(((long long)k.B * k.Hq * k.Sq + 3) / 4);
  return rot_dispatch(dtype, [&](auto dt) { return launch_here("fa_merge_kernel", fa_merge_kernel<decltype(dt)::value>, dim3(blocks), dim3(128), stream, k); });
}

// ---- prompts -----------------------------------------------------------------------------------
PackedShape shape_of(const fa_prompt_params* p) { return {p->dtype, p->Hq, p->Hkv, p->D, p->Dv, p->flags, p->scale}; }
// Query tiles of a CTA of the tcgen05 kernel; 0: the general kernel.  The host knows the rows and the requests, not their lengths.
//   * A few short prompts, whose rows fill no tile of 128 or whose CTAs of 64 rows the SMs hold at once: the general kernel, whose CTAs begin sooner.  (us, general /
//     one tile, eight prompts of 30 and 64 tokens: D 64 6.7 / 7.5 and 6.8 / 7.9, 32 / 8 heads 6.8 / 8.3 and 7.6 / 8.6, D 128 8.4 / 8.9 and 8.5 / 9.3; of 128 tokens 8.9 / 8.1.)
//     No more than 1024 keys in all, since they may be one prompt's (37.8 / 15.4).
//   * Else one tile, two CTAs on an SM, at head dims up to 64 (one / two: one prompt of 4096 tokens, 8 heads, 47.8 / 60.9, eight, 32 / 8 heads, 931 / 948), and above
//     where there are few tiles or short prompts (one of 4096, 8 heads, 62.4 / 66.1; 64 of 256, 32 / 8 heads, 155 / 165; eight of 1024 118.5 / 119.6).
//   * Two tiles, which share the loads of K and V, for long ones at head dims above 64 (32 / 8 heads: one of 2048 51.5 / 45.4, eight of 4096 1466 / 1297, eight pieces of 200 behind
//     4000 149 / 134).
int prompt_query_tiles(const fa_prompt_params* p) {
  const long long G = p->Hq / p->Hkv, B = std::max(p->B, 1), rows = p->tokens * G, sms = device_sm_count();
  if (p->keys <= std::min<long long>(64 * B, 1024) && (rows <= 64 * B || p->Hkv * (rows / 64 + B) <= 2 * sms)) return 0;
  long long keys = p->keys / B;
  if (p->window >= 0) keys = std::min<long long>(keys, (long long)p->window + 128);
  return p->D > 64 && keys >= 1536 && p->Hkv * ((rows + 127) / 128) >= 2 * sms ? 2 : 1;
}
// Parts of the rows' keys, each a CTA's, where the rows alone make a CTA for every other SM at most: as many as make two per SM, of 512 keys at least (what a row sees in the mean).
// (us, one part / this: 32 / 8 heads, D 128, pieces of 16 tokens behind 4000 57 / 18, eight behind 2000 33 / 22, one of 200 behind 32000 403 / 150; with more CTAs what the
// parts are written and read for costs more, eight of 64 behind 2000 36.9 / 36.9, 32 of 33 behind 500 38 / 72.)
int prompt_parts(const fa_prompt_params* p, int nq) {
  const long long B = std::max(p->B, 1), tiles = (p->tokens * (p->Hq / p->Hkv) + 127) / 128, ctas = p->Hkv * std::max<long long>(B, tiles), sms = device_sm_count();
  if (nq != 1 || 2 * ctas > sms) return 1;
  long long keys = (p->keys - std::min(p->tokens, p->keys) / 2) / B;
  if (p->window >= 0) keys = std::min<long long>(keys, (long long)p->window + 128);
  return (int)std::max<long long>(1, std::min<long long>({keys / 512, 2 * sms / ctas, 64}));
}
size_t prompt_bytes(const fa_prompt_params* p, int parts) {
  const size_t rows = (size_t)p->tokens * p->Hq;
  return parts > 1 ? (size_t)parts * (merge_up(rows * p->Dv * 4) + merge_up(rows * 8)) : 0;
}
int prompt_sizes(fa_module* m, const fa_prompt_params* p) {
  if (!m) return fail(FA_EINVAL, "module is null");
  if (!p) return fail(FA_EINVAL, "params is null");
  if (p->dtype < FA_F16 || p->dtype > FA_F32) return fail(FA_EINVAL, "unknown dtype");
  if (p->B < 0 || p->Hq <= 0 || p->Hkv <= 0 || p->tokens < 0 || p->keys < 0) return fail(FA_EINVAL, "Hq and Hkv must be positive, B, tokens and keys not negative");
  if (p->Hq % p->Hkv) return fail(FA_EINVAL, "Hq must be a multiple of Hkv");
  if (p->D <= 0 || p->D % 16 || p->Dv <= 0 || p->Dv % 16) return fail(FA_EUNSUPPORTED, "head dims must be positive multiples of 16");
  if (p->Dv > p->D) return fail(FA_EINVAL, "value head dim must not exceed the query/key head dim");
  if (p->D > 256) return fail(FA_EUNSUPPORTED, "head dim above 256 is not supported");
  if (p->tokens * (p->Hq / p->Hkv) > 0x7fffffffll - 65536 || p->keys > 0x7fffffffll - 65536) return fail(FA_EUNSUPPORTED, "tokens * Hq / Hkv and keys must stay below 2^31");
  if (p->B > 1 << 30) return fail(FA_EUNSUPPORTED, "more than 2^30 requests");
  return FA_OK;
}
void prompt_fill(fa_module* m, const fa_prompt_params* p, FaPackedParams& k) {
  memset(&k, 0, sizeof k);
  fill_buffers(m, k.mod_buf);
  k.q = cvt(p->q); k.k = cvt(p->k); k.v = cvt(p->v); k.o = cvt(p->o);
  k.lse = p->lse; k.starts = p->starts; k.key_starts = p->key_starts ? p->key_starts : p->starts; k.status = p->status;
  k.B = p->B; k.Hq = p->Hq; k.Hkv = p->Hkv; k.D = p->D; k.Dv = p->Dv;
  k.tokens = (int)p->tokens; k.keys = (int)p->keys;
  k.window = p->window < 0 ? -1 : std::min(p->window, 1 << 30);
  k.b_off = p->b_offset; k.h_off = p->h_offset; k.splits = 1;
  k.by_group = divide_by(p->Hq / p->Hkv); k.by_sq = divide_by(1);
  k.scale = p->scale;
}

}  // namespace

extern "C" {

int fa_prompt_prepare(fa_module* m, const fa_prompt_params* p) {
  if (int rc = prompt_sizes(m, p)) return rc;
  Kernel* kernel = nullptr;
  if (packed_tc_takes(shape_of(p), 1)) {
    for (int nq = 1; nq <= 2; ++nq)
      if (int rc = get_packed_tc_kernel(m, shape_of(p), 1, nq, &kernel)) return rc;
    if (int rc = get_packed_tc_kernel(m, shape_of(p), 3, 1, &kernel)) return rc;
  }
  // (also where the tcgen05 kernel would do: short prompts take this one, and strides that no tensor map takes)
  return get_packed_kernel(m, shape_of(p), false, &kernel);
}

size_t fa_prompt_workspace_bytes(const fa_prompt_params* p) {
  if (!p || p->Hkv <= 0 || p->Hq <= 0 || p->Hq % p->Hkv || p->tokens <= 0 || p->Dv <= 0) return 0;
  return packed_tc_takes(shape_of(p), p->keys) ? prompt_bytes(p, prompt_parts(p, prompt_query_tiles(p))) : 0;
}

int fa_prompt(fa_module* m, const fa_prompt_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = prompt_sizes(m, p)) return rc;
  if ((uintptr_t)workspace & 15) return fail(FA_EINVAL, "workspace must be 16-byte aligned");
  prof_reset();
  if (p->tokens == 0) return FA_OK;
  if (p->B > 0 && !p->starts) return fail(FA_EINVAL, "starts is null");
  const int es = esize(p->dtype);
  if (int rc = check_tensor(p->q, "q", es)) return rc;
  if (int rc = check_tensor(p->o, "o", es)) return rc;
  if (int rc = check_tensor(p->k, "k", es, p->keys > 0)) return rc;
  if (int rc = check_tensor(p->v, "v", es, p->keys > 0)) return rc;
  FaTcPackedHost L;
  prompt_fill(m, p, L.p);
  Kernel* kernel = nullptr;
  const long long rows = p->tokens * (p->Hq / p->Hkv);
  const int nq = packed_tc_takes(shape_of(p), p->keys) ? prompt_query_tiles(p) : 0;
  if (nq > 0 && packed_maps(shape_of(p), p->k, p->v, (int)p->keys, L)) {
    const int parts = prompt_parts(p, nq);
    if (int rc = get_packed_tc_kernel(m, shape_of(p), parts > 1 ? 3 : 1, nq, &kernel)) return rc;
    const dim3 grid = packed_grid(p->Hkv * parts, rows, 128 * nq, p->B), block(nq == 1 ? 256 : 384);
    if (parts == 1) return launch(kernel, grid, block, &L, stream);
    if (!workspace || workspace_bytes < prompt_bytes(p, parts)) return fail(FA_EWORKSPACE, "prompt attention workspace too small");
    L.p.splits = parts;
    L.p.part_o = (float*)workspace;
    L.p.part_ml = (float*)((char*)workspace + parts * merge_up((size_t)p->tokens * p->Hq * p->Dv * 4));
    if (int rc = launch(kernel, grid, block, &L, stream)) return rc;
    return launch_merge(p->dtype, FaMergeParams{L.p.part_o, L.p.part_ml, nullptr, nullptr, L.p.o, p->lse, 1, p->Hq, p->Hkv, (int)p->tokens, p->Dv, parts}, stream);
  }
  if (int rc = get_packed_kernel(m, shape_of(p), false, &kernel)) return rc;
  return launch(kernel, packed_grid(p->Hkv, rows, 64, p->B), dim3(128), &L.p, stream);
}

}  // extern "C"
