// Attention of prompts laid end to end (fa_prompt) and over a prefix that requests share (the first of the two parts of fa_paged with one; the other is the
// pages', and fa_prefix_merge_kernel joins them).  Kernels: kernels/fa_packed.cuh.  Part of flaxattn.cu.
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

// ---- general kernel: tiles of fa_packed.cuh ---------------------------------------------------
// Keys of a tile: as many as leave room for two CTAs on an SM.
int packed_bn(int dtype, int D) { return dtype == FA_F32 ? (D <= 64 ? 64 : D <= 128 ? 32 : 16) : D <= 128 ? 64 : 32; }
int get_packed_kernel(fa_module* m, const PackedShape& s, bool prefix, Kernel** k) {
  const int BN = packed_bn(s.dtype, s.D), es = esize(s.dtype);
  // (the map of fa_packed.cuh)
  const int smem = 64 * pitch(s.D, es) + 2 * BN * (pitch(s.D, es) + pitch(s.Dv, es)) + (s.dtype == FA_F32 ? 64 * pitch(BN, 4) : 0);
  return get_kernel(m, kernel_key(kIdPacked, {{s.dtype, 2}, {s.D, 9}, {s.Dv, 9}, {BN, 9}, {prefix ? 1 : 0, 1}}), "fa_packed.cuh",
                    [&] { return defs({{"FA_DTYPE", s.dtype}, {"FA_D", s.D}, {"FA_DV", s.Dv}, {"FA_BN", BN}, {"FA_PREFIX", prefix ? 1 : 0}}); },
                    "fa_packed_kernel", smem, k);
}

// items of `rows` rows for `n` rows of B requests, dealt over the y and z dimension of a grid (and those of rows of no request, in front and behind)
dim3 packed_grid(int heads, long long n, int rows, int B) {
  const long long items = n / rows + B + 2, y = std::min<long long>(items, 32768);
  return dim3((unsigned)heads, (unsigned)y, (unsigned)((items + y - 1) / y));
}

// ---- over a prefix -----------------------------------------------------------------------------
// The parts of a row (from the tiles of the prefix, not divided, with their maximum in log2 units and sum) and what the pages of its request gave (divided,
// with the same), joined:  o = sum_k 2^(m_k - m) o_k / sum_k 2^(m_k - m) l_k.  A warp per row.
struct FaMergeParams {
  const float *part_o, *part_ml;  // [parts, Hkv, tokens * G, ..]
  const float *own_o, *own_ml;    // [B, Hq, Sq, ..]
  FaTensor o;
  float* lse;
  int B, Hq, Hkv, Sq, Dv, parts;
};
template <int DT>
__global__ void __launch_bounds__(128) fa_prefix_merge_kernel(const __grid_constant__ FaMergeParams p) {
  grid_wait();
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5), n_rows = (long long)p.B * p.Hq * p.Sq;
  if (row >= n_rows) return;
  const int q = (int)(row % p.Sq), bh = (int)(row / p.Sq), h = bh % p.Hq, b = bh / p.Hq;
  const int G = p.Hq / p.Hkv, hk = h / G;
  const long long at = (long long)hk * p.B * p.Sq * G + ((long long)b * p.Sq + q) * G + (h - hk * G);
  const bool active = lane * 4 < p.Dv, second = lane * 4 + 128 < p.Dv;
  const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
  const auto weight = [](float m, float l, float top) { return l == 0.f ? 0.f : exp2f(m - (top == -INFINITY ? 0.f : top)); };
  // the pages' first, as sums: times l
  const float2 own = *(const float2*)(p.own_ml + row * 2);
  float m = own.y == 0.f ? -INFINITY : own.x, l = own.y;
  float4 x = active ? *(const float4*)(p.own_o + row * p.Dv + lane * 4) : zero, y = second ? *(const float4*)(p.own_o + row * p.Dv + lane * 4 + 128) : zero;
  const auto scale = [&](float f) {
    x.x *= f; x.y *= f; x.z *= f; x.w *= f;
    y.x *= f; y.y *= f; y.z *= f; y.w *= f;
  };
  scale(l);
  constexpr int U = 4;
  for (int k = 0; k < p.parts; k += U) {
    float2 ml[U];
    float4 u[U], v[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {  // (all of them on their way at once)
      const bool in = k + i < p.parts;
      const long long a = in ? (k + i) * n_rows + at : 0;
      ml[i] = in ? *(const float2*)(p.part_ml + a * 2) : make_float2(-INFINITY, 0.f);
      u[i] = in && active ? *(const float4*)(p.part_o + a * p.Dv + lane * 4) : zero;
      v[i] = in && second ? *(const float4*)(p.part_o + a * p.Dv + lane * 4 + 128) : zero;
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < U; ++i) top = fmaxf(top, ml[i].x);
    const float f = weight(m, l, top);
    l *= f;
    scale(f);
    m = top;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const float g = weight(ml[i].x, ml[i].y, top);
      l += g * ml[i].y;
      x.x += g * u[i].x; x.y += g * u[i].y; x.z += g * u[i].z; x.w += g * u[i].w;
      y.x += g * v[i].x; y.y += g * v[i].y; y.z += g * v[i].z; y.w += g * v[i].w;
    }
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
  if (lane == 0 && p.lse != nullptr) p.lse[row] = l == 0.f ? -INFINITY : ((m == -INFINITY ? 0.f : m) + log2f(l)) * 0.6931471805599453f;
}

PackedShape shape_of(const fa_paged_params* p) { return {p->dtype, p->Hq, p->Hkv, p->D, p->Dv, p->flags, p->scale}; }
// Parts that the prefix is cut into: as many as fill the SMs with CTAs of the heads' rows, but a tile each at least.
int prefix_parts(const fa_paged_params* p) {
  const long long rows = (long long)p->B * p->Sq * (p->Hq / p->Hkv), ctas = p->Hkv * ((rows + 63) / 64);
  const int tiles = (p->prefix_length + packed_bn(p->dtype, p->D) - 1) / packed_bn(p->dtype, p->D);
  return (int)std::max<long long>(1, std::min<long long>(std::min(tiles, 64), 2LL * device_sm_count() / ctas));
}
int prefix_fill(fa_module* m, const fa_paged_params* p, float* part_o, float* part_ml, FaPackedParams& k) {
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
  return FA_OK;
}
int launch_prefix(fa_module* m, const fa_paged_params* p, float* part_o, float* part_ml, void* stream) {
  FaPackedParams k;
  if (int rc = prefix_fill(m, p, part_o, part_ml, k)) return rc;
  Kernel* kernel = nullptr;
  if (int rc = get_packed_kernel(m, shape_of(p), true, &kernel)) return rc;
  const long long items = ((long long)k.tokens * (p->Hq / p->Hkv) + 63) / 64;
  if (items > 65535) return fail(FA_EUNSUPPORTED, "too many rows for a prefix");
  return launch(kernel, dim3((unsigned)p->Hkv, (unsigned)items, (unsigned)k.splits), dim3(128), &k, stream);
}
int launch_prefix_merge(const fa_paged_params* p, const float* part_o, const float* part_ml, const float* own_o, const float* own_ml, int parts, void* stream) {
  FaMergeParams k{part_o, part_ml, own_o, own_ml, cvt(p->o), p->lse, p->B, p->Hq, p->Hkv, p->Sq, p->Dv, parts};
  const unsigned blocks = (unsigned)(((long long)p->B * p->Hq * p->Sq + 3) / 4);
  return rot_dispatch(p->dtype, [&](auto dt) { return launch_here("fa_prefix_merge_kernel", fa_prefix_merge_kernel<decltype(dt)::value>, dim3(blocks), dim3(128), stream, k); });
}

// ---- prompts -----------------------------------------------------------------------------------
PackedShape shape_of(const fa_prompt_params* p) { return {p->dtype, p->Hq, p->Hkv, p->D, p->Dv, p->flags, p->scale}; }
int prompt_sizes(fa_module* m, const fa_prompt_params* p) {
  if (!m) return fail(FA_EINVAL, "module is null");
  if (!p) return fail(FA_EINVAL, "params is null");
  if (p->dtype < FA_F16 || p->dtype > FA_F32) return fail(FA_EINVAL, "unknown dtype");
  if (p->B < 0 || p->Hq <= 0 || p->Hkv <= 0 || p->tokens < 0 || p->keys < 0) return fail(FA_EINVAL, "Hq and Hkv must be positive, B, tokens and keys not negative");
  if (p->Hq % p->Hkv) return fail(FA_EINVAL, "Hq must be a multiple of Hkv");
  if (p->D <= 0 || p->D % 16 || p->Dv <= 0 || p->Dv % 16) return fail(FA_EUNSUPPORTED, "head dims must be positive multiples of 16");
  if (p->Dv > p->D) return fail(FA_EINVAL, "value head dim must not exceed the query/key head dim");
  if (p->D > 256) return fail(FA_EUNSUPPORTED, "head dim above 256 is not supported");
  if (p->tokens * (p->Hq / p->Hkv) > 0x7fffffffll - 65536 || p->keys > 0x7fffffffll - 65536 || p->B > 0x7fffffff - 1) return fail(FA_EUNSUPPORTED, "tokens * Hq / Hkv and keys must stay below 2^31");
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
  return get_packed_kernel(m, shape_of(p), false, &kernel);
}

int fa_prompt(fa_module* m, const fa_prompt_params* p, void* stream) {
  if (int rc = prompt_sizes(m, p)) return rc;
  prof_reset();
  if (p->tokens == 0) return FA_OK;
  if (p->B > 0 && !p->starts) return fail(FA_EINVAL, "starts is null");
  const int es = esize(p->dtype);
  if (int rc = check_tensor(p->q, "q", es)) return rc;
  if (int rc = check_tensor(p->o, "o", es)) return rc;
  if (int rc = check_tensor(p->k, "k", es, p->keys > 0)) return rc;
  if (int rc = check_tensor(p->v, "v", es, p->keys > 0)) return rc;
  FaPackedParams k;
  prompt_fill(m, p, k);
  Kernel* kernel = nullptr;
  if (int rc = get_packed_kernel(m, shape_of(p), false, &kernel)) return rc;
  return launch(kernel, packed_grid(p->Hkv, p->tokens * (p->Hq / p->Hkv), 64, p->B), dim3(128), &k, stream);
}

}  // extern "C"
