// Filling the pages: per-head q/k RMSNorm, rotate-half RoPE and the paged K/V write of packed QKV rows.
//
//   y = x * rsqrt(mean(x^2) + eps) * w     (heads with a norm weight; values pass unchanged)
//   o[d] = y[d] * cos[d] - y[d + D/2] * sin[d],   o[d + D/2] = y[d + D/2] * cos[d + D/2] + y[d] * sin[d + D/2]
//
// in fp32, rounded to bf16 once, at the store (q3t_qk_norm_rope_kv instead keeps the reference's rounding
// after every operation). Queries go to query_out, keys and values to the row's cache position.
//
// The kernel is bound by its bytes: every element is read and written once. D/8 lanes own a head; a lane
// holds 4 dims of the first half and the 4 dims that rotate with them in the second, so RoPE needs no
// exchange between lanes and the norm only the D/8-lane sum.
#include "common.cuh"
#include "host.cuh"
#include "paged.cuh"

using namespace q3t;

namespace {

struct WriteArgs {
  const __nv_bfloat16* qkv;
  int64_t qkv_stride;
  const __nv_bfloat16 *q_norm, *k_norm, *cos, *sin;
  float eps;
  int64_t table_len;
  const int64_t *rotary_positions, *cache_positions, *sequences;
  PageTable pages;
  __nv_bfloat16 *query_out, *key_pages, *value_pages;
  int64_t page_stride;
  int q_heads, kv_heads;
  int64_t rows;
  unsigned* status;
};

Q3T_DEV void load4(const __nv_bfloat16* p, float (&f)[4]) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
  const float2 a = __bfloat1622float2(h[0]), b = __bfloat1622float2(h[1]);
  f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
}
Q3T_DEV void store4(__nv_bfloat16* p, const float (&f)[4]) {
  uint2 v;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
  h[0] = __floats2bfloat162_rn(f[0], f[1]);
  h[1] = __floats2bfloat162_rn(f[2], f[3]);
  *reinterpret_cast<uint2*>(p) = v;
}

constexpr int kThreads = 128;

template <int D>
__global__ void __launch_bounds__(kThreads) paged_write_kernel(const WriteArgs a) {
  constexpr int L = D / 8;  // lanes of a head
  grid_dependency_wait();
  const int heads = a.q_heads + 2 * a.kv_heads;
  const int64_t unit = int64_t(blockIdx.x) * (kThreads / L) + threadIdx.x / L;
  const bool live = unit < a.rows * heads;
  const int64_t r = live ? unit / heads : 0;
  const int head = live ? int(unit % heads) : 0;
  const int d0 = int(threadIdx.x % L) * 4, d1 = d0 + D / 2;
  const int64_t sequence = a.sequences != nullptr ? a.sequences[r] : r;
  const bool padding = sequence < 0;
  int64_t rp = a.rotary_positions[r];
  const bool rp_ok = rp >= 0 && rp < a.table_len;
  if (!rp_ok) rp = rp < 0 ? 0 : a.table_len - 1;
  const bool is_q = head < a.q_heads, is_v = head >= a.q_heads + a.kv_heads;

  const __nv_bfloat16* src = a.qkv + r * a.qkv_stride + int64_t(head) * D;
  float x0[4], x1[4], c0[4], c1[4], s0[4], s1[4];
  load4(src + d0, x0);
  load4(src + d1, x1);
  load4(a.cos + rp * D + d0, c0);
  load4(a.cos + rp * D + d1, c1);
  load4(a.sin + rp * D + d0, s0);
  load4(a.sin + rp * D + d1, s1);
  float o0[4], o1[4];
  if (a.q_norm != nullptr) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) ss += x0[e] * x0[e] + x1[e] * x1[e];
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = rsqrtf(ss * (1.f / float(D)) + a.eps);
    const __nv_bfloat16* w = is_q ? a.q_norm : a.k_norm;
    float w0[4], w1[4];
    load4(w + d0, w0);
    load4(w + d1, w1);
#pragma unroll
    for (int e = 0; e < 4; ++e) o0[e] = x0[e] * inv * w0[e], o1[e] = x1[e] * inv * w1[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) o0[e] = x0[e], o1[e] = x1[e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float y0 = o0[e], y1 = o1[e];
    o0[e] = is_v ? x0[e] : y0 * c0[e] - y1 * s0[e];
    o1[e] = is_v ? x1[e] : y1 * c1[e] + y0 * s1[e];
  }
  if (!live || padding) return;
  if (!rp_ok && head == 0 && d0 == 0) raise_status(a.status, kStatusBadIndex);
  __nv_bfloat16* dst;
  if (is_q) {
    dst = a.query_out + (r * a.q_heads + head) * D;
  } else {
    const int64_t position = a.cache_positions[r];
    const int64_t page = a.pages.lookup(sequence, position);
    if (page < 0) {
      if (d0 == 0) raise_status(a.status, kStatusBadIndex);
      return;
    }
    const int h = head - a.q_heads - (is_v ? a.kv_heads : 0);
    dst = (is_v ? a.value_pages : a.key_pages) + page * a.page_stride +
          (int64_t(h) * a.pages.page_size + position % a.pages.page_size) * D;
  }
  store4(dst + d0, o0);
  store4(dst + d1, o1);
}

}  // namespace

extern "C" int q3t_paged_qk_norm_rope_kv(const q3t_paged_write* call, unsigned* status, void* stream) {
  const char* name = "paged_qk_norm_rope_kv";
  if (call == nullptr) return fail(Q3T_EINVAL, "%s: null pointer", name);
  const q3t_paged_write& p = *call;
  const q3t_paged_cache& c = p.cache;
  if (!p.qkv || !p.cos_table || !p.sin_table || !p.rotary_positions || !p.cache_positions || !p.query_out ||
      (p.q_norm_weight == nullptr) != (p.k_norm_weight == nullptr))
    return fail(Q3T_EINVAL, "%s: null pointer", name);
  if (const int rc = check_cache(name, c)) return rc;
  if (p.rows < 1 || p.q_heads < 1 || p.q_heads > 1024 || p.table_len < 1 ||
      (p.sequences == nullptr && c.table_rows < p.rows))
    return fail(Q3T_EINVAL, "%s: invalid geometry", name);
  const int64_t heads = p.q_heads + 2 * c.kv_heads;
  if (p.qkv_stride < heads * c.head_dim || p.qkv_stride % 8) return fail(Q3T_EINVAL, "%s: qkv stride", name);
  if (!aligned16(p.qkv) || !aligned16(p.q_norm_weight) || !aligned16(p.k_norm_weight) || !aligned16(p.cos_table) ||
      !aligned16(p.sin_table) || !aligned16(p.query_out))
    return fail(Q3T_EINVAL, "%s: 16-byte alignment", name);
  if (p.rows > (int64_t(1) << 31) / heads) return fail(Q3T_EINVAL, "%s: too many rows", name);
  const DeviceGuard guard(c.device);
  if (!guard.ok()) return fail(Q3T_ECUDA, "%s: no such device", name);
  WriteArgs a;
  a.qkv = static_cast<const __nv_bfloat16*>(p.qkv);
  a.qkv_stride = p.qkv_stride;
  a.q_norm = static_cast<const __nv_bfloat16*>(p.q_norm_weight);
  a.k_norm = static_cast<const __nv_bfloat16*>(p.k_norm_weight);
  a.cos = static_cast<const __nv_bfloat16*>(p.cos_table);
  a.sin = static_cast<const __nv_bfloat16*>(p.sin_table);
  a.eps = float(p.eps);
  a.table_len = p.table_len;
  a.rotary_positions = p.rotary_positions;
  a.cache_positions = p.cache_positions;
  a.sequences = p.sequences;
  a.pages = PageTable{c.page_table, c.table_stride, c.table_rows, c.table_columns, c.pages, int(c.page_size)};
  a.query_out = static_cast<__nv_bfloat16*>(p.query_out);
  a.key_pages = static_cast<__nv_bfloat16*>(const_cast<void*>(c.key_pages));
  a.value_pages = static_cast<__nv_bfloat16*>(const_cast<void*>(c.value_pages));
  a.page_stride = c.page_stride;
  a.q_heads = int(p.q_heads);
  a.kv_heads = int(c.kv_heads);
  a.rows = p.rows;
  a.status = status;
  const int64_t per_block = kThreads / (c.head_dim / 8);
  const dim3 grid(unsigned((p.rows * heads + per_block - 1) / per_block));
  return launch(c.head_dim == 128 ? paged_write_kernel<128> : paged_write_kernel<64>, grid, dim3(kThreads), 0, stream,
                true, name, a);
}
