// Filling the pages: per-head q/k RMSNorm, rotate-half RoPE and the paged K/V write of packed QKV rows.
//
//   y = x * rsqrt(mean(x^2) + eps) * w     (heads with a norm weight; values pass unchanged)
//   o[d] = y[d] * cos[d] - y[d + D/2] * sin[d],   o[d + D/2] = y[d + D/2] * cos[d + D/2] + y[d] * sin[d + D/2]
//
// in fp32, rounded to bf16 once, at the store (q3t_qk_norm_rope_kv instead keeps the reference's rounding
// after every operation). Queries go to query_out, keys and values to the row's cache position.
//
// The kernel is bound by its bytes: every element is read and written once. D/16 lanes own a head; a lane
// holds 8 dims of the first half and the 8 dims that rotate with them in the second, so RoPE needs no
// exchange between lanes and the norm only the D/16-lane sum. A lane takes HEADS heads of a row, whose loads
// are all on their way before the first is used, and reads the row's positions, cos and sin once for them.
//
// 3500 rows of 16 + 2 * 8 heads of 128 dims: 17.2 us for 65.8 MB, 3.8 TB/s; 16000 rows 4.8 TB/s; 1 to 64 rows 2.5 us. The
// same kernel that only copies takes 11 us for the 3500: what is between is the chain of positions, cos/sin and the head's
// sum in each thread, with as many threads as the registers allow. Fewer registers (a launch bound), two or eight heads to
// a lane, packed fp32 arithmetic, and rows brought into shared memory by a copying warp were all slower.
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

constexpr int kThreads = 128;

template <int D, int HEADS>
__global__ void __launch_bounds__(kThreads) paged_write_kernel(const WriteArgs a) {
  constexpr int L = D / 16;  // lanes of a head
  grid_dependency_wait();
  const int heads = a.q_heads + 2 * a.kv_heads, chunks = (heads + HEADS - 1) / HEADS;
  const unsigned unit = blockIdx.x * (kThreads / L) + threadIdx.x / L;
  const unsigned r = unit / unsigned(chunks);
  if (r >= a.rows) return;  // whole groups of L lanes leave; the sums below name the lanes of a group
  const int head0 = int(unit - r * chunks) * HEADS, d0 = int(threadIdx.x % L) * 8;
  const unsigned group = (L == 8 ? 0xffu : 0xfu) << (threadIdx.x & 31 & ~(L - 1));

  uint4 x[HEADS][2];
  const __nv_bfloat16* src = a.qkv + r * a.qkv_stride + int64_t(head0) * D + d0;
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    x[i][0] = x[i][1] = make_uint4(0u, 0u, 0u, 0u);
    if (head0 + i < heads) {
      x[i][0] = *reinterpret_cast<const uint4*>(src + i * D);
      x[i][1] = *reinterpret_cast<const uint4*>(src + i * D + D / 2);
    }
  }
  const int64_t sequence = a.sequences != nullptr ? a.sequences[r] : r;
  const int64_t position = a.cache_positions[r];
  int64_t rp = a.rotary_positions[r];
  const bool rp_ok = rp >= 0 && rp < a.table_len;
  if (!rp_ok) rp = rp < 0 ? 0 : a.table_len - 1;
  float c0[8], c1[8], s0[8], s1[8];
  unpack8(*reinterpret_cast<const uint4*>(a.cos + rp * D + d0), c0);
  unpack8(*reinterpret_cast<const uint4*>(a.cos + rp * D + D / 2 + d0), c1);
  unpack8(*reinterpret_cast<const uint4*>(a.sin + rp * D + d0), s0);
  unpack8(*reinterpret_cast<const uint4*>(a.sin + rp * D + D / 2 + d0), s1);
  if (sequence < 0) return;  // padding
  if (!rp_ok && head0 == 0 && d0 == 0) raise_status(a.status, kStatusBadIndex);
  int64_t at = -1;  // element offset of the row's position in a pool, head 0
  if (head0 + HEADS > a.q_heads) {
    int row;
    const int64_t page = a.pages.lookup(sequence, position, row);
    if (page >= 0) at = page * a.page_stride + int64_t(row) * D + d0;
    else if (d0 == 0) raise_status(a.status, kStatusBadIndex);
  }
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    const int head = head0 + i;
    if (head >= heads) break;
    __nv_bfloat16* dst = a.query_out + (int64_t(r) * a.q_heads + head) * D + d0;
    if (head >= a.q_heads) {
      const bool key = head < a.q_heads + a.kv_heads;
      const int h = head - a.q_heads - (key ? 0 : a.kv_heads);
      if (at < 0) continue;
      dst = (key ? a.key_pages : a.value_pages) + at + int64_t(h) * a.pages.page_size * D;
    }
    if (head < a.q_heads + a.kv_heads) {
      float y0[8], y1[8], o0[8], o1[8];
      unpack8(x[i][0], y0);
      unpack8(x[i][1], y1);
      if (a.q_norm != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += y0[e] * y0[e] + y1[e] * y1[e];
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(group, ss, o);
        const float inv = rsqrtf(ss * (1.f / float(D)) + a.eps);
        const __nv_bfloat16* w = head < a.q_heads ? a.q_norm : a.k_norm;
        float w0[8], w1[8];
        unpack8(*reinterpret_cast<const uint4*>(w + d0), w0);
        unpack8(*reinterpret_cast<const uint4*>(w + D / 2 + d0), w1);
#pragma unroll
        for (int e = 0; e < 8; ++e) y0[e] *= inv * w0[e], y1[e] *= inv * w1[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        o0[e] = y0[e] * c0[e] - y1[e] * s0[e];
        o1[e] = y1[e] * c1[e] + y0[e] * s1[e];
      }
      x[i][0] = pack8(o0);
      x[i][1] = pack8(o1);
    }
    *reinterpret_cast<uint4*>(dst) = x[i][0];
    *reinterpret_cast<uint4*>(dst + D / 2) = x[i][1];
  }
}

template <int D, int HEADS>
int launch_write(const WriteArgs& a, void* stream, const char* name) {
  constexpr int kUnits = kThreads / (D / 16);
  const int64_t units = a.rows * ((a.q_heads + 2 * a.kv_heads + HEADS - 1) / HEADS);
  return launch(paged_write_kernel<D, HEADS>, dim3(unsigned((units + kUnits - 1) / kUnits)), dim3(kThreads), 0, stream, true,
                name, a);
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
  // few rows: a lane per head for the shortest chain (1..64 rows of 32 heads 2.5 us against 3.7 with four); many: four
  // heads to a lane (3500 rows 17.2 us against 19.2)
  const bool few = p.rows * heads <= 32768;
  if (c.head_dim == 128) return few ? launch_write<128, 1>(a, stream, name) : launch_write<128, 4>(a, stream, name);
  return few ? launch_write<64, 1>(a, stream, name) : launch_write<64, 4>(a, stream, name);
}
