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
// exchange between lanes and the norm only the D/16-lane sum. A lane takes HEADS heads of one kind of a row, whose
// loads are all on their way before the first is used, and reads the row's positions, cos and sin once for them.
//
// 3887 rows of 16 + 2 * 8 heads of 128 dims: 15.1 us for 65.8 MB that are not in L2, 4.4 TB/s (13.1 where half of them are,
// 10.2 where all are); 16000 rows 5.3 TB/s; 1 to 64 rows 1.9 to 2.4 us. The same kernel that only copies takes 11.7 us for
// the 3887. With the weight, cos and sin unpacked and multiplied for every head the kernel was bound by its instructions;
// packed arithmetic on factors that four heads share leaves 37 % of the issue slots in use, and the loads' latency is the
// bound. Five CTAs an SM instead of what the registers would leave: 16.5 -> 15.1 us. Two or eight heads to a lane, a loop
// that fetches the next heads meanwhile (two of them in registers leave fewer warps), and rows brought into shared memory
// by a copying warp were all slower.
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

Q3T_DEV float2 unpack2(uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
Q3T_DEV uint32_t pack2(float2 v) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
struct Words {
  uint32_t w[4];
};
Q3T_DEV Words load8(const __nv_bfloat16* p) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  return {{v.x, v.y, v.z, v.w}};
}
// The same for what is read once: it leaves L1 to the weights, cos and sin (3887 rows, of which L2 holds half, as behind
// the projection that wrote them: 14.4 -> 13.1 us; with all of them in L2 no difference; from memory 14.6 -> 15.1).
Q3T_DEV Words load8_once(const __nv_bfloat16* p) {
  Words v;
  asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3])
               : "l"(p)
               : "memory");
  return v;
}
Q3T_DEV void store8(__nv_bfloat16* p, const Words& v) {
  *reinterpret_cast<uint4*>(p) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
}

template <int D, int HEADS>
__global__ void __launch_bounds__(kThreads, HEADS == 1 ? 1 : 5) paged_write_kernel(const WriteArgs a) {
  constexpr int L = D / 16;  // lanes of a head
  grid_dependency_wait();
  const int q_chunks = (a.q_heads + HEADS - 1) / HEADS, kv_chunks = (a.kv_heads + HEADS - 1) / HEADS;
  const int chunks = q_chunks + 2 * kv_chunks;
  const unsigned unit = blockIdx.x * (kThreads / L) + threadIdx.x / L;
  const unsigned r = unit / unsigned(chunks);
  if (r >= a.rows) return;  // whole groups of L lanes leave; the sums below name the lanes of a group
  int chunk = int(unit - r * chunks);
  const int kind = chunk < q_chunks ? 0 : chunk < q_chunks + kv_chunks ? 1 : 2;  // queries, keys, values
  if (kind > 0) chunk -= q_chunks + (kind - 1) * kv_chunks;
  const int head0 = chunk * HEADS, heads = min(HEADS, (kind > 0 ? a.kv_heads : a.q_heads) - head0);
  const int d0 = int(threadIdx.x % L) * 8;
  const unsigned group = (L == 8 ? 0xffu : 0xfu) << (threadIdx.x & 31 & ~(L - 1));

  // the loads that others depend on first, then all the others
  const int64_t sequence = a.sequences != nullptr ? a.sequences[r] : r;
  const int64_t position = a.cache_positions[r];
  int64_t rp = a.rotary_positions[r];
  Words x[HEADS][2];
  const int in_row = head0 + (kind > 0 ? a.q_heads + (kind - 1) * a.kv_heads : 0);
  const __nv_bfloat16* src = a.qkv + r * a.qkv_stride + int64_t(in_row) * D + d0;
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    x[i][0] = x[i][1] = {};
    if (i < heads) x[i][0] = load8_once(src + i * D), x[i][1] = load8_once(src + i * D + D / 2);
  }
  const bool rp_ok = rp >= 0 && rp < a.table_len;
  if (!rp_ok) rp = rp < 0 ? 0 : a.table_len - 1;
  Words c0 = {}, c1 = {}, s0 = {}, s1 = {};
  if (kind < 2) {
    c0 = load8(a.cos + rp * D + d0), c1 = load8(a.cos + rp * D + D / 2 + d0);
    s0 = load8(a.sin + rp * D + d0), s1 = load8(a.sin + rp * D + D / 2 + d0);
  }
  __nv_bfloat16* dst = a.query_out + (int64_t(r) * a.q_heads + head0) * D + d0;
  int64_t step = D;  // from head to head
  if (kind > 0) {
    int row;
    const int64_t page = a.pages.lookup(sequence, position, row);
    step *= a.pages.page_size;
    dst = page < 0 ? nullptr : (kind == 1 ? a.key_pages : a.value_pages) + page * a.page_stride + head0 * step + row * D + d0;
  }
  if (sequence < 0) return;  // padding
  if (d0 == 0 && (dst == nullptr || (!rp_ok && kind == 0 && head0 == 0))) raise_status(a.status, kStatusBadIndex);
  if (dst == nullptr) return;

  if (kind < 2) {
    // o0 = inv (x0 a + x1 b), o1 = inv (x1 c + x0 d): the weight goes into cos and sin once for the lane's heads, and inv
    // comes last, behind products that do not wait for the sum
    float2 fa[4], fb[4], fc[4], fd[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      fa[e] = unpack2(c0.w[e]), fb[e] = unpack2(s0.w[e] ^ 0x80008000u);  // -sin
      fc[e] = unpack2(c1.w[e]), fd[e] = unpack2(s1.w[e]);
    }
    if (a.q_norm != nullptr) {
      const __nv_bfloat16* w = kind == 0 ? a.q_norm : a.k_norm;
      const Words w0 = load8(w + d0), w1 = load8(w + D / 2 + d0);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 u = unpack2(w0.w[e]), v = unpack2(w1.w[e]);
        fa[e] = mul2(fa[e], u), fd[e] = mul2(fd[e], u);
        fb[e] = mul2(fb[e], v), fc[e] = mul2(fc[e], v);
      }
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      float2 x0[4], x1[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x0[e] = unpack2(x[i][0].w[e]), x1[e] = unpack2(x[i][1].w[e]);
      float inv = 1.f;
      if (a.q_norm != nullptr) {
        float2 squares = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 4; ++e) squares = fma2(x1[e], x1[e], fma2(x0[e], x0[e], squares));
        float sum = squares.x + squares.y;
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(group, sum, o);
        inv = rsqrtf(sum * (1.f / float(D)) + a.eps);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[i][0].w[e] = pack2(mul2(fma2(x0[e], fa[e], mul2(x1[e], fb[e])), {inv, inv}));
        x[i][1].w[e] = pack2(mul2(fma2(x1[e], fc[e], mul2(x0[e], fd[e])), {inv, inv}));
      }
    }
  }
#pragma unroll
  for (int i = 0; i < HEADS; ++i)
    if (i < heads) store8(dst + i * step, x[i][0]), store8(dst + i * step + D / 2, x[i][1]);
}

template <int D, int HEADS>
int launch_write(const WriteArgs& a, void* stream, const char* name) {
  constexpr int kUnits = kThreads / (D / 16);
  const int64_t units = a.rows * ((a.q_heads + HEADS - 1) / HEADS + 2 * ((a.kv_heads + HEADS - 1) / HEADS));
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
  // few rows: a lane per head for the shortest chain (64 rows of 32 heads of 128 dims 2.1 us against 2.7 with four, 512
  // rows 3.9 against 4.2); many: four heads to a lane share what a row needs once (1000 rows 5.9 us against 6.7, 3887 15.1
  // against 16.9)
  const bool few = p.rows * heads <= 24576;
  if (c.head_dim == 128) return few ? launch_write<128, 1>(a, stream, name) : launch_write<128, 4>(a, stream, name);
  return few ? launch_write<64, 1>(a, stream, name) : launch_write<64, 4>(a, stream, name);
}
