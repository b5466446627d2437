// Attention of one new token per sequence over a paged key/value cache.
//
//   out[r, h] = sum_j softmax_j(scale * q[r, h] . k_j) v_j,   j = 0 .. positions[r]
//
// A (row, key/value head) pair is read once for all query heads of its group (in passes of 8 where the
// group is wider). Warps are independent workers: each streams a contiguous run of 16-key steps through
// its own shared-memory FIFO and keeps its own online softmax, with no barrier until the end.
//
// The products run on mma.sync m16n8k16 with the keys as the 16 rows and the query heads as the 8 columns:
//   S^T[16 keys, 8 heads]  = K[16, D] Q^T[D, 8]          D/16 steps
//   O^T[D, 8 heads]       += V^T[D, 16] P^T[16, 8]       D/16 tiles of 16 dims
// so one or eight heads cost the same D/8 instructions per step and no accumulator row is wasted. (tcgen05
// needs 64 or 128 rows of A and a round trip through TMEM and shared memory for P; the kernel is bound by
// its key/value bytes at under 8 flops a byte, and these instructions are far from being the limit.)
//
// Which lane copies what is chosen so that a lane reads back from shared memory exactly the 16-byte units
// that it copied itself: unit u of lane l sits at [u][l]. That needs no swizzle, has no bank conflict and
// no synchronisation beyond the lane's own cp.async groups. With g = lane / 4, t = lane % 4:
//   K: units of keys g and g + 8 at dim chunks t, t + 4, ... (8 dims each). Q is loaded with the same
//      permutation of dims, so the dot product needs no reordering.
//   V: units of keys 2t, 2t+1, 2t+8, 2t+9 at dim chunk g (and g + 8): two keys' units become the A fragment
//      of O^T by byte permutes; row g of tile j is dim 8g + j, so a lane ends with 8 adjacent output dims.
#include "common.cuh"
#include "host.cuh"
#include "paged.cuh"

using namespace q3t;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kHeads = 8;  // query heads of a pass (columns of the products)

struct DecodeArgs {
  const __nv_bfloat16 *query, *keys, *values;
  int64_t query_stride, page_stride;
  PageTable pages;
  const int64_t* positions;
  __nv_bfloat16* out;
  int rows, q_heads, kv_heads, group, passes;
  int64_t context;
  float scale_log2;
  unsigned* status;
};

Q3T_DEV void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
Q3T_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
Q3T_DEV void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
Q3T_DEV uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
// C (16x8 fp32) += A (16x16 bf16) * B (16x8 bf16)
Q3T_DEV void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transpose of an 8x8 bf16 matrix held two adjacent columns per lane.
Q3T_DEV uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
Q3T_DEV uint32_t pack2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
Q3T_DEV uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// The online softmax of up to 8 query heads over a run of keys, spread over a warp: lane (g, t) holds heads
// 2t and 2t + 1; o[j] are tile j's outputs {dim row g of head 2t, of 2t + 1, dim row g + 8 of both}. m is a
// reference that the true maximum exceeds by at most 8 (in powers of two): it only moves when a score
// passes it by more, so most steps skip the rescale; o / l and the merge do not depend on it. l is this
// lane's share of the sum until finish().
template <int D>
struct Run {
  static constexpr int kTiles = D / 16;
  float o[kTiles][4];
  float m[2], l[2];

  Q3T_DEV void reset() {
#pragma unroll
    for (int j = 0; j < kTiles; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
  }
  Q3T_DEV void finish() {
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], x);
  }
};

template <int D, int W, int ST>
struct Cfg {
  static constexpr int kKUnits = D / 16, kVUnits = D / 16;       // 16-byte units of a lane per step
  static constexpr int kStepBytes = (kKUnits + kVUnits) * 512;   // 16 keys: K and V
  static constexpr int kRing = ST * kStepBytes;                  // a warp's FIFO
  static constexpr int kPart = kHeads * (D + 2);                 // floats of a run at rest: m, l and o per head
  static constexpr int kSmem = W * (kRing + kPart * 4);
};

// One step's 16-byte units of this lane, from the element offset of its first key.
template <int D>
Q3T_DEV void copy_step(uint32_t ring, const __nv_bfloat16* keys, const __nv_bfloat16* values, int64_t at, int g, int t) {
  constexpr int C = D / 32;  // K chunks per key and lane
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int j = 0; j < C; ++j)
      cp_async16(ring + (half * C + j) * 512, keys + at + (g + 8 * half) * D + (4 * j + t) * 8);
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
      cp_async16(ring + (2 * C + k * (D / 64) + c) * 512,
                 values + at + (2 * t + (k & 1) + 8 * (k >> 1)) * D + (g + 8 * c) * 8);
}

// One step from this lane's FIFO slot: 16 keys, of which the first `valid` count.
template <int D>
Q3T_DEV void attend_step(Run<D>& run, uint32_t ring, const uint4 (&q)[D / 32], int valid, float scale_log2, int g, int t) {
  constexpr int C = D / 32;
  // ---- S^T = K Q^T; even and odd steps accumulate apart: two chains
  float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
  for (int j = 0; j < C; ++j) {
    const uint4 lo = lds16(ring + j * 512), hi = lds16(ring + (C + j) * 512);
    mma(s[0], lo.x, hi.x, lo.y, hi.y, q[j].x, q[j].y);
    mma(s[1], lo.z, hi.z, lo.w, hi.w, q[j].z, q[j].w);
  }
  // p[e]: key g (e < 2) or g + 8, head 2t + (e & 1)
  float p[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) p[e] = (s[0][e] + s[1][e]) * scale_log2;
  const bool lo_ok = g < valid, hi_ok = g + 8 < valid;
  // ---- online softmax
  const bool past = (lo_ok && (!(p[0] <= run.m[0] + 8.f) || !(p[1] <= run.m[1] + 8.f))) ||
                    (hi_ok && (!(p[2] <= run.m[0] + 8.f) || !(p[3] <= run.m[1] + 8.f)));
  if (__any_sync(0xffffffffu, past)) {
    float f[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float top = fmaxf(lo_ok ? p[e] : -INFINITY, hi_ok ? p[e + 2] : -INFINITY);
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      const float m = fmaxf(run.m[e], top);
      f[e] = run.m[e] == m ? 1.f : exp2f(run.m[e] - m);
      run.m[e] = m;
      run.l[e] *= f[e];
    }
#pragma unroll
    for (int j = 0; j < Run<D>::kTiles; ++j) {
      run.o[j][0] *= f[0], run.o[j][1] *= f[1];
      run.o[j][2] *= f[0], run.o[j][3] *= f[1];
    }
  }
  // while every score so far is -inf, so is m: the weights are 0, not the NaN of -inf - -inf
  const float ref[2] = {run.m[0] == -INFINITY ? 0.f : run.m[0], run.m[1] == -INFINITY ? 0.f : run.m[1]};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    p[e] = (e < 2 ? lo_ok : hi_ok) ? exp2f(p[e] - ref[e & 1]) : 0.f;
    run.l[e & 1] += p[e];
  }
  // P^T as the B operand; its rounding to bf16 (2^-9 relative per weight) is that of a bf16 tensor product
  const uint32_t b0 = transpose8(pack2(p[0], p[1])), b1 = transpose8(pack2(p[2], p[3]));
  // ---- O^T += V^T P^T
  uint4 v[4][D / 64];
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      v[k][c] = lds16(ring + (2 * C + k * (D / 64) + c) * 512);
      // rows past the last key may hold anything, NaN too, and 0 * NaN is NaN
      if (valid < kStepKeys && 2 * t + (k & 1) + 8 * (k >> 1) >= valid) v[k][c] = make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
  for (int j = 0; j < D / 16; ++j) {
    // D = 128: dims 8g + j and 64 + 8g + j; D = 64: dims 8g + 2j and 8g + 2j + 1
    const int i0 = D == 128 ? j : 2 * j, i1 = D == 128 ? j : 2 * j + 1, c1 = D / 64 - 1;
    const uint32_t s0 = i0 & 1 ? 0x7632u : 0x5410u, s1 = i1 & 1 ? 0x7632u : 0x5410u;
    mma(run.o[j], __byte_perm(word(v[0][0], i0 / 2), word(v[1][0], i0 / 2), s0),
        __byte_perm(word(v[0][c1], i1 / 2), word(v[1][c1], i1 / 2), s1),
        __byte_perm(word(v[2][0], i0 / 2), word(v[3][0], i0 / 2), s0),
        __byte_perm(word(v[2][c1], i1 / 2), word(v[3][c1], i1 / 2), s1), b0, b1);
  }
}

// The query heads of a pass as the B fragments of S^T (zero columns past `heads`).
template <int D>
Q3T_DEV void load_query(uint4 (&q)[D / 32], const __nv_bfloat16* query, int heads, int g, int t) {
#pragma unroll
  for (int j = 0; j < D / 32; ++j)
    q[j] = g < heads ? *reinterpret_cast<const uint4*>(query + g * D + (4 * j + t) * 8) : make_uint4(0u, 0u, 0u, 0u);
}

// Dim of element e (0 .. 2 * D/16) of the lane's outputs of one head: o[e / 2][2 * (e & 1)].
// A run at rest in shared memory: [head][m, l, o of every dim].
template <int D>
Q3T_DEV void rest(const Run<D>& run, float* part, int heads, int g, int t) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int head = 2 * t + e;
    if (head >= heads) continue;
    float* to = part + head * (D + 2);
    if (g == 0) to[0] = run.m[e], to[1] = run.l[e];
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      to[2 + (D == 128 ? 8 * g + j : 8 * g + 2 * j)] = run.o[j][e];
      to[2 + (D == 128 ? 64 + 8 * g + j : 8 * g + 2 * j + 1)] = run.o[j][2 + e];
    }
  }
}

// One CTA per (row, key/value head, pass): its warps share the row's steps in contiguous runs and merge
// through shared memory. PROMPT: row r is a packed prompt row, whose sequence and position follow from
// row_offsets and start_positions.
struct PromptRows {
  const int64_t *row_offsets, *start_positions;
  int sequences;
};

template <int D, int W, int ST, bool PROMPT>
__global__ void __launch_bounds__(W * 32, 1) paged_attention_direct(const DecodeArgs a, const PromptRows pr) {
  using C = Cfg<D, W, ST>;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  grid_dependency_wait();
  const int units = a.kv_heads * a.passes;
  const int row = int(blockIdx.x / units), unit = int(blockIdx.x % units);
  const int head = unit / a.passes, pass = unit % a.passes;
  int64_t sequence = row, position;
  if constexpr (PROMPT) {
    int lo = 0, hi = pr.sequences;  // the last sequence that starts at or before the row
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pr.row_offsets[mid] <= row) lo = mid;
      else hi = mid;
    }
    if (row < pr.row_offsets[lo] || row >= pr.row_offsets[lo + 1]) return;  // a row of no sequence
    sequence = lo;
    position = pr.start_positions[lo] + (row - pr.row_offsets[lo]);
    if (position < 0) position = -1;
  } else {
    position = a.positions[row];
  }
  if (position < -1 || position >= a.context) {
    if (unit == 0 && threadIdx.x == 0) raise_status(a.status, kStatusBadIndex);
    position = position < -1 ? -1 : a.context - 1;
  }
  const int heads = min(kHeads, a.group - pass * kHeads);
  const int head0 = head * a.group + pass * kHeads;
  __nv_bfloat16* out = a.out + (int64_t(row) * a.q_heads + head0) * D;
  const int64_t steps = steps_of(position);
  if (steps == 0) {  // nothing to see: zeros
    for (int e = threadIdx.x; e < heads * D / 8; e += W * 32) reinterpret_cast<uint4*>(out)[e] = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  const int64_t first = split_begin(warp, steps, W), last = split_begin(warp + 1, steps, W);
  uint4 q[D / 32];
  load_query<D>(q, a.query + row * a.query_stride + int64_t(head0) * D, heads, g, t);
  Run<D> run;
  run.reset();
  const uint32_t ring = smem_u32(smem + warp * C::kRing) + lane * 16;
  float* parts = reinterpret_cast<float*>(smem + W * C::kRing);

  // element offset of step s, looked up 32 steps at a time, one per lane
  int64_t ahead = 0;
  auto look = [&](int64_t s) {
    int64_t at = 0;
    if (s + lane < last) {
      const int64_t p0 = (s + lane) * kStepKeys;
      int64_t page = a.pages.lookup(sequence, p0);
      if (page < 0) {
        raise_status(a.status, kStatusBadIndex);
        page = 0;
      }
      at = page * a.page_stride + (int64_t(head) * a.pages.page_size + p0 % a.pages.page_size) * D;
    }
    return at;
  };
  auto issue = [&](int64_t s) {
    if (s < last) {
      const int i = int(s - first) & 31;
      if (i == 0) ahead = look(s);
      const int64_t at = __shfl_sync(0xffffffffu, ahead, i);
      copy_step<D>(ring + uint32_t((s - first) % ST) * C::kStepBytes, a.keys, a.values, at, g, t);
    }
    cp_async_commit();
  };
  for (int i = 0; i < ST; ++i) issue(first + i);
  for (int64_t s = first; s < last; ++s) {
    cp_async_wait<ST - 1>();
    const int64_t left = position + 1 - s * kStepKeys;
    attend_step<D>(run, ring + uint32_t((s - first) % ST) * C::kStepBytes, q, left < kStepKeys ? int(left) : kStepKeys,
                   a.scale_log2, g, t);
    issue(s + ST);
  }
  run.finish();
  rest<D>(run, parts + warp * C::kPart, heads, g, t);
  __syncthreads();
  for (int e = threadIdx.x; e < heads * D / 2; e += W * 32) {
    const int i = e / (D / 2), d = e % (D / 2) * 2;
    const float* p = parts + i * (D + 2);
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, p[w * C::kPart]);
    float l = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float* x = p + w * C::kPart;
      const float f = exp2f(x[0] - top);  // a warp without steps rests at m = -inf, l = 0, o = 0
      l += x[1] * f;
      o0 += x[2 + d] * f;
      o1 += x[3 + d] * f;
    }
    *reinterpret_cast<uint32_t*>(out + i * D + d) = pack2(o0 / l, o1 / l);
  }
}

template <int D, int W, int ST, bool PROMPT>
int launch_direct(const DecodeArgs& a, const PromptRows& pr, void* stream, const char* name) {
  using C = Cfg<D, W, ST>;
  static PerDevice once;
  if (const int rc = smem_limit(once, paged_attention_direct<D, W, ST, PROMPT>, C::kSmem, name)) return rc;
  return launch(paged_attention_direct<D, W, ST, PROMPT>, dim3(unsigned(int64_t(a.rows) * a.kv_heads * a.passes)),
                dim3(W * 32), size_t(C::kSmem), stream, true, name, a, pr);
}

int fill(DecodeArgs& a, const char* name, const q3t_paged_cache& c, const void* query, int64_t query_stride,
         int64_t rows, int64_t q_heads, void* out, double scale, unsigned* status) {
  if (!query || !out) return fail(Q3T_EINVAL, "%s: null pointer", name);
  if (const int rc = check_cache(name, c)) return rc;
  if (rows < 1 || rows > (int64_t(1) << 30) || q_heads < 1 || q_heads > 1024 || q_heads % c.kv_heads)
    return fail(Q3T_EINVAL, "%s: invalid geometry", name);
  if (query_stride < q_heads * c.head_dim || query_stride % 8) return fail(Q3T_EINVAL, "%s: query stride", name);
  if (!aligned16(query) || !aligned16(out)) return fail(Q3T_EINVAL, "%s: 16-byte alignment", name);
  a.query = static_cast<const __nv_bfloat16*>(query);
  a.keys = static_cast<const __nv_bfloat16*>(c.key_pages);
  a.values = static_cast<const __nv_bfloat16*>(c.value_pages);
  a.query_stride = query_stride;
  a.page_stride = c.page_stride;
  a.pages = PageTable{c.page_table, c.table_stride, c.table_rows, c.table_columns, c.pages, int(c.page_size)};
  a.positions = nullptr;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.rows = int(rows);
  a.q_heads = int(q_heads);
  a.kv_heads = int(c.kv_heads);
  a.group = int(q_heads / c.kv_heads);
  a.passes = (a.group + kHeads - 1) / kHeads;
  a.context = c.table_columns * c.page_size;
  a.scale_log2 = float(scale) * kLog2e;
  a.status = status;
  if (rows * c.kv_heads * a.passes > (int64_t(1) << 31) - 1) return fail(Q3T_EINVAL, "%s: too many rows", name);
  return Q3T_OK;
}

}  // namespace

extern "C" size_t q3t_paged_decode_attention_workspace_bytes(int64_t rows, int64_t q_heads, int64_t kv_heads,
                                                             int64_t head_dim, int64_t context) {
  (void)rows, (void)q_heads, (void)kv_heads, (void)head_dim, (void)context;
  return 0;
}

extern "C" int q3t_paged_decode_attention(const q3t_paged_decode* call, unsigned* status, void* stream) {
  const char* name = "paged_decode_attention";
  if (call == nullptr) return fail(Q3T_EINVAL, "%s: null pointer", name);
  const q3t_paged_decode& p = *call;
  DecodeArgs a;
  if (const int rc = fill(a, name, p.cache, p.query, p.query_stride, p.rows, p.q_heads, p.out, p.scale, status)) return rc;
  if (!p.positions) return fail(Q3T_EINVAL, "%s: null pointer", name);
  if (p.cache.table_rows < p.rows) return fail(Q3T_EINVAL, "%s: the page table needs a row per query row", name);
  if (p.context < 1 || p.context > a.context) return fail(Q3T_EINVAL, "%s: context beyond the page table", name);
  const DeviceGuard guard(p.cache.device);
  if (!guard.ok()) return fail(Q3T_ECUDA, "%s: no such device", name);
  a.positions = p.positions;
  a.context = p.context;
  const PromptRows none = {};
  return p.cache.head_dim == 128 ? launch_direct<128, 8, 3, false>(a, none, stream, name)
                                 : launch_direct<64, 8, 6, false>(a, none, stream, name);
}

extern "C" size_t q3t_paged_prefill_attention_workspace_bytes(int64_t rows, int64_t sequences, int64_t q_heads,
                                                              int64_t kv_heads, int64_t head_dim, int64_t context) {
  (void)rows, (void)sequences, (void)q_heads, (void)kv_heads, (void)head_dim, (void)context;
  return 0;
}

extern "C" int q3t_paged_prefill_attention(const q3t_paged_prefill* call, unsigned* status, void* stream) {
  const char* name = "paged_prefill_attention";
  if (call == nullptr) return fail(Q3T_EINVAL, "%s: null pointer", name);
  const q3t_paged_prefill& p = *call;
  DecodeArgs a;
  if (const int rc = fill(a, name, p.cache, p.query, p.query_stride, p.rows, p.q_heads, p.out, p.scale, status)) return rc;
  if (!p.row_offsets || !p.start_positions) return fail(Q3T_EINVAL, "%s: null pointer", name);
  if (p.sequences < 1 || p.sequences > (int64_t(1) << 20) || p.cache.table_rows < p.sequences)
    return fail(Q3T_EINVAL, "%s: invalid geometry", name);
  const DeviceGuard guard(p.cache.device);
  if (!guard.ok()) return fail(Q3T_ECUDA, "%s: no such device", name);
  const PromptRows pr = {p.row_offsets, p.start_positions, int(p.sequences)};
  return p.cache.head_dim == 128 ? launch_direct<128, 8, 3, true>(a, pr, stream, name)
                                 : launch_direct<64, 8, 6, true>(a, pr, stream, name);
}
