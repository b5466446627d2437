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
// A step's keys of one head are 16 adjacent rows of a page, and so are its values: each cp.async instruction
// of a warp copies 512 adjacent bytes. (Copying instead what each lane will read back itself, 64-byte
// pieces of 8 rows, needs neither swizzle nor warp barrier, but ran at 5.0 TB/s instead of 6.7: the memory
// system takes one request per 128-byte line an instruction touches.) The 16-byte chunks of a row are
// permuted on their way so that no read has a bank conflict. With g = lane / 4, t = lane % 4 a lane reads
//   K: keys g and g + 8 at dim chunks t, t + 4, ... (8 dims each); chunk c of key k is at c ^ 4 (k % 2).
//      Q is loaded with the same permutation of dims, so the dot product needs no reordering;
//   V: keys 2t, 2t+1, 2t+8, 2t+9 at dim chunk g (and g + 8); chunk c of key k is at c ^ 2 (k / 2 % 4). Two
//      keys' chunks become the A fragment of O^T by byte permutes; row g of tile j is dim 8g + j, so a lane
//      ends with 8 adjacent output dims.
#include "common.cuh"
#include "host.cuh"
#include "paged.cuh"
#include "paged_prefill.cuh"

using namespace q3t;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRanks = 8;  // CTAs that share a row's keys, at most: the portable cluster size
constexpr int kHeads = 8;  // query heads of a pass (columns of the products)

struct DecodeArgs {
  const __nv_bfloat16 *query, *keys, *values;
  int64_t query_stride, page_stride;
  PageTable pages;
  const int64_t* positions;
  __nv_bfloat16* out;
  int rows, q_heads, kv_heads, group, passes;
  int ranks;  // CTAs of a cluster, which share an item's keys
  int64_t context;
  float scale_log2;
  unsigned* status;
};

Q3T_DEV void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
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
// 2^x, 2 ulp; results below 2^-126 are 0, which a weight may be.
Q3T_DEV float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
Q3T_DEV void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// Two floats at this CTA's shared address `addr`, from the cluster's CTA `rank`.
Q3T_DEV float2 ld_cluster2(uint32_t addr, int rank) {
  float2 v;
  asm volatile(
      "{\n\t.reg .b32 a;\n\t"
      "mapa.shared::cluster.u32 a, %2, %3;\n\t"
      "ld.shared::cluster.v2.f32 {%0, %1}, [a];\n\t}\n"
      : "=f"(v.x), "=f"(v.y)
      : "r"(addr), "r"(rank)
      : "memory");
  return v;
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
  static constexpr int kStepBytes = kStepKeys * 2 * D * 2;       // 16 keys: K and V
  static constexpr int kRing = ST * kStepBytes;                  // a warp's FIFO
  static constexpr int kPart = kHeads * (D + 2);                 // floats of a run at rest: m, l and o per head
  static constexpr int kSmem = W * kRing + kPart * 4;
};

// The places of a lane in a FIFO slot (bytes from its start; K at 0, V at D * 32).
template <int D>
struct Places {
  uint32_t put_k, put_v[D == 128 ? 4 : 2];  // unit 0 of the copies; V's permutation takes turns
  uint32_t get_k[2], get_v;                        // chunks 0 and 1 of key g; chunk g of key 2t

  Q3T_DEV explicit Places(int lane) {
    constexpr int R = D / 8;  // chunks (and lanes) of a row
    const int g = lane >> 2, t = lane & 3, key = lane / R, chunk = lane % R;
    put_k = key * 2 * D + ((chunk ^ (4 * (key & 1))) << 4);
    constexpr int V = D == 128 ? 4 : 2;
#pragma unroll
    for (int u = 0; u < V; ++u) put_v[u] = D * 32 + key * 2 * D + ((chunk ^ (2 * (((u * 32 / R + key) >> 1) & 3))) << 4);
    get_k[0] = g * 2 * D + t * 16 + 64 * (g & 1);
    get_k[1] = g * 2 * D + t * 16 + 64 * (1 - (g & 1));
    get_v = D * 32 + 2 * t * 2 * D + ((g ^ (2 * t)) << 4);
  }
};

// Copies one step, from the element offset of its first key; `lane8`: 8 * lane.
template <int D>
Q3T_DEV void copy_step(uint32_t slot, const __nv_bfloat16* keys, const __nv_bfloat16* values, int64_t at, const Places<D>& at_lane,
                       int lane8) {
  constexpr int V = D == 128 ? 4 : 2;
#pragma unroll
  for (int u = 0; u < D / 16; ++u) cp_async16(slot + at_lane.put_k + u * 512, keys + at + u * 256 + lane8);
#pragma unroll
  for (int u = 0; u < D / 16; ++u) cp_async16(slot + at_lane.put_v[u % V] + u * 512, values + at + u * 256 + lane8);
}

// One step from its FIFO slot: 16 keys, of which the first `valid` count; `masked`: this lane's columns see only the first
// sees.x and sees.y of them.
template <int D>
Q3T_DEV void attend_step(Run<D>& run, uint32_t slot, const Places<D>& at_lane, const uint4 (&q)[D / 32], int valid,
                         bool masked, int2 sees, float scale_log2, int g, int t) {
  constexpr int C = D / 32;
  // ---- S^T = K Q^T; even and odd steps accumulate apart: two chains
  float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  uint4 v[4][D / 64];
#pragma unroll
  for (int j = 0; j < C; ++j) {
    const uint32_t at = slot + at_lane.get_k[j & 1] + (j >> 1) * 128;
    const uint4 lo = lds16(at), hi = lds16(at + 16 * D);
    mma(s[0], lo.x, hi.x, lo.y, hi.y, q[j].x, q[j].y);
    mma(s[1], lo.z, hi.z, lo.w, hi.w, q[j].z, q[j].w);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int c = 0; c < D / 64; ++c) v[k][c] = lds16(slot + at_lane.get_v + (k & 1) * 2 * D + (k >> 1) * 16 * D + c * 128);
  // p[e]: key g (e < 2) or g + 8, head 2t + (e & 1)
  float p[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) p[e] = (s[0][e] + s[1][e]) * scale_log2;
  if (masked) {
    if (g >= sees.x) p[0] = -INFINITY;
    if (g >= sees.y) p[1] = -INFINITY;
    if (g + 8 >= sees.x) p[2] = -INFINITY;
    if (g + 8 >= sees.y) p[3] = -INFINITY;
    // rows past the last key may hold anything, NaN too, and 0 * NaN is NaN
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
        if (2 * t + (k & 1) + 8 * (k >> 1) >= valid) v[k][c] = make_uint4(0u, 0u, 0u, 0u);
  }
  // ---- online softmax
  const bool past = !(fmaxf(p[0], p[2]) <= run.m[0] + 8.f) || !(fmaxf(p[1], p[3]) <= run.m[1] + 8.f);
  if (__any_sync(0xffffffffu, past)) {
    float f[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float top = fmaxf(p[e], p[e + 2]);
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      const float m = fmaxf(run.m[e], top);
      f[e] = run.m[e] == m ? 1.f : exp2_fast(run.m[e] - m);
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
    p[e] = exp2_fast(p[e] - ref[e & 1]);
    run.l[e & 1] += p[e];
  }
  // P^T as the B operand; its rounding to bf16 (2^-8 relative per weight) is that of a bf16 tensor product
  const uint32_t b0 = transpose8(pack2(p[0], p[1])), b1 = transpose8(pack2(p[2], p[3]));
  // ---- O^T += V^T P^T
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

// One CTA per (row, key/value head, pass), or a cluster of `ranks`: the warps share the row's steps in contiguous runs,
// merge through shared memory, and a cluster's CTAs through distributed shared memory. 256 rows of 1..4096 keys, 16 query
// and 8 KV heads of 128 dims: 313 us for 2.17 GB, 6.9 TB/s (a plain read of memory reaches 7.1).
// PROMPT: the item's rows are up to `pack` consecutive packed rows of one sequence, whose heads fill the eight columns (4
// rows of two heads): the form of the prompt attention for few rows and for what its tiled kernel does not take
// (prompt_plan).
struct PromptRows {
  const int64_t *row_offsets, *start_positions;
  int sequences;
  int pack;    // rows of an item at most
  int inverse; // (i * inverse) >> 8 is column i's row in its pack (i < 8): 256 / group rounded up, 0 for packs of one row
  int packs;   // items of a (KV head, pass) at most
  bool look;   // few enough sequences to look at all of them at once
};
constexpr int kLookRounds = 4;  // of 32 sequences

// Sequence, first row, row count and first position of number `index`, for a whole warp; false: there is none. Offsets
// that make no sense are flagged by the first CTA and own nothing. Up to 128 sequences take one round of loads where a
// search takes one for each halving.
Q3T_DEV bool locate(const PromptRows& pr, int rows, int index, bool first, unsigned* status, int64_t& sequence, int& row,
                    int& count, int64_t& position) {
  const int lane = threadIdx.x & 31;
  sequence = -1;
  if (pr.look) {
    int64_t lo[kLookRounds], hi[kLookRounds], start[kLookRounds];
#pragma unroll
    for (int i = 0; i < kLookRounds; ++i) {
      const int s = 32 * i + lane;
      lo[i] = hi[i] = start[i] = 0;
      if (s < pr.sequences) lo[i] = pr.row_offsets[s], hi[i] = pr.row_offsets[s + 1], start[i] = pr.start_positions[s];
    }
    int before = 0;
#pragma unroll
    for (int i = 0; i < kLookRounds; ++i) {
      if (32 * i >= pr.sequences) continue;
      const bool sound = lo[i] >= 0 && lo[i] <= hi[i] && hi[i] <= rows;
      if (first && !sound) raise_status(status, kStatusBadIndex);
      const int items = sound ? (int(hi[i] - lo[i]) + pr.pack - 1) / pr.pack : 0;
      int sum = items;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += other;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + sum > index);
      if (hit != 0 && sequence < 0) {
        const int src = __ffs(hit) - 1, skip = (index - before - (sum - items)) * pr.pack;
        sequence = 32 * i + src;
        row = __shfl_sync(0xffffffffu, int(lo[i]) + skip, src);
        count = __shfl_sync(0xffffffffu, min(pr.pack, int(hi[i] - lo[i]) - skip), src);
        position = __shfl_sync(0xffffffffu, clamped_start(start[i]) + skip, src);
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
  } else {
    int lo = 0, hi = pr.sequences;  // the last sequence that starts at or before the row
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pr.row_offsets[mid] <= index) lo = mid;
      else hi = mid;
    }
    const int64_t begin = pr.row_offsets[lo], end = pr.row_offsets[lo + 1];
    if (begin >= 0 && begin <= index && index < end && end <= rows) {
      sequence = lo;
      row = index;
      count = 1;
      position = clamped_start(pr.start_positions[lo]) + (index - begin);
    }
    for (int s = threadIdx.x; first && s < pr.sequences; s += blockDim.x)
      if (pr.row_offsets[s] < 0 || pr.row_offsets[s] > pr.row_offsets[s + 1] || pr.row_offsets[s + 1] > rows)
        raise_status(status, kStatusBadIndex);
  }
  return sequence >= 0;
}

template <int D, int W, int ST, bool PROMPT>
__global__ void __launch_bounds__(W * 32, W == 4 ? 3 : 1) paged_attention_direct(const DecodeArgs a, const PromptRows pr) {
  using C = Cfg<D, W, ST>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  grid_dependency_wait();
  const int units = a.kv_heads * a.passes, ranks = a.ranks;
  const int item = int(blockIdx.x) / ranks, rank = int(blockIdx.x) % ranks;
  const int unit = item % units;
  const int head = unit / a.passes, pass = unit % a.passes;
  int row = item / units, count = 1;  // rows of the item
  int64_t sequence = row, position;   // position: of the first row, then of the last
  if constexpr (PROMPT) {
    if (!locate(pr, a.rows, row, blockIdx.x == 0, a.status, sequence, row, count, position)) return;  // as do all its CTAs
  } else {
    position = a.positions[row];
  }
  const int64_t position0 = position;
  position += count - 1;
  if (position >= a.context || (!PROMPT && position < -1)) {
    if (unit == 0 && threadIdx.x == 0) raise_status(a.status, kStatusBadIndex);
    position = position < -1 ? -1 : a.context - 1;
  }
  const int heads = min(kHeads, a.group - pass * kHeads), columns = PROMPT ? count * heads : heads;
  const int head0 = head * a.group + pass * kHeads;
  // column i: row (of the pack) and head; where its output begins
  auto row_of_column = [&](int i) { return PROMPT ? (i * pr.inverse) >> 8 : 0; };
  auto out_of = [&](int i) {
    const int r = row_of_column(i);
    return a.out + (int64_t(row + r) * a.q_heads + head0 + i - r * heads) * D;
  };
  const int64_t steps = steps_of(position);
  if (steps == 0) {  // nothing to see: zeros
    for (int e = rank * W * 32 + threadIdx.x; e < columns * D / 8; e += ranks * W * 32)
      reinterpret_cast<uint4*>(out_of(e / (D / 8)))[e % (D / 8)] = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  // the CTAs that share the row: no more than give every warp a step
  const int sharing = int(split_parts((steps + W - 1) / W, ranks));
  if (rank >= sharing && sharing == 1) return;
  const int64_t r0 = rank < sharing ? split_begin(rank, steps, sharing) : steps;
  const int64_t r1 = rank < sharing ? split_begin(rank + 1, steps, sharing) : steps;
  const int64_t first = r0 + split_begin(warp, r1 - r0, W), last = r0 + split_begin(warp + 1, r1 - r0, W);
  uint4 q[D / 32];
  const int row_g = row_of_column(g);
  load_query<D>(q, a.query + (row + row_g) * a.query_stride + int64_t(head0 - row_g * heads) * D, columns, g, t);
  // keys that columns 2t and 2t + 1 see of the item's last step (16 more of the one before)
  int2 sees = {kStepKeys, kStepKeys};
  if constexpr (PROMPT) {
    auto of = [&](int i) {
      const int64_t n = min(position0 + row_of_column(i), position) + 1 - (steps - 1) * kStepKeys;
      return int(max(n, int64_t(-2 * kStepKeys)));
    };
    sees = make_int2(of(2 * t), of(2 * t + 1));
  }
  Run<D> run;
  run.reset();
  const uint32_t ring = smem_u32(smem + warp * C::kRing);
  const Places<D> at_lane(lane);

  // element offset of step first + i, looked up 32 steps at a time, one per lane
  const int own = int(last - first);
  int64_t ahead = 0;
  auto look = [&](int i) {
    int64_t at = 0;
    if (i + lane < own) {
      const int64_t p0 = (first + i + lane) * kStepKeys;
      int row_there;
      int64_t page = a.pages.lookup(sequence, p0, row_there);
      if (page < 0) {
        raise_status(a.status, kStatusBadIndex);
        page = 0;
      }
      at = page * a.page_stride + (int64_t(head) * a.pages.page_size + row_there) * D;
    }
    return at;
  };
  auto issue = [&](int i, uint32_t slot) {
    if (i < own) {
      if ((i & 31) == 0) ahead = look(i);
      copy_step<D>(slot, a.keys, a.values, __shfl_sync(0xffffffffu, ahead, i & 31), at_lane, 8 * lane);
    }
    cp_async_commit();
  };
  for (int i = 0; i < ST; ++i) issue(i, ring + i * C::kStepBytes);
  const int tail = int(position % kStepKeys) + 1;
  uint32_t slot = ring;
  for (int i = 0; i < own; ++i) {
    cp_async_wait<ST - 1>();
    __syncwarp();  // the other lanes' copies too
    const int valid = first + i + 1 == steps ? tail : kStepKeys;
    if constexpr (PROMPT) {  // up to 8 consecutive positions: only the last two steps hold keys that some row does not see
      const bool near = first + i + 2 >= steps;
      const int more = first + i + 1 == steps ? 0 : kStepKeys;
      attend_step<D>(run, slot, at_lane, q, valid, near, make_int2(sees.x + more, sees.y + more), a.scale_log2, g, t);
    } else {
      attend_step<D>(run, slot, at_lane, q, valid, valid < kStepKeys, make_int2(valid, valid), a.scale_log2, g, t);
    }
    __syncwarp();  // every lane has read the slot
    issue(i + ST, slot);
    slot = slot + C::kStepBytes == ring + C::kRing ? ring : slot + C::kStepBytes;
  }
  run.finish();
  __syncwarp();
  rest<D>(run, reinterpret_cast<float*>(smem + warp * C::kRing), columns, g, t);  // the FIFO is drained
  __syncthreads();
  // a row before the first key is zero
  auto store = [&](int i, int d, float o0, float o1, float l) {
    const bool none = PROMPT && position0 + row_of_column(i) < 0;
    *reinterpret_cast<uint32_t*>(out_of(i) + d) = none ? 0u : pack2(o0 / l, o1 / l);
  };
  float* mine = reinterpret_cast<float*>(smem + W * C::kRing);
  for (int e = threadIdx.x; e < columns * D / 2; e += W * 32) {
    const int i = e / (D / 2), d = e % (D / 2) * 2;
    const float* p = reinterpret_cast<const float*>(smem) + i * (D + 2);
    constexpr int kNext = C::kRing / 4;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, p[w * kNext]);
    float l = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float* x = p + w * kNext;
      const float f = x[0] == top ? 1.f : exp2_fast(x[0] - top);  // a warp without steps rests at m = -inf, l = o = 0
      l += x[1] * f;
      o0 += x[2 + d] * f;
      o1 += x[3 + d] * f;
    }
    if (sharing == 1) {
      store(i, d, o0, o1, l);
    } else {
      float* to = mine + i * (D + 2);
      if (d == 0) to[0] = top, to[1] = l;
      to[2 + d] = o0;
      to[3 + d] = o1;
    }
  }
  if (sharing == 1) return;
  // ---- the cluster's CTAs join their runs through distributed shared memory, in the order of their keys
  cluster_sync();
  for (int e = rank * W * 32 + threadIdx.x; e < columns * D / 2; e += ranks * W * 32) {
    const int i = e / (D / 2), d = e % (D / 2) * 2;
    const uint32_t at = smem_u32(mine + i * (D + 2));
    float m[kRanks], sum[kRanks];
    float2 o[kRanks];
    float top = -INFINITY;
#pragma unroll
    for (int r = 0; r < kRanks; ++r) {
      m[r] = -INFINITY, sum[r] = 0.f, o[r] = make_float2(0.f, 0.f);
      if (r < sharing) {
        const float2 ml = ld_cluster2(at, r);
        m[r] = ml.x, sum[r] = ml.y;
        o[r] = ld_cluster2(at + 8 + 4 * d, r);
      }
      top = fmaxf(top, m[r]);
    }
    float l = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
    for (int r = 0; r < kRanks; ++r) {
      const float f = m[r] == top ? 1.f : exp2_fast(m[r] - top);
      l += sum[r] * f;
      o0 += o[r].x * f;
      o1 += o[r].y * f;
    }
    store(i, d, o0, o1, l);
  }
  cluster_sync();  // no CTA leaves while its shared memory is read
}

template <int D, int W, int ST, bool PROMPT>
int launch_direct(DecodeArgs& a, const PromptRows& pr, int ranks, void* stream, const char* name) {
  using C = Cfg<D, W, ST>;
  static PerDevice once;
  if (const int rc = smem_limit(once, paged_attention_direct<D, W, ST, PROMPT>, C::kSmem, name)) return rc;
  a.ranks = ranks;
  return launch_cluster(paged_attention_direct<D, W, ST, PROMPT>,
                        dim3(unsigned(int64_t(PROMPT ? pr.packs : a.rows) * a.kv_heads * a.passes * ranks)), dim3(W * 32), size_t(C::kSmem),
                        ranks, stream, name, a, pr);
}

// Many rows, or long ones: the steps of all rows and KV heads, end to end, are cut into one even range per CTA (one CTA
// per SM) and each range into one run per warp, wherever rows begin and end: no SM waits for a longer row, whatever
// the lengths are. A run that covers its item (row, KV head, pass) whole writes the output; the others rest in shared
// memory and are merged there; what two CTAs share goes through the workspace to a second, dependent launch.
// The order of every merge follows from the ranges alone, so results repeat bit for bit.
struct SplitArgs {
  int parts;      // CTAs = ranges
  int heads;      // query heads of a pass at most
  float* partial;   // workspace: [parts][2][heads][D + 2]: the item a range begins inside of (0) or ends inside of (1)
};

struct Resting {  // a run in shared memory
  int64_t begin, end;  // its item's steps
  int row, unit, valid;
};

constexpr int kSplitRows = 4096;  // prefix sums in shared memory

template <int D, int W, int ST>
__host__ __device__ constexpr int split_smem(int heads, int rows) {
  return W * (Cfg<D, W, ST>::kRing + heads * (D + 2) * 4 + 2 * int(sizeof(Resting))) + (rows + 1 + W) * 4;
}

template <int D>
Q3T_DEV void store_rows(const Run<D>& run, __nv_bfloat16* out, int heads, int g, int t) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int head = 2 * t + e;
    if (head >= heads) continue;
    const float inv = 1.f / run.l[e];
    float f[8], h[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      f[j] = (D == 128 ? run.o[j % (D / 16)][e] : run.o[j / 2][e + 2 * (j & 1)]) * inv;
      h[j] = run.o[j % (D / 16)][e + 2] * inv;
    }
    *reinterpret_cast<uint4*>(out + head * D + 8 * g) = pack8(f);
    if (D == 128) *reinterpret_cast<uint4*>(out + head * D + 64 + 8 * g) = pack8(h);
  }
}

template <int D, int W, int ST>
__global__ void __launch_bounds__(W * 32, 1) paged_decode_split(const DecodeArgs a, const SplitArgs sp) {
  using C = Cfg<D, W, ST>;
  constexpr int kThreads = W * 32;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int part = sp.heads * (D + 2);
  float* parts = reinterpret_cast<float*>(smem + W * C::kRing);
  // where a warp's runs rest: the first (0) apart from its FIFO, which still fills; the last (1) in the FIFO
  auto rests = [&](int k) { return k & 1 ? reinterpret_cast<float*>(smem + (k >> 1) * C::kRing) : parts + (k >> 1) * part; };
  Resting* resting = reinterpret_cast<Resting*>(parts + W * part);
  int32_t* prefix = reinterpret_cast<int32_t*>(resting + 2 * W);
  int32_t* warp_sums = prefix + a.rows + 1;
  grid_dependency_wait();

  // ---- steps before every row; rows with no key get their zeros here
  int32_t carry = 0;
  for (int r0 = 0; r0 < a.rows; r0 += kThreads) {
    const int r = r0 + int(threadIdx.x);
    int32_t steps = 0;
    if (r < a.rows) {
      int64_t position = a.positions[r];
      if (position < -1 || position >= a.context) {
        if (blockIdx.x == 0) raise_status(a.status, kStatusBadIndex);
        position = position < -1 ? -1 : a.context - 1;
      }
      steps = int32_t(steps_of(position));
    }
    int32_t sum = steps;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t other = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += other;
    }
    if (lane == 31) warp_sums[warp] = sum;
    __syncthreads();
    int32_t before = carry, all = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int32_t v = warp_sums[w];
      if (w < warp) before += v;
      all += v;
    }
    if (r < a.rows) prefix[r] = before + sum - steps;
    carry += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) prefix[a.rows] = carry;
  if (threadIdx.x < 2 * W) resting[threadIdx.x].valid = 0;
  __syncthreads();
  for (int r = blockIdx.x; r < a.rows; r += sp.parts)
    if (prefix[r] == prefix[r + 1])
      for (int e = threadIdx.x; e < a.q_heads * D / 8; e += kThreads)
        reinterpret_cast<uint4*>(a.out + int64_t(r) * a.q_heads * D)[e] = make_uint4(0u, 0u, 0u, 0u);
  const int units = a.kv_heads * a.passes;
  const int64_t total = int64_t(carry) * units;
  const int64_t ranges = split_parts(total, sp.parts);
  if (int64_t(blockIdx.x) >= ranges) return;
  const int64_t c0 = split_begin(blockIdx.x, total, ranges), c1 = split_begin(blockIdx.x + 1, total, ranges);
  const int64_t f0 = c0 + split_begin(warp, c1 - c0, W), f1 = c0 + split_begin(warp + 1, c1 - c0, W);

  // ---- the issuing side: pages are looked up 32 steps at a time, one per lane, a window ahead of their use
  struct Window {
    int32_t page;
    int64_t inner;
  };
  auto look = [&](int64_t f) {
    Window w = {0, 0};
    f += lane;
    if (f < f1) {
      const int r = row_of(prefix, a.rows, f, units);
      const int32_t n = prefix[r + 1] - prefix[r];
      const int32_t in_row = int32_t(f - int64_t(prefix[r]) * units);
      const int32_t unit = in_row / n, p0 = (in_row - unit * n) * kStepKeys, column = p0 / a.pages.page_size;
      w.page = a.pages.table[r * a.pages.stride + column];
      w.inner = (int64_t(unit / a.passes) * a.pages.page_size + (p0 - column * a.pages.page_size)) * D;
    }
    return w;
  };
  const uint32_t ring = smem_u32(smem + warp * C::kRing);
  const Places<D> at_lane(lane);
  const int count = int(f1 - f0);
  Window next = look(f0);
  int64_t ahead = 0;
  auto issue = [&](int i, uint32_t slot) {
    if (i < count) {
      if ((i & 31) == 0) {
        int64_t page = next.page;
        if (page < 0 || page >= a.pages.pages) {
          raise_status(a.status, kStatusBadIndex);
          page = 0;
        }
        ahead = page * a.page_stride + next.inner;
        next = look(f0 + i + 32);
      }
      copy_step<D>(slot, a.keys, a.values, __shfl_sync(0xffffffffu, ahead, i & 31), at_lane, 8 * lane);
    }
    cp_async_commit();
  };
  for (int i = 0; i < ST; ++i) issue(i, ring + i * C::kStepBytes);

  // ---- the computing side
  uint4 q[D / 32];
  Run<D> run;
  int row = 0, unit = 0, heads = 0, tail = 0;
  int64_t begin = 0, end = f0;
  int from = 0, until = 0;  // this warp's steps of the item, as indexes of its own
  uint32_t slot = ring;
  for (int i = 0; i < count; ++i) {
    if (i == until) {  // a new item
      row = row_of(prefix, a.rows, end, units);
      const int64_t base = int64_t(prefix[row]) * units;
      const int32_t n = prefix[row + 1] - prefix[row];
      unit = int32_t(end - base) / n;
      begin = base + int64_t(unit) * n;
      end = begin + n;
      from = i;
      until = end < f1 ? int(end - f0) : count;
      tail = int(min(a.positions[row], a.context - 1) % kStepKeys) + 1;
      const int pass = unit % a.passes;
      heads = min(kHeads, a.group - pass * kHeads);
      load_query<D>(q, a.query + row * a.query_stride + int64_t(unit / a.passes * a.group + pass * kHeads) * D, heads, g, t);
      run.reset();
    }
    cp_async_wait<ST - 1>();
    __syncwarp();  // the other lanes' copies too
    const int valid = f0 + i + 1 == end ? tail : kStepKeys;
    attend_step<D>(run, slot, at_lane, q, valid, valid < kStepKeys, make_int2(valid, valid), a.scale_log2, g, t);
    __syncwarp();  // every lane has read the slot
    issue(i + ST, slot);
    slot = slot + C::kStepBytes == ring + C::kRing ? ring : slot + C::kStepBytes;
    if (i + 1 == until) {
      run.finish();
      if (f0 + from == begin && f0 + until == end) {
        const int head0 = unit / a.passes * a.group + unit % a.passes * kHeads;
        store_rows<D>(run, a.out + (int64_t(row) * a.q_heads + head0) * D, heads, g, t);
      } else {
        const int at = 2 * warp + (from > 0);
        __syncwarp();
        rest<D>(run, rests(at), heads, g, t);
        if (lane == 0) resting[at] = {begin, end, row, unit, 1};
      }
    }
  }
  __syncthreads();

  // ---- merge what rests: runs of one item are neighbours
  for (int k = 0; k < 2 * W;) {
    if (!resting[k].valid) {
      ++k;
      continue;
    }
    const Resting it = resting[k];
    int last = k + 1;
    while (last < 2 * W && (!resting[last].valid || resting[last].begin == it.begin)) ++last;
    const int pass = it.unit % a.passes, n = min(kHeads, a.group - pass * kHeads);
    const bool whole = it.begin >= c0 && it.end <= c1;
    float* to = sp.partial + (int64_t(blockIdx.x) * 2 + (it.begin > c0)) * part;
    __nv_bfloat16* out = a.out + (int64_t(it.row) * a.q_heads + it.unit / a.passes * a.group + pass * kHeads) * D;
    for (int e = threadIdx.x; e < n * D / 2; e += kThreads) {
      const int i = e / (D / 2), d = e % (D / 2) * 2;
      float top = -INFINITY;
      for (int s = k; s < last; ++s)
        if (resting[s].valid) top = fmaxf(top, rests(s)[i * (D + 2)]);
      float l = 0.f, o0 = 0.f, o1 = 0.f;
      for (int s = k; s < last; ++s) {
        if (!resting[s].valid) continue;
        const float* x = rests(s) + i * (D + 2);
        const float f = x[0] == top ? 1.f : exp2f(x[0] - top);
        l += x[1] * f;
        o0 += x[2 + d] * f;
        o1 += x[3 + d] * f;
      }
      if (whole) {
        *reinterpret_cast<uint32_t*>(out + i * D + d) = pack2(o0 / l, o1 / l);
      } else {
        if (d == 0) to[i * (D + 2)] = top, to[i * (D + 2) + 1] = l;
        to[i * (D + 2) + 2 + d] = o0;
        to[i * (D + 2) + 3 + d] = o1;
      }
    }
    k = last;
  }
}

// The items that several ranges share: one CTA joins their partial runs in the order of the ranges. It finds them from
// the positions alone, before it waits for the launch that it depends on (that one has waited for everything before it),
// and up to kAtOnce parts are read in one round of loads (3 rows of 20000..65535 keys: 84.3 -> 79.7 us in all). No CTA
// leaves before the wait: what follows this launch may rely on its end for the end of both.
constexpr int kJoinThreads = 256, kAtOnce = 8;

template <int D>
__global__ void __launch_bounds__(kJoinThreads) paged_decode_join(const DecodeArgs a, const SplitArgs sp) {
  extern __shared__ float weight[];  // [heads][parts], then [heads] sums
  __shared__ int sums[2][kJoinThreads / 32];
  const int units = a.kv_heads * a.passes, row = int(blockIdx.x / units), unit = int(blockIdx.x % units);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto steps = [&](int r) { return int(steps_of(min(a.positions[r], a.context - 1))); };
  int before = 0, all = 0;
  for (int r = threadIdx.x; r < a.rows; r += kJoinThreads) {
    const int n = steps(r);
    all += n;
    before += r < row ? n : 0;
  }
  const int n = steps(row);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  if (lane == 0) sums[0][warp] = all, sums[1][warp] = before;
  __syncthreads();
  all = before = 0;
#pragma unroll
  for (int w = 0; w < kJoinThreads / 32; ++w) all += sums[0][w], before += sums[1][w];
  if (n == 0) {
    grid_dependency_wait();
    return;
  }
  const int64_t total = int64_t(all) * units, begin = int64_t(before) * units + int64_t(unit) * n;
  const int64_t ranges = split_parts(total, sp.parts);
  const int first = int(split_owner(begin, total, ranges)), last = int(split_owner(begin + n - 1, total, ranges));
  if (first == last) {
    grid_dependency_wait();
    return;
  }
  const int pass = unit % a.passes, heads = min(kHeads, a.group - pass * kHeads), part = sp.heads * (D + 2);
  // ranges after the first begin inside the item
  const int slot = begin > split_begin(first, total, ranges);
  auto at = [&](int i) { return sp.partial + (int64_t(first + i) * 2 + (i == 0 ? slot : 0)) * part; };
  const int count = last - first + 1, head0 = unit / a.passes * a.group + pass * kHeads;
  __nv_bfloat16* out = a.out + (int64_t(row) * a.q_heads + head0) * D;
  grid_dependency_wait();
  if (count <= kAtOnce) {
    for (int e = threadIdx.x; e < heads * D / 2; e += kJoinThreads) {
      const int h = e / (D / 2), d = e % (D / 2) * 2;
      float2 ml[kAtOnce], o[kAtOnce];
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        ml[i] = make_float2(-INFINITY, 0.f), o[i] = make_float2(0.f, 0.f);
        if (i < count) {
          const float* p = at(i) + h * (D + 2);
          ml[i] = *reinterpret_cast<const float2*>(p);
          o[i] = *reinterpret_cast<const float2*>(p + 2 + d);
        }
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) top = fmaxf(top, ml[i].x);
      float l = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const float f = ml[i].x == top ? 1.f : exp2_fast(ml[i].x - top);
        l += ml[i].y * f;
        o0 += o[i].x * f;
        o1 += o[i].y * f;
      }
      *reinterpret_cast<uint32_t*>(out + h * D + d) = pack2(o0 / l, o1 / l);
    }
    return;
  }
  float* total_l = weight + sp.heads * sp.parts;
  for (int h = warp; h < heads; h += kJoinThreads / 32) {
    float top = -INFINITY, l = 0.f;
    for (int i = lane; i < count; i += 32) top = fmaxf(top, at(i)[h * (D + 2)]);
    top = warp_max(top);
    for (int i = lane; i < count; i += 32) {
      const float m = at(i)[h * (D + 2)], f = m == top ? 1.f : exp2_fast(m - top);
      weight[h * sp.parts + i] = f;
      l += at(i)[h * (D + 2) + 1] * f;
    }
    l = warp_sum(l);
    if (lane == 0) total_l[h] = l;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < heads * D / 2; e += kJoinThreads) {
    const int h = e / (D / 2), d = e % (D / 2) * 2;
    float o0 = 0.f, o1 = 0.f;
#pragma unroll 8
    for (int i = 0; i < count; ++i) {
      const float2 v = *reinterpret_cast<const float2*>(at(i) + h * (D + 2) + 2 + d);
      o0 += v.x * weight[h * sp.parts + i];
      o1 += v.y * weight[h * sp.parts + i];
    }
    *reinterpret_cast<uint32_t*>(out + h * D + d) = pack2(o0 / total_l[h], o1 / total_l[h]);
  }
}

struct SplitPlan {
  int parts, heads;
  size_t bytes;
};
SplitPlan split_plan(int64_t group, int64_t head_dim) {
  SplitPlan p;
  p.parts = sm_count();
  p.heads = int(group < kHeads ? group : kHeads);
  p.bytes = size_t(p.parts) * 2 * p.heads * (head_dim + 2) * 4;
  return p;
}

// How a decode call runs, from sizes that the host knows (lengths stay on the device). Measured with 16 query and 8
// KV heads of 128 dims, in a graph:
// - items (row, KV head, pass) up to one per SM: 8 warps per CTA, and clusters while they too find an SM each
//   (1 row of 1000 keys: 10.3 us with 4 warps, 8.4 with 8, 5.0 with clusters of 8; 8 rows of 1000: 10.6, 8.6 and
//   7.2 with clusters of 2, but 11.9 with 512 CTAs in clusters of 8: a CTA that finds nothing to do still costs, so
//   that a cluster is no larger than the context has steps for);
// - more items: CTAs of 4 warps, three to an SM, one per item (256 rows of 50..150 keys: 26.9 us against 54.9 with 8
//   warps; 64 rows of 64..2048: 52, as good);
// - contexts that would keep one CTA busy for long: the split kernel. With equal lengths the two are even (64 rows of
//   4000..8192: 254 us split, 257 direct; 256 rows of 1..4096: 329 and 313), but one row of 8192 keys among 63 of 200
//   takes 80 us direct and 25 split, one of 32768 among 7 takes 83 and 36.
struct DecodePlan {
  bool split;
  int ranks;   // direct: CTAs per item
  bool wide;   // direct: 8 warps per CTA instead of 4
};
DecodePlan decode_plan(int64_t rows, int64_t q_heads, int64_t kv_heads, int64_t context) {
  const int64_t units = kv_heads * ((q_heads / kv_heads + kHeads - 1) / kHeads), items = rows * units;
  DecodePlan p = {false, 1, items <= sm_count()};
  while (p.wide && p.ranks < kRanks && items * p.ranks * 2 <= sm_count() && context > 128 * p.ranks) p.ranks *= 2;
  const int64_t steps = steps_of(context - 1);
  // 32-bit step counts of a row and of one unit over all rows
  p.split = context > p.ranks * (p.wide ? 8192 : 4096) && rows <= kSplitRows && steps < (int64_t(1) << 26) &&
            steps * (rows > units ? rows : units) < (int64_t(1) << 31);
  return p;
}

// Whether a prompt call goes by rows, as a decode call does, instead of in tiles: a tile takes as long for one row as for
// 128, but a pass over the keys serves no more than the eight columns of the products. With 16 query and 8 KV heads of 128
// dims, tiles and rows: one prompt of 13 rows 7.2 us and 4.0, 64 rows 7.5 and 4.7, 200 rows 10.9 and 7.7, 300 rows 10.9 and
// 12.8; 48 rows behind 1000 keys 20.1 and 9.7, 200 behind 1800 26.4 and 27.6; 16 behind 4000 25.9 and 14.9, 64 behind 6000
// 28.9 and 32.0, 16 behind 24000 45.6 and 59.2. The host knows the table's columns only, not the rows' keys.
struct PromptPlan {
  bool by_rows, look;
  int pack;
  int64_t packs;
  DecodePlan how;
};
PromptPlan prompt_plan(int64_t rows, int64_t sequences, int64_t q_heads, int64_t kv_heads, int64_t capacity) {
  const int64_t group = q_heads / kv_heads;
  PromptPlan p;
  p.look = sequences <= 32 * kLookRounds && rows <= (int64_t(1) << 20);
  const int64_t units = kv_heads * ((group + kHeads - 1) / kHeads);
  // several rows' heads share a pass where it is long or the rows are many (16 rows behind 2000 keys 13.4 us alone and 10.6
  // together; behind 500 6.7 and 7.5, 13 rows 3.9 and 4.6: finding the packs and fewer CTAs cost more than they save)
  const bool many = rows * units > 3 * sm_count() || capacity > 768;
  p.pack = many && p.look && group <= kHeads ? int(kHeads / group) : 1;
  // every sequence may end inside a pack
  p.packs = rows / p.pack + sequences < rows ? rows / p.pack + sequences : rows;
  p.how = decode_plan(p.packs, q_heads, kv_heads, capacity);
  p.by_rows = p.packs * units <= 3 * sm_count() && capacity <= (p.how.wide ? 6144 * p.how.ranks : 2048);
  return p;
}

template <int D, int W, int ST>
int launch_split(const DecodeArgs& a, void* workspace, void* stream, const char* name) {
  static PerDevice once;
  constexpr int kMost = 232448;
  if (const int rc = smem_limit(once, paged_decode_split<D, W, ST>, kMost, name)) return rc;
  const SplitPlan p = split_plan(a.group, D);
  const SplitArgs sp = {p.parts, p.heads, static_cast<float*>(workspace)};
  if (const int rc = launch(paged_decode_split<D, W, ST>, dim3(unsigned(p.parts)), dim3(W * 32),
                            size_t(split_smem<D, W, ST>(p.heads, a.rows)), stream, true, name, a, sp))
    return rc;
  return launch(paged_decode_join<D>, dim3(unsigned(int64_t(a.rows) * a.kv_heads * a.passes)), dim3(kJoinThreads),
                size_t(p.heads) * (p.parts + 1) * 4, stream, true, name, a, sp);
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
  a.ranks = 1;
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
  if (rows < 1 || q_heads < 1 || kv_heads < 1 || head_dim < 1 || !decode_plan(rows, q_heads, kv_heads, context).split)
    return 0;
  return split_plan(q_heads / kv_heads, head_dim).bytes;
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
  const DecodePlan how = decode_plan(p.rows, p.q_heads, p.cache.kv_heads, p.context);
  const bool d128 = p.cache.head_dim == 128;
  if (how.split) {
    const SplitPlan plan = split_plan(a.group, p.cache.head_dim);
    if (p.workspace == nullptr || p.workspace_bytes < int64_t(plan.bytes) || !aligned16(p.workspace))
      return fail(Q3T_ESPACE, "%s: workspace of %zu bytes (16-byte aligned) needed", name, plan.bytes);
    return d128 ? launch_split<128, 8, 2>(a, p.workspace, stream, name)
                : launch_split<64, 8, 4>(a, p.workspace, stream, name);
  }
  const PromptRows none = {};
  if (how.wide)
    return d128 ? launch_direct<128, 8, 2, false>(a, none, how.ranks, stream, name)
                : launch_direct<64, 8, 4, false>(a, none, how.ranks, stream, name);
  return d128 ? launch_direct<128, 4, 2, false>(a, none, 1, stream, name)
              : launch_direct<64, 4, 4, false>(a, none, 1, stream, name);
}

extern "C" size_t q3t_paged_prefill_attention_workspace_bytes(int64_t rows, int64_t sequences, int64_t q_heads,
                                                              int64_t kv_heads, int64_t head_dim, int64_t context) {
  if (rows < 1 || sequences < 1 || q_heads < 1 || kv_heads < 1 || q_heads < kv_heads || head_dim < 1) return 0;
  return prompt_plan(rows, sequences, q_heads, kv_heads, context).by_rows
             ? 0
             : prefill_tiles_workspace(rows, sequences, q_heads, kv_heads, head_dim, context);
}

extern "C" int q3t_paged_prefill_attention_form(int64_t rows, int64_t sequences, int64_t q_heads, int64_t kv_heads,
                                                int64_t head_dim, int64_t context) {
  if (rows < 1 || sequences < 1 || kv_heads < 1 || q_heads < kv_heads || head_dim < 1 || context < 1)
    return fail(Q3T_EINVAL, "paged_prefill_attention_form: invalid geometry");
  if (prompt_plan(rows, sequences, q_heads, kv_heads, context).by_rows || !prefill_tiles_supported(rows, context, 1.)) return 0;
  return prefill_tiles_workspace(rows, sequences, q_heads, kv_heads, head_dim, context) > 0 ? 2 : 1;
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
  const PromptPlan plan = prompt_plan(p.rows, p.sequences, p.q_heads, p.cache.kv_heads, a.context);
  if (!plan.by_rows && prefill_tiles_supported(p.rows, a.context, p.scale)) return launch_prefill_tiles(p, status, stream, name);
  const PromptRows pr = {p.row_offsets, p.start_positions, int(p.sequences), plan.pack,
                         plan.pack > 1 ? int(255 / a.group + 1) : 0, int(plan.packs), plan.look};
  const DecodePlan& how = plan.how;
  const bool d128 = p.cache.head_dim == 128;
  if (how.wide || !plan.by_rows)
    return d128 ? launch_direct<128, 8, 2, true>(a, pr, how.ranks, stream, name)
                : launch_direct<64, 8, 4, true>(a, pr, how.ranks, stream, name);
  return d128 ? launch_direct<128, 4, 2, true>(a, pr, 1, stream, name)
              : launch_direct<64, 4, 4, true>(a, pr, 1, stream, name);
}
