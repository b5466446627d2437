// Causal attention of packed prompts over a paged key/value cache, on tcgen05 tensor cores.
//
//   out[r, h] = sum_j softmax_j(scale * q[r, h] . k_j) v_j,   j = 0 .. position of row r in its sequence
//
// A CTA owns two query tiles of 128 rows for one KV head: 2 x 128 / G consecutive positions times the G query heads of
// the group, position-major, so one K/V tile serves all heads of the group. It streams the sequence's keys in tiles of
// 128 through TMA (pieces of gcd(page_size, 128) rows: each lies in one page) and keeps the scores on chip:
//
//   S_t = Q_t K^T      tcgen05.mma 128 x 128 x D into TMEM
//   P_t = 2^(S_t scale log2e - m)   one thread per query row; bf16, over S_t's own TMEM columns
//   O_t += P_t V       tcgen05.mma 128 x D x 128, P from TMEM, V as the MN-major operand
//
// Warps 4-7 and 8-11 are the softmax of tile 0 and 1, warp 0 loads, warp 1 issues the products, warp 3 hands out the
// work: while one tile's weights are computed the tensor cores run the other's products. m is a reference that the
// row's maximum exceeds by at most 8 (powers of two), so O in TMEM is rescaled only when a maximum moves by more; O / l
// does not depend on it. P's rounding to bf16 is that of a bf16 tensor product; S, m, l and O stay in fp32.
//
// One prompt of 8191 rows with 32 query and 8 KV heads of 128 dims: 510 us in a stream of calls, 1080 TFLOP/s, under the
// power cap; 432 to 454 us in a short run (1270 to 1210). A pair of 128 x 128 key tiles takes 3150 cycles of which the tensor cores work 2080: scores, the first half of
// the weights, their product and the next scores wait for one another, and there is no TMEM for a third tile.
//
// Work comes in one of two ways (the host picks by sizes):
// - items (query tile pair, KV head) in turn: a CTA whose item's loads are nearly out takes over one that has not been
//   launched yet, so items go to the SMs as those get free, and the next one's loads and first products overlap the last
//   one's softmax and stores (16 prompts of 256 rows 20.1 us; before the hand-over was made leaner 22.4, against 23.9 with
//   a CTA each);
// - one even range of all items' key tiles per CTA, one CTA per SM. An item that a range covers only in part leaves O, m
//   and l in the workspace, and a second, dependent launch joins the parts in the order of their keys (results repeat
//   bit for bit). Parts are never smaller than kLeast tiles: short items move to one range whole.
#include "common.cuh"
#include "exp2_poly.cuh"
#include "host.cuh"
#include "paged.cuh"
#include "paged_prefill.cuh"

using namespace q3t;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTileKeys = 128, kTileRows = 128;
constexpr int kStages = 2;  // of K, and of V
constexpr int kThreads = 384;
constexpr int kLeast = 4;          // key tiles of a part
constexpr int kFixed = 2;          // what an item costs beside its key tiles, in key tiles
constexpr int kAhead = 2;          // key tiles of an item that are still to be loaded when the next one is asked for
constexpr int kPlanTiles = 2048;   // query tile pairs that a range plan holds, and entries of the numbers of whole items
constexpr int kPlanSequences = 1024;
// Query tile pairs that a sequence is counted with at most: kThreads sequences and all before them stay within 32 bits. A
// sequence of more has 230 GB of queries and outputs at the least (4 rows of 43 heads of 64 dims a pair).
constexpr int kMostPairs = 5 << 20;
static_assert(int64_t(kThreads) * kMostPairs + (int64_t(1) << 28) / 4 + (1 << 20) < (int64_t(1) << 31), "32 bits");

struct PrefillArgs {
  PageTable pages;
  const int64_t *row_offsets, *start_positions;
  __nv_bfloat16* out;
  int rows, sequences, q_heads, kv_heads, group;
  int heads;    // query heads of a tile: the group, in passes of 64 where it is wider
  int passes, positions;  // passes over the group; positions of a tile
  int piece;    // rows of a TMA box: gcd(page_size, 128)
  int capacity; // positions that a page table row can hold
  bool out_32;  // out is 32-byte aligned
  int parts;    // ranges, one per CTA; 0: whole items in turn
  int pairs;    // query tile pairs at most
  int shift, groups;  // the CTA keeps the numbers behind every 2^shift sequences
  struct Segment* shared_segments;  // workspace: [parts][2], what a range left unfinished at its start (0) and end (1)
  float* partial;                   // workspace: [parts][2][D / 4][256 rows][4], then [256][2] (m, l)
  float scale_log2;
  unsigned* status;
};

// A run of key tiles of one item.
struct Segment {
  int sequence, row, count;            // the tile pair's first packed row and rows (positions); count 0: no more work
  int head, head0, heads;              // KV head; first query head and query heads of the pass
  int tile0, key_tiles, all_tiles;     // key tiles of the run, and of the item
  int slot;                            // -1: the whole item; else where the run's O, m and l wait for the join
  int position;                        // of the first row (a start past +-2^30 as that)
  int tiles[2], keys;                  // key tiles of each query tile, and keys, counted from the run's first key on
};

template <int D>
struct Smem {
  static constexpr int kTile = 128 * D * 2;  // a query, key or value tile: D / 64 blocks of 128 rows x 128 bytes
  static constexpr int kBlock = 128 * 128;
  static constexpr int kK = 2 * kTile, kV = kK + kStages * kTile, kPlan = kV + kStages * kTile;
  static constexpr int kBar = kPlan + (kPlanTiles + 1 + kPlanSequences + 1) * 4 + 8;
  static constexpr int kBytes = (kBar + 15) / 16 * 16 + 512 + 1024;
};

struct Bars {
  uint64_t q_full[2], q_free[2], k_full[kStages], v_full[kStages], turn[2], s_full[2], p_full[2][2], o_done[2], o_free[2],
      segment_full[2], segment_free[2], loaded, takeover, done;
  alignas(16) uint4 response;
  Segment segments[2];
  int sums[kThreads / 32];
  uint32_t tmem;
};

// floats of a part in the workspace
template <int D>
constexpr int kPartFloats = 256 * (D + 2);

// One 4-D tiled load; x * 2 bytes is a multiple of 16 (0 or 64 elements).
Q3T_DEV void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}
// The issuing warp stays converged and computes every operand warp-uniformly (tcgen05.mma takes them from uniform
// registers); `leader` is set in one lane, which alone issues. With the addresses computed by a single lane instead,
// moving them over took longer than the products (100 cycles an instruction of 64).
Q3T_DEV bool elect_one() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(e));
  return e != 0;
}
// Descriptor words: start address, leading stride | stride 1024, version 1, 128-byte swizzle (see umma_desc_sw128).
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
Q3T_DEV uint64_t desc_of(uint32_t lo) { return (uint64_t(kDescHi) << 32) | lo; }
// K-major operand at `addr`; its next 16 columns are 2 further on.
Q3T_DEV uint32_t desc_k(uint32_t addr) { return (addr >> 4) | (1u << 16); }
// MN-major operand: 64 columns x 8 rows per 1024-byte atom, the next 64 columns `block` bytes on; the next 16 rows
// are 128 further on.
Q3T_DEV uint32_t desc_mn(uint32_t addr, uint32_t block) { return (addr >> 4) | ((block >> 4) << 16); }
// D[tmem] (+)= A[smem] * B[smem]
Q3T_DEV void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, bool add, bool leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(desc_of(a_lo)), "l"(desc_of(b_lo)), "r"(idesc), "r"(uint32_t(add)), "r"(uint32_t(leader))
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]: A bf16, two values of a row per 32-bit column.
Q3T_DEV void mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, bool add, bool leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(desc_of(b_lo)), "r"(idesc), "r"(uint32_t(add)), "r"(uint32_t(leader))
      : "memory");
}
Q3T_DEV void commit_if(uint64_t* bar, bool leader) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar)),
      "r"(uint32_t(leader))
      : "memory");
}
Q3T_DEV void tmem_ld32(uint32_t addr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
Q3T_DEV void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
      : "memory");
}
// Waits for tcgen05.ld; the 32 registers pass through, so that nothing reads (or moves) them before. With more than 32,
// the others pass through an empty statement behind the wait.
template <bool WAIT = true>
Q3T_DEV void tmem_ld_wait(float* v) {
  if constexpr (WAIT) asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  asm volatile(""
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]),
                 "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]),
                 "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]),
                 "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
               :
               : "memory");
}
Q3T_DEV void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
Q3T_DEV float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The largest of three; NaN where one of them is.
Q3T_DEV float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
Q3T_DEV float max2(float a, float b) {
  float c;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}
// Moves registers between the warpgroups: the CTA is launched with kThreads * 168, and 56 + 2 * 224 = 3 * 168.
constexpr int kRegsLoad = 56, kRegsSoftmax = 224;
static_assert(kRegsLoad + 2 * kRegsSoftmax == 3 * 168, "register shares must add up to the launch's");
Q3T_DEV uint32_t pack2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// Asks for a CTA of this grid that has not been launched yet; the answer comes through `bar`. After a refusal it is not
// asked again.
Q3T_DEV void try_take_over(uint4* response, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   smem_u32(response)),
               "r"(smem_u32(bar))
               : "memory");
}
Q3T_DEV bool taken_over(const uint4* response, int& block) {
  uint32_t yes, x;
  ulonglong2 r;
  asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(r.x), "=l"(r.y) : "r"(smem_u32(response)) : "memory");
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\tmov.b128 r, {%2, %3};\n\tmov.u32 %1, 0;\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\tselp.u32 %0, 1, 0, p;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}\n"
      : "=r"(yes), "=r"(x)
      : "l"(r.x), "l"(r.y));
  block = int(x);
  return yes != 0;
}
// 32 bytes to memory, in one store where the address allows it.
Q3T_DEV void store32(void* to, const uint32_t* w, bool aligned) {
  if (aligned) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(to)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    reinterpret_cast<uint4*>(to)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}
// A bounded wait of a whole warp: every lane leaves with the same answer.
Q3T_DEV bool warp_wait(uint64_t* bar, int phase, unsigned* status, unsigned bits) {
  return __all_sync(0xffffffffu, mbar_wait(bar, phase & 1, status, bits));
}

// The packed rows of sequence s and the first of them; 0 where the offsets make no sense.
Q3T_DEV int rows_of(const PrefillArgs& a, int s, int& first) {
  const int64_t lo = a.row_offsets[s], hi = a.row_offsets[s + 1];
  if (lo >= 0 && hi <= a.rows && hi > lo) {
    first = int(lo);
    return int(hi - lo);
  }
  if (hi != lo) raise_status(a.status, kStatusBadIndex);
  first = 0;
  return 0;
}
// Keys that rows up to position `end` - 1 see (what the table cannot hold is cut off), and their tiles.
Q3T_DEV int keys_of(const PrefillArgs& a, int64_t end) { return end < 0 ? 0 : int(end < a.capacity ? end : a.capacity); }
Q3T_DEV int key_tiles_of(const PrefillArgs& a, int64_t end) { return (keys_of(a, end) + kTileKeys - 1) / kTileKeys; }

// Query tile pairs are numbered from the last of the last sequence backwards, so that those with the most keys
// come first. One warp finds the sequence, rows and key tiles of number `index`; count 0: there is none. `before`: where the
// CTA has it, the numbers behind every 2^shift sequences, the last one first, of which 32 at once are looked at; without it
// all are (past 32 sequences that is too slow: 20000 of 2..6 rows, 8 KV heads, take 4.6 ms, and 169 with a look at all of
// them for every item).
Q3T_DEV Segment find_tile(const PrefillArgs& a, const int32_t* before, int index, int unit, int lane) {
  const int span = 2 * a.positions;
  Segment t = {};
  int base = a.sequences - 1, stop = 0;  // the first sequence to look at
  if (before != nullptr) {
    const int i = row_of(before, a.groups, index, 1);
    base -= i << a.shift;
    stop = max(0, base + 1 - (1 << a.shift));
    index -= before[i];
  }
  for (; base >= stop; base -= 32) {
    const int s = base - lane;
    int n = 0, first = 0, tiles = 0;
    int64_t start = 0;
    if (s >= 0) {
      start = clamped_start(a.start_positions[s]);
      n = rows_of(a, s, first);
    }
    tiles = (n + span - 1) / span;
    int sum = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += other;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, sum > index);
    if (hit == 0) {
      index -= __shfl_sync(0xffffffffu, sum, 31);
      continue;
    }
    const int src = __ffs(hit) - 1;
    const int in_sequence = ((tiles - 1) - (index - (sum - tiles))) * span;  // counted from the sequence's last tile
    t.sequence = base - src;
    t.row = __shfl_sync(0xffffffffu, first + in_sequence, src);
    t.count = __shfl_sync(0xffffffffu, min(span, n - in_sequence), src);
    // no table holds 2^30 positions and no call has as many rows: 32 bits tell all that matters
    const int64_t most = int64_t(1) << 30;
    t.position = __shfl_sync(0xffffffffu, int(max(-most, min(most, start + in_sequence))), src);
    t.all_tiles = key_tiles_of(a, t.position + t.count);
    t.key_tiles = t.all_tiles;
    t.slot = -1;
    const int pass = unit % a.passes;
    t.head = unit / a.passes;
    t.head0 = t.head * a.group + pass * a.heads;
    t.heads = min(a.heads, a.group - pass * a.heads);
    if (lane == 0 && t.position + t.count > a.capacity) raise_status(a.status, kStatusBadIndex);
    break;
  }
  return t;
}

// Completes a run: what its query tiles see of it. One warp does it for all others, off their way.
Q3T_DEV void shape(const PrefillArgs& a, Segment& t) {
  t.keys = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int count = max(0, min(a.positions, t.count - i * a.positions));
    const int end = count > 0 ? keys_of(a, t.position + i * a.positions + count) - t.tile0 * kTileKeys : 0;
    t.tiles[i] = max(0, min(t.key_tiles, (end + kTileKeys - 1) / kTileKeys));
    t.keys = max(t.keys, min(end, t.key_tiles * kTileKeys));
  }
}

// Inclusive sum over the CTA; `sums` holds one value per warp.
Q3T_DEV int block_sum(int v, int* sums, int warp, int lane, int& all) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int other = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += other;
  }
  if (lane == 31) sums[warp] = v;
  __syncthreads();
  all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    const int s = sums[w];
    if (w < warp) v += s;
    all += s;
  }
  __syncthreads();
  return v;
}

// Where range `i` of `parts` begins among `total` units of work (an item: its key tiles and kFixed), moved
// to an item's end where less than kLeast tiles would be cut off.
Q3T_DEV int64_t range_begin(const int32_t* prefix, int pairs, int units, int64_t i, int64_t total, int64_t parts) {
  const int64_t at = split_begin(i, total, parts);
  if (at <= 0 || at >= total) return at;
  const int e = row_of(prefix, pairs, at, units);
  const int n = prefix[e + 1] - prefix[e];
  const int64_t base = int64_t(prefix[e]) * units;
  const int64_t item = base + (at - base) / n * n;
  const int o = int(at - item);
  // an item's fixed cost stands at its beginning
  if (n < 2 * kLeast + kFixed ? 2 * o <= n : o < kLeast + kFixed) return item;
  if (n < 2 * kLeast + kFixed || n - o < kLeast) return item + n;
  return at;
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    paged_prefill_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                         const __grid_constant__ CUtensorMap tmv, const PrefillArgs a) {
  using M = Smem<D>;
  constexpr int kHalves = D / 64;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Bars* bars = reinterpret_cast<Bars*>(smem + (M::kBar + 15) / 16 * 16);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int units = a.kv_heads * a.passes;
  int given = 0;  // warp 3: segments handed out
  // set up while the launch before may still run: none of it reads what that one writes
  if (warp == 1) {
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&bars->q_full[i], 1);
        mbar_init(&bars->q_free[i], 1);
        mbar_init(&bars->s_full[i], 1);
        mbar_init(&bars->turn[i], 1);
        mbar_init(&bars->p_full[i][0], 128);
        mbar_init(&bars->p_full[i][1], 128);
        mbar_init(&bars->o_done[i], 1);
        mbar_init(&bars->o_free[i], 128);
        mbar_init(&bars->segment_full[i], 1);
        mbar_init(&bars->segment_free[i], 10);  // warps that read it: loads, products, eight of softmax
      }
      for (int i = 0; i < kStages; ++i) {
        mbar_init(&bars->k_full[i], 1);
        mbar_init(&bars->v_full[i], 1);
      }
      mbar_init(&bars->loaded, 1);
      mbar_init(&bars->takeover, 1);
      mbar_init(&bars->done, 1);
      fence_mbar_init();
    }
  } else if (warp == 0 && lane == 0) {
    prefetch_tmap(&tmq);
    prefetch_tmap(&tmk);
    prefetch_tmap(&tmv);
  }
  __syncthreads();
  grid_dependency_wait();
  if (warp == 2) {  // behind the wait: the launch before may need the columns until its end
    tmem_alloc(&bars->tmem, 512);
    tmem_relinquish();
  }
  // ---- the plan: the numbers behind every sequence, where it takes more than a look to find one; for ranges, the work
  // before every query tile pair, for one unit
  int32_t* prefix = reinterpret_cast<int32_t*>(smem + M::kPlan);
  int32_t* before = nullptr;
  int pairs = 0;
  if (a.parts > 0 || a.sequences > 32) {
    before = a.parts > 0 ? prefix + kPlanTiles + 1 : prefix;
    const int span = 2 * a.positions;
    for (int s0 = 0; s0 < a.sequences; s0 += kThreads) {
      const int s = a.sequences - 1 - s0 - int(threadIdx.x);
      int first, n = s >= 0 ? rows_of(a, s, first) : 0, all;
      // offsets that run backwards may make sequences overlap: no more pairs are listed than rows in order can have
      n = min(min((n + span - 1) / span, a.pairs), kMostPairs);
      const int sum = block_sum(n, bars->sums, warp, lane, all), i = a.sequences - 1 - s;
      if (s >= 0 && (i & ((1 << a.shift) - 1)) == 0) before[i >> a.shift] = min(pairs + sum - n, a.pairs);
      pairs = min(pairs + all, a.pairs);
    }
    __syncthreads();
    int work = 0;
    for (int e0 = 0; a.parts > 0 && e0 < pairs; e0 += kThreads) {
      const int e = e0 + int(threadIdx.x);
      int cost = 0, all;
      if (e < pairs) {
        const int i = row_of(before, a.sequences, e, 1), s = a.sequences - 1 - i;
        int first;
        const int n = rows_of(a, s, first), tile = (n + span - 1) / span - 1 - (e - before[i]);
        cost = kFixed + key_tiles_of(a, clamped_start(a.start_positions[s]) + min(n, (tile + 1) * span));
      }
      const int sum = block_sum(cost, bars->sums, warp, lane, all);
      if (e < pairs) prefix[e] = work + sum - cost;
      work += all;
    }
    if (a.parts > 0 && threadIdx.x == 0) prefix[pairs] = work;
  }
  if (a.parts == 0 && warp == 3) {  // the CTA's first item
    Segment seg = find_tile(a, before, int(blockIdx.x) / units, int(blockIdx.x) % units, lane);
    shape(a, seg);
    if (lane == 0 && seg.count > 0) {
      bars->segments[0] = seg;
      mbar_arrive(&bars->segment_full[0]);
    }
    given = seg.count > 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;

  // The next segment of work, for one warp, read where it stands (the softmax loop needs every register, and a copy is
  // on the way of the first loads) and handed back with `leave`; null: none, or a wait gave up.
  int taken = 0;
  auto take = [&](bool& ok) -> const Segment* {
    ok = ok && warp_wait(&bars->segment_full[taken & 1], taken >> 1, a.status, kStatusFlagTimeout);
    const Segment* seg = &bars->segments[taken & 1];
    return ok && seg->count > 0 ? seg : nullptr;
  };
  auto leave = [&] {
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars->segment_free[taken & 1]);
    ++taken;
  };
  bool ok = true;

  if (warp >= 4) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    // ---------------- softmax: thread = query row = TMEM lane
    const int t = (warp >> 2) - 1, m = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + (uint32_t((warp & 3) * 32) << 16);
    const uint32_t s_at = lanes + 128 * t;  // this tile's scores and weights; its output 256 columns on
    const int p = m / a.heads, h = m - p * a.heads;
    int done = 0, outs = 0;  // key tiles and outputs so far
    while (const Segment* taken_segment = take(ok)) {
      const Segment& seg = *taken_segment;
      int key_tiles, seen0;  // of this query tile; keys that the row sees from the segment's first on
      const bool real = p < min(a.positions, seg.count - t * a.positions) && h < seg.heads;  // others hold anything
      {
        key_tiles = seg.tiles[t];
        const int position = seg.position + t * a.positions + p;
        seen0 = max(-1, min(position, a.capacity - 1)) + 1 - seg.tile0 * kTileKeys;
      }
      float top = -INFINITY, sum = 0.f;
      for (int j = 0; j < key_tiles; ++j, ++done) {
        if (!warp_wait(&bars->s_full[t], done, a.status, kStatusMmaTimeout)) {
          ok = false;
          break;
        }
        tc_fence_after();
        float s[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s_at + 32 * c, s + 32 * c);
#pragma unroll
        for (int c = 0; c < 4; ++c) c == 0 ? tmem_ld_wait<true>(s) : tmem_ld_wait<false>(s + 32 * c);
        const int seen = seen0 - j * kTileKeys;  // keys of this tile that the row sees
        if (__any_sync(0xffffffffu, seen < kTileKeys)) {
#pragma unroll
          for (int i = 0; i < 128; ++i) s[i] = i < seen ? s[i] : -INFINITY;
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 128; i += 2) mx[i / 2 & 3] = max3(mx[i / 2 & 3], s[i], s[i + 1]);
        const float now = max2(max3(mx[0], mx[1], mx[2]), mx[3]) * a.scale_log2;
        // a NaN among the scores becomes the maximum, and with it the sum: the row has no value, wherever the NaN stands
        if (__any_sync(0xffffffffu, !(now <= top + 8.f) && real)) {
          const float to = max2(top, now);
          const float f = to == top ? 1.f : exp2_fast(top - to);
          top = to;
          sum *= f;
          if (j > 0) {  // the products up to tile j - 1 are done: s_full says so
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              float o[16];
              tmem_ld16(s_at + 256 + c, o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] *= f;
              tmem_st16(s_at + 256 + c, reinterpret_cast<const uint32_t*>(o));
            }
          }
        }
        const float ref = top == -INFINITY ? 0.f : top;
        const float2 scale2 = make_float2(a.scale_log2, a.scale_log2), ref2 = make_float2(-ref, -ref);
        float2 part[2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
        for (int quarter = 0; quarter < 4; ++quarter) {
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float2 x = fma2(make_float2(s[32 * quarter + 2 * i], s[32 * quarter + 2 * i + 1]), scale2, ref2);
            if ((i & 7) == 3) {  // one in eight: 3 % for long prompts, -3 % for prompts of a few rows; one in four is no faster
              x = exp2_poly(x);
            } else {
              x.x = exp2_fast(x.x);
              x.y = exp2_fast(x.y);
            }
            part[i & 1] = add2(part[i & 1], x);
            w[i] = pack2(x.x, x.y);
          }
          tmem_st16(s_at + 16 * quarter, w);
          if (quarter & 1) {
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(&bars->p_full[t][quarter >> 1]);
          }
        }
        sum += (part[0].x + part[0].y) + (part[1].x + part[1].y);
      }
      if (ok && key_tiles > 0) {
        ok = warp_wait(&bars->o_done[t], outs, a.status, kStatusMmaTimeout);
        ++outs;
      }
      if (!ok) break;
      tc_fence_after();
      const bool none = seg.position + t * a.positions + p < 0;  // the row sees nothing
      if (seg.slot < 0) {
        // ---- O / l: each thread its row, a whole sector (16 dims) a store. A row without keys is 0; a maximum of +inf
        // leaves no value.
        const float inv = none ? 0.f : top == INFINITY ? NAN : 1.f / sum;
        __nv_bfloat16* to = a.out + ((int64_t(seg.row) + t * a.positions + p) * a.q_heads + seg.head0 + h) * D;
#pragma unroll 1  // the code runs once an item: short is faster than unrolled, which waits for its instructions
        for (int c = 0; c < D / 32; ++c, to += 32) {
          float o[32];
          if (key_tiles > 0) {  // uniform over the warp
            tmem_ld32(s_at + 256 + 32 * c, o);
            tmem_ld_wait(o);
          }
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = none ? 0u : pack2(o[2 * i] * inv, o[2 * i + 1] * inv);
          if (real) {
            store32(to, w, a.out_32);
            store32(to + 16, w + 8, a.out_32);
          }
        }
      } else {
        float* part = a.partial + (int64_t(blockIdx.x) * 2 + seg.slot) * kPartFloats<D>;
        const int row = t * 128 + m;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          if (key_tiles > 0) {
            tmem_ld32(s_at + 256 + 32 * c, o);
            tmem_ld_wait(o);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *reinterpret_cast<float4*>(part + ((8 * c + i) * 256 + row) * 4) =
                key_tiles > 0 ? make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        *reinterpret_cast<float2*>(part + 256 * D + 2 * row) = make_float2(top, sum);
      }
      tc_fence_before();
      if (key_tiles > 0) mbar_arrive(&bars->o_free[t]);
      leave();
    }
    tc_fence_before();
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsLoad));
    if (warp == 0) {
      // ---------------- loads. Lane: (piece of a key tile, 64-dim block)
      const int pieces = kTileKeys / a.piece, piece = lane / kHalves, half = lane % kHalves;
      int n = 0, loaded = 0, queries[2] = {0, 0};  // key tiles so far; loads begun; query tiles so far
      while (const Segment* taken_segment = take(ok)) {
        const Segment& seg = *taken_segment;
        const int keys = seg.keys;
        const int signal = max(0, seg.key_tiles - 1 - kAhead);  // the tile at which the next item is asked for
        if (signal == 0 && lane == 0) mbar_arrive(&bars->loaded);
        const int key0 = seg.tile0 * kTileKeys;
        auto page_of = [&](int j) {  // the page of this lane's piece of tile j, and its row there
          int2 at = make_int2(int(a.pages.pages), 0);  // past the pool: a load of zeros
          const int key = j * kTileKeys + piece * a.piece;
          if (piece < pieces && key < keys) {
            int row;
            const int64_t page = a.pages.lookup(seg.sequence, key0 + key, row);
            if (page >= 0) at = make_int2(int(page), row);
            else raise_status(a.status, kStatusBadIndex);
          }
          return at;
        };
        int2 next = page_of(0);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (!ok || seg.tiles[t] == 0) continue;
          if (queries[t] > 0) ok = warp_wait(&bars->q_free[t], queries[t] - 1, a.status, kStatusMmaTimeout);
          if (!ok) break;
          ++queries[t];
          if (lane == 0) {
            mbar_expect_tx(&bars->q_full[t], uint32_t(a.heads * a.positions * 128 * kHalves));
            for (int h = 0; h < kHalves; ++h)
              tma_load_3d(smem + t * M::kTile + h * M::kBlock, &tmq, &bars->q_full[t], h * 64,
                          seg.head0, seg.row + t * a.positions, policy_evict_first());
          }
        }
        for (int j = 0; j < seg.key_tiles && ok; ++j, ++n) {
          const int s = n % kStages;
          if (j > 0 && j == signal && lane == 0) mbar_arrive(&bars->loaded);
          const int2 at = next;
          const int wanted = min(pieces, (keys - j * kTileKeys + a.piece - 1) / a.piece);  // pieces that hold a key
          const uint32_t bytes = uint32_t(wanted * a.piece * 128 * kHalves);
#pragma unroll
          for (int v = 0; v < 2 && ok; ++v) {
            // turn i of the products has read key tile i and value tile i - 1
            const int turn = n - kStages + v;
            if (n >= kStages) ok = warp_wait(&bars->turn[turn & 1], turn >> 1, a.status, kStatusMmaTimeout);
            if (!ok) break;
            uint64_t* full = v ? &bars->v_full[s] : &bars->k_full[s];
            if (lane == 0) mbar_expect_tx(full, bytes);
            __syncwarp();
            if (piece < wanted)
              tma_load_4d(smem + (v ? M::kV : M::kK) + s * M::kTile + half * M::kBlock + piece * a.piece * 128, v ? &tmv : &tmk,
                          full, half * 64, at.y, seg.head, at.x);
            ++loaded;
          }
          if (j + 1 < seg.key_tiles) next = page_of(j + 1);
        }
        if (!ok) break;
        leave();
      }
      if (!ok) {  // loads still in flight land before the CTA leaves
        for (int t = 0; t < 2; ++t)
          if (queries[t] > 0) mbar_wait(&bars->q_full[t], (queries[t] - 1) & 1, a.status, kStatusTmaTimeout);
        for (int i = max(0, loaded - 2 * kStages); i < loaded; ++i)
          mbar_wait(i & 1 ? &bars->v_full[(i / 2) % kStages] : &bars->k_full[(i / 2) % kStages], (i / 2 / kStages) & 1, a.status,
                    kStatusTmaTimeout);
      }
    } else if (warp == 1) {
      // ---------------- products (TMEM column 0 is the allocation's first: it is all of TMEM)
      constexpr uint32_t idesc_s = umma_idesc_bf16(128, kTileKeys);
      constexpr uint32_t idesc_o = umma_idesc_bf16(128, D) | (1u << 16);  // V MN-major
      const uint32_t base = smem_u32(smem);
      const bool leader = elect_one();
      int n = 0, weights[2] = {0, 0}, queries[2] = {0, 0};  // key tiles, weight tiles and query tiles so far
      auto wait = [&](uint64_t* bar, int phase, unsigned bit) { ok = ok && warp_wait(bar, phase, a.status, bit); };
      auto scores = [&](int t, int s) {
        const uint32_t q = desc_k(base + t * M::kTile), k = desc_k(base + M::kK + s * M::kTile);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const uint32_t step = (i >> 2) * (M::kBlock >> 4) + 2 * (i & 3);
          mma_ss(128 * t, q + step, k + step, idesc_s, i > 0, leader);
        }
        commit_if(&bars->s_full[t], leader);
      };
      while (const Segment* taken_segment = take(ok)) {
        const Segment& seg = *taken_segment;
        const int key_tiles = __shfl_sync(0xffffffffu, seg.key_tiles, 0);  // so that the compiler knows them uniform
        const int tiles[2] = {__shfl_sync(0xffffffffu, seg.tiles[0], 0), __shfl_sync(0xffffffffu, seg.tiles[1], 0)};
        const int keys = __shfl_sync(0xffffffffu, seg.keys, 0);
        leave();
        if (key_tiles == 0) continue;
        wait(&bars->k_full[n % kStages], n / kStages, kStatusTmaTimeout);
        for (int t = 0; t < 2; ++t) {
          if (tiles[t] == 0) continue;
          wait(&bars->q_full[t], queries[t], kStatusTmaTimeout);
          tc_fence_after();
          if (!ok) break;
          scores(t, n % kStages);
          if (tiles[t] == 1) commit_if(&bars->q_free[t], leader);
        }
        if (ok) commit_if(&bars->turn[n & 1], leader);
        for (int j = 0; j < key_tiles && ok; ++j, ++n) {
          const int s = n % kStages, sn = (n + 1) % kStages;
          wait(&bars->v_full[s], n / kStages, kStatusTmaTimeout);
          const int valid = keys - j * kTileKeys;
          if (ok && valid < kTileKeys) {
            // value rows past the last key hold anything, or were not loaded: their weights are 0, and 0 * NaN is NaN
            for (int e = lane; e < (kTileKeys - valid) * 8 * kHalves; e += 32) {
              const int h = e % kHalves, c = e / kHalves;
              *reinterpret_cast<uint4*>(smem + M::kV + s * M::kTile + h * M::kBlock + valid * 128 + c * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_async_shared();
            __syncwarp();
          }
          const uint32_t v = desc_mn(base + M::kV + s * M::kTile, M::kBlock);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (j >= tiles[t]) continue;
            // the last output of this query tile has been read
            if (j == 0 && queries[t] > 0) wait(&bars->o_free[t], queries[t] - 1, kStatusMmaTimeout);
#pragma unroll
            for (int part = 0; part < 2; ++part) {  // the first 64 keys' weights come before the others are computed
              wait(&bars->p_full[t][part], weights[t], kStatusMmaTimeout);
              tc_fence_after();
              if (!ok) continue;
#pragma unroll
              for (int i = 4 * part; i < 4 * part + 4; ++i)
                mma_ts(256 + 128 * t, 128 * t + 8 * i, v + 128 * i, idesc_o, j > 0 || i > 0, leader);
            }
            if (!ok) continue;
            ++weights[t];
            if (j + 1 < tiles[t]) {
              wait(&bars->k_full[sn], (n + 1) / kStages, kStatusTmaTimeout);  // behind the products just issued
              if (!ok) continue;
              scores(t, sn);
              if (j + 2 == tiles[t]) commit_if(&bars->q_free[t], leader);
            } else {
              commit_if(&bars->o_done[t], leader);
            }
          }
          if (ok && j + 1 < key_tiles) commit_if(&bars->turn[(n + 1) & 1], leader);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) queries[t] += tiles[t] > 0;
      }
      if (lane == 0) {  // every product is done before TMEM is released
        umma_commit(&bars->done);
        mbar_wait(&bars->done, 0, a.status, kStatusMmaTimeout);
      }
    } else if (warp == 3) {
      // ---------------- work
      Segment seg;
      auto give = [&](Segment& g) {
        shape(a, g);
        if (given >= 2) ok = warp_wait(&bars->segment_free[given & 1], (given >> 1) - 1, a.status, kStatusFlagTimeout);
        if (!ok) return;
        if (lane == 0) {
          bars->segments[given & 1] = g;
          mbar_arrive(&bars->segment_full[given & 1]);  // releases what the lane wrote
        }
        ++given;
      };
      if (a.parts == 0) {
        // The first item was handed out above. More: take over CTAs of this grid that have not been launched yet, so the
        // items still go to the SMs one by one, as those get free: asked for shortly before an item's last loads are out
        // (16 prompts of 40..400 rows 22.5 us, 23.1 when asked for behind them), and never two ahead.
        int items = given;
        for (int i = 0; ok; ++i) {
          if (items > 0) ok = warp_wait(&bars->loaded, items - 1, a.status, kStatusFlagTimeout);
          if (ok && given >= 2) ok = warp_wait(&bars->segment_free[given & 1], (given >> 1) - 1, a.status, kStatusFlagTimeout);
          if (!ok) break;
          if (lane == 0) {
            mbar_expect_tx(&bars->takeover, 16);
            try_take_over(&bars->response, &bars->takeover);
          }
          ok = warp_wait(&bars->takeover, i, a.status, kStatusFlagTimeout);
          int block = 0;
          if (!ok || !taken_over(&bars->response, block)) break;
          fence_async_shared();  // every lane's read of the answer comes before the next one is written over it
          __syncwarp();
          seg = find_tile(a, before, block / units, block % units, lane);
          if (seg.count > 0) {
            give(seg);
            ++items;
          }
        }
      } else {
        Segment* left = a.shared_segments + blockIdx.x * 2;  // what this range leaves to the join
        if (lane == 0) left[0].count = left[1].count = 0;
        const int64_t total = int64_t(prefix[pairs]) * units;
        const int64_t parts = split_parts(total / kLeast > 1 ? total / kLeast : 1, a.parts);
        const int64_t f1 = int64_t(blockIdx.x) < parts ? range_begin(prefix, pairs, units, blockIdx.x + 1, total, parts) : 0;
        int64_t f = int64_t(blockIdx.x) < parts ? range_begin(prefix, pairs, units, blockIdx.x, total, parts) : 0;
        while (f < f1 && ok) {
          const int e = row_of(prefix, pairs, f, units), n = prefix[e + 1] - prefix[e];
          const int64_t base = int64_t(prefix[e]) * units;
          const int unit = int((f - base) / n);
          const int64_t item = base + int64_t(unit) * n, end = item + n < f1 ? item + n : f1;
          seg = find_tile(a, before, e, unit, lane);
          seg.tile0 = f > item ? int(f - item) - kFixed : 0;
          seg.key_tiles = int(end - item) - kFixed - seg.tile0;
          seg.slot = f > item ? 0 : end < item + n ? 1 : -1;
          if (seg.count > 0) give(seg);
          if (lane == 0 && seg.slot >= 0) left[seg.slot] = seg;
          f = end;
        }
      }
      seg = {};
      if (ok) give(seg);
    }
  }
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of an item that several ranges share: CTA (i, eighth) the 32 rows of the item that range i began and
// did not end. Its parts are slot 1 of range i and slot 0 of the ranges after it, up to the item's end.
template <int D>
__global__ void __launch_bounds__(256) paged_prefill_join(const PrefillArgs a) {
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const Segment* segments = a.shared_segments + blockIdx.x * 2 + 1;
  const Segment first = segments[0];
  if (first.count == 0) return;
  int parts = 1;
  for (int base = 1; first.key_tiles < first.all_tiles; base += 32) {  // 32 ranges at a time
    const bool there = int(blockIdx.x) + base + lane < a.parts;
    const bool last = !there || segments[2 * (base + lane) - 1].tile0 + segments[2 * (base + lane) - 1].key_tiles >= first.all_tiles;
    const unsigned hit = __ballot_sync(0xffffffffu, last);
    parts = base + (hit ? __ffs(hit) : 32);
    if (hit) break;
  }
  parts = min(parts, a.parts - int(blockIdx.x));
  const int row = blockIdx.y * 32 + (threadIdx.x & 31), chunk0 = (threadIdx.x >> 5) * (D / 32);  // of D / 4
  const int t = row >> 7, p = (row & 127) / a.heads, h = (row & 127) - p * a.heads;
  const int count = max(0, min(a.positions, first.count - t * a.positions));
  if (p >= count || h >= first.heads) return;
  auto part_of = [&](int i) { return a.partial + (int64_t(blockIdx.x + i) * 2 + (i == 0)) * kPartFloats<D>; };
  float top = -INFINITY;
#pragma unroll 4
  for (int i = 0; i < parts; ++i) top = fmaxf(top, part_of(i)[256 * D + 2 * row]);
  float l = 0.f, v[D / 8] = {};
  for (int i = 0; i < parts; ++i) {
    const float* part = part_of(i);
    const float2 ml = *reinterpret_cast<const float2*>(part + 256 * D + 2 * row);
    const float f = ml.x == top ? 1.f : exp2_fast(ml.x - top);
    l += ml.y * f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const float4 o = *reinterpret_cast<const float4*>(part + ((chunk0 + c) * 256 + row) * 4);
      v[4 * c] += o.x * f;
      v[4 * c + 1] += o.y * f;
      v[4 * c + 2] += o.z * f;
      v[4 * c + 3] += o.w * f;
    }
  }
  const bool none = first.position + t * a.positions + p < 0;
  const float inv = top == INFINITY ? NAN : 1.f / l;
  __nv_bfloat16* out = a.out + (int64_t(first.row + t * a.positions + p) * a.q_heads + first.head0 + h) * D + chunk0 * 4;
#pragma unroll
  for (int c = 0; c < D / 64; ++c) {
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = none ? 0.f : v[8 * c + e] * inv;
    *reinterpret_cast<uint4*>(out + 8 * c) = pack8(w);
  }
}

template <int D>
int launch_prefill(const q3t_paged_prefill& p, const PrefillArgs& a, int64_t blocks, void* stream, const char* name) {
  const q3t_paged_cache& c = p.cache;
  CUtensorMap tmq, tmk, tmv;
  if (const int rc = make_map_bf16_strided(&tmq, p.query, {D, p.q_heads, p.rows, 1}, {D, p.query_stride, 0},
                                           {64, a.heads, a.positions, 1}, 3))
    return rc;
  for (int v = 0; v < 2; ++v)
    if (const int rc = make_map_bf16_strided(v ? &tmv : &tmk, v ? c.value_pages : c.key_pages,
                                             {D, c.page_size, c.kv_heads, c.pages}, {D, c.page_size * D, c.page_stride},
                                             {64, a.piece, 1, 1}, 4))
      return rc;
  static PerDevice once;
  if (const int rc = smem_limit(once, paged_prefill_kernel<D>, Smem<D>::kBytes, name)) return rc;
  if (const int rc = launch(paged_prefill_kernel<D>, dim3(unsigned(blocks)), dim3(kThreads), size_t(Smem<D>::kBytes), stream,
                            true, name, tmq, tmk, tmv, a))
    return rc;
  if (a.parts == 0) return Q3T_OK;
  return launch(paged_prefill_join<D>, dim3(unsigned(a.parts), 8), dim3(256), 0, stream, true, name, a);
}

// Bytes of the segments at the workspace's start; what follows is read and written in whole lines.
size_t segment_bytes(int parts) { return (size_t(parts) * 2 * sizeof(Segment) + 255) / 256 * 256; }

// How a call runs, from sizes that the host knows.
struct PrefillPlan {
  int heads, passes, positions;
  int64_t pairs, items;  // at most: every sequence may end inside a pair of tiles
  int parts;      // ranges; 0: one item per CTA
  size_t bytes;
};
PrefillPlan prefill_plan(int64_t rows, int64_t sequences, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t capacity) {
  PrefillPlan p;
  const int64_t group = q_heads / kv_heads;
  p.heads = int(group < 64 ? group : 64);
  p.passes = int((group + p.heads - 1) / p.heads);
  p.positions = kTileRows / p.heads;
  p.pairs = rows / (2 * p.positions) + sequences;
  p.items = p.pairs * kv_heads * p.passes;
  // Ranges pay where items are few and may be long: 4 chunks of 100..700 rows behind 2000..8000 keys 148 us in turn, 117 in
  // ranges; 512 rows behind 16000 keys 221 and 77. With many items they only add the
  // plan and the join (one prompt of 4096 rows and 32 heads: 128 and 137; one of 2048 and 16 heads: 36 and 44).
  const int64_t tiles = (capacity + kTileKeys - 1) / kTileKeys, sms = sm_count();
  const bool few = (tiles >= 32 && p.items <= 3 * sms) || (tiles >= 16 && p.items <= sms / 4);
  p.parts = few && p.pairs <= kPlanTiles && sequences <= kPlanSequences && p.pairs * (tiles + kFixed) < (int64_t(1) << 31) ? int(sms) : 0;
  p.bytes = p.parts == 0 ? 0 : segment_bytes(p.parts) + size_t(p.parts) * 2 * 256 * (head_dim + 2) * 4;
  return p;
}

}  // namespace

namespace q3t {

bool prefill_tiles_supported(int64_t rows, int64_t capacity, double scale) {
  // an item of 2^26 keys takes a second, half of what a wait may take
  return scale > 0. && scale < 1e30 && capacity <= (int64_t(1) << 26) && rows < (int64_t(1) << 28);
}

size_t prefill_tiles_workspace(int64_t rows, int64_t sequences, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                               int64_t capacity) {
  return prefill_plan(rows, sequences, q_heads, kv_heads, head_dim, capacity).bytes;
}

int launch_prefill_tiles(const q3t_paged_prefill& p, unsigned* status, void* stream, const char* name) {
  const q3t_paged_cache& c = p.cache;
  const PrefillPlan plan = prefill_plan(p.rows, p.sequences, p.q_heads, c.kv_heads, c.head_dim, c.table_columns * c.page_size);
  if (plan.bytes > 0 && (p.workspace == nullptr || p.workspace_bytes < int64_t(plan.bytes) || !aligned16(p.workspace)))
    return fail(Q3T_ESPACE, "%s: workspace of %zu bytes (16-byte aligned) needed", name, plan.bytes);
  if (plan.items > 2147483647) return fail(Q3T_EINVAL, "%s: too many rows", name);
  PrefillArgs a;
  a.pages = PageTable{c.page_table, c.table_stride, c.table_rows, c.table_columns, c.pages, int(c.page_size)};
  a.row_offsets = p.row_offsets;
  a.start_positions = p.start_positions;
  a.out = static_cast<__nv_bfloat16*>(p.out);
  a.rows = int(p.rows);
  a.sequences = int(p.sequences);
  a.q_heads = int(p.q_heads);
  a.kv_heads = int(c.kv_heads);
  a.group = int(p.q_heads / c.kv_heads);
  a.heads = plan.heads;
  a.passes = plan.passes;
  a.positions = plan.positions;
  a.piece = 16;
  while (a.piece < kTileKeys && c.page_size % (2 * a.piece) == 0) a.piece *= 2;
  a.capacity = int(c.table_columns * c.page_size);
  a.scale_log2 = float(p.scale) * kLog2e;
  a.status = status;
  a.out_32 = (reinterpret_cast<uintptr_t>(p.out) & 31u) == 0;
  a.parts = plan.parts;
  a.pairs = int(plan.pairs);
  a.shift = group_shift(p.sequences, kPlanTiles);  // 0 for ranges, whose sequences are fewer
  a.groups = groups_of(p.sequences, a.shift);
  a.shared_segments = static_cast<Segment*>(p.workspace);
  a.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(p.workspace) + segment_bytes(plan.parts));
  const int64_t blocks = plan.parts > 0 ? plan.parts : plan.items;
  return c.head_dim == 128 ? launch_prefill<128>(p, a, blocks, stream, name) : launch_prefill<64>(p, a, blocks, stream, name);
}

}  // namespace q3t
