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
// Warps 4-7 and 8-11 are the softmax of tile 0 and 1, warp 0 loads, warp 1 issues the products: while one tile's
// weights are computed the tensor cores run the other's products. m is a reference that the row's maximum exceeds by at
// most 8 (powers of two), so O in TMEM is rescaled only when a maximum moves by more; O / l does not depend on it.
// P's rounding to bf16 is that of a bf16 tensor product; S, m, l and O stay in fp32.
#include "common.cuh"
#include "host.cuh"
#include "paged.cuh"
#include "paged_prefill.cuh"

using namespace q3t;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTileKeys = 128, kTileRows = 128;
constexpr int kStages = 2;  // of K, and of V
constexpr int kThreads = 384;

struct PrefillArgs {
  PageTable pages;
  const int64_t *row_offsets, *start_positions;
  __nv_bfloat16* out;
  int rows, sequences, q_heads, kv_heads, group;
  int heads;    // query heads of a tile: the group, in passes of 64 where it is wider
  int passes, positions;  // passes over the group; positions of a tile
  int piece;    // rows of a TMA box: gcd(page_size, 128)
  int capacity; // positions that a page table row can hold
  float scale_log2;
  unsigned* status;
};

template <int D>
struct Smem {
  static constexpr int kTile = 128 * D * 2;  // a query, key or value tile: D / 64 blocks of 128 rows x 128 bytes
  static constexpr int kBlock = 128 * 128;
  static constexpr int kK = 2 * kTile, kV = kK + kStages * kTile, kBar = kV + kStages * kTile;
  static constexpr int kBytes = kBar + 256 + 1024;
};

struct Bars {
  uint64_t q_full[2], k_full[kStages], v_full[kStages], turn[2], s_full[2], p_full[2][2], o_done[2], done;
  uint32_t tmem;
};

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
Q3T_DEV void tmem_st32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(addr)
      : "memory");
}
Q3T_DEV void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
Q3T_DEV void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
Q3T_DEV float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two fp32 operations in one instruction.
Q3T_DEV float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
Q3T_DEV float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
Q3T_DEV float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Moves registers between the warpgroups: the CTA is launched with kThreads * 168, and 56 + 2 * 224 = 3 * 168.
constexpr int kRegsLoad = 56, kRegsSoftmax = 224;
static_assert(kRegsLoad + 2 * kRegsSoftmax == 3 * 168, "register shares must add up to the launch's");
Q3T_DEV uint32_t pack2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// A bounded wait of a whole warp: every lane leaves with the same answer.
Q3T_DEV bool warp_wait(uint64_t* bar, int phase, unsigned* status, unsigned bits) {
  return __all_sync(0xffffffffu, mbar_wait(bar, phase & 1, status, bits));
}

// What a CTA works on. Work items are numbered from the last tile of the last sequence backwards, so that
// the tiles with the most keys start first.
struct Tile {
  int sequence, row, count;  // first packed row and rows (positions)
  int64_t position;          // of the first row
};

// Found by one warp; count 0: no such tile.
Q3T_DEV Tile find_tile(const PrefillArgs& a, int index, int lane) {
  const int span = 2 * a.positions;
  for (int base = a.sequences - 1; base >= 0; base -= 32) {
    const int s = base - lane;
    int n = 0, first = 0, tiles = 0;
    if (s >= 0) {
      const int64_t lo = a.row_offsets[s], hi = a.row_offsets[s + 1];
      if (lo >= 0 && hi <= a.rows && hi > lo) {
        first = int(lo);
        n = int(hi - lo);
        tiles = (n + span - 1) / span;
      } else if (hi != lo) {
        raise_status(a.status, kStatusBadIndex);
      }
    }
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
    Tile t;
    const int tile = (tiles - 1) - (index - (sum - tiles));  // counted from the sequence's last tile
    t.sequence = __shfl_sync(0xffffffffu, s, src);
    t.row = __shfl_sync(0xffffffffu, first + tile * span, src);
    t.count = __shfl_sync(0xffffffffu, min(span, n - tile * span), src);
    const int in_sequence = __shfl_sync(0xffffffffu, tile * span, src);
    t.position = a.start_positions[t.sequence] + in_sequence;
    return t;
  }
  return Tile{0, 0, 0, 0};
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    paged_prefill_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                         const __grid_constant__ CUtensorMap tmv, const PrefillArgs a) {
  using M = Smem<D>;
  constexpr int kHalves = D / 64;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Bars* bars = reinterpret_cast<Bars*>(smem + M::kBar);
  __shared__ Tile shared_tile;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int units = a.kv_heads * a.passes, unit = int(blockIdx.x % units), head = unit / a.passes;
  const int head0 = head * a.group + unit % a.passes * a.heads;  // first query head
  grid_dependency_wait();
  if (warp == 0) {
    const Tile found = find_tile(a, int(blockIdx.x / units), lane);
    if (lane == 0) shared_tile = found;
  } else if (warp == 1) {
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&bars->q_full[i], 1);
        mbar_init(&bars->s_full[i], 1);
        mbar_init(&bars->turn[i], 1);
        mbar_init(&bars->p_full[i][0], 128);
        mbar_init(&bars->p_full[i][1], 128);
        mbar_init(&bars->o_done[i], 1);
      }
      for (int i = 0; i < kStages; ++i) {
        mbar_init(&bars->k_full[i], 1);
        mbar_init(&bars->v_full[i], 1);
      }
      mbar_init(&bars->done, 1);
      fence_mbar_init();
    }
  }
  __syncthreads();
  const Tile tile = shared_tile;
  if (tile.count == 0) return;
  if (warp == 2) {
    tmem_alloc(&bars->tmem, 512);
    tmem_relinquish();
  }
  // rows, last key + 1 and key tiles of each query tile; keys that the table cannot hold are cut off
  int count[2], key_end[2], tiles[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    count[t] = max(0, min(a.positions, tile.count - t * a.positions));
    const int64_t end = tile.position + t * a.positions + count[t];
    if (count[t] > 0 && end > a.capacity && threadIdx.x == 0) raise_status(a.status, kStatusBadIndex);
    key_end[t] = count[t] == 0 || end < 0 ? 0 : int(end < a.capacity ? end : a.capacity);
    tiles[t] = (key_end[t] + kTileKeys - 1) / kTileKeys;
  }
  const int key_tiles = max(tiles[0], tiles[1]), keys = max(key_end[0], key_end[1]);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;

  if (warp >= 4) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    // ---------------- softmax: thread = query row = TMEM lane
    const int t = (warp >> 2) - 1, m = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + (uint32_t((warp & 3) * 32) << 16);
    const uint32_t s_at = lanes + 128 * t, o_at = lanes + 256 + 128 * t;
    const int p = m / a.heads, h = m % a.heads;
    const bool real = p < count[t] && unit % a.passes * a.heads + h < a.group;
    const int64_t position = tile.position + t * a.positions + p;
    const int last = int(position < -1 ? -1 : position < a.capacity ? position : a.capacity - 1);  // last key seen
    float top = -INFINITY, sum = 0.f;
    bool ok = true;
    for (int j = 0; j < tiles[t]; ++j) {
      if (!warp_wait(&bars->s_full[t], j, a.status, kStatusMmaTimeout)) {
        ok = false;
        break;
      }
      tc_fence_after();
      float s[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(s_at + 32 * c, s + 32 * c);
      tmem_ld_wait();
      const int seen = last + 1 - j * kTileKeys;  // keys of this tile that the row sees
      if (__any_sync(0xffffffffu, seen < kTileKeys)) {
#pragma unroll
        for (int i = 0; i < 128; ++i) s[i] = i < seen ? s[i] : -INFINITY;
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 128; i += 2) mx[i / 2 & 3] = max3(mx[i / 2 & 3], s[i], s[i + 1]);
      const float now = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale_log2;
      if (__any_sync(0xffffffffu, now > top + 8.f || (top == -INFINITY && now > top))) {
        const float to = fmaxf(top, now);
        const float f = to == top ? 1.f : exp2_fast(top - to);
        top = to;
        sum *= f;
        if (j > 0) {  // the products up to tile j - 1 are done: s_full says so
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            float o[32];
            tmem_ld32(o_at + 32 * c, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= f;
            tmem_st32(o_at + 32 * c, reinterpret_cast<const uint32_t*>(o));
          }
        }
      }
      const float ref = top == -INFINITY ? 0.f : top;
      const float2 scale2 = make_float2(a.scale_log2, a.scale_log2), ref2 = make_float2(-ref, -ref);
      float2 part[2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t w[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          float2 x = fma2(make_float2(s[64 * c + 2 * i], s[64 * c + 2 * i + 1]), scale2, ref2);
          x.x = exp2_fast(x.x);
          x.y = exp2_fast(x.y);
          part[i & 1] = add2(part[i & 1], x);
          w[i] = pack2(x.x, x.y);
        }
        tmem_st32(s_at + 32 * c, w);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&bars->p_full[t][c]);
      }
      sum += (part[0].x + part[0].y) + (part[1].x + part[1].y);
    }
    // ---- O / l
    if (tiles[t] > 0) ok = ok && warp_wait(&bars->o_done[t], 0, a.status, kStatusMmaTimeout);
    tc_fence_after();
    __nv_bfloat16* to = a.out + (int64_t(tile.row + t * a.positions + p) * a.q_heads + head0 + h) * D;
    const float inv = last < 0 ? 0.f : 1.f / sum;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      float o[32];
      if (tiles[t] > 0 && ok) {  // uniform over the warp
        tmem_ld32(o_at + 32 * c, o);
        tmem_ld_wait();
      }
      if (real && ok) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = last < 0 ? 0.f : o[8 * i + e] * inv;
          *reinterpret_cast<uint4*>(to + 32 * c + 8 * i) = pack8(v);
        }
      }
    }
    tc_fence_before();
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsLoad));
  if (warp == 0) {
    // ---------------- loads
    bool ok = true;
    if (lane == 0) {
      for (int t = 0; t < 2; ++t) {
        if (tiles[t] == 0) continue;
        mbar_expect_tx(&bars->q_full[t], uint32_t(a.heads * a.positions * 128 * kHalves));
        for (int h = 0; h < kHalves; ++h)
          tma_load_3d(smem + t * M::kTile + h * M::kBlock, &tmq, &bars->q_full[t], h * 64, head0,
                      tile.row + t * a.positions, policy_evict_first());
      }
    }
    // lane: (piece of the tile, 64-dim block)
    const int pieces = kTileKeys / a.piece, piece = lane / kHalves, half = lane % kHalves;
    auto page_of = [&](int j) {  // the page of this lane's piece of tile j, and its row there
      int2 at = make_int2(int(a.pages.pages), 0);  // past the pool: a load of zeros
      const int key = j * kTileKeys + piece * a.piece;
      if (piece < pieces && key < keys) {
        const int64_t page = a.pages.lookup(tile.sequence, key);
        if (page >= 0) at = make_int2(int(page), key % a.pages.page_size);
        else raise_status(a.status, kStatusBadIndex);
      }
      return at;
    };
    int2 next = page_of(0);
    int loaded = 0;
    for (int j = 0; j < key_tiles && ok; ++j) {
      const int s = j % kStages;
      const int2 at = next;
      const int wanted = min(pieces, (keys - j * kTileKeys + a.piece - 1) / a.piece);  // pieces that hold a key
      const uint32_t bytes = uint32_t(wanted * a.piece * 128 * kHalves);
#pragma unroll
      for (int v = 0; v < 2 && ok; ++v) {
        // turn i of the products has read key tile i and value tile i - 1
        const int turn = j - kStages + v;
        if (j >= kStages) ok = warp_wait(&bars->turn[turn & 1], turn >> 1, a.status, kStatusMmaTimeout);
        if (!ok) break;
        uint64_t* full = v ? &bars->v_full[s] : &bars->k_full[s];
        if (lane == 0) mbar_expect_tx(full, bytes);
        __syncwarp();
        if (piece < wanted)
          tma_load_4d(smem + (v ? M::kV : M::kK) + s * M::kTile + half * M::kBlock + piece * a.piece * 128, v ? &tmv : &tmk,
                      full, half * 64, at.y, head, at.x);
        ++loaded;
      }
      if (j + 1 < key_tiles) next = page_of(j + 1);
    }
    if (!ok)  // loads still in flight land before the CTA leaves
      for (int i = max(0, loaded - 2 * kStages); i < loaded; ++i)
        mbar_wait(i & 1 ? &bars->v_full[(i / 2) % kStages] : &bars->k_full[(i / 2) % kStages], (i / 2 / kStages) & 1, a.status,
                  kStatusTmaTimeout);
  } else if (warp == 1) {
    // ---------------- products (TMEM column 0 is the allocation's first: it is all of TMEM)
    constexpr uint32_t idesc_s = umma_idesc_bf16(128, kTileKeys);
    constexpr uint32_t idesc_o = umma_idesc_bf16(128, D) | (1u << 16);  // V MN-major
    const uint32_t base = smem_u32(smem);
    const bool leader = elect_one();
    bool ok = true;
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
    if (key_tiles > 0) {
      wait(&bars->k_full[0], 0, kStatusTmaTimeout);
      for (int t = 0; t < 2; ++t) {
        if (tiles[t] == 0) continue;
        wait(&bars->q_full[t], 0, kStatusTmaTimeout);
        tc_fence_after();
        if (ok) scores(t, 0);
      }
      if (ok) commit_if(&bars->turn[0], leader);
    }
    for (int j = 0; j < key_tiles && ok; ++j) {
      const int s = j % kStages, phase = j / kStages, sn = (j + 1) % kStages;
      wait(&bars->v_full[s], phase, kStatusTmaTimeout);
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
      if (j + 1 < key_tiles) wait(&bars->k_full[sn], (j + 1) / kStages, kStatusTmaTimeout);
      const uint32_t v = desc_mn(base + M::kV + s * M::kTile, M::kBlock);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (j >= tiles[t]) continue;
#pragma unroll
        for (int half = 0; half < 2; ++half) {  // the first 64 keys' weights come before the others are computed
          wait(&bars->p_full[t][half], j, kStatusMmaTimeout);
          tc_fence_after();
          if (!ok) continue;
#pragma unroll
          for (int i = 4 * half; i < 4 * half + 4; ++i)
            mma_ts(256 + 128 * t, 128 * t + 8 * i, v + 128 * i, idesc_o, j > 0 || i > 0, leader);
        }
        if (!ok) continue;
        if (j + 1 < tiles[t]) scores(t, sn);
        else commit_if(&bars->o_done[t], leader);
      }
      if (ok) commit_if(&bars->turn[(j + 1) & 1], leader);
    }
    if (lane == 0) {  // every product is done before TMEM is released
      umma_commit(&bars->done);
      mbar_wait(&bars->done, 0, a.status, kStatusMmaTimeout);
    }
  }
  }
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
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
  return launch(paged_prefill_kernel<D>, dim3(unsigned(blocks)), dim3(kThreads), size_t(Smem<D>::kBytes), stream, true, name,
                tmq, tmk, tmv, a);
}

}  // namespace

namespace q3t {

bool prefill_tiles_supported(const q3t_paged_prefill& p) {
  const q3t_paged_cache& c = p.cache;
  return p.scale > 0. && p.scale < 1e30 && c.table_columns * c.page_size < (int64_t(1) << 30) && p.rows < (int64_t(1) << 28);
}

int launch_prefill_tiles(const q3t_paged_prefill& p, unsigned* status, void* stream, const char* name) {
  const q3t_paged_cache& c = p.cache;
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
  a.heads = a.group < 64 ? a.group : 64;
  a.passes = (a.group + a.heads - 1) / a.heads;
  a.positions = kTileRows / a.heads;
  a.piece = 16;
  while (a.piece < kTileKeys && c.page_size % (2 * a.piece) == 0) a.piece *= 2;
  a.capacity = int(c.table_columns * c.page_size);
  a.scale_log2 = float(p.scale) * kLog2e;
  a.status = status;
  // every sequence may end inside a tile
  const int64_t tiles = p.rows / (2 * a.positions) + p.sequences, blocks = tiles * a.kv_heads * a.passes;
  if (blocks > 2147483647) return fail(Q3T_EINVAL, "%s: too many rows", name);
  return c.head_dim == 128 ? launch_prefill<128>(p, a, blocks, stream, name) : launch_prefill<64>(p, a, blocks, stream, name);
}

}  // namespace q3t
