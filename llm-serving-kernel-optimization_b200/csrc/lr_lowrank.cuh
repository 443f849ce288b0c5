// lr_lowrank.cuh -- rows times a short inner dimension (up to 128), added to or
// combined with base rows: the second half of the low-rank adapters and the row
// gradient of the gate projection.
#pragma once

#include "lr_common.cuh"

namespace lr {

constexpr int kAdWarps = 8;
constexpr int kAdThreads = kAdWarps * 32;
constexpr int kMaxRank = 128;

LR_DEVICE void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                       uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same with a zero accumulator.
LR_DEVICE void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                             uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

LR_DEVICE uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
LR_DEVICE uint32_t cluster_nctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
// Of every thread of the cluster; the barrier takes a warp's lanes together.
LR_DEVICE void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;"
               ::: "memory");
}
LR_DEVICE float ld_cluster_f32(uint32_t saddr, uint32_t rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
// Plain 16-byte read that leaves L1 alone (rows read once; may be written in place later).
LR_DEVICE uint4 ld_row(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}

LR_DEVICE uint2 ld_row8(const __half* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];"
               : "=r"(v.x), "=r"(v.y)
               : "l"(p)
               : "memory");
  return v;
}

// Read-only loads that stay where they are issued (ahead of their use).
LR_DEVICE uint4 ld_ahead16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
LR_DEVICE uint2 ld_ahead8(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
LR_DEVICE void cp_async_16(void* smem, const void* gmem) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem)), "l"(gmem)
               : "memory");
}
// Zeros instead of a copy where !ok (gmem is then not read).
LR_DEVICE void cp_async_16_zfill(void* smem, const void* gmem, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem)), "l"(gmem),
               "r"(ok ? 16 : 0)
               : "memory");
}
LR_DEVICE void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
LR_DEVICE void cp_async_wait_group() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// Arrives on an mbarrier when this thread's earlier cp.async have landed.
LR_DEVICE void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
LR_DEVICE void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// ---------------------------------------------------------------------------
// a window's groups
// ---------------------------------------------------------------------------
struct Groups {
  int32_t adapter[64];  // per row: its adapter, -1 none, -2 past the last row
  int32_t group[64];    // per row: its group, -1 for no group
  int32_t first[64];    // per group: its first row
  int n;
  int uniform;          // every row has the same adapter
};

// Warp 0 groups the W <= 64 rows from row0 by adapter.  Rows without one make
// a group of their own when `with_none`.  The caller synchronises the block.
template <int W>
LR_DEVICE void group_rows(Groups& s, const int32_t* __restrict__ index, long row0, long R, int n,
                          bool with_none, int32_t* err) {
  const int lane = threadIdx.x & 31;
  int a[2], lead[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int t = u * 32 + lane;
    a[u] = -2;
    if (t < W && row0 + t < R) {
      a[u] = __ldcg(index + row0 + t);
      if (a[u] < -1 || a[u] >= n) {
        report(err, LR_DEVERR_BAD_ADAPTER);
        a[u] = -1;
      }
    }
    const unsigned peers = __match_any_sync(0xffffffffu, a[u]);
    lead[u] = u * 32 + __ffs(peers) - 1;
  }
  const int lowest = with_none ? -1 : 0;
  unsigned la = __ballot_sync(0xffffffffu, lead[0] == lane && a[0] >= lowest);
  if (W > 32) {  // a group of the upper rows may have started in the lower ones
    for (unsigned m = la; m; m &= m - 1) {
      const int r = __ffs(m) - 1;
      const int ar = __shfl_sync(0xffffffffu, a[0], r);
      if (a[1] == ar) lead[1] = r;
    }
  }
  const unsigned lb = __ballot_sync(0xffffffffu, W > 32 && lead[1] == 32 + lane && a[1] >= lowest);
  const unsigned long long leaders = la | (static_cast<unsigned long long>(lb) << 32);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int t = u * 32 + lane;
    if (t < W) {
      const int slot = __popcll(leaders & ((1ull << lead[u]) - 1));
      s.adapter[t] = a[u];
      s.group[t] = a[u] >= lowest ? slot : -1;
      if (a[u] >= lowest && lead[u] == t) s.first[slot] = t;
    }
  }
  const int a0 = __shfl_sync(0xffffffffu, a[0], 0);
  const bool same = __all_sync(0xffffffffu, (a[0] == a0 || a[0] == -2) && (a[1] == a0 || a[1] == -2));
  if (lane == 0) {
    s.n = __popcll(leaders);
    s.uniform = same && a0 >= 0;
  }
}

// Warps per group (a power of two) when g groups share the block's warps.
LR_DEVICE int warps_per_group(int g) { return g <= 1 ? 8 : g <= 2 ? 4 : g <= 4 ? 2 : 1; }

// Powers of two that take a largest finite value m into [2^14, 2^15) and back, both
// normal numbers: 2^-113 to 2^126.  Below 2^-112 m stays under 2^14; two fp16 terms
// then leave 2^-25 of 2^-126 over, less than fp32's own spacing.
LR_DEVICE void half_range_scale(float m, float& up, float& down) {
  const int ex = m > 0.f ? min(126, 141 - int(__float_as_uint(m) >> 23)) : 0;
  up = __uint_as_float(unsigned(127 + ex) << 23);
  down = __uint_as_float(unsigned(127 - ex) << 23);
}

// ---------------------------------------------------------------------------
// expand: out[row] = base[row] + s_a v[row] . B_a^T   (or the SwiGLU of two)
// ---------------------------------------------------------------------------
// mma m16n8k16 with the window's rows as M (MT tiles of 16) and output columns
// as N.  v enters as two fp16 terms of the row scaled by a power of two to
// [2^14, 2^15) (value and remainder: 2^-22 of the row's largest, no overflow),
// so v is not rounded to fp16.  The terms are written to shared memory in
// fragment order: one 16-byte read is a lane's A operand.  n-tile j, column c
// stands for output column (c >> 1) * 8 + 2 j + (c & 1) of the warp's 32: a lane
// ends with 8 neighbouring columns of its two rows, one 16-byte read of the base
// and one store each.
// 16384 x 14336, rank 32: 175 to 190 us, 5 TB/s of base in and out (floor 143), HBM
// 64 % and the tensor pipe 32 % busy; of the 126 instructions around 16 rows x 32
// columns 16 are mma and 44 convert, add and round, under the power cap's clock.
// Largest sizes taken: row numbers plus a tile, and 64 rows' offsets, stay in 32 bits.
constexpr int kMaxRows = 0x7fffffff - 1023;
constexpr int kMaxColumns = 1 << 26;
constexpr uint64_t kCopyWaitNs = 1000000000ull;  // bound of every wait for a copy

enum ExpandMode : int {
  kExpandAdd = 0,      // base + delta
  kExpandSwiglu = 1,   // silu(base + delta) * (base2 + delta2)
  kExpandProduct = 2,  // delta alone, every row with entry 0 of b (no index)
  kExpandProduct32 = 3,  // the same, out in fp32
};

constexpr bool is_product(int mode) {
  return mode == kExpandProduct || mode == kExpandProduct32;
}

struct ExpandArgs {
  const float* v;  // [bank][R][r]
  const __half* b[2];  // [n][N][ldb], zero past r
  const float* scale[2];
  const int32_t* index;
  const __half* base[2];  // the base rows; gate and up rows for SwiGLU
  void* out;  // fp16; fp32 for kExpandProduct32
  long R;
  int N, n, r, ldb;
  int groups_per_chunk;  // 32-column groups of a block
  bool in_place;
  int32_t* err;
};

// The weights of a warp's 32 columns stay in registers while its row tiles pass.
// RV is the rank rounded up to 16 (8-byte loads: one mma step), 32, 64 or 128
// (16-byte loads: two steps per 32).
template <int RV>
struct RankTile {
  static constexpr int kPer = RV == 16 ? 4 : 8;     // rank values of a lane's load
  static constexpr int kLoads = RV == 16 ? 1 : RV / 32;
  static constexpr int kSteps = RV / 16;            // mma steps
  uint32_t w[kSteps][4][2];

  // Columns n0 + (g >> 1) * 8 + 2 j + (g & 1); bp points at (that column for j = 0, tq * kPer).
  // With a distance of 1: columns n0 + 4 g + j.
  template <int DISTANCE = 2>
  LR_DEVICE void load(const __half* __restrict__ bp, int ldb, bool ok, int tq) {
#pragma unroll
    for (int b = 0; b < kLoads; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = ok && b * 32 + tq * kPer < ldb;
        const __half* q = bp + (unsigned(DISTANCE * j) * unsigned(ldb) + b * 32);
        if (RV == 16) {
          uint2 v = make_uint2(0, 0);
          if (in) v = ld_ahead8(q);
          w[0][j][0] = v.x;
          w[0][j][1] = v.y;
        } else {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (in) v = ld_ahead16(q);
          w[2 * b][j][0] = v.x;
          w[2 * b][j][1] = v.y;
          w[(2 * b + 1) % kSteps][j][0] = v.z;
          w[(2 * b + 1) % kSteps][j][1] = v.w;
        }
      }
  }

  // acc = the row tile's two terms (`lo` after `hi`: [step][lane]) . weights
  LR_DEVICE void multiply(float (&acc)[4][4], const uint4* hi, const uint4* lo) const {
#pragma unroll
    for (int t = 0; t < kSteps; ++t) {
      const uint4 a = hi[t * 32];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (t == 0)
          mma_f16_first(acc[j], a.x, a.y, a.z, a.w, w[t][j][0], w[t][j][1]);
        else
          mma_f16(acc[j], a.x, a.y, a.z, a.w, w[t][j][0], w[t][j][1]);
      }
    }
#pragma unroll
    for (int t = 0; t < kSteps; ++t) {
      const uint4 a = lo[t * 32];
#pragma unroll
      for (int j = 0; j < 4; ++j) mma_f16(acc[j], a.x, a.y, a.z, a.w, w[t][j][0], w[t][j][1]);
    }
  }

  // The weights as the A operand (32 columns) and 8 rows' terms as B: `v` holds
  // [step][lane] of (value, value, remainder, remainder).
  LR_DEVICE void multiply_rows(float (&acc)[2][4], const uint4* v) const {
#pragma unroll
    for (int t = 0; t < kSteps; ++t) {
      const uint4 q = v[t * 32];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (t == 0)
          mma_f16_first(acc[i], w[t][2 * i][0], w[t][2 * i + 1][0], w[t][2 * i][1],
                        w[t][2 * i + 1][1], q.x, q.y);
        else
          mma_f16(acc[i], w[t][2 * i][0], w[t][2 * i + 1][0], w[t][2 * i][1],
                  w[t][2 * i + 1][1], q.x, q.y);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
        mma_f16(acc[i], w[t][2 * i][0], w[t][2 * i + 1][0], w[t][2 * i][1], w[t][2 * i + 1][1],
                q.z, q.w);
    }
  }
};

// Place of rank values (c, c + 1), c even, of row t among a window's fragments
// [row tile][step][lane][4 words]: the words of a lane are (row g, first k),
// (row g + 8, first k), (row g, second k), (row g + 8, second k).
template <int RV>
LR_DEVICE int fragment_word(int t, int c) {
  const int m = t >> 4, h = (t >> 3) & 1, g = t & 7;
  int step, tq, kh;
  if (RV == 16) {
    step = 0;
    tq = c >> 2;
    kh = (c >> 1) & 1;
  } else {
    step = (c >> 5) * 2 + ((c >> 2) & 1);
    tq = (c >> 3) & 3;
    kh = (c >> 1) & 1;
  }
  return ((m * (RV / 16) + step) * 32 + g * 4 + tq) * 4 + kh * 2 + h;
}

// Windows of 16 rows: groups whose weights are in flight together.
template <int RV, int MODE>
constexpr int expand_ahead() {
  // as many as 64 registers hold; SwiGLU's two banks leave room for half of that
  return MODE == kExpandSwiglu ? (RV == 16 ? 2 : 1) : RV <= 64 ? 128 / RV : 1;
}

// Larger windows stream the base rows: stages of the window's rows x 224 columns
// by cp.async of a producer warp, a row per instruction, to seven consumer warps of
// 32 columns.  (A ninth warp for the producer would cost the others a quarter of
// their registers at two blocks on an SM: 18 warps do not spread over its four
// parts.)  Without base rows all eight warps consume.
template <int MODE>
constexpr int consumers() {
  return is_product(MODE) ? kAdWarps : kAdWarps - 1;
}
constexpr int kTilePitch = (kAdWarps - 1) * 64;  // bytes, 64 mod 128: neighbouring rows in
                                                 // different banks
template <int MODE>
constexpr int tile_stages() {
  return MODE == kExpandSwiglu ? 2 : 3;
}

template <int RV, int MT, int MODE>
constexpr int expand_base_bytes() {
  return is_product(MODE) || MT == 1
             ? 0
             : tile_stages<MODE>() * (MODE == kExpandSwiglu ? 2 : 1) * MT * 16 * kTilePitch;
}

template <int RV, int MT, int MODE>
constexpr int expand_smem_bytes() {
  return expand_base_bytes<RV, MT, MODE>() + (MODE == kExpandSwiglu ? 2 : 1) * 2 * MT * 16 * RV * 2;
}

// Two blocks on an SM (128 registers a thread) where the weights leave room for it.
template <int RV, int MT, int MODE>
constexpr int expand_min_blocks() {
  return RV <= (MODE == kExpandSwiglu ? (MT == 1 ? 32 : 16) : 64) ? 2 : 1;
}

template <int MODE>
struct ExpandOut {
  using type = __half;
};
template <>
struct ExpandOut<kExpandProduct32> {
  using type = float;
};

// Eight results of a row of the fp32 product, unrounded.
LR_DEVICE void store_product32(float* to, const float (&acc)[1][4][4], int h, float fac) {
  float4 o[2];
  o[0] = make_float4(acc[0][0][2 * h] * fac, acc[0][0][2 * h + 1] * fac, acc[0][1][2 * h] * fac,
                     acc[0][1][2 * h + 1] * fac);
  o[1] = make_float4(acc[0][2][2 * h] * fac, acc[0][2][2 * h + 1] * fac, acc[0][3][2 * h] * fac,
                     acc[0][3][2 * h + 1] * fac);
  reinterpret_cast<float4*>(to)[0] = o[0];
  reinterpret_cast<float4*>(to)[1] = o[1];
}

// Eight results of a row: base (and base2) with the scaled sums of both banks.
template <int MODE, int BANKS>
LR_DEVICE uint4 expand_epilogue(const float (&acc)[BANKS][4][4], int h, const float (&fac)[BANKS],
                                const uint4 (&base)[BANKS]) {
  float o[BANKS][8];
#pragma unroll
  for (int bk = 0; bk < BANKS; ++bk) {
    const __half2* bh = reinterpret_cast<const __half2*>(&base[bk]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 b2 = is_product(MODE) ? make_float2(0.f, 0.f) : __half22float2(bh[j]);
      o[bk][2 * j] = fmaf(acc[bk][j][2 * h], fac[bk], b2.x);
      o[bk][2 * j + 1] = fmaf(acc[bk][j][2 * h + 1], fac[bk], b2.y);
    }
  }
  if (MODE == kExpandSwiglu) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[0][i] = silu_f32(o[0][i]) * o[BANKS - 1][i];
  }
  return pack_half8(o[0]);
}

template <int RV, int MT, int MODE>
__global__ void __launch_bounds__(kAdThreads, expand_min_blocks<RV, MT, MODE>())
    expand_kernel(ExpandArgs p) {
  constexpr int W = 16 * MT;
  constexpr int BANKS = MODE == kExpandSwiglu ? 2 : 1;
  constexpr int kTerm = W * RV / 8;  // uint4 of one term of v
  constexpr int kTileGroups = consumers<MODE>(), kTileStages = tile_stages<MODE>();
  constexpr int kProducer = kTileGroups;  // the producer warp
  extern __shared__ __align__(128) unsigned char s_dyn[];  // base rows, then v
  uint4* s_v = reinterpret_cast<uint4*>(s_dyn + expand_base_bytes<RV, MT, MODE>());
  // s_v: [bank][hi, lo][row tile][step][lane]
  __shared__ uint64_t s_full[kTileStages], s_empty[kTileStages];
  __shared__ int s_abort;
  __shared__ Groups s;
  __shared__ float s_fac[BANKS][W];
  // Only v comes from the launch before (shrink, which lets this one start after its
  // own wait): index, base rows and weights are read ahead of that launch's end.
  // A product's weights are its predecessor's, too.
  if (is_product(MODE)) {
    pdl_wait();
    pdl_trigger();
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  const long row0 = long(blockIdx.x) * W;
  const int nrows = int(min(long(W), p.R - row0));
  const int cg0 = blockIdx.y * p.groups_per_chunk;
  const int cg1 = min(cg0 + p.groups_per_chunk, (p.N + 31) / 32);
  if (!is_product(MODE) && warp == 0)
    group_rows<W>(s, p.index, row0, p.R, p.n, !p.in_place, nullptr);
  if (MT > 1 && !is_product(MODE) && threadIdx.x == 32) {
    for (int i = 0; i < kTileStages; ++i) {
      mbar_init(s_full + i, 32);  // the producer's lanes
      mbar_init(s_empty + i, kTileGroups);
    }
    s_abort = 0;
    fence_mbarrier_init();
  }
  __syncthreads();
  const bool stream = MT > 1 && !is_product(MODE) && s.n > 0;

  // Producer: tiles [first, last) of the base rows, each as soon as its stage has
  // been read.  The first stages start ahead of everything else.
  const int n_tiles = (cg1 - cg0 + kTileGroups - 1) / kTileGroups;
  const auto produce = [&](int first, int last) {
    for (int i = first; i < last; ++i) {
      const int st = i % kTileStages, round = i / kTileStages, cg = cg0 + i * kTileGroups;
      if (round > 0 &&
          !mbar_wait_warp(s_empty + st, (round - 1) & 1, &s_abort, p.err, kCopyWaitNs))
        return;
      if (lane < kTileGroups * 4 && cg * 32 + lane * 8 < p.N) {
#pragma unroll
        for (int bk = 0; bk < BANKS; ++bk) {
          const __half* from = p.base[bk] + size_t(row0) * p.N + cg * 32 + lane * 8;
          unsigned char* to = s_dyn + (st * BANKS + bk) * W * kTilePitch + lane * 16;
#pragma unroll 8
          for (int t = 0; t < nrows; ++t)
            cp_async_16(to + t * kTilePitch, from + size_t(unsigned(t) * unsigned(p.N)));
        }
      }
      cp_async_arrive(s_full + st);
    }
  };
  if (stream && warp == kProducer) produce(0, min(n_tiles, kTileStages));

  // Windows of 16 rows: the weights of groups [g0, g0 + S) for column group c.
  constexpr int S = MT == 1 ? expand_ahead<RV, MODE>() : 1;
  const int n_groups = is_product(MODE) ? 1 : s.n;
  RankTile<RV> wt[S][BANKS];
  const auto group_weights = [&](int c, int g0) {
    const int nr = c * 32 + (g >> 1) * 8;
#pragma unroll
    for (int u = 0; u < S; ++u) {
      const int ad = is_product(MODE) ? 0
                     : g0 + u < n_groups    ? s.adapter[s.first[g0 + u]]
                                            : -1;
#pragma unroll
      for (int bk = 0; bk < BANKS; ++bk)
        wt[u][bk].load(p.b[bk] + (size_t(max(ad, 0)) * p.N + nr + (g & 1)) * p.ldb +
                           tq * RankTile<RV>::kPer,
                       p.ldb, ad >= 0 && c < cg1 && nr < p.N, tq);
    }
  };
  // The first ones are in flight while v is prepared where the registers allow it
  // (SwiGLU and rank 64 lose more to spills).
  constexpr bool EARLY = MT == 1 && RV == 16 && MODE == kExpandAdd;
  if (EARLY) group_weights(cg0 + warp, 0);
  if (!is_product(MODE)) {
    pdl_wait();
    pdl_trigger();
  }
  {  // v: fp32 -> scaled (value, remainder) pairs in fragment order
    constexpr int LPR = kAdThreads / W;               // lanes of a row
    constexpr int EL = (RV / 2 + LPR - 1) / LPR;      // pairs of a lane
    const int t = threadIdx.x / LPR, q = threadIdx.x % LPR;
    const int ad = is_product(MODE) ? (t < nrows ? 0 : -1) : s.adapter[t];
#pragma unroll
    for (int bk = 0; bk < BANKS; ++bk) {
      const float* row = p.v + (size_t(bk) * p.R + row0 + t) * p.r;
      float val[EL][2];
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < EL; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int c = 2 * (i * LPR + q) + e;
          val[i][e] = ad >= 0 && c < p.r ? __ldcg(row + c) : 0.f;
          const float a = fabsf(val[i][e]);
          if (a < INFINITY) m = fmaxf(m, a);
        }
#pragma unroll
      for (int o = 1; o < LPR; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      float up, down;
      half_range_scale(m, up, down);
      uint32_t* hi = reinterpret_cast<uint32_t*>(s_v + 2 * bk * kTerm);
      uint32_t* lo = hi + 4 * kTerm;
#pragma unroll
      for (int i = 0; i < EL; ++i) {
        const int c = 2 * (i * LPR + q);
        if (c < RV) {
          __half h[2], l[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float x = val[i][e] * up;
            h[e] = __float2half_rn(x);
            const float hf = __half2float(h[e]);
            l[e] = __float2half_rn(fabsf(hf) < INFINITY ? x - hf : 0.f);
          }
          const int at = fragment_word<RV>(t, c);
          hi[at] = __half_as_ushort(h[0]) | (uint32_t(__half_as_ushort(h[1])) << 16);
          lo[at] = __half_as_ushort(l[0]) | (uint32_t(__half_as_ushort(l[1])) << 16);
        }
      }
      if (q == 0)
        s_fac[bk][t] = ad >= 0 ? (p.scale[bk] ? __ldg(p.scale[bk] + ad) : 1.f) * down : 0.f;
    }
  }
  __syncthreads();

  const unsigned n8 = 8u * unsigned(p.N);
  if (MT > 1) {
    // Every consumer takes its 32 of a tile's columns for all rows: a window's groups
    // one after the other (one for a prompt), each on its own row tiles.
    if (!is_product(MODE) && warp == kProducer) {
      if (stream) produce(min(n_tiles, kTileStages), n_tiles);
      cp_async_wait_all();  // leave no copy behind
      return;
    }
    float fac[2 * MT][BANKS];
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i)
#pragma unroll
      for (int bk = 0; bk < BANKS; ++bk) fac[i][bk] = s_fac[bk][g + 8 * i];
    using Out = typename ExpandOut<MODE>::type;
    Out* out = static_cast<Out*>(p.out) + size_t(row0 + g) * p.N + (cg0 + warp) * 32 + tq * 8;
    const unsigned char* bp = s_dyn + g * kTilePitch + warp * 64 + tq * 16;
    const uint4* vp = s_v + lane;
    unsigned st = 0, parity = 0;

    const auto arrived = [&]() {
      return is_product(MODE) ||
             mbar_wait_warp(s_full + st, parity, &s_abort, p.err, kCopyWaitNs);
    };
    // One group's rows of the tile of column group c.  `whole`: the window is one
    // group and `grp` is not looked at; `last`: the tile is not read again.
    const auto multiply = [&](const RankTile<RV>(&wt)[BANKS], int c, const bool whole, int grp,
                              bool last) {
      const bool cok = c < cg1 && c * 32 + tq * 8 < p.N;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        bool mine[2] = {g + 16 * m < nrows, g + 16 * m + 8 < nrows};
        if (!whole) {
          mine[0] = s.group[g + 16 * m] == grp;
          mine[1] = s.group[g + 16 * m + 8] == grp;
        }
        uint4 bs[2][BANKS];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int bk = 0; bk < BANKS; ++bk)
            if (!is_product(MODE))
              bs[h][bk] = *reinterpret_cast<const uint4*>(
                  bp + ((st * BANKS + bk) * W + 16 * m + 8 * h) * kTilePitch);
        if (m == MT - 1 && !is_product(MODE) && last) {
          __syncwarp();
          if (lane == 0) mbar_arrive(s_empty + st);
        }
        if (!whole && !__any_sync(0xffffffffu, mine[0] || mine[1])) continue;
        float acc[BANKS][4][4];
#pragma unroll
        for (int bk = 0; bk < BANKS; ++bk) {
          const uint4* hi = vp + 2 * bk * kTerm + m * (RV / 16) * 32;
          wt[bk].multiply(acc[bk], hi, hi + kTerm);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if constexpr (MODE == kExpandProduct32) {
            if (cok && mine[h])
              store_product32(out + size_t(unsigned(2 * m + h) * n8), acc, h, fac[2 * m + h][0]);
          } else {
            const uint4 o = expand_epilogue<MODE, BANKS>(acc, h, fac[2 * m + h], bs[h]);
            if (cok && mine[h])
              *reinterpret_cast<uint4*>(out + size_t(unsigned(2 * m + h) * n8)) = o;
          }
        }
      }
    };
    const auto advance = [&]() {
      out += kTileGroups * 32;
      if (++st == kTileStages) {
        st = 0;
        parity ^= 1;
      }
    };
    const int end = cg0 + warp + n_tiles * kTileGroups;
    int c = cg0 + warp;
    if (is_product(MODE) || s.uniform) {
      const int ad = is_product(MODE) ? 0 : s.adapter[0];
      const __half* wp[BANKS];
#pragma unroll
      for (int bk = 0; bk < BANKS; ++bk)
        wp[bk] = p.b[bk] + (size_t(ad) * p.N + c * 32 + (g >> 1) * 8 + (g & 1)) * p.ldb +
                 tq * RankTile<RV>::kPer;
      const size_t wstep = size_t(kTileGroups) * 32 * p.ldb;
      const auto weights = [&](RankTile<RV>(&wt)[BANKS], int cw) {
#pragma unroll
        for (int bk = 0; bk < BANKS; ++bk) {
          wt[bk].load(wp[bk], p.ldb, cw < cg1 && cw * 32 + (g >> 1) * 8 < p.N, tq);
          wp[bk] += wstep;
        }
      };
      // the next column group's weights load while one is multiplied
      RankTile<RV> w0[BANKS], w1[BANKS];
      if (RV <= (is_product(MODE) ? 32 : 64) && MODE != kExpandSwiglu) {
        weights(w0, c);
        while (true) {
          weights(w1, c + kTileGroups);
          if (!arrived()) break;
          multiply(w0, c, true, 0, true);
          advance();
          if ((c += kTileGroups) >= end) break;
          weights(w0, c + kTileGroups);
          if (!arrived()) break;
          multiply(w1, c, true, 0, true);
          advance();
          if ((c += kTileGroups) >= end) break;
        }
      } else {
        for (; c < end; c += kTileGroups) {
          weights(w0, c);
          if (!arrived()) break;
          multiply(w0, c, true, 0, true);
          advance();
        }
      }
      return;
    }
    if (n_groups == 0) return;
    for (; c < end; c += kTileGroups) {
      if (!arrived()) break;
      for (int grp = 0; grp < n_groups; ++grp) {
        const int ad = s.adapter[s.first[grp]];
        const int nr = c * 32 + (g >> 1) * 8;
        RankTile<RV> wt[BANKS];  // zeros for the rows without an adapter
#pragma unroll
        for (int bk = 0; bk < BANKS; ++bk)
          wt[bk].load(p.b[bk] + (size_t(max(ad, 0)) * p.N + nr + (g & 1)) * p.ldb +
                          tq * RankTile<RV>::kPer,
                      p.ldb, ad >= 0 && c < cg1 && nr < p.N, tq);
        multiply(wt, c, false, grp, grp == n_groups - 1);
      }
      advance();
    }
    return;
  }

  // Windows of 16 rows: a warp takes its column groups for all of them.  The window's
  // groups come S at a time, all their weights in flight; each is multiplied with
  // every row and kept for its own, so the base rows are finished once, by all lanes.
  int gid[2];
  bool none[2];
  float fac[2][BANKS];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int t = g + 8 * h;
    gid[h] = is_product(MODE) ? (t < nrows ? 0 : -1) : s.group[t];
    none[h] = !is_product(MODE) && s.adapter[t] < 0;
#pragma unroll
    for (int bk = 0; bk < BANKS; ++bk) fac[h][bk] = s_fac[bk][t];
  }
  const size_t row_off = size_t(row0 + g) * p.N + tq * 8;
  for (int c = cg0 + warp; c < cg1; c += kAdWarps) {
    const bool cok = c * 32 + tq * 8 < p.N;
    const size_t off = row_off + c * 32;
    uint4 bs[2][BANKS];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int bk = 0; bk < BANKS; ++bk)
        if (!is_product(MODE) && cok && gid[h] >= 0)
          bs[h][bk] = ld_row(reinterpret_cast<const uint4*>(p.base[bk] + off + h * n8));
    float acc[BANKS][4][4];
#pragma unroll
    for (int bk = 0; bk < BANKS; ++bk)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[bk][j][i] = 0.f;
    for (int g0 = 0; g0 < n_groups; g0 += S) {
      if (!EARLY || g0 > 0 || c > cg0 + warp) group_weights(c, g0);
#pragma unroll
      for (int u = 0; u < S; ++u) {
        if (g0 + u >= n_groups) break;
#pragma unroll
        for (int bk = 0; bk < BANKS; ++bk) {
          float mine[4][4];
          const uint4* hi = s_v + lane + 2 * bk * kTerm;
          wt[u][bk].multiply(mine, hi, hi + kTerm);
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc[bk][j][i] = gid[i >> 1] == g0 + u ? mine[j][i] : acc[bk][j][i];
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (!cok || gid[h] < 0) continue;
      if constexpr (MODE == kExpandProduct32) {
        store_product32(static_cast<float*>(p.out) + off + h * n8, acc, h, fac[h][0]);
      } else {
        uint4 o = expand_epilogue<MODE, BANKS>(acc, h, fac[h], bs[h]);
        if (MODE == kExpandAdd && none[h]) o = bs[h][0];
        *reinterpret_cast<uint4*>(static_cast<__half*>(p.out) + off + h * n8) = o;
      }
    }
  }
}

// Up to 256 rows: windows of 8 rows.  A block's (request, column group) pairs are
// split evenly over its warps in that order, so a warp streams one adapter's columns
// (or two's), the weights and base rows of the next S column groups in flight.  The
// weights are the A operand (16 columns a tile), the window's rows B: half the
// products of a tile of 16 rows, of which a request has one or two; rows of other
// requests are multiplied too and not stored.  A lane ends with 4 neighbouring
// columns of rows 2 tq and 2 tq + 1.  Against 16-row tiles with every group in
// every warp, a pass with shrink outside graphs (in a captured one, whose launches
// carry no programmatic edge, 17 and 33 us): 64 rows of 64 adapters of rank 16, N 14336, 15.5
// us (15.9), of rank 32 21.6 (27); 128 expert rows of SwiGLU pairs 31.5 (32.2), in
// neighbouring pairs 25.3 (27.2); one token, 4096 x 4096, rank 64, 7.5 (8.6).
// Powers of two of warps to a group left warps idle: 33.7 for the expert rows.
// Column groups in flight: twice as many spill registers, half as many leave the
// memory idle (decode batch 20 and 16.5 us against 15).
template <int RV, int MODE>
constexpr int expand_rows_ahead() {
  constexpr int n = (MODE == kExpandSwiglu ? 32 : 64) / RV;
  return n > 0 ? n : 1;
}

template <int RV, int MODE>
constexpr int expand_rows_min_blocks() {
  return RV <= (MODE == kExpandSwiglu ? 32 : 64) ? 2 : 1;
}

template <int RV, int MODE>
__global__ void __launch_bounds__(kAdThreads, expand_rows_min_blocks<RV, MODE>())
    expand_rows_kernel(ExpandArgs p) {
  constexpr int W = 8, BANKS = MODE == kExpandSwiglu ? 2 : 1;
  constexpr int S = expand_rows_ahead<RV, MODE>();
  __shared__ uint4 s_v[BANKS][RV / 16][32];
  __shared__ float s_fac[BANKS][W];
  __shared__ Groups s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  const long row0 = long(blockIdx.x) * W;
  const int cg0 = blockIdx.y * p.groups_per_chunk;
  const int cg1 = min(cg0 + p.groups_per_chunk, (p.N + 31) / 32);
  // as in expand_kernel: only v comes from the launch before
  if (warp == 0) group_rows<W>(s, p.index, row0, p.R, p.n, !p.in_place, nullptr);
  __syncthreads();
  // (group, column group) items in order, an eighth of them to each warp: a warp
  // streams the columns of one or two groups
  const int cols = cg1 - cg0;
  const int first = s.n * cols * warp / kAdWarps, last = s.n * cols * (warp + 1) / kAdWarps;
  RankTile<RV> wt[S][BANKS];
  uint2 bs[S][BANKS][2];
  const size_t row_off = size_t(row0 + 2 * tq) * p.N + 4 * g;
  int left = last - first;                       // items to load
  int lgrp = first / cols, lc = cg0 + first % cols;  // the next one
  int lad = -1;
  bool lmine[2] = {false, false};
  const __half* wp[BANKS];
  const __half* bp[BANKS];
#pragma unroll
  for (int bk = 0; bk < BANKS; ++bk) bp[bk] = p.base[bk] + row_off + lc * 32;
  const auto enter = [&]() {
    if (left > 0) {
      lad = s.adapter[s.first[lgrp]];
      lmine[0] = s.group[2 * tq] == lgrp;
      lmine[1] = s.group[2 * tq + 1] == lgrp;
    }
#pragma unroll
    for (int bk = 0; bk < BANKS; ++bk)
      wp[bk] = p.b[bk] + (size_t(max(lad, 0)) * p.N + lc * 32 + 4 * g) * p.ldb +
               tq * RankTile<RV>::kPer;
  };
  enter();
  const unsigned wstep = 32u * unsigned(p.ldb);
  const auto load = [&](RankTile<RV>(&w)[BANKS], uint2(&base)[BANKS][2]) {
    const bool in = left > 0 && lc * 32 + 4 * g < p.N;
#pragma unroll
    for (int bk = 0; bk < BANKS; ++bk) {
      w[bk].template load<1>(wp[bk], p.ldb, in && lad >= 0, tq);
      wp[bk] += wstep;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (in && lmine[h]) base[bk][h] = ld_row8(bp[bk] + h * size_t(p.N));
      bp[bk] += 32;
    }
    --left;
    if (++lc == cg1) {
      lc = cg0;
      ++lgrp;
#pragma unroll
      for (int bk = 0; bk < BANKS; ++bk) bp[bk] -= cols * 32;
      enter();
    }
  };
#pragma unroll
  for (int u = 0; u < S; ++u) load(wt[u], bs[u]);  // in flight while v is prepared
  pdl_wait();
  pdl_trigger();
  {  // v: a warp per row, fp32 -> scaled (value, remainder) pairs in fragment order
    constexpr int EL = (RV / 2 + 31) / 32;  // pairs of a lane
    const int ad = s.adapter[warp];  // of row `warp`
#pragma unroll
    for (int bk = 0; bk < BANKS; ++bk) {
      const float* row = p.v + (size_t(bk) * p.R + row0 + warp) * p.r;
      float val[EL][2];
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < EL; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int c = 2 * (i * 32 + lane) + e;
          val[i][e] = ad >= 0 && c < p.r ? __ldcg(row + c) : 0.f;
          const float a = fabsf(val[i][e]);
          if (a < INFINITY) m = fmaxf(m, a);
        }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      float up, down;
      half_range_scale(m, up, down);
#pragma unroll
      for (int i = 0; i < EL; ++i) {
        const int c = 2 * (i * 32 + lane);
        if (c < RV) {
          __half h[2], l[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float x = val[i][e] * up;
            h[e] = __float2half_rn(x);
            const float hf = __half2float(h[e]);
            l[e] = __float2half_rn(fabsf(hf) < INFINITY ? x - hf : 0.f);
          }
          const int step = RV == 16 ? 0 : (c >> 5) * 2 + ((c >> 2) & 1);
          const int q = RV == 16 ? c >> 2 : (c >> 3) & 3;
          uint32_t* to = reinterpret_cast<uint32_t*>(&s_v[bk][step][warp * 4 + q]) + ((c >> 1) & 1);
          to[0] = __half_as_ushort(h[0]) | (uint32_t(__half_as_ushort(h[1])) << 16);
          to[2] = __half_as_ushort(l[0]) | (uint32_t(__half_as_ushort(l[1])) << 16);
        }
      }
      if (lane == 0)
        s_fac[bk][warp] = ad >= 0 ? (p.scale[bk] ? __ldg(p.scale[bk] + ad) : 1.f) * down : 0.f;
    }
  }
  __syncthreads();
  float fac[2][BANKS];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int bk = 0; bk < BANKS; ++bk) fac[h][bk] = s_fac[bk][2 * tq + h];
  const int gid[2] = {s.group[2 * tq], s.group[2 * tq + 1]};
  const bool none[2] = {s.adapter[2 * tq] < 0, s.adapter[2 * tq + 1] < 0};
  int i = first, grp = i / cols, c = cg0 + i % cols;
  __half* out = static_cast<__half*>(p.out) + row_off + c * 32;
  while (i < last) {
#pragma unroll
    for (int u = 0; u < S; ++u) {
      if (i >= last) break;
      float acc[BANKS][2][4];
#pragma unroll
      for (int bk = 0; bk < BANKS; ++bk) wt[u][bk].multiply_rows(acc[bk], &s_v[bk][0][lane]);
      const bool cok = c * 32 + 4 * g < p.N;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float o[BANKS][4];
#pragma unroll
        for (int bk = 0; bk < BANKS; ++bk) {
          const __half2* b2 = reinterpret_cast<const __half2*>(&bs[u][bk][h]);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float2 f = __half22float2(b2[x]);
            o[bk][2 * x] = fmaf(acc[bk][x][h], fac[h][bk], f.x);
            o[bk][2 * x + 1] = fmaf(acc[bk][x][2 + h], fac[h][bk], f.y);
          }
        }
        if (MODE == kExpandSwiglu) {
#pragma unroll
          for (int x = 0; x < 4; ++x) o[0][x] = silu_f32(o[0][x]) * o[BANKS - 1][x];
        }
        const __half2 lo = __floats2half2_rn(o[0][0], o[0][1]);
        const __half2 hi = __floats2half2_rn(o[0][2], o[0][3]);
        uint2 r = make_uint2(reinterpret_cast<const uint32_t&>(lo),
                             reinterpret_cast<const uint32_t&>(hi));
        if (MODE == kExpandAdd && none[h]) r = bs[u][0][h];
        if (cok && gid[h] == grp)
          *reinterpret_cast<uint2*>(out + h * size_t(p.N)) = r;
      }
      load(wt[u], bs[u]);
      ++i;
      out += 32;
      if (++c == cg1) {
        c = cg0;
        ++grp;
        out -= cols * 32;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
constexpr long kTargetBlocks = 148;

template <int RV, int MT, int MODE>
static int launch_expand(ExpandArgs p, cudaStream_t stream) {
  if (p.R > kMaxRows || p.N > kMaxColumns) return LR_ERR_INVALID_ARGUMENT;
  constexpr int W = 16 * MT;
  constexpr int smem = expand_smem_bytes<RV, MT, MODE>();
  auto kern = expand_kernel<RV, MT, MODE>;
  static unsigned long long configured = 0;
  if (const int rc = set_dyn_smem_once(kern, smem, configured)) return rc;
  const long windows = (p.R + W - 1) / W;
  const int cgs = (p.N + 31) / 32;
  int gpc = consumers<MODE>();
  if (MT == 1 || is_product(MODE)) {
    // one wave of two blocks per SM where that leaves a warp 1 to 16 groups
    const long per = (windows * cgs + 2 * kTargetBlocks * 8 - 1) / (2 * kTargetBlocks * 8);
    gpc = int(per < 1 ? 1 : per > 16 ? 16 : per) * 8;
  } else {
    // one tile's columns per block, more while the grid stays above eight blocks per SM
    while (gpc < 50 && windows * ((cgs + 2 * gpc - 1) / (2 * gpc)) >= 8 * kTargetBlocks) gpc *= 2;
  }
  p.groups_per_chunk = gpc;
  if (windows > 0x7fffffffL || (cgs + gpc - 1) / gpc > 65535) return LR_ERR_INVALID_ARGUMENT;
  return launch_pdl(kern, dim3(unsigned(windows), (cgs + gpc - 1) / gpc),
                    dim3(kAdThreads), smem, stream, p);
}

template <int RV, int MODE>
static int launch_expand_rows(ExpandArgs p, cudaStream_t stream) {
  if (p.N > kMaxColumns) return LR_ERR_INVALID_ARGUMENT;
  const long windows = (p.R + 7) / 8;
  const int cgs = (p.N + 31) / 32;
  // one wave of two blocks per SM
  const long fit = (windows * cgs + 2 * kTargetBlocks - 1) / (2 * kTargetBlocks);
  const int gpc = int(fit < 4 ? 4 : fit > 128 ? 128 : fit);
  p.groups_per_chunk = gpc;
  if ((cgs + gpc - 1) / gpc > 65535) return LR_ERR_INVALID_ARGUMENT;
  return launch_pdl(expand_rows_kernel<RV, MODE>, dim3(unsigned(windows), (cgs + gpc - 1) / gpc),
                    dim3(kAdThreads), 0, stream, p);
}

constexpr long kSmallRows = 256;  // up to here windows of 8 rows

// Row windows of 64 (32 for SwiGLU), or of 16 while the larger ones would leave
// fewer than two blocks of 256 columns for an SM.
template <int MODE>
static int run_expand(const ExpandArgs& p, cudaStream_t stream) {
  constexpr int MT = MODE == kExpandSwiglu ? 2 : 4;
  const long blocks = (p.R + 16 * MT - 1) / (16 * MT) * ((p.N + 255) / 256);
  const bool small = blocks < 2 * kTargetBlocks;
  if constexpr (!is_product(MODE)) {
    if (p.R <= kSmallRows)
      return p.r <= 16   ? launch_expand_rows<16, MODE>(p, stream)
             : p.r <= 32 ? launch_expand_rows<32, MODE>(p, stream)
             : p.r <= 64 ? launch_expand_rows<64, MODE>(p, stream)
                         : launch_expand_rows<128, MODE>(p, stream);
  }
  if (p.r <= 16)
    return small ? launch_expand<16, 1, MODE>(p, stream) : launch_expand<16, MT, MODE>(p, stream);
  if (p.r <= 32)
    return small ? launch_expand<32, 1, MODE>(p, stream) : launch_expand<32, MT, MODE>(p, stream);
  if (p.r <= 64)
    return small ? launch_expand<64, 1, MODE>(p, stream) : launch_expand<64, MT, MODE>(p, stream);
  return small ? launch_expand<128, 1, MODE>(p, stream) : launch_expand<128, MT, MODE>(p, stream);
}

}  // namespace lr
