// lr_adapters.cu -- low-rank adapters of many requests beside a shared projection (sm_100a).
//
// Row t of x carries an adapter number a = index[t] (-1: none):
//   out_t = base_t + s_a (x_t A_a^T) B_a^T
// or, beside a SwiGLU expert's two projections,
//   out_t = silu(gate_t + D_gate) * (up_t + D_up).
// Two launches: `shrink` writes v = x A^T (rank values per row, fp32), `expand`
// adds v B^T to the base rows.  Rows are taken in windows of neighbours; a
// window's rows are grouped by adapter inside the block (no sort of the batch,
// no host involvement), and the block's 8 warps are dealt out to its groups:
// one group (a prompt's rows) gets all warps, eight groups (decode) a warp each.
// Work is bound by memory: a row costs 2 (K + 2N) bytes and 2 r (K + N)
// operations, so mma.sync with fragments loaded straight into registers keeps
// up and needs no staging through shared memory.
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
LR_DEVICE void cluster_sync() {
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

LR_DEVICE void cp_async_16(void* smem, const void* gmem) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem)), "l"(gmem)
               : "memory");
}
LR_DEVICE void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
LR_DEVICE void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// silu(gate) * up of eight fp16 values
LR_DEVICE uint4 swiglu8(const uint4& gate, const uint4& up) {
  const __half2* a = reinterpret_cast<const __half2*>(&gate);
  const __half2* b = reinterpret_cast<const __half2*>(&up);
  float o[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = __half22float2(a[i]), y = __half22float2(b[i]);
    o[2 * i] = silu_f32(x.x) * y.x;
    o[2 * i + 1] = silu_f32(x.y) * y.y;
  }
  return pack_half8(o);
}

// ---------------------------------------------------------------------------
// a window's groups
// ---------------------------------------------------------------------------
struct Groups {
  int32_t adapter[64];  // per row: its adapter, -1 none, -2 past the last row
  int32_t group[64];    // per row: its group, -1 for no group
  int32_t first[64];    // per group: its first row
  int n;
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
      a[u] = __ldg(index + row0 + t);
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
  if (lane == 0) s.n = __popcll(leaders);
}

// Warps per group (a power of two) when g groups share the block's warps.
LR_DEVICE int warps_per_group(int g) { return g <= 1 ? 8 : g <= 2 ? 4 : g <= 4 ? 2 : 1; }

// ---------------------------------------------------------------------------
// shrink: v[row][r] = x[row] . A_a^T
// ---------------------------------------------------------------------------
// mma m16n8k16 with the rank as M (RB blocks of 16) and the window's rows as N
// (NT tiles of 8).  A lane's 16-byte loads hold 8 neighbouring k of a row; the
// k axis of the product is taken in that order for both operands, so 32 k are
// two mma steps with no shuffle.  K is split over the cluster's blocks and over
// the warps of a group; the parts are added in a fixed order through
// (distributed) shared memory.
struct ShrinkArgs {
  const __half* x;
  const __half* a[2];
  const int32_t* index;
  float* v;  // [bank][R][r]
  long R;
  int K, n, r;
  int32_t* err;
};

template <int RB, int NT>
__global__ void __launch_bounds__(kAdThreads) adapter_shrink_kernel(ShrinkArgs p, int rank_groups) {
  constexpr int W = 8 * NT;
  constexpr int RK = 16 * RB;
  constexpr int PITCH = W + 2;
  // k-blocks whose loads are in flight together: 12 to 16 16-byte loads per lane
  constexpr int U = NT == 1 ? (RB == 1 ? 4 : RB == 2 ? 3 : 2) : (RB == 4 ? 1 : 2);
  extern __shared__ float s_part[];  // [kAdWarps][RK][PITCH]
  __shared__ Groups s;
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  const int cs = int(cluster_nctarank()), cr = int(cluster_ctarank());
  const long row0 = long(blockIdx.x / cs) * W;
  const int bank = blockIdx.y / rank_groups, rank0 = (blockIdx.y % rank_groups) * RK;
  const int per_round = kAdWarps / gridDim.z;  // groups a block takes at a time
  if (warp == 0) group_rows<W>(s, p.index, row0, p.R, p.n, false, bank == 0 ? p.err : nullptr);
  __syncthreads();
  const int nb = (p.K + 31) / 32;
  for (int base = blockIdx.z * per_round; base < s.n; base += kAdWarps) {
    const int ng = min(per_round, s.n - base);
    const int wpg = warps_per_group(ng);
    const int grp = warp / wpg, sub = warp % wpg;
    float acc[RB][NT][4];
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[i][j][c] = 0.f;
    if (grp < ng) {
      const int slot = base + grp;
      const int ad = s.adapter[s.first[slot]];
      // Rank rows past r and rows of other groups read a valid row instead: their
      // products land in values that nobody takes.
      const __half* ap = (bank ? p.a[1] : p.a[0]) + size_t(ad) * p.r * p.K + tq * 8;
      const __half* arow[2 * RB];
#pragma unroll
      for (int i = 0; i < 2 * RB; ++i) {
        const int rk = rank0 + i * 8 + g;
        arow[i] = ap + size_t(rk < p.r ? rk : 0) * p.K;
      }
      const __half* xrow[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int t = s.group[j * 8 + g] == slot ? j * 8 + g : s.first[slot];
        xrow[j] = p.x + size_t(row0 + t) * p.K + tq * 8;
      }
      auto load = [&](uint4(&av)[2 * RB], uint4(&xv)[NT], int kb) {
#pragma unroll
        for (int i = 0; i < 2 * RB; ++i)
          av[i] = __ldg(reinterpret_cast<const uint4*>(arow[i] + kb * 32));
#pragma unroll
        for (int j = 0; j < NT; ++j)
          xv[j] = ld_row(reinterpret_cast<const uint4*>(xrow[j] + kb * 32));
      };
      auto multiply = [&](const uint4(&av)[2 * RB], const uint4(&xv)[NT]) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < RB; ++i) {
            const uint4 lo = av[2 * i], hi = av[2 * i + 1], x = xv[j];
            mma_f16(acc[i][j], lo.x, hi.x, lo.y, hi.y, x.x, x.y);
            mma_f16(acc[i][j], lo.z, hi.z, lo.w, hi.w, x.z, x.w);
          }
      };
      const int part = cr * wpg + sub, parts = cs * wpg;
      const int kb0 = int(long(nb) * part / parts), kb1 = int(long(nb) * (part + 1) / parts);
      const int kfull = min(kb1, p.K / 32);  // a last block of fewer than 32 k comes apart
      int kb = kb0;
      for (; kb + U <= kfull; kb += U) {
        uint4 av[U][2 * RB], xv[U][NT];
#pragma unroll
        for (int u = 0; u < U; ++u) load(av[u], xv[u], kb + u);
#pragma unroll
        for (int u = 0; u < U; ++u) multiply(av[u], xv[u]);
      }
      for (; kb < kb1; ++kb) {
        uint4 av[2 * RB], xv[NT];
#pragma unroll
        for (int i = 0; i < 2 * RB; ++i) av[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < NT; ++j) xv[j] = make_uint4(0, 0, 0, 0);
        if (kb * 32 + tq * 8 < p.K) load(av, xv, kb);
        __syncwarp();
        multiply(av, xv);
      }
    }
    float* mine = s_part + size_t(warp) * RK * PITCH;
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int c = 0; c < 2; ++c)
          *reinterpret_cast<float2*>(mine + (i * 16 + g + 8 * c) * PITCH + j * 8 + 2 * tq) =
              make_float2(acc[i][j][2 * c], acc[i][j][2 * c + 1]);
    __syncthreads();
    // warps of a group, then blocks of the cluster, in order
    for (int o = threadIdx.x; o < W * RK; o += kAdThreads) {
      const int t = o / RK, i = o % RK;
      const int gt = s.group[t] - base;
      if (s.group[t] < 0 || gt < 0 || gt >= ng || rank0 + i >= p.r) continue;
      float* at = s_part + (size_t(gt * wpg) * RK + i) * PITCH + t;
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < kAdWarps; ++u)
        if (u < wpg) sum += at[u * RK * PITCH];
      if (cs == 1)
        p.v[(size_t(bank) * p.R + row0 + t) * p.r + rank0 + i] = sum;
      else
        *at = sum;
    }
    if (cs > 1) {
      cluster_sync();
      for (int o = cr * kAdThreads + threadIdx.x; o < W * RK; o += cs * kAdThreads) {
        const int t = o / RK, i = o % RK;
        const int gt = s.group[t] - base;
        if (s.group[t] < 0 || gt < 0 || gt >= ng || rank0 + i >= p.r) continue;
        const uint32_t at = smem_u32(s_part + (size_t(gt * wpg) * RK + i) * PITCH + t);
        float q[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) q[c] = c < cs ? ld_cluster_f32(at, c) : 0.f;
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < 8; ++c) sum += q[c];
        p.v[(size_t(bank) * p.R + row0 + t) * p.r + rank0 + i] = sum;
      }
      cluster_sync();  // the parts stay until every block of the cluster has read them
    } else {
      __syncthreads();
    }
  }
}

// ---------------------------------------------------------------------------
// expand: out[row] = base[row] + s_a v[row] . B_a^T   (or the SwiGLU of two)
// ---------------------------------------------------------------------------
// mma m16n8k16 with the window's rows as M (MT tiles of 16) and output columns
// as N.  v enters as two fp16 terms of the row scaled by a power of two to
// [2^14, 2^15) (value and remainder: 2^-22 of the row's largest, no overflow),
// so v is not rounded to fp16.  n-tile j, column c stands for output column
// (c >> 1) * 8 + 2 j + (c & 1) of the warp's 32: a lane ends with 8 neighbouring
// columns of its two rows, one 16-byte load of the base and one store each.
struct ExpandArgs {
  const float* v;       // [bank][R][r]
  const __half* b[2];
  const float* scale[2];
  const int32_t* index;
  const __half* base[2];  // the base rows; gate and up rows for SwiGLU
  __half* out;
  long R;
  int N, n, r;
  int groups_per_chunk;  // 32-column groups of a block
  bool in_place;
};

// The weights of a warp's 32 columns stay in registers while its row tiles pass.
// RV is the rank rounded up to 16 (8-byte loads: one mma step), 32, 64 or 128
// (16-byte loads: two steps per 32).
template <int RV>
struct RankTile {
  static constexpr int kPer = RV == 16 ? 4 : 8;     // rank values of a lane's load
  static constexpr int kLoads = RV == 16 ? 1 : RV / 32;
  static constexpr int kWords = kPer / 2;
  uint32_t w[kLoads][4][kWords];

  // Columns n0 + (g >> 1) * 8 + 2 j + (g & 1); bp points at (that column for j = 0, tq * kPer).
  LR_DEVICE void load(const __half* __restrict__ bp, int r, bool ok, int tq) {
#pragma unroll
    for (int b = 0; b < kLoads; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = ok && b * 32 + tq * kPer < r;
        const __half* q = bp + size_t(2 * j) * r + b * 32;
        if (RV == 16) {
          uint2 v = make_uint2(0, 0);
          if (in) v = __ldg(reinterpret_cast<const uint2*>(q));
          w[b][j][0] = v.x;
          w[b][j][1] = v.y;
        } else {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (in) v = __ldg(reinterpret_cast<const uint4*>(q));
          w[b][j][0] = v.x;
          w[b][j][1] = v.y;
          w[b][j][kWords - 2] = v.z;
          w[b][j][kWords - 1] = v.w;
        }
      }
  }

  // acc += rows (two fp16 terms, `lo` after `hi`) . weights; hi points at (row g, tq * kPer).
  LR_DEVICE void multiply(float (&acc)[4][4], const __half* hi, const __half* lo, int pitch) const {
#pragma unroll
    for (int b = 0; b < kLoads; ++b)
#pragma unroll
      for (int term = 0; term < 2; ++term) {
        const __half* q = (term ? lo : hi) + b * 32;
        if (RV == 16) {
          const uint2 a0 = *reinterpret_cast<const uint2*>(q);
          const uint2 a1 = *reinterpret_cast<const uint2*>(q + 8 * pitch);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mma_f16(acc[j], a0.x, a1.x, a0.y, a1.y, w[b][j][0], w[b][j][1]);
        } else {
          const uint4 a0 = *reinterpret_cast<const uint4*>(q);
          const uint4 a1 = *reinterpret_cast<const uint4*>(q + 8 * pitch);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            mma_f16(acc[j], a0.x, a1.x, a0.y, a1.y, w[b][j][0], w[b][j][1]);
            mma_f16(acc[j], a0.z, a1.z, a0.w, a1.w, w[b][j][kWords - 2], w[b][j][kWords - 1]);
          }
        }
      }
  }
};

// Base rows in flight per warp: a ring over column groups, or (one row tile) as
// many column groups at once as their weights' registers allow.
template <int RV, int MT, bool SWIGLU>
constexpr int expand_stages() {
  return MT > 1 ? (RV <= 32 ? 3 : 2) : RV == 16 ? (SWIGLU ? 4 : 8) : RV == 32 ? (SWIGLU ? 2 : 4) : RV == 64 && !SWIGLU ? 2 : 1;
}

template <int RV, int MT, bool SWIGLU>
__global__ void __launch_bounds__(kAdThreads, RV <= 64 && !SWIGLU ? 2 : 1)
    adapter_expand_kernel(ExpandArgs p) {
  constexpr int W = 16 * MT;
  constexpr int BANKS = SWIGLU ? 2 : 1;
  constexpr int PITCH = RV + 8;
  constexpr int S = expand_stages<RV, MT, SWIGLU>();
  constexpr bool AHEAD = RV <= 64 && !SWIGLU;
  extern __shared__ __align__(16) unsigned char s_dyn[];
  uint4* s_ring = reinterpret_cast<uint4*>(s_dyn);  // [warp][S][bank][2 MT][lane]
  __half* s_v = reinterpret_cast<__half*>(s_ring + kAdWarps * S * BANKS * MT * 2 * 32);
  // s_v: [bank][hi, lo][W][PITCH]
  __shared__ Groups s;
  __shared__ float s_fac[BANKS][W];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  const long row0 = long(blockIdx.x) * W;
  if (warp == 0) group_rows<W>(s, p.index, row0, p.R, p.n, !p.in_place, nullptr);
  __syncthreads();
  {  // v: fp32 -> scaled (value, remainder) pairs
    constexpr int LPR = kAdThreads / W;  // lanes of a row
    constexpr int EL = (RV + LPR - 1) / LPR;
    const int t = threadIdx.x / LPR, q = threadIdx.x % LPR;
    const int ad = s.adapter[t];
#pragma unroll
    for (int bk = 0; bk < BANKS; ++bk) {
      const float* row = p.v + (size_t(bk) * p.R + row0 + t) * p.r;
      float val[EL];
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < EL; ++i) {
        const int c = i * LPR + q;
        val[i] = ad >= 0 && c < p.r ? __ldcg(row + c) : 0.f;
        m = fmaxf(m, fabsf(val[i]));
      }
#pragma unroll
      for (int o = 1; o < LPR; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      // 2^ex takes the row's largest into [2^14, 2^15); both powers are normal numbers
      int ex = 0;
      if (m > 0.f && m < INFINITY) ex = max(-100, min(100, 141 - int(__float_as_uint(m) >> 23)));
      const float up = __uint_as_float(unsigned(127 + ex) << 23);
      const float down = __uint_as_float(unsigned(127 - ex) << 23);
      __half* hi = s_v + (2 * bk * W + t) * PITCH;
      __half* lo = hi + W * PITCH;
#pragma unroll
      for (int i = 0; i < EL; ++i) {
        const int c = i * LPR + q;
        if (c < RV) {
          const float x = val[i] * up;
          const __half h = __float2half_rn(x);
          const float hf = __half2float(h);
          hi[c] = h;
          lo[c] = __float2half_rn(fabsf(hf) < INFINITY ? x - hf : 0.f);
        }
      }
      if (q == 0)
        s_fac[bk][t] = ad >= 0 ? (p.scale[bk] ? __ldg(p.scale[bk] + ad) : 1.f) * down : 0.f;
    }
  }
  __syncthreads();
  const int cg0 = blockIdx.y * p.groups_per_chunk;
  const int cg1 = min(cg0 + p.groups_per_chunk, (p.N + 31) / 32);
  for (int base = 0; base < s.n; base += kAdWarps) {
    const int ng = min(kAdWarps, s.n - base);
    const int wpg = warps_per_group(ng);
    const int grp = warp / wpg, sub = warp % wpg;
    if (grp >= ng) continue;
    const int slot = base + grp;
    const int ad = s.adapter[s.first[slot]];
    unsigned rows_ok = 0, tiles = 0;  // this lane's member rows, the warp's used row tiles
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (s.group[m * 16 + g + 8 * h] == slot) rows_ok |= 1u << (2 * m + h);
      if (__any_sync(0xffffffffu, (rows_ok >> (2 * m)) & 3u)) tiles |= 1u << m;
    }
    // This lane's rows: (m, h) is 16 m + 8 h rows below the first.
    const size_t row_off = size_t(row0 + g) * p.N;
    const auto at = [&](int m, int h) { return size_t(unsigned(16 * m + 8 * h) * unsigned(p.N)); };
    if (ad < 0) {  // no adapter: the base rows as they are
      for (int c = cg0 + sub; c < cg1; c += wpg) {
        const int nc = c * 32 + tq * 8;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (!((rows_ok >> (2 * m + h)) & 1u) || nc >= p.N) continue;
            uint4 v = ld_row(reinterpret_cast<const uint4*>(p.base[0] + row_off + at(m, h) + nc));
            if (SWIGLU)
              v = swiglu8(v, ld_row(reinterpret_cast<const uint4*>(p.base[BANKS - 1] + row_off +
                                                                    at(m, h) + nc)));
            *reinterpret_cast<uint4*>(p.out + row_off + at(m, h) + nc) = v;
          }
      }
      continue;
    }
    // Column group c's base rows go to stage st of this lane's own slots.
    uint4* slots = s_ring + warp * (S * BANKS * MT * 2 * 32) + lane;
    const auto fetch = [&](int c, int st) {
      const int nc = c * 32 + tq * 8;
      if (c < cg1 && nc < p.N) {
#pragma unroll
        for (int bk = 0; bk < BANKS; ++bk)
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if ((rows_ok >> (2 * m + h)) & 1u)
                cp_async_16(slots + ((st * BANKS + bk) * MT * 2 + 2 * m + h) * 32,
                            p.base[bk] + row_off + at(m, h) + nc);
      }
      cp_async_commit();
    };
    const auto weights = [&](RankTile<RV>(&wt)[BANKS], int c) {
      const int nr = c * 32 + (g >> 1) * 8;
#pragma unroll
      for (int bk = 0; bk < BANKS; ++bk)
        wt[bk].load(p.b[bk] + (size_t(ad) * p.N + nr + (g & 1)) * p.r + tq * RankTile<RV>::kPer,
                    p.r, c < cg1 && nr < p.N, tq);
    };
    const auto finish = [&](const RankTile<RV>(&wt)[BANKS], int c, int st) {
      const int nc = c * 32 + tq * 8;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (!((tiles >> m) & 1u)) continue;
        float acc[BANKS][4][4];
#pragma unroll
        for (int bk = 0; bk < BANKS; ++bk) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[bk][j][i] = 0.f;
          const __half* hi = s_v + (2 * bk * W + m * 16 + g) * PITCH + tq * RankTile<RV>::kPer;
          wt[bk].multiply(acc[bk], hi, hi + W * PITCH, PITCH);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (!((rows_ok >> (2 * m + h)) & 1u) || nc >= p.N) continue;
          float o[BANKS][8];
#pragma unroll
          for (int bk = 0; bk < BANKS; ++bk) {
            const uint4 bs = slots[((st * BANKS + bk) * MT * 2 + 2 * m + h) * 32];
            const __half2* bh = reinterpret_cast<const __half2*>(&bs);
            const float f = s_fac[bk][m * 16 + g + 8 * h];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 b2 = __half22float2(bh[j]);
              o[bk][2 * j] = fmaf(acc[bk][j][2 * h], f, b2.x);
              o[bk][2 * j + 1] = fmaf(acc[bk][j][2 * h + 1], f, b2.y);
            }
          }
          if (SWIGLU) {
#pragma unroll
            for (int i = 0; i < 8; ++i) o[0][i] = silu_f32(o[0][i]) * o[BANKS - 1][i];
          }
          *reinterpret_cast<uint4*>(p.out + row_off + at(m, h) + nc) = pack_half8(o[0]);
        }
      }
    };
    if (MT == 1) {  // S column groups at a time, all their loads in flight
      for (int c0 = cg0 + sub; c0 < cg1; c0 += wpg * S) {
        RankTile<RV> wt[S][BANKS];
#pragma unroll
        for (int u = 0; u < S; ++u) {
          fetch(c0 + u * wpg, u);
          weights(wt[u], c0 + u * wpg);
        }
        cp_async_wait<0>();
#pragma unroll
        for (int u = 0; u < S; ++u)
          if (c0 + u * wpg < cg1) finish(wt[u], c0 + u * wpg, u);
      }
    } else {  // a ring of S stages of base rows, the next group's weights in registers
      RankTile<RV> wt[BANKS];
      int c = cg0 + sub, st = 0;
#pragma unroll
      for (int u = 0; u < S - 1; ++u) fetch(c + u * wpg, u);
      if (AHEAD) weights(wt, c);
      for (; c < cg1; c += wpg) {
        fetch(c + (S - 1) * wpg, st == 0 ? S - 1 : st - 1);
        if (AHEAD) {
          RankTile<RV> next[BANKS];
          weights(next, c + wpg);
          cp_async_wait<S - 1>();
          finish(wt, c, st);
#pragma unroll
          for (int bk = 0; bk < BANKS; ++bk) wt[bk] = next[bk];
        } else {
          weights(wt, c);
          cp_async_wait<S - 1>();
          finish(wt, c, st);
        }
        st = st == S - 1 ? 0 : st + 1;
      }
      cp_async_wait<0>();
    }
  }
}

// ---------------------------------------------------------------------------
// adapter numbers of the expert rows
// ---------------------------------------------------------------------------
// Row r of expert e's segment from token t uses the bank's entry adapter[t] * E + e;
// rows past the segment's kept slots and tokens without an adapter get -1.
__global__ void __launch_bounds__(256)
    adapter_rows_kernel(const int32_t* __restrict__ adapter, int T, int n,
                        const int32_t* __restrict__ source_idx,
                        const int32_t* __restrict__ offsets,
                        const int32_t* __restrict__ kept_counts, long S, int E,
                        int32_t* __restrict__ index, int32_t* err) {
  pdl_wait();
  pdl_trigger();
  const long r = long(blockIdx.x) * 256 + threadIdx.x;
  if (r >= S) return;
  int lo = 0, hi = E;  // the last e with offsets[e] <= r
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(offsets + mid) <= r) lo = mid; else hi = mid;
  }
  int out = -1;
  if (r < long(__ldg(offsets + lo)) + __ldg(kept_counts + lo)) {
    const int t = __ldg(source_idx + r);
    if (t < 0 || t >= T) {
      report(err, LR_DEVERR_BAD_TOKEN);
    } else {
      const int a = __ldg(adapter + t);
      if (a < -1 || a >= n)
        report(err, LR_DEVERR_BAD_ADAPTER);
      else if (a >= 0)
        out = a * E + lo;
    }
  }
  index[r] = out;
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Launch with a cluster of `cluster` blocks along x, programmatic as launch_pdl.
template <typename... KArgs, typename... Args>
static int launch_cluster(void (*kern)(KArgs...), dim3 grid, unsigned cluster, size_t smem,
                          cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kAdThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(stream, &cs) != cudaSuccess) cs = cudaStreamCaptureStatusNone;
  cfg.numAttrs = cs == cudaStreamCaptureStatusNone ? 2 : 1;
  LR_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...));
  return 0;
}

constexpr long kSmallRows = 256;  // up to here windows of 8 (shrink) and 16 rows (expand)
constexpr long kTargetBlocks = 148;

template <int RB, int NT>
static int launch_shrink(const ShrinkArgs& p, int banks, cudaStream_t stream) {
  constexpr int W = 8 * NT, RK = 16 * RB;
  constexpr int smem = kAdWarps * RK * (W + 2) * int(sizeof(float));
  auto kern = adapter_shrink_kernel<RB, NT>;
  static unsigned long long configured = 0;
  if (const int rc = set_dyn_smem_once(kern, smem, configured)) return rc;
  const long windows = (p.R + W - 1) / W;
  const int rank_groups = (p.r + RK - 1) / RK;
  // fill the SMs by splitting K over a cluster, then a window's groups over blocks
  unsigned cs = 1, gs = 1;
  while (cs < 8 && windows * rank_groups * banks * cs < kTargetBlocks) cs *= 2;
  while (gs < 4 && gs < p.R && windows * rank_groups * banks * cs * gs < kTargetBlocks) gs *= 2;
  if (windows * cs > 0x7fffffffL) return LR_ERR_INVALID_ARGUMENT;
  return launch_cluster(kern, dim3(unsigned(windows * cs), rank_groups * banks, gs), cs, smem,
                        stream, p, rank_groups);
}

template <int RV, int MT, bool SWIGLU>
static int launch_expand(ExpandArgs p, cudaStream_t stream) {
  constexpr int W = 16 * MT;
  constexpr int banks = SWIGLU ? 2 : 1;
  constexpr int smem = kAdWarps * expand_stages<RV, MT, SWIGLU>() * banks * MT * 2 * 32 * 16 +
                       banks * 2 * W * (RV + 8) * int(sizeof(__half));
  auto kern = adapter_expand_kernel<RV, MT, SWIGLU>;
  static unsigned long long configured = 0;
  if (const int rc = set_dyn_smem_once(kern, smem, configured)) return rc;
  const long windows = (p.R + W - 1) / W;
  const int cgs = (p.N + 31) / 32;
  // 256 columns per block, more while the grid stays above eight blocks per SM
  int gpc = 8;
  while (gpc < 64 && windows * ((cgs + 2 * gpc - 1) / (2 * gpc)) >= 8 * kTargetBlocks) gpc *= 2;
  p.groups_per_chunk = gpc;
  if (windows > 0x7fffffffL) return LR_ERR_INVALID_ARGUMENT;
  return launch_pdl(kern, dim3(unsigned(windows), (cgs + gpc - 1) / gpc), dim3(kAdThreads), smem,
                    stream, p);
}

static int run_shrink(const ShrinkArgs& p, int banks, cudaStream_t stream) {
  const bool small = p.R <= kSmallRows;
  if (p.r <= 16)
    return small ? launch_shrink<1, 1>(p, banks, stream) : launch_shrink<1, 4>(p, banks, stream);
  if (p.r <= 32)
    return small ? launch_shrink<2, 1>(p, banks, stream) : launch_shrink<2, 4>(p, banks, stream);
  return small ? launch_shrink<4, 1>(p, banks, stream) : launch_shrink<4, 4>(p, banks, stream);
}

template <bool SWIGLU>
static int run_expand(const ExpandArgs& p, cudaStream_t stream) {
  constexpr int MT = SWIGLU ? 2 : 4;
  const bool small = p.R <= kSmallRows;
  if (p.r <= 16)
    return small ? launch_expand<16, 1, SWIGLU>(p, stream) : launch_expand<16, MT, SWIGLU>(p, stream);
  if (p.r <= 32)
    return small ? launch_expand<32, 1, SWIGLU>(p, stream) : launch_expand<32, MT, SWIGLU>(p, stream);
  if (p.r <= 64)
    return small ? launch_expand<64, 1, SWIGLU>(p, stream) : launch_expand<64, MT, SWIGLU>(p, stream);
  return small ? launch_expand<128, 1, SWIGLU>(p, stream) : launch_expand<128, MT, SWIGLU>(p, stream);
}

static int check_adapter_args(const void* x, long R, int K, const int32_t* index, int n, int r,
                              int N) {
  if (R < 0 || R > 0x7fffffffL || K <= 0 || K % 8 != 0 || N <= 0 || N % 8 != 0 || n < 1 || r < 8 ||
      r > kMaxRank || r % 8 != 0)
    return LR_ERR_INVALID_ARGUMENT;
  if (R > 0 && (!x || !index || !aligned16(x))) return LR_ERR_INVALID_ARGUMENT;
  return LR_OK;
}

static bool bank_ok(const void* a, const void* b) { return a && b && aligned16(a) && aligned16(b); }

}  // namespace lr

// ===========================================================================
// C ABI
// ===========================================================================
using namespace lr;

extern "C" size_t lr_adapter_workspace_bytes(int num_rows, int rank, int num_banks) {
  if (num_rows < 1 || rank < 1 || num_banks < 1) return 0;
  return size_t(num_rows) * rank * num_banks * sizeof(float);
}

extern "C" int lr_adapter_add(const void* x, int R, int K, const int32_t* index, int num_adapters,
                              const void* a, const void* b, const float* scale, int rank, int N,
                              const void* base, void* out, void* workspace, size_t workspace_bytes,
                              int32_t* err, lr_stream_t stream) {
  if (const int rc = check_adapter_args(x, R, K, index, num_adapters, rank, N)) return rc;
  if (R == 0) return LR_OK;
  if (!bank_ok(a, b) || !base || !out || !aligned16(base) || !aligned16(out))
    return LR_ERR_INVALID_ARGUMENT;
  if (!workspace || workspace_bytes < lr_adapter_workspace_bytes(R, rank, 1))
    return LR_ERR_WORKSPACE;
  ShrinkArgs sp{static_cast<const __half*>(x), {static_cast<const __half*>(a), nullptr}, index,
                static_cast<float*>(workspace), R, K, num_adapters, rank, err};
  if (const int rc = run_shrink(sp, 1, stream)) return rc;
  ExpandArgs ep{sp.v, {static_cast<const __half*>(b), nullptr}, {scale, nullptr}, index,
                {static_cast<const __half*>(base), nullptr}, static_cast<__half*>(out), R, N,
                num_adapters, rank, 0, base == out};
  return run_expand<false>(ep, stream);
}

extern "C" int lr_adapter_swiglu(const void* x, int R, int K, const int32_t* index,
                                 int num_adapters, const void* a_gate, const void* b_gate,
                                 const float* scale_gate, const void* a_up, const void* b_up,
                                 const float* scale_up, int rank, int N, const void* gate,
                                 const void* up, void* out, void* workspace,
                                 size_t workspace_bytes, int32_t* err, lr_stream_t stream) {
  if (const int rc = check_adapter_args(x, R, K, index, num_adapters, rank, N)) return rc;
  if (R == 0) return LR_OK;
  if (!bank_ok(a_gate, b_gate) || !bank_ok(a_up, b_up) || !gate || !up || !out ||
      !aligned16(gate) || !aligned16(up) || !aligned16(out))
    return LR_ERR_INVALID_ARGUMENT;
  if (!workspace || workspace_bytes < lr_adapter_workspace_bytes(R, rank, 2))
    return LR_ERR_WORKSPACE;
  ShrinkArgs sp{static_cast<const __half*>(x),
                {static_cast<const __half*>(a_gate), static_cast<const __half*>(a_up)}, index,
                static_cast<float*>(workspace), R, K, num_adapters, rank, err};
  if (const int rc = run_shrink(sp, 2, stream)) return rc;
  ExpandArgs ep{sp.v, {static_cast<const __half*>(b_gate), static_cast<const __half*>(b_up)},
                {scale_gate, scale_up}, index,
                {static_cast<const __half*>(gate), static_cast<const __half*>(up)},
                static_cast<__half*>(out), R, N, num_adapters, rank, 0, false};
  return run_expand<true>(ep, stream);
}

extern "C" int lr_adapter_rows(const int32_t* adapter_ids, int T, int num_adapters,
                               const int32_t* source_idx, const int32_t* offsets,
                               const int32_t* kept_counts, int S, int E, int32_t* index,
                               int32_t* err, lr_stream_t stream) {
  if (T < 0 || S < 0 || E < 1 || num_adapters < 1 || long(num_adapters) * E > 0x7fffffffL)
    return LR_ERR_INVALID_ARGUMENT;
  if (S == 0) return LR_OK;
  if (!adapter_ids || !source_idx || !offsets || !kept_counts || !index)
    return LR_ERR_INVALID_ARGUMENT;
  return launch_pdl(adapter_rows_kernel, dim3((unsigned(S) + 255) / 256), dim3(256), 0, stream,
                    adapter_ids, T, num_adapters, source_idx, offsets, kept_counts, long(S), E,
                    index, err);
}
