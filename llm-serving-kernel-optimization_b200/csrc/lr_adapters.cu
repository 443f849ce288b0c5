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
// The floor is memory: a row costs 2 (K + 2N) bytes and 2 r (K + N) operations.
// mma.sync keeps up with that (its pipe is 22 to 32 % busy in the large batches).
#include "lr_lowrank.cuh"

namespace lr {

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

// The window's groups [base0, s.n) in rounds: a round's groups share the block's
// warps, 2^n warps splitting K for a group.
template <int RB, int NT>
LR_DEVICE void shrink_groups(const ShrinkArgs& p, const Groups& s, float* s_part, long row0,
                             int bank, int rank0, int base0, int per_round) {
  constexpr int W = 8 * NT;
  constexpr int RK = 16 * RB;
  constexpr int PITCH = W + 2;
  // k-blocks whose loads are in flight together: 12 to 16 16-byte loads per lane
  constexpr int U = NT == 1 ? (RB == 1 ? 4 : RB == 2 ? 3 : 2) : 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  const int cs = int(cluster_nctarank()), cr = int(cluster_ctarank());
  const int nb = (p.K + 31) / 32;
  for (int base = base0; base < s.n; base += kAdWarps) {
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

// Small batches: windows of 8 rows; the grid's z deals a window's groups out to
// blocks.  64 rows x 4096 with an adapter of rank 16 each: 8 us, most of it the
// chain index, A, cluster, result (8.4 MB of A are 1.3 us of HBM).
template <int RB>
__global__ void __launch_bounds__(kAdThreads) adapter_shrink_kernel(ShrinkArgs p, int rank_groups) {
  constexpr int RK = 16 * RB;
  extern __shared__ __align__(128) unsigned char s_dyn[];  // [kAdWarps][RK][10] floats
  __shared__ Groups s;
  const int cs = int(cluster_nctarank());
  const long row0 = long(blockIdx.x / cs) * 8;
  const int bank = blockIdx.y / rank_groups, rank0 = (blockIdx.y % rank_groups) * RK;
  const int per_round = kAdWarps / gridDim.z;  // groups a block takes at a time
  pdl_wait();
  pdl_trigger();
  if (threadIdx.x < 32)
    group_rows<8>(s, p.index, row0, p.R, p.n, false, bank == 0 ? p.err : nullptr);
  __syncthreads();
  shrink_groups<RB, 1>(p, s, reinterpret_cast<float*>(s_dyn), row0, bank, rank0,
                       blockIdx.z * per_round, per_round);
}

// Larger batches: windows of 64 rows.  A group (a prompt's rows) streams tiles of
// 128 k, its rows of x and its adapter's rows of A, through a ring of cp.async
// stages; warp w multiplies 32 of the 128 k (w & 3) for half of the rows (w >> 2).
// The groups of a window that up to three requests share go to the two blocks of
// the grid's z (one of them leaves at once otherwise: its slot is free while the
// others stream); a window of more groups takes its halves through shrink_groups.
// 16384 x 4096, rank 32: 36 to 44 us (x alone is 21 us of HBM; A, read again by every
// window, is half as much from L2); 49 us where requests meet inside windows.  A bulk
// copy for each of these 256-byte rows took 127 us; a tensor map that moves a whole
// tile was not tried.  Registers (128, a few bytes spilled) and 256 working blocks on
// 296 places hold it where it is: HBM at 48 %, issue slots at 40 %.
constexpr int kTileK = 128;
constexpr int kTileKPitch = kTileK * 2 + 64;  // bytes; neighbouring rows in different banks

constexpr int kShrinkStages = 3;

template <int RB>
constexpr int shrink_smem_bytes() {
  constexpr int ring = kShrinkStages * (64 + 16 * RB) * kTileKPitch;
  constexpr int part = kAdWarps * 16 * RB * 34 * int(sizeof(float));
  return ring > part ? ring : part;
}

template <int RB>
__global__ void __launch_bounds__(kAdThreads, 2)
    adapter_shrink_stream_kernel(ShrinkArgs p, int rank_groups) {
  constexpr int RK = 16 * RB, S = kShrinkStages, PITCH = 34;
  constexpr int kStageBytes = (64 + RK) * kTileKPitch;
  extern __shared__ __align__(128) unsigned char s_dyn[];  // ring, then the warps' sums
  __shared__ Groups s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  const int cs = int(cluster_nctarank()), cr = int(cluster_ctarank());
  const long row0 = long(blockIdx.x / cs) * 64;
  const int bank = blockIdx.y / rank_groups, rank0 = (blockIdx.y % rank_groups) * RK;
  float* s_part = reinterpret_cast<float*>(s_dyn);
  pdl_wait();
  pdl_trigger();
  if (warp == 0) group_rows<64>(s, p.index, row0, p.R, p.n, false, bank == 0 ? p.err : nullptr);
  __syncthreads();
  if (s.n > 3) {
    if (blockIdx.z > 0) return;
    for (int half = 0; half < 2; ++half) {
      __syncthreads();
      if (warp == 0)
        group_rows<32>(s, p.index, row0 + 32 * half, p.R, p.n, false, nullptr);
      __syncthreads();
      shrink_groups<RB, 4>(p, s, s_part, row0 + 32 * half, bank, rank0, 0, kAdWarps);
    }
    return;
  }
  const int all = (p.K + kTileK - 1) / kTileK;
  const int tile0 = int(long(all) * cr / cs), tiles = int(long(all) * (cr + 1) / cs) - tile0;
  const int ranks = min(RK, p.r - rank0);
  const int kq = warp & 3, half = warp >> 2;
  for (int grp = blockIdx.z; grp < s.n; grp += gridDim.z) {
    const __half* ap = (bank ? p.a[1] : p.a[0]) + (size_t(s.adapter[s.first[grp]]) * p.r + rank0) * p.K;
    const auto fetch = [&](int i) {  // tile i into its stage: 16 lanes per row, zeros past the ends
      if (i < tiles) {
        const int k = (tile0 + i) * kTileK + (threadIdx.x & 15) * 8;
        unsigned char* to = s_dyn + (i % S) * kStageBytes + (threadIdx.x & 15) * 16;
#pragma unroll
        for (int u = 0; u < 64 + RK; u += 16) {
          const int row = u + (threadIdx.x >> 4);
          const bool ok = k < p.K && (u < 64 ? s.group[row] == grp : row - 64 < ranks);
          const __half* from = u < 64 ? p.x + size_t(row0 + row) * p.K : ap + size_t(row - 64) * p.K;
          cp_async_16_zfill(to + row * kTileKPitch, ok ? from + k : p.x, ok);
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < S - 1; ++i) fetch(i);
    float acc[RB][4][4];
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[i][j][c] = 0.f;
    for (int i = 0; i < tiles; ++i) {
      cp_async_wait_group<S - 2>();
      __syncthreads();
      fetch(i + S - 1);  // into the stage read one tile ago
      const int st = i % S;
      const unsigned char* from = s_dyn + st * kStageBytes + kq * 64 + tq * 16;
      uint4 av[2 * RB], xv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        xv[j] = *reinterpret_cast<const uint4*>(from + (half * 32 + j * 8 + g) * kTileKPitch);
#pragma unroll
      for (int j = 0; j < 2 * RB; ++j)
        av[j] = *reinterpret_cast<const uint4*>(from + (64 + j * 8 + g) * kTileKPitch);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < RB; ++r) {
          const uint4 lo = av[2 * r], hi = av[2 * r + 1], x = xv[j];
          mma_f16(acc[r][j], lo.x, hi.x, lo.y, hi.y, x.x, x.y);
          mma_f16(acc[r][j], lo.z, hi.z, lo.w, hi.w, x.z, x.w);
        }
    }
    cp_async_wait_all();
    __syncthreads();  // every tile is read: the ring becomes the warps' sums [warp][RK][PITCH]
    float* mine = s_part + warp * RK * PITCH;
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < 2; ++c)
          *reinterpret_cast<float2*>(mine + (i * 16 + g + 8 * c) * PITCH + j * 8 + 2 * tq) =
              make_float2(acc[i][j][2 * c], acc[i][j][2 * c + 1]);
    __syncthreads();
    // the four k-quarters, then the blocks of the cluster, in order
    for (int o = threadIdx.x; o < 64 * RK; o += kAdThreads) {
      const int t = o / RK, i = o % RK;
      if (s.group[t] != grp || i >= ranks) continue;
      float* at = s_part + ((t >> 5) * 4 * RK + i) * PITCH + (t & 31);
      const float sum = ((at[0] + at[RK * PITCH]) + at[2 * RK * PITCH]) + at[3 * RK * PITCH];
      if (cs == 1)
        p.v[(size_t(bank) * p.R + row0 + t) * p.r + rank0 + i] = sum;
      else
        *at = sum;
    }
    if (cs > 1) {
      cluster_sync();
      for (int o = cr * kAdThreads + threadIdx.x; o < 64 * RK; o += cs * kAdThreads) {
        const int t = o / RK, i = o % RK;
        if (s.group[t] != grp || i >= ranks) continue;
        const uint32_t at = smem_u32(s_part + ((t >> 5) * 4 * RK + i) * PITCH + (t & 31));
        float q[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) q[c] = c < cs ? ld_cluster_f32(at, c) : 0.f;
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < 8; ++c) sum += q[c];
        p.v[(size_t(bank) * p.R + row0 + t) * p.r + rank0 + i] = sum;
      }
      cluster_sync();  // the sums stay until every block of the cluster has read them
    } else {
      __syncthreads();
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

// Blocks are made to fill one wave of two per SM: K is split over a cluster, and a
// small batch's window over blocks of its groups.
template <int RB>
static int launch_shrink_small(const ShrinkArgs& p, int banks, cudaStream_t stream) {
  constexpr int RK = 16 * RB;
  const long windows = (p.R + 7) / 8;
  const int rank_groups = (p.r + RK - 1) / RK;
  const long blocks = windows * rank_groups * banks;
  unsigned cs = 1, gs = 1;
  while (cs < 8 && blocks * cs * 2 <= 2 * kTargetBlocks) cs *= 2;
  while (gs < 4 && gs < p.R && blocks * cs * gs * 2 <= 2 * kTargetBlocks) gs *= 2;
  return launch_cluster(adapter_shrink_kernel<RB>,
                        dim3(unsigned(windows * cs), rank_groups * banks, gs), cs,
                        kAdWarps * RK * 10 * sizeof(float), stream, p, rank_groups);
}

// Clusters of 8 wait long for eight free SMs next to one another: only where the
// grid stays under half a block per SM (1111 rows, K 2048, rank 64: 35 us against
// 21 with clusters of 4; 400 rows, K 4096, rank 16: 13 against 15).
template <int RB>
static int launch_shrink_stream(const ShrinkArgs& p, int banks, cudaStream_t stream) {
  constexpr int RK = 16 * RB, smem = shrink_smem_bytes<RB>();
  auto kern = adapter_shrink_stream_kernel<RB>;
  static unsigned long long configured = 0;
  if (const int rc = set_dyn_smem_once(kern, smem, configured)) return rc;
  const long windows = (p.R + 63) / 64;
  const int rank_groups = (p.r + RK - 1) / RK;
  const long blocks = windows * rank_groups * banks;
  unsigned cs = 1;
  while (cs < 8 && blocks * cs * 2 <= (cs < 4 ? 2 * kTargetBlocks : kTargetBlocks / 2)) cs *= 2;
  if (windows * cs > 0x7fffffffL) return LR_ERR_INVALID_ARGUMENT;
  return launch_cluster(kern, dim3(unsigned(windows * cs), rank_groups * banks, 2), cs, smem,
                        stream, p, rank_groups);
}

// Ranks above 32 (64 in small batches) are taken in parts, each reading x again:
// one kernel for rank 64 measured the same time in four times the registers.
static int run_shrink(const ShrinkArgs& p, int banks, cudaStream_t stream) {
  if (p.R > kSmallRows)
    return p.r <= 16 ? launch_shrink_stream<1>(p, banks, stream)
                     : launch_shrink_stream<2>(p, banks, stream);
  return p.r <= 16   ? launch_shrink_small<1>(p, banks, stream)
         : p.r <= 32 ? launch_shrink_small<2>(p, banks, stream)
                     : launch_shrink_small<4>(p, banks, stream);
}

static int check_adapter_args(const void* x, long R, int K, const int32_t* index, int n, int r,
                              int N) {
  if (R < 0 || R > kMaxRows || K <= 0 || K % 8 != 0 || K > kMaxColumns || N <= 0 || N % 8 != 0 ||
      N > kMaxColumns || n < 1 || r < 8 || r > kMaxRank || r % 8 != 0)
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
  if (!aligned16(workspace)) return LR_ERR_INVALID_ARGUMENT;
  ShrinkArgs sp{static_cast<const __half*>(x), {static_cast<const __half*>(a), nullptr}, index,
                static_cast<float*>(workspace), R, K, num_adapters, rank, err};
  if (const int rc = run_shrink(sp, 1, stream)) return rc;
  ExpandArgs ep{sp.v, {static_cast<const __half*>(b), nullptr}, {scale, nullptr}, index,
                {static_cast<const __half*>(base), nullptr}, out, R, N,
                num_adapters, rank, rank, 0, base == out, err};
  return run_expand<kExpandAdd>(ep, stream);
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
  if (!aligned16(workspace)) return LR_ERR_INVALID_ARGUMENT;
  ShrinkArgs sp{static_cast<const __half*>(x),
                {static_cast<const __half*>(a_gate), static_cast<const __half*>(a_up)}, index,
                static_cast<float*>(workspace), R, K, num_adapters, rank, err};
  if (const int rc = run_shrink(sp, 2, stream)) return rc;
  ExpandArgs ep{sp.v, {static_cast<const __half*>(b_gate), static_cast<const __half*>(b_up)},
                {scale_gate, scale_up}, index,
                {static_cast<const __half*>(gate), static_cast<const __half*>(up)},
                out, R, N, num_adapters, rank, rank, 0, false, err};
  return run_expand<kExpandSwiglu>(ep, stream);
}

extern "C" int lr_adapter_rows(const int32_t* adapter_ids, int T, int num_adapters,
                               const int32_t* source_idx, const int32_t* offsets,
                               const int32_t* kept_counts, int S, int E, int32_t* index,
                               int32_t* err, lr_stream_t stream) {
  if (T < 0 || S < 0 || S > kMaxRows || E < 1 || num_adapters < 1 ||
      long(num_adapters) * E > 0x7fffffffL)
    return LR_ERR_INVALID_ARGUMENT;
  if (S == 0) return LR_OK;
  if (!adapter_ids || !source_idx || !offsets || !kept_counts || !index)
    return LR_ERR_INVALID_ARGUMENT;
  return launch_pdl(adapter_rows_kernel, dim3((unsigned(S) + 255) / 256), dim3(256), 0, stream,
                    adapter_ids, T, num_adapters, source_idx, offsets, kept_counts, long(S), E,
                    index, err);
}
