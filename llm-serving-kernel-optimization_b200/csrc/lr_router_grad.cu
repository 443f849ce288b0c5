// lr_router_grad.cu -- the router's training path (sm_100a): top-k gating with
// the balance loss and per-expert counts, and the gradients of the gate
// projection, the dispatch and the weighted combine.
//
// With p = softmax(l_t), the selected set s_t (k largest logits, ties towards
// the lowest expert), q = sum_{s_t} p + 1e-9, w_j = p_j / q, counts c_e and the
// n live tokens:
//   loss   = lbw * E * sum_e f_e P_e,  f_e = c_e / (n k),  P_e = sum_t p_te / n
//   dp_e   = [e in s_t] (dw_e - sum_j dw_j w_j) / q  +  dloss * lbw * E * f_e / n
//   dl_e   = p_e (dp_e - sum_i p_i dp_i)              (f is a constant, as in the loss)
//   dW     = dl^T h,  dh = dl W,  db = sum_t dl
//   dy_row = w dout_t,  dw = <dout_t, y_row>,  dx_t = sum_j dpermuted[row_j]
#include <type_traits>

#include "lr_lowrank.cuh"

namespace lr {

// ---------------------------------------------------------------------------
// top-k gating + balance loss + counts
// ---------------------------------------------------------------------------
// A token's logits are spread over LPT lanes, 8 per lane in two float4 pieces
// (lane l holds experts c*4*LPT + 4l + r, c < 2, r < 4), so a warp reads whole
// rows.  Selection is k rounds of a maximum over (ordered logit, lowest expert
// first) keys.  Probability sums and counts stay in registers over a lane's
// tokens, go through shuffles and shared memory to one partial per block and
// expert, and are summed over blocks in double in block order: no atomics.
// 262144 tokens x 8 experts take 10 us (12.6 MB, 2 us of HBM: a warp has no loads in
// flight ahead of its next round, of which it has one or two) and 8192 x 64 top-6
// takes 8; one thread per token with 64 experts in registers took 60 at 777 tokens.
constexpr int kGateThreads = 512;
constexpr int kGateBlocksMax = 296;  // 2 per SM

struct GatingParts {
  double* psum;    // [E][B]
  int32_t* count;  // [E + 1][B], row E: live tokens
};

// Larger key = larger logit, then lower expert; NaN below every number.
LR_DEVICE unsigned long long select_key(float v, int e) {
  uint32_t u = __float_as_uint(v + 0.f);  // -0 -> +0: they tie
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  if (v != v) u = 0u;
  return (static_cast<unsigned long long>(u) << 32) | (0xffffffffu - unsigned(e));
}

template <int LPT>
LR_DEVICE float group_sum(float v) {
#pragma unroll
  for (int o = 1; o < LPT; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int LPT>
LR_DEVICE float group_max(float v) {
#pragma unroll
  for (int o = 1; o < LPT; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// This lane's 8 logits of row t (-inf past E) and their softmax.
template <int LPT>
LR_DEVICE void row_softmax(const float* __restrict__ logits, int t, bool valid, int E, bool vec,
                           int l, float (&v)[8], float (&p)[8]) {
  const float* row = logits + size_t(valid ? t : 0) * E;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int e0 = c * 4 * LPT + 4 * l;
    if (vec) {
      float4 q = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (valid && e0 < E) q = __ldg(reinterpret_cast<const float4*>(row + e0));
      v[4 * c] = q.x;
      v[4 * c + 1] = q.y;
      v[4 * c + 2] = q.z;
      v[4 * c + 3] = q.w;
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        v[4 * c + r] = (valid && e0 + r < E) ? __ldg(row + e0 + r) : -INFINITY;
    }
  }
  float m = v[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) m = fmaxf(m, v[i]);
  m = group_max<LPT>(m);
  float z = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = (i >> 2) * 4 * LPT + 4 * l + (i & 3);
    p[i] = e < E ? expf(v[i] - m) : 0.f;
    z += p[i];
  }
  z = group_sum<LPT>(z);
#pragma unroll
  for (int i = 0; i < 8; ++i) p[i] = p[i] / z;
}

// counts[0..E), counts[E] = live tokens, and the loss, from totals in double: a
// thread per expert for the divisions, one for the sum in expert order.
LR_DEVICE void write_gating_stats(int E, int k, float lbw, double* s_p, const int32_t* s_c,
                                  int32_t* __restrict__ counts, float* __restrict__ aux) {
  const int n = s_c[E];
  for (int e = threadIdx.x; e <= E; e += blockDim.x) {
    counts[e] = s_c[e];
    if (e < E) s_p[e] = n > 0 ? (double(s_c[e]) / (double(n) * k)) * (s_p[e] / n) : 0.0;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double a = 0.0;
    for (int e = 0; e < E; ++e) a += s_p[e];
    aux[0] = static_cast<float>(double(lbw) * E * a);
  }
}

template <int LPT>
__global__ void __launch_bounds__(kGateThreads)
    balanced_gating_kernel(const float* __restrict__ logits, const uint8_t* __restrict__ mask,
                           int T, int E, int k, float lbw, bool vec,
                           int32_t* __restrict__ expert_ids, float* __restrict__ gate_w,
                           int32_t* __restrict__ counts, float* __restrict__ aux,
                           GatingParts parts) {
  constexpr int kW = kGateThreads / 32;
  __shared__ float s_p[kW][8 * LPT];
  __shared__ int32_t s_c[kW][8 * LPT + 1];
  __shared__ double s_tp[8 * LPT];
  __shared__ int32_t s_tc[8 * LPT + 1];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int l = lane % LPT;
  const int per_warp = 32 / LPT;
  float psum[8];
  int cnt[8];
  int live_n = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    psum[i] = 0.f;
    cnt[i] = 0;
  }
  const long stride = long(gridDim.x) * kW * per_warp;
  for (long tb = (long(blockIdx.x) * kW + warp) * per_warp; tb < T; tb += stride) {
    const int t = int(tb) + lane / LPT;
    const bool valid = t < T;
    const bool live = valid && (mask == nullptr || mask[t] != 0);
    float v[8], p[8];
    row_softmax<LPT>(logits, t, valid, E, vec, l, v, p);
    unsigned taken = 0;  // this lane's selected experts
    int ids[kMaxTopK];
    float ps[kMaxTopK];
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < kMaxTopK; ++j) {
      if (j < k) {
        unsigned long long best = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int e = (i >> 2) * 4 * LPT + 4 * l + (i & 3);
          const unsigned long long key = select_key(v[i], e);
          if (e < E && !((taken >> i) & 1u) && key > best) best = key;
        }
#pragma unroll
        for (int o = 1; o < LPT; o <<= 1) {
          const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
          if (other > best) best = other;
        }
        const int e = int(0xffffffffu - unsigned(best));
        const int owner = (e >> 2) % LPT, i = (e >> 2) / LPT * 4 + (e & 3);
        if (owner == l) taken |= 1u << i;
        float pe = 0.f;
#pragma unroll
        for (int x = 0; x < 8; ++x)
          if (x == i) pe = p[x];
        pe = __shfl_sync(0xffffffffu, pe, (lane & ~(LPT - 1)) + owner);
        ids[j] = e;
        ps[j] = pe;
        q += pe;
      }
    }
    const float denom = q + 1e-9f;
    if (valid) {
#pragma unroll
      for (int j = 0; j < kMaxTopK; ++j) {
        if (j < k && j % LPT == l) {
          const size_t s = size_t(t) * k + j;
          expert_ids[s] = ids[j];
          gate_w[s] = live ? ps[j] / denom : 0.f;
        }
      }
    }
    if (live) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        psum[i] += p[i];
        cnt[i] += (taken >> i) & 1u;
      }
      live_n += l == 0;
    }
  }
  // lanes with the same experts, then warps, then blocks
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int o = LPT; o < 32; o <<= 1) {
      psum[i] += __shfl_xor_sync(0xffffffffu, psum[i], o);
      cnt[i] += __shfl_xor_sync(0xffffffffu, cnt[i], o);
    }
    if (lane < LPT) {
      const int e = (i >> 2) * 4 * LPT + 4 * l + (i & 3);
      s_p[warp][e] = psum[i];
      s_c[warp][e] = cnt[i];
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) live_n += __shfl_xor_sync(0xffffffffu, live_n, o);
  if (lane == 0) s_c[warp][8 * LPT] = live_n;
  __syncthreads();
  for (int e = threadIdx.x; e <= 8 * LPT; e += kGateThreads) {
    double ps = 0.0;
    int c = 0;
    for (int w = 0; w < kW; ++w) {
      if (e < 8 * LPT) ps += double(s_p[w][e]);
      c += s_c[w][e];
    }
    const int row = e == 8 * LPT ? E : e;  // the live count moves up to row E
    if (gridDim.x == 1) {
      if (e < E) s_tp[e] = ps;
      if (e < E || e == 8 * LPT) s_tc[row] = c;
    } else if (e < E || e == 8 * LPT) {
      if (e < E) parts.psum[size_t(e) * gridDim.x + blockIdx.x] = ps;
      parts.count[size_t(row) * gridDim.x + blockIdx.x] = c;
    }
  }
  if (gridDim.x > 1) return;
  __syncthreads();
  write_gating_stats(E, k, lbw, s_tp, s_tc, counts, aux);
}

// One block: totals over the B blocks' partials, a warp per expert (5 us; a ticket
// and a last block in the kernel above would need a memset before it instead).
__global__ void __launch_bounds__(1024)
    gating_stats_kernel(GatingParts parts, int B, int E, int k, float lbw,
                        int32_t* __restrict__ counts, float* __restrict__ aux) {
  __shared__ double s_tp[64];
  __shared__ int32_t s_tc[65];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  for (int e = threadIdx.x >> 5; e <= E; e += 32) {
    double ps = 0.0;
    int c = 0;
    for (int b = lane; b < B; b += 32) {
      if (e < E) ps += parts.psum[size_t(e) * B + b];
      c += parts.count[size_t(e) * B + b];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      ps += __shfl_xor_sync(0xffffffffu, ps, o);
      c += __shfl_xor_sync(0xffffffffu, c, o);
    }
    if (lane == 0) {
      if (e < E) s_tp[e] = ps;
      s_tc[e] = c;
    }
  }
  __syncthreads();
  write_gating_stats(E, k, lbw, s_tp, s_tc, counts, aux);
}

// The gradient in the logits: the softmax is taken again from the logits (one
// read, nothing kept from the forward but the ids), one launch, no reductions
// across tokens.  With `csr` the counts are the differences of CSR offsets and
// every token is live.
// dl is a difference of nearly equal terms where a router is balanced or one
// expert takes all of a token's weight, so the terms are taken relative to the
// first selected expert's (0): adding a constant to dp changes nothing, and with
// d'_j = dw_j - dw_0, c' = sum_j d'_j w_j, sum_j w_j = 1 - 1e-9 / q,
//   dp_i - dp_0 = bal_i - bal_0 + (i selected ? d'_i : c' - dw_0 1e-9 / q) / q,
// bal_i = dloss lbw E (f_i - 1/E) / n with the difference in double.
// Forward, statistics and this: 27 us at 262144 x 8, 19 at 8192 x 64 top-6.
template <int LPT>
__global__ void __launch_bounds__(kGateThreads)
    balanced_gating_backward_kernel(const float* __restrict__ logits,
                                    const uint8_t* __restrict__ mask,
                                    const int32_t* __restrict__ expert_ids,
                                    const int32_t* __restrict__ counts, int csr,
                                    const float* __restrict__ d_w, const float* __restrict__ d_aux,
                                    int T, int E, int k, float lbw, bool vec,
                                    float* __restrict__ d_logits) {
  constexpr int kW = kGateThreads / 32;
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int l = lane % LPT;
  const int per_warp = 32 / LPT;
  const int n = csr ? T : counts[E];
  __shared__ float s_bal[8 * LPT];  // the loss' gradient in p_e
  if (threadIdx.x < 8 * LPT) {
    const int e = threadIdx.x;
    float b = 0.f;
    if (d_aux && e < E && n > 0) {
      const int c = csr ? counts[e + 1] - counts[e] : counts[e];
      b = d_aux[0] * float(double(lbw) * (double(E) * c / (double(n) * k) - 1.0) / n);
    }
    s_bal[e] = b;
  }
  __syncthreads();
  float bal[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) bal[i] = s_bal[(i >> 2) * 4 * LPT + 4 * l + (i & 3)];
  const long stride = long(gridDim.x) * kW * per_warp;
  for (long tb = (long(blockIdx.x) * kW + warp) * per_warp; tb < T; tb += stride) {
    const int t = int(tb) + lane / LPT;
    const bool valid = t < T;
    const bool live = valid && (mask == nullptr || mask[t] != 0);
    float v[8], p[8], dw[8];
    row_softmax<LPT>(logits, t, valid, E, vec, l, v, p);
    unsigned taken = 0;
    float dw0 = 0.f, bal0 = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[i] = 0.f;
    if (d_w) {
      int first = 0;
#pragma unroll
      for (int j = 0; j < kMaxTopK; ++j) {
        if (j < k) {
          const size_t s = size_t(valid ? t : 0) * k + j;
          const int e = __ldg(expert_ids + s);
          const float g = __ldg(d_w + s);
          if (j == 0) {
            first = e;
            dw0 = g;
          }
          if ((e >> 2) % LPT == l) {
            const int i = (e >> 2) / LPT * 4 + (e & 3);
            taken |= 1u << i;
#pragma unroll
            for (int x = 0; x < 8; ++x)
              if (x == i) dw[x] = g - dw0;
          }
        }
      }
      bal0 = s_bal[first & (8 * LPT - 1)];
    }
    float q = 0.f, c = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if ((taken >> i) & 1u) {
        q += p[i];
        c = fmaf(dw[i], p[i], c);
      }
    }
    q = group_sum<LPT>(q) + 1e-9f;
    c = group_sum<LPT>(c) / q;
    const float rest = d_w ? (c - dw0 * (1e-9f / q)) / q : 0.f;
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      dw[i] = (bal[i] - bal0) + (((taken >> i) & 1u) ? dw[i] / q : rest);
      dot = fmaf(p[i], dw[i], dot);
    }
    dot = group_sum<LPT>(dot);
    if (!valid) continue;  // the loop bound is the same for the whole warp
    float* row = d_logits + size_t(t) * E;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int e0 = h * 4 * LPT + 4 * l;
      float g[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) g[r] = live ? p[4 * h + r] * (dw[4 * h + r] - dot) : 0.f;
      if (vec) {
        if (e0 < E) *reinterpret_cast<float4*>(row + e0) = make_float4(g[0], g[1], g[2], g[3]);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (e0 + r < E) row[e0 + r] = g[r];
      }
    }
  }
}

static int gating_blocks(int T, int E) {
  const int lpt = E <= 8 ? 1 : E <= 16 ? 2 : E <= 32 ? 4 : 8;
  const long per_block = kGateThreads / lpt;
  const long b = (T + per_block - 1) / per_block;
  return int(b < 1 ? 1 : b > kGateBlocksMax ? kGateBlocksMax : b);
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
static size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

// ---------------------------------------------------------------------------
// gate projection: gradients
// ---------------------------------------------------------------------------
// fp32 gradients meet fp16 rows and weights: they go in as two terms (rounded, and
// rounded remainder: 2^-22 left over), so no rounding beyond fp32's is added.
LR_DEVICE void split_tf32(float v, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(v));
  const float h = __uint_as_float(hi);
  const float r = fabsf(h) < INFINITY ? v - h : 0.f;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(r));
}

LR_DEVICE void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

LR_DEVICE void half8_bits(const uint4& v, uint32_t (&f)[8]) {
  const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = __half22float2(h[i]);
    f[2 * i] = __float_as_uint(x.x);
    f[2 * i + 1] = __float_as_uint(x.y);
  }
}

// dW[E,d] = dl^T h on mma.sync m16n8k16 fp16 with tokens as the k axis.  dl is
// split once, per chunk of 128 tokens and expert, into two fp16 terms of the
// column scaled by a power of two to [2^14, 2^15) (2^-22 of the column's largest
// is left over); rows g and g + 8 of an m-tile are the value and the remainder of
// expert g, so one instruction multiplies both and their sums stay apart until
// the chunk is done.  Every chunk is added to fp32 totals: a tensor-core chain is
// 8 steps long.
constexpr int kChunk = 128;     // tokens of a scale, and of a tensor-core chain
constexpr int kStage = 64;      // tokens of a pipeline stage
constexpr int kDwCols = 256;    // columns of h per block, 32 per warp
constexpr int kDwStages = 3;
constexpr int kHPitch = kDwCols * 2 + 16;  // bytes: ldmatrix rows in different banks

// The scaled terms in fragment order [16-token step][8-expert tile][lane], the
// powers of two that undo the scaling [chunk][E8], column sums [chunk][E8], and
// the transposed weight [d][E8] (zero past E) for the row gradient.  Blocks
// [0, chunks * groups) split dl, a chunk and 64 experts each; the rest transpose
// 64 columns each.  6 to 8 us beside the products' 20 to 25.
struct SplitArgs {
  const float* dl;
  const __half* wg;
  int T, d, E, E8;
  int split_blocks, groups;
  uint4* frag;
  float* down;
  float* colsum;  // nullable
  __half* wt;
};

__global__ void __launch_bounds__(256) gate_split_kernel(SplitArgs p) {
  __shared__ float s_dl[kChunk][65];
  __shared__ float s_red[4][64];
  __shared__ float s_up[64];
  pdl_wait();
  pdl_trigger();
  if (int(blockIdx.x) >= p.split_blocks) {
    const int c0 = (blockIdx.x - p.split_blocks) * 64;
    __half(*s_w)[66] = reinterpret_cast<__half(*)[66]>(&s_dl[0][0]);  // [expert][column]
    for (int e0 = 0; e0 < p.E8; e0 += 64) {
      __syncthreads();
      for (int i = threadIdx.x; i < 64 * 64; i += 256) {
        const int e = e0 + (i >> 6), c = c0 + (i & 63);
        s_w[i >> 6][i & 63] = e < p.E && c < p.d ? p.wg[size_t(e) * p.d + c] : __half(0.f);
      }
      __syncthreads();
      for (int i = threadIdx.x; i < 64 * 64; i += 256) {
        const int c = c0 + (i >> 6), e = e0 + (i & 63);
        if (c < p.d && e < p.E8) p.wt[size_t(c) * p.E8 + e] = s_w[i & 63][i >> 6];
      }
    }
    return;
  }
  const int chunk = blockIdx.x / p.groups, e0 = (blockIdx.x % p.groups) * 64;
  const int ne = min(64, p.E - e0), ne8 = min(64, p.E8 - e0);
  const long t0 = long(chunk) * kChunk;
  const int lg = ne8 <= 8 ? 3 : ne8 <= 16 ? 4 : ne8 <= 32 ? 5 : 6;  // columns read: 2^lg >= ne8
#pragma unroll 8
  for (int i = threadIdx.x; i < (kChunk << lg); i += 256) {
    const int t = i >> lg, e = i & ((1 << lg) - 1);
    s_dl[t][e] = t0 + t < p.T && e < ne ? __ldg(p.dl + size_t(t0 + t) * p.E + e0 + e) : 0.f;
  }
  __syncthreads();
  {
    const int e = threadIdx.x & 63, q = threadIdx.x >> 6;
    float m = 0.f, sum = 0.f;
    if (e < ne8) {
      for (int t = q; t < kChunk; t += 4) {
        const float a = fabsf(s_dl[t][e]);
        if (a < INFINITY) m = fmaxf(m, a);
        sum += s_dl[t][e];
      }
    }
    s_red[q][e] = m;
    __syncthreads();
    if (q == 0) {
      m = fmaxf(fmaxf(s_red[0][e], s_red[1][e]), fmaxf(s_red[2][e], s_red[3][e]));
      float down;
      half_range_scale(m, s_up[e], down);
      if (e < ne8) p.down[size_t(chunk) * p.E8 + e0 + e] = down;
    }
    __syncthreads();
    s_red[q][e] = sum;
    __syncthreads();
    if (q == 0 && p.colsum && e < ne8)
      p.colsum[size_t(chunk) * p.E8 + e0 + e] =
          (s_red[0][e] + s_red[1][e]) + (s_red[2][e] + s_red[3][e]);
  }
  // a thread writes a lane's A operand: 4 tokens of an expert, value and remainder
  const int tiles = p.E8 / 8, my_tiles = ne8 / 8;
  for (int i = threadIdx.x; i < (kChunk / 16) * my_tiles * 32; i += 256) {
    const int lane = i & 31, tile = (i >> 5) % my_tiles, step = (i >> 5) / my_tiles;
    const int e = tile * 8 + (lane >> 2), tq = lane & 3;
    uint32_t w[4];
#pragma unroll
    for (int half_k = 0; half_k < 2; ++half_k) {
      unsigned short h[2], l[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float x = s_dl[step * 16 + half_k * 8 + 2 * tq + u][e] * s_up[e];
        const __half hi = __float2half_rn(x);
        const float hf = __half2float(hi);
        h[u] = __half_as_ushort(hi);
        l[u] = __half_as_ushort(__float2half_rn(fabsf(hf) < INFINITY ? x - hf : 0.f));
      }
      w[2 * half_k] = h[0] | (uint32_t(h[1]) << 16);
      w[2 * half_k + 1] = l[0] | (uint32_t(l[1]) << 16);
    }
    p.frag[((size_t(chunk) * (kChunk / 16) + step) * tiles + e0 / 8 + tile) * 32 + lane] =
        make_uint4(w[0], w[1], w[2], w[3]);
  }
}

LR_DEVICE void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t saddr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(saddr));
}

// A block: 256 columns of h, up to 64 experts (blockIdx.z), a range of chunks.
// Stages of 64 tokens (rows of h and dl fragments) come in by cp.async, three
// deep.  Reading h bounds it with 8 experts (16384 x 4096: 24 us, 5.5 TB/s).  With 64
// (8111 x 2048: 21 us, 5 of HBM) 252 registers leave 8 warps on an SM, each of which
// reads all fragments of the 2 x 64 gradient rows from shared memory; the tensor pipe
// is 34 % busy.  tcgen05 (M = 128 fits) was not tried.  tf32 products of the unsplit
// gradients took 38 and 117 us.
template <int MTL>
__global__ void __launch_bounds__(256)
    gate_dw_kernel(const __half* __restrict__ h, const uint4* __restrict__ frag,
                   const float* __restrict__ down, int T, int d, int E, int E8, int chunks,
                   int chunks_per_block, float* __restrict__ part) {
  constexpr int kFragBytes = (kStage / 16) * MTL * 512;
  constexpr int kHBytes = kStage * kHPitch;
  extern __shared__ __align__(128) unsigned char s_dyn[];  // [stage][h rows, fragments]
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  const int d0 = blockIdx.x * kDwCols, e0 = blockIdx.z * 64;
  const int tiles = E8 / 8;
  const int c0 = blockIdx.y * chunks_per_block, c1 = min(chunks, c0 + chunks_per_block);
  const int stages = (c1 - c0) * (kChunk / kStage);
  const auto fetch = [&](int i) {
    if (i < stages) {
      unsigned char* sh = s_dyn + (i % kDwStages) * (kHBytes + kFragBytes);
      const long t0 = long(c0) * kChunk + long(i) * kStage;
#pragma unroll
      for (int u = 0; u < kStage / 8; ++u) {  // a warp per row
        const int t = u * 8 + warp, c = d0 + lane * 8;
        const bool ok = t0 + t < T && c < d;
        cp_async_16_zfill(sh + t * kHPitch + lane * 16, h + size_t(ok ? t0 + t : 0) * d + (ok ? c : 0),
                          ok);
      }
      const uint4* fp = frag + (t0 / 16) * tiles * 32 + (e0 / 8) * 32;
      for (int x = threadIdx.x; x < (kStage / 16) * MTL * 32; x += 256) {
        const int step = x / (MTL * 32), in = x % (MTL * 32);
        const bool ok = e0 / 8 + in / 32 < tiles;
        cp_async_16_zfill(sh + kHBytes + x * 16, fp + (ok ? step * tiles * 32 + in : 0), ok);
      }
    }
    cp_async_commit();
  };
  float total[MTL][4][2];
#pragma unroll
  for (int m = 0; m < MTL; ++m)
#pragma unroll
    for (int n = 0; n < 4; ++n) total[m][n][0] = total[m][n][1] = 0.f;
#pragma unroll
  for (int i = 0; i < kDwStages - 1; ++i) fetch(i);
  float acc[MTL][4][4];
  for (int i = 0; i < stages; ++i) {
    cp_async_wait_group<kDwStages - 2>();
    __syncthreads();
    fetch(i + kDwStages - 1);
    if (i % (kChunk / kStage) == 0) {
#pragma unroll
      for (int m = 0; m < MTL; ++m)
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[m][n][c] = 0.f;
    }
    const unsigned char* sh = s_dyn + (i % kDwStages) * (kHBytes + kFragBytes);
    const uint32_t hrow = smem_u32(sh) + (lane & 15) * kHPitch + warp * 64 + (lane >> 4) * 16;
    const uint4* fr = reinterpret_cast<const uint4*>(sh + kHBytes) + lane;
#pragma unroll
    for (int step = 0; step < kStage / 16; ++step) {
      uint32_t b[2][4];
      ldmatrix_x4_trans(b[0], hrow + step * 16 * kHPitch);
      ldmatrix_x4_trans(b[1], hrow + step * 16 * kHPitch + 32);
#pragma unroll
      for (int m = 0; m < MTL; ++m) {
        const uint4 a = fr[(step * MTL + m) * 32];
#pragma unroll
        for (int n = 0; n < 4; ++n)
          mma_f16(acc[m][n], a.x, a.y, a.z, a.w, b[n >> 1][(n & 1) * 2], b[n >> 1][(n & 1) * 2 + 1]);
      }
    }
    if (i % (kChunk / kStage) == kChunk / kStage - 1) {
      const int chunk = c0 + i / (kChunk / kStage);
#pragma unroll
      for (int m = 0; m < MTL; ++m) {
        const int e = e0 + m * 8 + g;
        const float f = e < E8 ? __ldg(down + size_t(chunk) * E8 + e) : 0.f;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          total[m][n][0] = fmaf(acc[m][n][0] + acc[m][n][2], f, total[m][n][0]);
          total[m][n][1] = fmaf(acc[m][n][1] + acc[m][n][3], f, total[m][n][1]);
        }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MTL; ++m) {
    const int e = e0 + m * 8 + g;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int c = d0 + warp * 32 + n * 8 + 2 * tq;
      if (e < E && c < d)
        *reinterpret_cast<float2*>(part + (size_t(blockIdx.y) * E + e) * d + c) =
            make_float2(total[m][n][0], total[m][n][1]);
    }
  }
}

// out[i] = sum over the token ranges of part[s][i], in range order; the bias
// gradient from the chunks' column sums, a warp per expert.
__global__ void __launch_bounds__(256)
    sum_parts_kernel(const float* __restrict__ part, long n4, int splits, long blocks,
                     float* __restrict__ out, const float* __restrict__ colsum, int chunks, int E,
                     int E8, float* __restrict__ out_b) {
  pdl_wait();
  pdl_trigger();
  if (blockIdx.x >= blocks) {
    const int e = int(blockIdx.x - blocks) * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    float s = 0.f;
    if (e < E)
      for (int c = lane; c < chunks; c += 32) s += colsum[size_t(c) * E8 + e];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (e < E && lane == 0) out_b[e] = s;
    return;
  }
  // 32 columns of four; warp w adds ranges w, w + 8, ..., then the warps in order
  __shared__ float4 s_sum[8][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long i = long(blockIdx.x) * 32 + lane;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (i < n4) {
    const float4* q = reinterpret_cast<const float4*>(part) + i;
#pragma unroll 4
    for (int k = warp; k < splits; k += 8) {
      const float4 v = __ldcg(q + size_t(k) * n4);
      s.x += v.x;
      s.y += v.y;
      s.z += v.z;
      s.w += v.w;
    }
  }
  s_sum[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && i < n4) {
#pragma unroll
    for (int w = 1; w < 8; ++w) {
      const float4 v = s_sum[w][lane];
      s.x += v.x;
      s.y += v.y;
      s.z += v.z;
      s.w += v.w;
    }
    reinterpret_cast<float4*>(out)[i] = s;
  }
}

// A row gradient: rounded to fp16, or fp32 as it is.
LR_DEVICE void store_dh(__half* to, float v) { *to = __float2half_rn(v); }
LR_DEVICE void store_dh(float* to, float v) { *to = v; }
LR_DEVICE void store_dh8(__half* to, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(to) = pack_half8(v);
}
LR_DEVICE void store_dh8(float* to, const float (&v)[8]) {
  reinterpret_cast<float4*>(to)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(to)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// dh[T,d] = dl W for more experts than the low-rank kernel takes (128).
// fp32 gradients go in as two tf32 terms.  A warp owns MT*16 tokens x 64 columns; experts are
// the k axis.  n-tile j takes column g*8 + j of the lane's 16-byte weight load,
// so a lane ends with 16 neighbouring columns of its rows.
template <int MT, typename DH>
__global__ void __launch_bounds__(256)
    gate_dh_kernel(const float* __restrict__ dl, const __half* __restrict__ wg, int T, int d, int E,
                   DH* __restrict__ dh) {
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  const int t0 = blockIdx.x * (16 * MT);
  const int d0 = (blockIdx.y * 8 + warp) * 64;
  if (d0 >= d) return;
  const bool dok = d0 + g * 8 < d;
  float acc[MT][8][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][j][i] = 0.f;
  for (int e0 = 0; e0 < E; e0 += 8) {
    uint32_t b[2][8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int e = e0 + tq + 4 * u;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (e < E && dok) v = __ldg(reinterpret_cast<const uint4*>(wg + size_t(e) * d + d0 + g * 8));
      half8_bits(v, b[u]);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = t0 + m * 16 + g + 8 * (i & 1);
        const int e = e0 + tq + 4 * (i >> 1);
        split_tf32((t < T && e < E) ? __ldg(dl + size_t(t) * E + e) : 0.f, hi[i], lo[i]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        mma_tf32(acc[m][j], hi, b[0][j], b[1][j]);
        mma_tf32(acc[m][j], lo, b[0][j], b[1][j]);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int t = t0 + m * 16 + g + 8 * r;
      if (t >= T) continue;
#pragma unroll
      for (int half_i = 0; half_i < 2; ++half_i) {  // columns (2tq) * 8 .. and (2tq + 1) * 8 ..
        const int c = d0 + (2 * tq + half_i) * 8;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = acc[m][j][2 * r + half_i];
        if (c < d) store_dh8(dh + size_t(t) * d + c, v);
      }
    }
}

// All three gradients of a small batch (up to 256 tokens, 64 experts) in one launch,
// on CUDA cores in fp32: a block owns 64 columns, dl and its columns of W lie in
// shared memory.  The four launches above cost such a batch more time on the host
// than on the GPU (64 tokens x 256, 8 experts: 11 us against 3).
constexpr int kSmallGateTokens = 256;
constexpr int kSmallGateExperts = 64;

template <typename DH>
__global__ void __launch_bounds__(256)
    gate_backward_small_kernel(const __half* __restrict__ h, const __half* __restrict__ wg,
                               const float* __restrict__ dl, int T, int d, int E,
                               DH* __restrict__ dh, float* __restrict__ dw,
                               float* __restrict__ db) {
  extern __shared__ __align__(128) unsigned char s_dyn[];
  const int EP = (E + 3) & ~3;                       // zeros past E
  float* s_dl = reinterpret_cast<float*>(s_dyn);     // [T][EP]
  float* s_w = s_dl + T * EP;                        // [EP][64]
  pdl_wait();
  pdl_trigger();
  const int c = threadIdx.x & 63, q = threadIdx.x >> 6;
  const int col = blockIdx.x * 64 + c;
  for (int i = threadIdx.x; i < T * EP; i += 256) {
    const int t = i / EP, e = i % EP;
    s_dl[i] = e < E ? __ldg(dl + size_t(t) * E + e) : 0.f;
  }
  if (dh)
    for (int e = q; e < EP; e += 4)
      s_w[e * 64 + c] = e < E && col < d ? __half2float(wg[size_t(e) * d + col]) : 0.f;
  __syncthreads();
  if (dh && col < d) {
    for (int t0 = q; t0 < T; t0 += 16) {  // tokens t0, t0 + 4, t0 + 8, t0 + 12
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      for (int e = 0; e < EP; e += 4) {
        const float w0 = s_w[e * 64 + c], w1 = s_w[(e + 1) * 64 + c];
        const float w2 = s_w[(e + 2) * 64 + c], w3 = s_w[(e + 3) * 64 + c];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (t0 + 4 * u < T) {
            const float4 g = *reinterpret_cast<const float4*>(s_dl + (t0 + 4 * u) * EP + e);
            acc[u] = fmaf(g.x, w0, acc[u]);
            acc[u] = fmaf(g.y, w1, acc[u]);
            acc[u] = fmaf(g.z, w2, acc[u]);
            acc[u] = fmaf(g.w, w3, acc[u]);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (t0 + 4 * u < T) store_dh(dh + size_t(t0 + 4 * u) * d + col, acc[u]);
    }
  }
  if (dw && col < d) {
    // experts 16 g + 4 q .. 16 g + 4 q + 3 of groups g
    float acc[kSmallGateExperts / 16][4];
#pragma unroll
    for (int g = 0; g < kSmallGateExperts / 16; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[g][i] = 0.f;
#pragma unroll 4
    for (int t = 0; t < T; ++t) {
      const float x = __half2float(h[size_t(t) * d + col]);
#pragma unroll
      for (int g = 0; g < kSmallGateExperts / 16; ++g) {
        if (16 * g + 4 * q < EP) {
          const float4 v = *reinterpret_cast<const float4*>(s_dl + t * EP + 16 * g + 4 * q);
          acc[g][0] = fmaf(v.x, x, acc[g][0]);
          acc[g][1] = fmaf(v.y, x, acc[g][1]);
          acc[g][2] = fmaf(v.z, x, acc[g][2]);
          acc[g][3] = fmaf(v.w, x, acc[g][3]);
        }
      }
    }
#pragma unroll
    for (int g = 0; g < kSmallGateExperts / 16; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = 16 * g + 4 * q + i;
        if (e < E) dw[size_t(e) * d + col] = acc[g][i];
      }
  }
  if (db && blockIdx.x == 0 && threadIdx.x < E) {
    float sum = 0.f;
    for (int t = 0; t < T; ++t) sum += s_dl[t * EP + threadIdx.x];
    db[threadIdx.x] = sum;
  }
}

// fp32 -> fp16, n values (a multiple of 8).
__global__ void __launch_bounds__(256)
    round_half_kernel(const float4* __restrict__ src, uint4* __restrict__ dst, long n8) {
  pdl_wait();
  pdl_trigger();
  const long i = long(blockIdx.x) * 256 + threadIdx.x;
  if (i >= n8) return;
  const float4 a = src[2 * i], b = src[2 * i + 1];
  const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  dst[i] = pack_half8(v);
}

struct GatePlan {
  int E8, chunks, groups, per_block, splits;
  size_t frag, down, colsum, wt, part, bytes;  // workspace offsets
};

// Token ranges of the weight gradient: as many chunks per block as keep the SMs
// full (two blocks on each up to 32 experts, whose stages leave room for two).
static GatePlan gate_plan(int T, int d, int E) {
  GatePlan p;
  p.E8 = (E + 7) & ~7;
  p.groups = (E + 63) / 64;
  p.chunks = (T + kChunk - 1) / kChunk;
  const long cols = long((d + kDwCols - 1) / kDwCols) * p.groups;
  const long fill = E > 32 ? kTargetBlocks : 2 * kTargetBlocks;
  p.per_block = int((p.chunks * cols + fill - 1) / fill);
  p.splits = (p.chunks + p.per_block - 1) / p.per_block;
  if (cols * p.splits > fill && p.splits > 1) {  // no few blocks in a wave of their own
    p.per_block = int((p.chunks + p.splits - 2) / (p.splits - 1));
    p.splits = (p.chunks + p.per_block - 1) / p.per_block;
  }
  p.frag = 0;
  p.down = p.frag + size_t(p.chunks) * (kChunk / 16) * (p.E8 / 8) * 512;
  p.colsum = p.down + align256(size_t(p.chunks) * p.E8 * sizeof(float));
  p.wt = p.colsum + align256(size_t(p.chunks) * p.E8 * sizeof(float));
  p.part = p.wt + align256(size_t(d) * p.E8 * sizeof(__half));
  p.bytes = p.part + (p.splits > 1 ? size_t(p.splits) * E * d * sizeof(float) : 0);
  return p;
}

template <int MTL>
static int launch_dw(const __half* h, const uint4* frag, const float* down, int T, int d, int E,
                     const GatePlan& gp, float* part, cudaStream_t stream) {
  constexpr int smem = kDwStages * (kStage * kHPitch + (kStage / 16) * MTL * 512);
  auto kern = gate_dw_kernel<MTL>;
  static unsigned long long configured = 0;
  if (const int rc = set_dyn_smem_once(kern, smem, configured)) return rc;
  const dim3 grid((d + kDwCols - 1) / kDwCols, gp.splits, gp.groups);
  return launch_pdl(kern, grid, dim3(256), smem, stream, h, frag, down, T, d, E, gp.E8, gp.chunks,
                    gp.per_block, part);
}

// ---------------------------------------------------------------------------
// weighted combine: gradients
// ---------------------------------------------------------------------------
// HBM bounds it: 16384 tokens x 2 slots x 4096 in 107 us, 6.3 TB/s; the weights'
// gradient alone 70 us.
// WPT warps share a token's row: the row of dout is read once, each kept slot's
// y row once, dy written once; the dot products are summed over lanes and warps
// in a fixed order.  Rows no slot keeps (the tail of an over-full expert's
// segment) are zero-filled by the warps of the tokens with the same numbers.  With
// one of the two gradients alone (frozen experts: DW) the other's bytes stay away.
template <int WPT, bool DY, bool DW>
__global__ void __launch_bounds__(256)
    combine_backward_kernel(const uint4* __restrict__ dout, const uint4* __restrict__ y,
                            const float* __restrict__ gate_w, const int32_t* __restrict__ slot_pos,
                            const int32_t* __restrict__ offsets,
                            const int32_t* __restrict__ kept_counts, int E, int T, int k, int d8,
                            uint4* __restrict__ dy, float* __restrict__ d_w) {
  constexpr int kTok = 8 / WPT;
  __shared__ float s_dot[8][kMaxTopK];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = warp % WPT;
  const long t = long(blockIdx.x) * kTok + warp / WPT;
  const bool valid = t < T;
  int my_pos = -1;
  float my_w = 0.f;
  if (valid && lane < k) {
    my_pos = __ldg(slot_pos + size_t(t) * k + lane);
    my_w = __ldg(gate_w + size_t(t) * k + lane);
  }
  int pos[kMaxTopK];
  float w[kMaxTopK], dot[kMaxTopK];
#pragma unroll
  for (int j = 0; j < kMaxTopK; ++j) {
    pos[j] = __shfl_sync(0xffffffffu, my_pos, j);
    w[j] = __shfl_sync(0xffffffffu, my_w, j);
    dot[j] = 0.f;
  }
  if (valid) {
    constexpr int U = 2;
    for (int c0 = part * 32 * U; c0 < d8; c0 += WPT * 32 * U) {
      uint4 g[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = c0 + u * 32 + lane;
        if (c < d8) g[u] = ld_stream(dout + size_t(t) * d8 + c);
      }
#pragma unroll
      for (int j = 0; j < kMaxTopK; ++j) {
        if (j < k && pos[j] >= 0) {
          uint4 v[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int c = c0 + u * 32 + lane;
            if (DW && c < d8) v[u] = ld_stream(y + size_t(pos[j]) * d8 + c);
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int c = c0 + u * 32 + lane;
            if (c < d8) {
              const __half2* gh = reinterpret_cast<const __half2*>(&g[u]);
              const __half2* vh = reinterpret_cast<const __half2*>(&v[u]);
              float o[8];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 a = __half22float2(gh[i]);
                if (DW) {
                  const float2 b = __half22float2(vh[i]);
                  dot[j] = fmaf(a.x, b.x, dot[j]);
                  dot[j] = fmaf(a.y, b.y, dot[j]);
                }
                o[2 * i] = w[j] * a.x;
                o[2 * i + 1] = w[j] * a.y;
              }
              if (DY) dy[size_t(pos[j]) * d8 + c] = pack_half8(o);
            }
          }
        }
      }
    }
    // rows that no slot keeps
    for (int j = 0; DY && j < k; ++j) {
      const long r = t * k + j;
      bool drop = false;
      for (int e = lane; e < E; e += 32)
        drop = drop || (r >= long(__ldg(offsets + e)) + __ldg(kept_counts + e) &&
                        r < __ldg(offsets + e + 1));
      if (__any_sync(0xffffffffu, drop)) {
        for (int c = part * 32 + lane; c < d8; c += WPT * 32)
          dy[size_t(r) * d8 + c] = make_uint4(0, 0, 0, 0);
      }
    }
  }
  if (!DW) return;
#pragma unroll
  for (int j = 0; j < kMaxTopK; ++j) {
    if (j < k) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], o);
      if (lane == 0) s_dot[warp][j] = dot[j];
    }
  }
  __syncthreads();
  if (valid && part == 0 && lane < k) {
    float s = 0.f;
#pragma unroll
    for (int p = 0; p < WPT; ++p) s += s_dot[warp + p][lane];
    d_w[size_t(t) * k + lane] = s;
  }
}

}  // namespace lr

// ===========================================================================
// C ABI
// ===========================================================================
using namespace lr;

static bool gating_args_ok(int T, int E, int k) {
  return T >= 0 && T <= kMaxRows && E >= 1 && E <= 64 && k >= 1 && k <= kMaxTopK && k <= E;
}

extern "C" size_t lr_balanced_gating_workspace_bytes(int num_tokens, int num_experts) {
  if (num_tokens < 1 || num_experts < 1) return 0;
  const size_t B = gating_blocks(num_tokens, num_experts);
  if (B == 1) return 0;
  return align256(B * num_experts * sizeof(double)) + B * (num_experts + 1) * sizeof(int32_t);
}

extern "C" int lr_balanced_gating(const float* logits, const uint8_t* token_mask, int T, int E,
                                  int k, float load_balance_weight, int32_t* expert_ids,
                                  float* gate_weights, int32_t* counts, float* aux_loss,
                                  void* workspace, size_t workspace_bytes, lr_stream_t stream) {
  if (!gating_args_ok(T, E, k) || !counts || !aux_loss) return LR_ERR_INVALID_ARGUMENT;
  if (T == 0) {
    LR_CUDA_TRY(cudaMemsetAsync(counts, 0, (E + 1) * sizeof(int32_t), stream));
    LR_CUDA_TRY(cudaMemsetAsync(aux_loss, 0, sizeof(float), stream));
    return LR_OK;
  }
  if (!logits || !expert_ids || !gate_weights) return LR_ERR_INVALID_ARGUMENT;
  const int B = gating_blocks(T, E);
  GatingParts parts{nullptr, nullptr};
  if (B > 1) {
    if (!workspace || workspace_bytes < lr_balanced_gating_workspace_bytes(T, E))
      return LR_ERR_WORKSPACE;
    if (!aligned16(workspace)) return LR_ERR_INVALID_ARGUMENT;  // it starts with doubles
    parts.psum = static_cast<double*>(workspace);
    parts.count = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) +
                                             align256(size_t(B) * E * sizeof(double)));
  }
  const bool vec = E % 4 == 0 && aligned16(logits);
  auto run = [&](auto kern) {
    return launch_pdl(kern, dim3(B), dim3(kGateThreads), 0, stream, logits, token_mask, T, E, k,
                      load_balance_weight, vec, expert_ids, gate_weights, counts, aux_loss, parts);
  };
  const int rc = E <= 8    ? run(balanced_gating_kernel<1>)
                 : E <= 16 ? run(balanced_gating_kernel<2>)
                 : E <= 32 ? run(balanced_gating_kernel<4>)
                           : run(balanced_gating_kernel<8>);
  if (rc != LR_OK || B == 1) return rc;
  return launch_pdl(gating_stats_kernel, dim3(1), dim3(1024), 0, stream, parts, B, E, k,
                    load_balance_weight, counts, aux_loss);
}

extern "C" int lr_balanced_gating_backward(const float* logits, const uint8_t* token_mask,
                                           const int32_t* expert_ids, const int32_t* counts,
                                           int counts_are_offsets, const float* d_weights,
                                           const float* d_aux, int T, int E, int k,
                                           float load_balance_weight, float* d_logits,
                                           lr_stream_t stream) {
  if (!gating_args_ok(T, E, k)) return LR_ERR_INVALID_ARGUMENT;
  if (T == 0) return LR_OK;
  if (!logits || !counts || !d_logits || (d_weights && !expert_ids))
    return LR_ERR_INVALID_ARGUMENT;
  if (counts_are_offsets && token_mask) return LR_ERR_INVALID_ARGUMENT;
  const bool vec = E % 4 == 0 && aligned16(logits) && aligned16(d_logits);
  const int B = gating_blocks(T, E);
  auto run = [&](auto kern) {
    return launch_pdl(kern, dim3(B), dim3(kGateThreads), 0, stream, logits, token_mask, expert_ids,
                      counts, counts_are_offsets, d_weights, d_aux, T, E, k, load_balance_weight,
                      vec, d_logits);
  };
  return E <= 8    ? run(balanced_gating_backward_kernel<1>)
         : E <= 16 ? run(balanced_gating_backward_kernel<2>)
         : E <= 32 ? run(balanced_gating_backward_kernel<4>)
                   : run(balanced_gating_backward_kernel<8>);
}

extern "C" int lr_round_half(const float* src, void* dst, long long n, lr_stream_t stream) {
  if (n < 0 || n % 8 != 0) return LR_ERR_INVALID_ARGUMENT;
  if (n == 0) return LR_OK;
  if (!src || !dst || !aligned16(src) || !aligned16(dst)) return LR_ERR_INVALID_ARGUMENT;
  return launch_pdl(round_half_kernel, dim3(unsigned((n / 8 + 255) / 256)), dim3(256), 0, stream,
                    reinterpret_cast<const float4*>(src), static_cast<uint4*>(dst), long(n / 8));
}

extern "C" size_t lr_gate_backward_workspace_bytes(int num_tokens, int d_model, int num_experts) {
  if (num_tokens < 1 || d_model < 1 || num_experts < 1) return 0;
  if (num_tokens <= kSmallGateTokens && num_experts <= kSmallGateExperts) return 0;
  return gate_plan(num_tokens, d_model, num_experts).bytes;
}

// DH: the type of d_h.
template <typename DH>
static int gate_backward(const void* h, const void* wg, const float* d_logits, int T, int d, int E,
                         void* d_h, float* d_wg, float* d_bias, void* workspace,
                         size_t workspace_bytes, lr_stream_t stream) {
  if (T < 0 || T > kMaxRows || d <= 0 || d % 16 != 0 || d > kMaxColumns || E < 1 ||
      E > 256)
    return LR_ERR_INVALID_ARGUMENT;
  if (d_bias && !d_wg) return LR_ERR_INVALID_ARGUMENT;
  if (T == 0) {
    if (d_wg) LR_CUDA_TRY(cudaMemsetAsync(d_wg, 0, size_t(E) * d * sizeof(float), stream));
    if (d_bias) LR_CUDA_TRY(cudaMemsetAsync(d_bias, 0, size_t(E) * sizeof(float), stream));
    return LR_OK;
  }
  if (!d_logits || (d_h && !wg) || (d_wg && !h)) return LR_ERR_INVALID_ARGUMENT;
  if (!aligned16(h) || !aligned16(wg) || !aligned16(d_h) || !aligned16(d_wg))
    return LR_ERR_INVALID_ARGUMENT;
  if (!d_wg && !d_h) return LR_OK;
  if (T <= kSmallGateTokens && E <= kSmallGateExperts) {
    const int ep = (E + 3) & ~3;
    static unsigned long long configured = 0;
    if (const int rc = set_dyn_smem_once(
            gate_backward_small_kernel<DH>,
            (kSmallGateTokens + 64) * kSmallGateExperts * int(sizeof(float)), configured))
      return rc;
    return launch_pdl(gate_backward_small_kernel<DH>, dim3((d + 63) / 64), dim3(256),
                      size_t(T + 64) * ep * sizeof(float), stream,
                      static_cast<const __half*>(h), static_cast<const __half*>(wg), d_logits, T,
                      d, E, static_cast<DH*>(d_h), d_wg, d_bias);
  }
  const GatePlan gp = gate_plan(T, d, E);
  if (!workspace || !aligned16(workspace) || workspace_bytes < gp.bytes) return LR_ERR_WORKSPACE;
  if (gp.splits > 65535) return LR_ERR_INVALID_ARGUMENT;
  char* ws = static_cast<char*>(workspace);
  const bool low_rank = d_h && E <= kMaxRank;
  SplitArgs sp;
  sp.dl = d_logits;
  sp.wg = static_cast<const __half*>(wg);
  sp.T = T;
  sp.d = d;
  sp.E = E;
  sp.E8 = gp.E8;
  sp.groups = gp.groups;
  sp.split_blocks = d_wg ? gp.chunks * gp.groups : 0;
  sp.frag = reinterpret_cast<uint4*>(ws + gp.frag);
  sp.down = reinterpret_cast<float*>(ws + gp.down);
  sp.colsum = d_bias ? reinterpret_cast<float*>(ws + gp.colsum) : nullptr;
  sp.wt = reinterpret_cast<__half*>(ws + gp.wt);
  const int blocks = sp.split_blocks + (low_rank ? (d + 63) / 64 : 0);
  if (blocks > 0)
    if (const int rc = launch_pdl(gate_split_kernel, dim3(blocks), dim3(256), 0, stream, sp))
      return rc;
  if (d_h) {
    if (low_rank) {
      ExpandArgs ep{};
      ep.v = d_logits;
      ep.b[0] = sp.wt;
      ep.out = d_h;
      ep.R = T;
      ep.N = d;
      ep.n = 1;
      ep.r = E;
      ep.ldb = gp.E8;
      constexpr int kMode = std::is_same<DH, float>::value ? kExpandProduct32 : kExpandProduct;
      if (const int rc = run_expand<kMode>(ep, stream)) return rc;
    } else {
      constexpr int MT = 2;
      const dim3 grid((T + 16 * MT - 1) / (16 * MT), (d + 511) / 512);
      if (const int rc = launch_pdl(gate_dh_kernel<MT, DH>, grid, dim3(256), 0, stream, d_logits,
                                    static_cast<const __half*>(wg), T, d, E,
                                    static_cast<DH*>(d_h)))
        return rc;
    }
  }
  if (d_wg) {
    float* part = gp.splits > 1 ? reinterpret_cast<float*>(ws + gp.part) : d_wg;
    const __half* hp = static_cast<const __half*>(h);
    const int rc = E <= 8    ? launch_dw<1>(hp, sp.frag, sp.down, T, d, E, gp, part, stream)
                   : E <= 16 ? launch_dw<2>(hp, sp.frag, sp.down, T, d, E, gp, part, stream)
                   : E <= 32 ? launch_dw<4>(hp, sp.frag, sp.down, T, d, E, gp, part, stream)
                             : launch_dw<8>(hp, sp.frag, sp.down, T, d, E, gp, part, stream);
    if (rc != LR_OK) return rc;
    const long n4 = gp.splits > 1 ? long(E) * d / 4 : 0;
    const long sum_blocks = (n4 + 31) / 32, bias_blocks = d_bias ? (E + 7) / 8 : 0;
    if (sum_blocks + bias_blocks > 0)
      return launch_pdl(sum_parts_kernel, dim3(unsigned(sum_blocks + bias_blocks)), dim3(256), 0,
                        stream, static_cast<const float*>(part), n4, gp.splits, sum_blocks, d_wg,
                        static_cast<const float*>(sp.colsum), gp.chunks, E, gp.E8, d_bias);
  }
  return LR_OK;
}

extern "C" int lr_gate_backward(const void* h, const void* wg, const float* d_logits, int T, int d,
                                int E, void* d_h, float* d_wg, float* d_bias, void* workspace,
                                size_t workspace_bytes, lr_stream_t stream) {
  return gate_backward<__half>(h, wg, d_logits, T, d, E, d_h, d_wg, d_bias, workspace,
                               workspace_bytes, stream);
}

extern "C" int lr_gate_backward_rows32(const void* h, const void* wg, const float* d_logits, int T,
                                       int d, int E, float* d_h, float* d_wg, float* d_bias,
                                       void* workspace, size_t workspace_bytes,
                                       lr_stream_t stream) {
  return gate_backward<float>(h, wg, d_logits, T, d, E, d_h, d_wg, d_bias, workspace,
                              workspace_bytes, stream);
}

extern "C" int lr_combine_backward(const void* d_out, const void* y, const float* gate_weights,
                                   const int32_t* slot_pos, const int32_t* offsets,
                                   const int32_t* kept_counts, int T, int k, int d, int E,
                                   void* d_y, float* d_weights, lr_stream_t stream) {
  if (T < 0 || k < 1 || k > kMaxTopK || long(T) * k > kMaxRows || d <= 0 || d % 8 != 0 || E < 1)
    return LR_ERR_INVALID_ARGUMENT;
  if (T == 0) return LR_OK;
  if (!d_out || !y || !gate_weights || !slot_pos || !offsets || !kept_counts)
    return LR_ERR_INVALID_ARGUMENT;
  if (!aligned16(d_out) || !aligned16(y) || !aligned16(d_y)) return LR_ERR_INVALID_ARGUMENT;
  const int d8 = d / 8;
  auto run = [&](auto kern, int wpt) {
    const int per = 8 / wpt;
    return launch_pdl(kern, dim3((T + per - 1) / per), dim3(256), 0, stream,
                      static_cast<const uint4*>(d_out), static_cast<const uint4*>(y), gate_weights,
                      slot_pos, offsets, kept_counts, E, T, k, d8, static_cast<uint4*>(d_y),
                      d_weights);
  };
  if (!d_y && !d_weights) return LR_OK;
  if (!d_y)
    return T < 2368 ? run(combine_backward_kernel<8, false, true>, 8)
                    : run(combine_backward_kernel<1, false, true>, 1);
  if (!d_weights)
    return T < 2368 ? run(combine_backward_kernel<8, true, false>, 8)
                    : run(combine_backward_kernel<1, true, false>, 1);
  return T < 2368 ? run(combine_backward_kernel<8, true, true>, 8)
                  : run(combine_backward_kernel<1, true, true>, 1);
}
