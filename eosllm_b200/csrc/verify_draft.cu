// verify_draft.cu -- verification of drafted tokens against the target's
// probabilities, from given random numbers.
//
// Sequence i has k_i drafted tokens x_0 .. x_{k-1}, target rows p_0 .. p_k,
// draft rows q_0 .. q_{k-1} and uniform numbers u_0 .. u_{K-1} and u_K.  The
// leading drafts with u_j q_j(x_j) < p_j(x_j) are accepted (accepting with
// probability min(1, p/q)); the products are compared exactly (f64).  After
// the first rejection, at a, one token is drawn from max(p_a - q_a, 0), or,
// where that leaves nothing, from p_a; after k acceptances it is drawn from
// p_k.  The draw is the lowest v with C_v > u_K C_last for the running sum C
// of the weights in f64 (weights that are not positive and finite count 0; where
// u C_last lies within rounding of a running sum, a neighbour of it may be drawn).
// Tokens so drawn are distributed as the target's own.
#include "eos_common.cuh"
#include "eos_kernels.h"

namespace eos {

struct VerifyParams {
  const float* p;  // [n_seq][K + 1][stride]
  const float* q;  // [n_seq][K][stride]
  uint64_t stride;
  const uint32_t* drafts;   // [n_seq][K]
  const uint32_t* n_draft;  // [n_seq], nullptr: K each
  const float* u;           // [n_seq][K + 1]
  uint32_t max_draft, n_vocab;
  uint32_t* tokens;   // [n_seq][K + 1]
  uint32_t* n_token;  // [n_seq]
};

__device__ __forceinline__ double vd_weight(float p, float q, bool residual) {
  if (residual) {
    const double d = (double)p - (double)q;
    return (d > 0.0 && d < (double)INFINITY) ? d : 0.0;
  }
  return (p > 0.0f && p < INFINITY) ? (double)p : 0.0;
}

// Four neighbouring weights v .. v + 3 of [.., hi) (0 beyond).
template <bool VEC>
__device__ __forceinline__ void vd_weights4(const float* p, const float* q, uint32_t v, uint32_t hi, bool residual,
                                            double* w) {
  float a[4] = {0.0f, 0.0f, 0.0f, 0.0f}, b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (VEC && v + 4u <= hi) {
    const float4 x = __ldg(reinterpret_cast<const float4*>(p + v));
    a[0] = x.x, a[1] = x.y, a[2] = x.z, a[3] = x.w;
    if (residual) {
      const float4 y = __ldg(reinterpret_cast<const float4*>(q + v));
      b[0] = y.x, b[1] = y.y, b[2] = y.z, b[3] = y.w;
    }
  } else {
#pragma unroll
    for (uint32_t e = 0; e < 4u; ++e)
      if (v + e < hi) {
        a[e] = __ldg(p + v + e);
        if (residual) b[e] = __ldg(q + v + e);
      }
  }
#pragma unroll
  for (uint32_t e = 0; e < 4u; ++e) w[e] = vd_weight(a[e], b[e], residual);
}

constexpr uint32_t kVdThreads = 512, kVdWarps = kVdThreads / 32, kVdMaxCluster = 8;

__device__ __forceinline__ void vd_cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ void vd_cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
  vd_cluster_wait();
}
// Address of a shared variable in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t vd_map(const void* p, uint32_t rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;"
      : "=r"(a)
      : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return a;
}

// One cluster of CTAs per sequence; CTA c and in it warp w own the row's
// contiguous slices in order.  A first pass sums the slices and tells every CTA
// the others' sums; the warp whose slice crosses the cut goes over it once
// more (from L1 or L2).  Reading one or two rows once is what bounds it for
// many sequences, the chain of three reads (draft, its probabilities, the
// row) for few: so few sequences get eight CTAs each.  One sequence of 4 drafts
// and 32000 tokens: 5.8 us; 64 of 7: 10.3 us, of which the 8.2 MB read take 1.3;
// the rest are the two reads before it and the barriers between (64 sequences:
// per instruction a warp waits ten slots at barriers and six on memory).
template <bool VEC, uint32_t NC>
__global__ void __launch_bounds__(kVdThreads) verify_draft_kernel(const VerifyParams a) {
  __shared__ uint32_t s_taken;
  __shared__ double s_sum[kVdWarps];
  __shared__ uint32_t s_last[kVdWarps];
  __shared__ double c_sum[NC];
  __shared__ uint32_t c_last[NC];
  // this CTA runs: the others may write into its shared memory (nothing to be made visible yet)
  asm volatile("barrier.cluster.arrive.relaxed.aligned;");
  const uint32_t i = blockIdx.x / NC, cta = blockIdx.x % NC;
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const uint32_t kk = a.max_draft;
  uint32_t k = a.n_draft != nullptr ? a.n_draft[i] : kk;
  if (k > kk) k = kk;
  const float* prow = a.p + (size_t)i * (kk + 1u) * a.stride;
  const float* qrow = a.q + (size_t)i * kk * a.stride;
  const float* urow = a.u + (size_t)i * (kk + 1u);
  const double u = (double)urow[kk];
  if (warp == 0) {  // 32 drafts at a time: the first that is not accepted
    uint32_t taken = k;
    for (uint32_t t0 = 0; t0 < k; t0 += 32u) {
      const uint32_t t = t0 + lane;
      bool good = t >= k;
      if (t < k) {
        const uint32_t x = a.drafts[(size_t)i * kk + t];
        if (x < a.n_vocab)
          good = (double)urow[t] * (double)qrow[t * a.stride + x] < (double)prow[t * a.stride + x];
      }
      const uint32_t bad = __ballot_sync(0xffffffffu, !good);
      if (bad) {
        taken = t0 + (uint32_t)__ffs((int)bad) - 1u;
        break;
      }
    }
    if (lane == 0) s_taken = taken;
  }
  __syncthreads();
  const uint32_t taken = s_taken;
  const float* pr = prow + taken * a.stride;
  const float* qr = qrow + taken * a.stride;
  // slices in steps of 128 elements (four per lane)
  const uint32_t steps = (a.n_vocab + 127u) / 128u, per = (steps + NC * kVdWarps - 1u) / (NC * kVdWarps);
  const uint32_t s_lo = (cta * kVdWarps + warp) * per;
  const uint32_t lo = s_lo < steps ? s_lo * 128u : a.n_vocab;
  const uint32_t hi = lo + per * 128u < a.n_vocab ? lo + per * 128u : a.n_vocab;
  bool residual = taken < k;
  vd_cluster_wait();  // every CTA of the cluster runs
  for (;;) {  // (a second time where p_a <= q_a everywhere: draw from p_a)
    double sum = 0.0;
    uint32_t last = 0;  // 1 + the last index with weight
#pragma unroll 4
    for (uint32_t v0 = lo; v0 < hi; v0 += 128u) {
      const uint32_t v = v0 + lane * 4u;
      double w[4];
      vd_weights4<VEC>(pr, qr, v, hi, residual, w);
#pragma unroll
      for (uint32_t e = 0; e < 4u; ++e) {
        sum += w[e];
        if (w[e] > 0.0) last = v + e + 1u;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    last = __reduce_max_sync(0xffffffffu, last);
    if (lane == 0) {
      s_sum[warp] = sum;
      s_last[warp] = last;
    }
    __syncthreads();
    if (tid < NC) {  // this CTA's sum into every CTA
      double t = 0.0;
      uint32_t e = 0;
#pragma unroll
      for (uint32_t w = 0; w < kVdWarps; ++w) {
        t += s_sum[w];
        e = s_last[w] > e ? s_last[w] : e;
      }
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(vd_map(&c_sum[cta], tid)), "d"(t) : "memory");
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(vd_map(&c_last[cta], tid)), "r"(e) : "memory");
    }
    vd_cluster_sync();
    double sums[NC], total = 0.0;
    uint32_t ends[NC], end = 0;
#pragma unroll
    for (uint32_t c = 0; c < NC; ++c) {
      sums[c] = c_sum[c];
      ends[c] = c_last[c];
      total += sums[c];
      end = ends[c] > end ? ends[c] : end;
    }
    if (end == 0 && residual) {
      residual = false;
      vd_cluster_sync();  // every CTA has read the sums
      continue;
    }
    const double cut = u * total;
    // The slice that crosses the cut or, past every rounding, holds the last weight.  Sums in another order may fall on
    // the other side of the cut, so who draws is decided once: every CTA finds the first CTA by the same additions, and
    // that one's warps find the first warp, or the last with weight; its last weight in turn where none crosses there.
    double base = 0.0, run = 0.0;
    uint32_t chosen = NC;
#pragma unroll
    for (uint32_t c = 0; c < NC; ++c) {
      if (chosen == NC && ends[c] != 0 && (run + sums[c] > cut || ends[c] == end)) {
        chosen = c;
        base = run;
      }
      run += sums[c];
    }
    uint32_t pick = kVdWarps;
    if (chosen == cta)
      for (uint32_t w = 0; w < kVdWarps; ++w) {
        if (s_last[w] != 0 && (base + s_sum[w] > cut || s_last[w] == c_last[cta])) {
          pick = w;
          break;
        }
        base += s_sum[w];
      }
    if (warp == pick) {
      uint32_t tok = s_last[pick] - 1u;
      double at = base;
      for (uint32_t v0 = lo; v0 < hi; v0 += 128u) {
        const uint32_t v = v0 + lane * 4u;
        double w[4];
        vd_weights4<VEC>(pr, qr, v, hi, residual, w);
        const double mine = (w[0] + w[1]) + (w[2] + w[3]);
        double c = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double t = __shfl_up_sync(0xffffffffu, c, o);
          if ((int)lane >= o) c += t;
        }
        double s = at + (c - mine);
        uint32_t hit = 4u;
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e) {
          s += w[e];
          if (hit == 4u && w[e] > 0.0 && s > cut) hit = e;
        }
        const uint32_t any = __ballot_sync(0xffffffffu, hit < 4u);
        if (any) {
          const uint32_t src = (uint32_t)__ffs((int)any) - 1u;
          tok = v0 + src * 4u + __shfl_sync(0xffffffffu, hit, (int)src);
          break;
        }
        at += __shfl_sync(0xffffffffu, c, 31);
      }
      if (lane == 0) a.tokens[(size_t)i * (kk + 1u) + taken] = tok;
    }
    if (cta == 0 && tid == 0) {
      if (end == 0) a.tokens[(size_t)i * (kk + 1u) + taken] = 0xffffffffu;  // no weight at all
      a.n_token[i] = taken + (end != 0 ? 1u : 0u);
    }
    break;
  }
  if (cta == 0)
    for (uint32_t t = tid; t <= kk; t += kVdThreads)
      if (t != taken) a.tokens[(size_t)i * (kk + 1u) + t] = t < taken ? a.drafts[(size_t)i * kk + t] : 0xffffffffu;
  vd_cluster_sync();  // no CTA leaves while another may still write into it
}

cudaError_t launch_verify_draft(const float* p, const float* q, uint64_t stride, const uint32_t* drafts,
                                const uint32_t* n_draft, uint32_t max_draft, const float* u, uint32_t n_seq,
                                uint32_t n_vocab, uint32_t* tokens, uint32_t* n_token, cudaStream_t st) {
  if (n_seq == 0) return cudaSuccess;
  const VerifyParams a{p, q, stride, drafts, n_draft, u, max_draft, n_vocab, tokens, n_token};
  // as many CTAs per sequence (1, 2, 4 or 8) as keep two per SM, each warp with a step to do
  uint32_t n_cta = 1;
  while (n_cta < kVdMaxCluster && 2ull * n_cta * n_seq <= 2u * kSms && 2u * n_cta * kVdWarps * 128u <= n_vocab) n_cta *= 2u;
  const bool vec = ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q)) & 15u) == 0 && stride % 4u == 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(n_seq * n_cta);
  cfg.blockDim = dim3(kVdThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = n_cta;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  void (*const fn[2][4])(const VerifyParams) = {
      {verify_draft_kernel<false, 1>, verify_draft_kernel<false, 2>, verify_draft_kernel<false, 4>, verify_draft_kernel<false, 8>},
      {verify_draft_kernel<true, 1>, verify_draft_kernel<true, 2>, verify_draft_kernel<true, 4>, verify_draft_kernel<true, 8>}};
  return cudaLaunchKernelEx(&cfg, fn[vec][n_cta == 8u ? 3 : n_cta / 2u], a);
}

}  // namespace eos
