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
// of the weights in f64 (weights that are not positive and finite count 0).
// Tokens so drawn are distributed as the target's own.
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

constexpr uint32_t kVdThreads = 1024, kVdWarps = kVdThreads / 32;

// One CTA per sequence; warp w owns the w-th contiguous slice of the row.
__global__ void __launch_bounds__(kVdThreads) verify_draft_kernel(const VerifyParams a) {
  __shared__ uint32_t s_taken;
  __shared__ double s_sum[kVdWarps];
  __shared__ uint32_t s_last[kVdWarps];
  const uint32_t i = blockIdx.x, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const uint32_t kk = a.max_draft;
  uint32_t k = a.n_draft != nullptr ? a.n_draft[i] : kk;
  if (k > kk) k = kk;
  const float* prow = a.p + (size_t)i * (kk + 1u) * a.stride;
  const float* qrow = a.q + (size_t)i * kk * a.stride;
  if (tid == 0) {
    uint32_t t = 0;
    for (; t < k; ++t) {
      const uint32_t x = a.drafts[(size_t)i * kk + t];
      if (x >= a.n_vocab) break;
      const double lhs = (double)a.u[(size_t)i * (kk + 1u) + t] * (double)qrow[t * a.stride + x];
      if (!(lhs < (double)prow[t * a.stride + x])) break;
    }
    s_taken = t;
  }
  __syncthreads();
  const uint32_t taken = s_taken;
  const float* pr = prow + taken * a.stride;
  const float* qr = qrow + taken * a.stride;
  const double u = (double)a.u[(size_t)i * (kk + 1u) + kk];
  const uint32_t per = ((a.n_vocab + kVdThreads - 1u) / kVdThreads) * 32u;  // a warp's slice
  const uint32_t lo = warp * per < a.n_vocab ? warp * per : a.n_vocab;
  const uint32_t hi = lo + per < a.n_vocab ? lo + per : a.n_vocab;
  bool residual = taken < k;
  for (;;) {
    double sum = 0.0;
    uint32_t last = 0;  // 1 + the last index with weight
    for (uint32_t v = lo + lane; v < hi; v += 32u) {
      const double w = vd_weight(pr[v], residual ? qr[v] : 0.0f, residual);
      sum += w;
      if (w > 0.0) last = v + 1u;
    }
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    last = __reduce_max_sync(0xffffffffu, last);
    if (lane == 0) {
      s_sum[warp] = sum;
      s_last[warp] = last;
    }
    __syncthreads();
    double total = 0.0;
    uint32_t end = 0;
    for (uint32_t w = 0; w < kVdWarps; ++w) {
      total += s_sum[w];
      end = s_last[w] > end ? s_last[w] : end;
    }
    if (end == 0 && residual) {  // p_a <= q_a everywhere: draw from p_a
      residual = false;
      __syncthreads();
      continue;
    }
    const double cut = u * total;
    // the warp whose slice crosses the cut, or, past every rounding, the last one with weight
    double before = 0.0;
    uint32_t pick = kVdWarps;
    double base = 0.0;
    for (uint32_t w = 0; w < kVdWarps; ++w) {
      if (s_last[w] != 0 && (before + s_sum[w] > cut || s_last[w] == end)) {
        pick = w;
        base = before;
        break;
      }
      before += s_sum[w];
    }
    if (tid == 0) {
      if (pick == kVdWarps) a.tokens[(size_t)i * (kk + 1u) + taken] = 0xffffffffu;  // no weight at all
      a.n_token[i] = taken + (pick < kVdWarps ? 1u : 0u);
    }
    if (warp == pick) {
      double run = base;
      uint32_t tok = s_last[pick] - 1u;
      for (uint32_t v0 = lo; v0 < hi; v0 += 32u) {
        const uint32_t v = v0 + lane;
        double w = v < hi ? vd_weight(pr[v], residual ? qr[v] : 0.0f, residual) : 0.0;
        double c = w;
        for (int o = 1; o < 32; o <<= 1) {
          const double t = __shfl_up_sync(0xffffffffu, c, o);
          if ((int)lane >= o) c += t;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, w > 0.0 && run + c > cut);
        if (hit) {
          tok = v0 + (uint32_t)__ffs((int)hit) - 1u;
          break;
        }
        run += __shfl_sync(0xffffffffu, c, 31);
      }
      if (lane == 0) a.tokens[(size_t)i * (kk + 1u) + taken] = tok;
    }
    break;
  }
  for (uint32_t t = tid; t <= kk; t += kVdThreads)
    if (t != taken) a.tokens[(size_t)i * (kk + 1u) + t] = t < taken ? a.drafts[(size_t)i * kk + t] : 0xffffffffu;
  
}

cudaError_t launch_verify_draft(const float* p, const float* q, uint64_t stride, const uint32_t* drafts,
                                const uint32_t* n_draft, uint32_t max_draft, const float* u, uint32_t n_seq,
                                uint32_t n_vocab, uint32_t* tokens, uint32_t* n_token, cudaStream_t st) {
  if (n_seq == 0) return cudaSuccess;
  const VerifyParams a{p, q, stride, drafts, n_draft, u, max_draft, n_vocab, tokens, n_token};
  verify_draft_kernel<<<n_seq, kVdThreads, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace eos
