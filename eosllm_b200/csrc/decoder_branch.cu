// decoder_branch.cu -- kernels of the decoder's 8-bit cache mode and of its
// branches (several sequences that continue the same tokens): RoPE on rows whose
// positions are in device memory, and probabilities from logits.
#include "decoder_internal.h"

namespace eos {

struct RopeRowsParams {
  float* qkv;           // [m][(heads + kvl) HD]: q heads, k heads, v heads
  const uint32_t* pos;  // position of sequence i's first row
  uint32_t per_seq;     // rows of a sequence
  uint32_t heads, width;  // q and k heads; floats of a row
  uint32_t* len_out;    // nullptr, or receives pos[0] + 1
  float base;
};

// One CTA per row: thread t rotates pairs t, t + 256, ... of the q and k heads,
// in place.
template <int HD>
__global__ void __launch_bounds__(256) rope_rows_kernel(const RopeRowsParams p) {
  const uint32_t row = blockIdx.x, seq = row / p.per_seq;
  const uint32_t pos = p.pos[seq] + (row - seq * p.per_seq);
  float* r = p.qkv + (size_t)row * p.width;
  for (uint32_t t = threadIdx.x; t < p.heads * (HD / 2u); t += 256u) {
    const uint32_t head = t / (HD / 2u), i = 2u * (t % (HD / 2u));
    float x0 = r[head * HD + i], x1 = r[head * HD + i + 1u];
    rope_pair<HD>(x0, x1, i, pos, p.base);
    r[head * HD + i] = x0;
    r[head * HD + i + 1u] = x1;
  }
  if (p.len_out != nullptr && row == 0 && threadIdx.x == 0) *p.len_out = pos + 1u;
}

cudaError_t launch_rope_rows(float* qkv, uint32_t m, uint32_t per_seq, uint32_t hl, uint32_t kvl, uint32_t hd,
                             const uint32_t* pos, float base, uint32_t* len_out, cudaStream_t st) {
  if (m == 0) return cudaSuccess;
  const RopeRowsParams p{qkv, pos, per_seq, hl + kvl, (hl + 2u * kvl) * hd, len_out, base};
  if (hd == 64) rope_rows_kernel<64><<<m, 256, 0, st>>>(p);
  else if (hd == 128) rope_rows_kernel<128><<<m, 256, 0, st>>>(p);
  else if (hd == 256) rope_rows_kernel<256><<<m, 256, 0, st>>>(p);
  else return cudaErrorInvalidValue;
  return cudaGetLastError();
}

// One CTA per row: p = softmax(logits / temperature), in place; temperature 0:
// 1 at the row's largest logit (the lowest of equals), 0 elsewhere.  The row
// (a few hundred KB) stays in L2 between its passes.
__global__ void __launch_bounds__(1024) logit_probs_kernel(float* x, uint32_t n, float inv_t) {
  __shared__ float red[32];
  __shared__ uint32_t redi[32];
  float* r = x + (size_t)blockIdx.x * n;
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  float best = -INFINITY;
  uint32_t at = 0xffffffffu;
  for (uint32_t i = tid; i < n; i += 1024u)
    if (r[i] > best) {
      best = r[i];
      at = i;
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float b = __shfl_xor_sync(0xffffffffu, best, o);
    const uint32_t a = __shfl_xor_sync(0xffffffffu, at, o);
    if (b > best || (b == best && a < at)) {
      best = b;
      at = a;
    }
  }
  if (lane == 0) {
    red[warp] = best;
    redi[warp] = at;
  }
  __syncthreads();
  for (int w = 0; w < 32; ++w)
    if (red[w] > best || (red[w] == best && redi[w] < at)) {
      best = red[w];
      at = redi[w];
    }
  if (inv_t == 0.0f) {
    for (uint32_t i = tid; i < n; i += 1024u) r[i] = i == at ? 1.0f : 0.0f;
    return;
  }
  __syncthreads();
  float sum = 0.0f;
  for (uint32_t i = tid; i < n; i += 1024u) sum += expf((r[i] - best) * inv_t);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) red[warp] = sum;
  __syncthreads();
  float tot = 0.0f;
  for (int w = 0; w < 32; ++w) tot += red[w];
  const float inv = 1.0f / tot;
  for (uint32_t i = tid; i < n; i += 1024u) r[i] = expf((r[i] - best) * inv_t) * inv;
}

cudaError_t launch_logit_probs(float* logits, uint32_t rows, uint32_t n, float temperature, cudaStream_t st) {
  if (rows == 0) return cudaSuccess;
  // (the reciprocal of a temperature below 2^-128 is no f32; at the largest one different logits are as far apart)
  const float inv_t = temperature > 0.0f ? fminf(1.0f / temperature, 3.402823466e38f) : 0.0f;
  logit_probs_kernel<<<rows, 1024, 0, st>>>(logits, n, inv_t);
  return cudaGetLastError();
}

// Draft probabilities of drafts that were not drawn: 1 at the token.
__global__ void one_hot_kernel(float* q, const uint32_t* tokens, uint32_t n) {
  const uint32_t r = blockIdx.y, i = blockIdx.x * 256u + threadIdx.x;
  if (i < n) q[(size_t)r * n + i] = i == tokens[r] ? 1.0f : 0.0f;
}

cudaError_t launch_one_hot(float* q, const uint32_t* tokens, uint32_t rows, uint32_t n, cudaStream_t st) {
  if (rows == 0) return cudaSuccess;
  one_hot_kernel<<<dim3((n + 255u) / 256u, rows), 256, 0, st>>>(q, tokens, n);
  return cudaGetLastError();
}

}  // namespace eos
