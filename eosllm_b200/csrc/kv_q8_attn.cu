// kv_q8_attn.cu -- attention of a batch of sequences that share a prefix,
// over the 8-bit paged cache (layout: kv_q8.cuh).
//
// Row t of the n_i rows of sequence i, head h, kv head g = h n_kv / n_head:
//   S_j = scale <q, k_j> over the prefix's tokens and the sequence's own
//   tokens 0 .. len_i - n_i + t;  out = sum_j softmax(S)_j v_j;  no token
//   visible: out = 0.
#include "eos_kernels.h"
#include "kv_q8.cuh"

namespace eos {

struct KvAttnParams {
  KvRows rows;
  const uint8_t* pages;
  const uint32_t* prefix_table;
  const uint32_t* prefix_len;
  const uint32_t* table;
  const uint32_t* seq_len;
  uint32_t max_prefix, table_stride, max_len;
  uint32_t n_pages, n_head, n_kv_head;
  const float* q;
  float* out;
  uint64_t q_stride, out_stride;
  float scale_log2;  // scale * log2(e)
  uint32_t* err;
};

// One CTA of 128 threads per (row, head): a page at a time, thread = token
// for the scores, thread = dimension (HD / 128 each) for the values.
template <uint32_t HD>
__global__ void __launch_bounds__(128) kv_attn_simple_kernel(const KvAttnParams p) {
  __shared__ float qs[HD], ps[kKvPage], red[4];
  const uint32_t r = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  const uint32_t i = kv_row_seq(p.rows, r);
  if (i >= p.rows.n_seq) return;
  const uint32_t r0 = kv_row_start(p.rows, i), r1 = kv_row_start(p.rows, i + 1u);
  const uint32_t g = (uint32_t)(((uint64_t)h * p.n_kv_head) / p.n_head);
  for (uint32_t d = tid; d < HD; d += 128u) qs[d] = p.q[r * p.q_stride + h * HD + d];
  constexpr uint32_t ND = (HD + 127u) / 128u;
  float o[ND] = {}, m = -INFINITY, l = 0.0f;
  for (uint32_t part = 0; part < 2; ++part) {
    uint32_t len = 0;
    if (part == 0) {
      len = p.prefix_len != nullptr ? *p.prefix_len : 0u;
      if (len > p.max_prefix) {
        report(p.err, EOS_DEVERR_RANGE);
        len = p.max_prefix;
      }
    } else {
      uint32_t all = p.seq_len[i];
      if (all > p.max_len) {
        report(p.err, EOS_DEVERR_RANGE);
        all = p.max_len;
      }
      const int64_t seen = (int64_t)all - (int64_t)(r1 - r0) + 1 + (int64_t)(r - r0);
      len = seen > 0 ? (uint32_t)seen : 0u;
    }
    const uint32_t* table = part == 0 ? p.prefix_table : p.table + (size_t)i * p.table_stride;
    for (uint32_t t0 = 0; t0 < len; t0 += kKvPage) {
      const uint32_t page = table[t0 / kKvPage];
      if (page >= p.n_pages) {
        report(p.err, EOS_DEVERR_RANGE);
        continue;
      }
      const uint8_t* blk = p.pages + ((size_t)page * p.n_kv_head + g) * kv_block_bytes(HD);
      __syncthreads();
      const bool on = t0 + tid < len;
      float s = -INFINITY, vs = 0.0f;
      if (on) {
        float acc = 0.0f;
        for (uint32_t d = 0; d < HD; ++d) acc = fmaf((float)(int8_t)blk[kv_k_offset<HD>(tid, d)], qs[d], acc);
        s = acc * *reinterpret_cast<const float*>(blk + kv_scale_offset<HD>(tid, 0)) * p.scale_log2;
        vs = *reinterpret_cast<const float*>(blk + kv_scale_offset<HD>(tid, 1));
      }
      float cm = s;
      for (int sh = 16; sh > 0; sh >>= 1) cm = fmaxf(cm, __shfl_xor_sync(0xffffffffu, cm, sh));
      if ((tid & 31u) == 0) red[tid >> 5] = cm;
      __syncthreads();
      const float nm = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
      const float mu = nm == -INFINITY ? 0.0f : nm;
      const float f = exp2f(m - mu), e = on ? exp2f(s - mu) : 0.0f;
      float ls = e;
      for (int sh = 16; sh > 0; sh >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, sh);
      ps[tid] = on ? e * vs : 0.0f;
      __syncthreads();
      if ((tid & 31u) == 0) red[tid >> 5] = ls;
      __syncthreads();
      l = fmaf(l, f, red[0] + red[1] + red[2] + red[3]);
      m = nm;
#pragma unroll
      for (uint32_t x = 0; x < ND; ++x) {
        const uint32_t d = x * 128u + tid;
        o[x] *= f;
        if (d < HD)
          for (uint32_t t = 0; t < kKvPage; ++t)
            if (t0 + t < len) o[x] = fmaf(ps[t], (float)(int8_t)blk[kv_v_offset<HD>(t, d)], o[x]);
      }
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (uint32_t x = 0; x < ND; ++x) {
    const uint32_t d = x * 128u + tid;
    if (d < HD) p.out[r * p.out_stride + h * HD + d] = o[x] * inv;
  }
}

size_t kv_attn_scratch_bytes(const KvPool&, const KvAttnBatch&, uint32_t) { return 16; }

cudaError_t launch_kv_attn(const KvPool& kv, const KvAttnBatch& b, const float* q, uint64_t q_stride, float* out,
                           uint64_t out_stride, uint32_t n_head, float scale, void*, uint32_t* err,
                           cudaStream_t st) {
  if (b.n_rows == 0 || b.n_seq == 0) return cudaSuccess;
  KvAttnParams p{};
  p.rows = KvRows{b.row0, b.n_seq, b.n_rows, b.row0 ? 0u : b.n_rows / b.n_seq};
  p.pages = kv.pages;
  p.prefix_table = b.prefix_table;
  p.prefix_len = b.prefix_len;
  p.table = b.table;
  p.seq_len = b.seq_len;
  p.max_prefix = b.max_prefix;
  p.table_stride = b.table_stride;
  p.max_len = b.max_len;
  p.n_pages = kv.n_pages;
  p.n_head = n_head;
  p.n_kv_head = kv.n_kv_head;
  p.q = q;
  p.out = out;
  p.q_stride = q_stride;
  p.out_stride = out_stride;
  p.scale_log2 = (float)((double)scale * 1.4426950408889634);
  p.err = err;
  const dim3 grid(b.n_rows, n_head);
  if (kv.head_dim == 64) kv_attn_simple_kernel<64><<<grid, 128, 0, st>>>(p);
  else if (kv.head_dim == 128) kv_attn_simple_kernel<128><<<grid, 128, 0, st>>>(p);
  else kv_attn_simple_kernel<256><<<grid, 128, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace eos
