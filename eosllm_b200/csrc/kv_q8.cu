// kv_q8.cu -- the 8-bit paged key/value cache: rows quantised as they are
// written, and read back (layout and quantizer: kv_q8.cuh).
#include "eos_kernels.h"
#include "kv_q8.cuh"

namespace eos {

struct KvCopyParams {
  KvRows rows;
  float* k;  // row r, head h at k + r * row_stride + h * HD
  float* v;
  uint64_t row_stride;
  uint8_t* pages;
  const uint32_t* table;  // page of tokens [128 j, 128 j + 128) of sequence i: table[i * table_stride + j]
  const uint32_t* pos;    // position of sequence i's first row
  uint32_t table_stride, n_pages, n_kv_head;
  uint32_t* err;
};

// Block of (row r, head h) and the row's slot in the page; nullptr when the
// row belongs to no sequence or its position or page is out of range (the
// latter two are reported).
__device__ __forceinline__ uint8_t* kv_locate(const KvCopyParams& p, uint32_t r, uint32_t h, uint32_t hd,
                                              uint32_t& slot) {
  const uint32_t i = kv_row_seq(p.rows, r);
  if (i >= p.rows.n_seq) return nullptr;
  const uint64_t at = (uint64_t)p.pos[i] + (r - kv_row_start(p.rows, i));
  if (at >= (uint64_t)p.table_stride * kKvPage) {
    report(p.err, EOS_DEVERR_RANGE);
    return nullptr;
  }
  const uint32_t page = p.table[(size_t)i * p.table_stride + (uint32_t)(at / kKvPage)];
  if (page >= p.n_pages) {
    report(p.err, EOS_DEVERR_RANGE);
    return nullptr;
  }
  slot = (uint32_t)(at % kKvPage);
  return p.pages + ((size_t)page * p.n_kv_head + h) * kv_block_bytes(hd);
}

// One warp per (row, head): lane l holds elements l E .. l E + E - 1.
template <uint32_t HD>
__global__ void __launch_bounds__(256) kv_write_rows_kernel(const KvCopyParams p) {
  constexpr uint32_t E = HD / 32u;
  const uint64_t w = (uint64_t)blockIdx.x * 8u + (threadIdx.x >> 5);
  const uint32_t lane = threadIdx.x & 31u;
  if (w >= (uint64_t)p.rows.n_rows * p.n_kv_head) return;  // warp-uniform
  const uint32_t r = (uint32_t)(w / p.n_kv_head), h = (uint32_t)(w % p.n_kv_head);
  uint32_t slot;
  uint8_t* blk = kv_locate(p, r, h, HD, slot);
  if (blk == nullptr) return;
#pragma unroll
  for (uint32_t which = 0; which < 2; ++which) {
    const float* src = (which ? p.v : p.k) + r * p.row_stride + h * HD + lane * E;
    float x[E];
    uint32_t amax = 0;
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) {
      x[e] = src[e];
      const uint32_t b = __float_as_uint(x[e]) & 0x7fffffffu;
      amax = b > amax ? b : amax;
    }
    const KvRowScale s = kv_row_scale(__reduce_max_sync(0xffffffffu, amax));
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) {
      const uint32_t d = lane * E + e;
      blk[which ? kv_v_offset<HD>(slot, d) : kv_k_offset<HD>(slot, d)] = (uint8_t)kv_quant(x[e], s);
    }
    if (lane == 0) *reinterpret_cast<float*>(blk + kv_scale_offset<HD>(slot, which)) = s.scale;
  }
}

template <uint32_t HD>
__global__ void __launch_bounds__(256) kv_read_rows_kernel(const KvCopyParams p) {
  constexpr uint32_t E = HD / 32u;
  const uint64_t w = (uint64_t)blockIdx.x * 8u + (threadIdx.x >> 5);
  const uint32_t lane = threadIdx.x & 31u;
  if (w >= (uint64_t)p.rows.n_rows * p.n_kv_head) return;  // warp-uniform
  const uint32_t r = (uint32_t)(w / p.n_kv_head), h = (uint32_t)(w % p.n_kv_head);
  uint32_t slot;
  const uint8_t* blk = kv_locate(p, r, h, HD, slot);
  if (blk == nullptr) return;
#pragma unroll
  for (uint32_t which = 0; which < 2; ++which) {
    float* dst = (which ? p.v : p.k) + r * p.row_stride + h * HD + lane * E;
    const float s = *reinterpret_cast<const float*>(blk + kv_scale_offset<HD>(slot, which));
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) {
      const uint32_t d = lane * E + e;
      const int8_t q = (int8_t)blk[which ? kv_v_offset<HD>(slot, d) : kv_k_offset<HD>(slot, d)];
      dst[e] = __fmul_rn((float)q, s);
    }
  }
}

namespace {
KvCopyParams copy_params(const KvPool& kv, const KvRowSet& rs, const float* k, const float* v, uint64_t row_stride,
                         uint32_t* err) {
  KvCopyParams p{};
  p.rows = KvRows{rs.row0, rs.n_seq, rs.n_rows, rs.row0 ? 0u : rs.n_rows / rs.n_seq};
  p.k = const_cast<float*>(k);
  p.v = const_cast<float*>(v);
  p.row_stride = row_stride;
  p.pages = kv.pages;
  p.table = rs.table;
  p.pos = rs.pos;
  p.table_stride = rs.table_stride;
  p.n_pages = kv.n_pages;
  p.n_kv_head = kv.n_kv_head;
  p.err = err;
  return p;
}
}  // namespace

cudaError_t launch_kv_write(const KvPool& kv, const KvRowSet& rs, const float* k, const float* v, uint64_t row_stride,
                            uint32_t* err, cudaStream_t st) {
  if (rs.n_rows == 0 || rs.n_seq == 0) return cudaSuccess;
  const KvCopyParams p = copy_params(kv, rs, k, v, row_stride, err);
  const uint32_t grid = (uint32_t)(((uint64_t)rs.n_rows * kv.n_kv_head + 7u) / 8u);
  if (kv.head_dim == 64) kv_write_rows_kernel<64><<<grid, 256, 0, st>>>(p);
  else if (kv.head_dim == 128) kv_write_rows_kernel<128><<<grid, 256, 0, st>>>(p);
  else kv_write_rows_kernel<256><<<grid, 256, 0, st>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_kv_read(const KvPool& kv, const KvRowSet& rs, float* k, float* v, uint64_t row_stride,
                           uint32_t* err, cudaStream_t st) {
  if (rs.n_rows == 0 || rs.n_seq == 0) return cudaSuccess;
  const KvCopyParams p = copy_params(kv, rs, k, v, row_stride, err);
  const uint32_t grid = (uint32_t)(((uint64_t)rs.n_rows * kv.n_kv_head + 7u) / 8u);
  if (kv.head_dim == 64) kv_read_rows_kernel<64><<<grid, 256, 0, st>>>(p);
  else if (kv.head_dim == 128) kv_read_rows_kernel<128><<<grid, 256, 0, st>>>(p);
  else kv_read_rows_kernel<256><<<grid, 256, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace eos
