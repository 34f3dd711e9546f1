// kv_q8.cu -- the 8-bit paged key/value cache: rows quantised as they are
// written, and read back (layout and quantizer: kv_q8.cuh).  Both directions
// share their kernels: one for a few rows per sequence, one for many.
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
  uint32_t r0, r1, pos;
  const uint32_t i = kv_find(p.rows, p.pos, [&](uint32_t, uint32_t start) { return start <= r; }, r0, r1, pos);
  if (i >= p.rows.n_seq || r < r0 || r >= r1) return nullptr;
  const uint64_t at = (uint64_t)pos + (r - r0);
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

// Byte e of four words as one word.
__device__ __forceinline__ uint32_t kv_pick_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t e) {
  const uint32_t sel = e | ((e + 4u) << 4);
  return __byte_perm(__byte_perm(a, b, sel), __byte_perm(c, d, sel), 0x5410);
}
__device__ __forceinline__ float4 kv_value4(uint32_t w, float s) {
  return make_float4(__fmul_rn((float)(int8_t)w, s), __fmul_rn((float)(int8_t)(w >> 8), s),
                     __fmul_rn((float)(int8_t)(w >> 16), s), __fmul_rn((float)(int8_t)(w >> 24), s));
}

// ---- a few rows per sequence (a decode step) -----------------------------------
// One warp per (row, head); lane l holds elements 4 l + 128 c .. + 3.  A row's
// value bytes lie HD / 4 sectors apart, so this moves a sector per byte: right
// for a token or a few, where a launch is what counts.
template <uint32_t HD, bool READ>
__global__ void __launch_bounds__(128) kv_rows_kernel(const KvCopyParams p) {
  constexpr uint32_t C = HD <= 128u ? 1u : HD / 128u;
  const uint64_t w = (uint64_t)blockIdx.x * 4u + (threadIdx.x >> 5);
  const uint32_t lane = threadIdx.x & 31u;
  if (w >= (uint64_t)p.rows.n_rows * p.n_kv_head) return;  // warp-uniform
  const uint32_t r = (uint32_t)(w / p.n_kv_head), h = (uint32_t)(w % p.n_kv_head);
  const bool on = HD >= 128u || lane < HD / 4u;
  const size_t at = r * p.row_stride + h * HD + lane * 4u;
  float4 x[2][C];
  if (!READ) {  // the loads fly while the slot is looked up
#pragma unroll
    for (uint32_t which = 0; which < 2; ++which)
#pragma unroll
      for (uint32_t c = 0; c < C; ++c)
        x[which][c] = on ? *reinterpret_cast<const float4*>((which ? p.v : p.k) + at + c * 128u)
                         : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  uint32_t slot;
  uint8_t* blk = kv_locate(p, r, h, HD, slot);
  if (blk == nullptr) return;
#pragma unroll
  for (uint32_t which = 0; which < 2; ++which) {
    float* sc = reinterpret_cast<float*>(blk + kv_scale_offset<HD>(slot, which));
    if (READ) {
      const float s = *sc;
#pragma unroll
      for (uint32_t c = 0; c < C; ++c) {
        const uint32_t d = lane * 4u + c * 128u;
        uint32_t q = 0;
        if (on && which == 0) q = *reinterpret_cast<const uint32_t*>(blk + kv_k_offset<HD>(slot, d));
        if (on && which == 1)
#pragma unroll
          for (uint32_t e = 0; e < 4u; ++e) q |= (uint32_t)blk[kv_v_offset<HD>(slot, d + e)] << (8u * e);
        if (on) *reinterpret_cast<float4*>((which ? p.v : p.k) + at + c * 128u) = kv_value4(q, s);
      }
    } else {
      float amax = 0.0f;
#pragma unroll
      for (uint32_t c = 0; c < C; ++c) amax = kv_absmax4(amax, x[which][c]);
      const KvRowScale s = kv_row_scale(amax);
#pragma unroll
      for (uint32_t c = 0; c < C; ++c) {
        const uint32_t d = lane * 4u + c * 128u, q = kv_quant4(x[which][c], s);
        if (on && which == 0) *reinterpret_cast<uint32_t*>(blk + kv_k_offset<HD>(slot, d)) = q;
        if (on && which == 1)
#pragma unroll
          for (uint32_t e = 0; e < 4u; ++e) blk[kv_v_offset<HD>(slot, d + e)] = (uint8_t)(q >> (8u * e));
      }
      if (lane == 0) *sc = s.scale;
    }
  }
}

// ---- many rows: a quarter of a page per CTA --------------------------------------
// One CTA of 256 threads per (32-token quarter, head).  Warp g has tokens g, g +
// 8, g + 16, g + 24 -- the four that are neighbours in a value row -- and a
// lane four neighbouring elements of each, so both layouts are whole words:
// a key row's word is a token's four elements, a value row's word an element's
// four tokens (a 4 x 4 byte transpose in registers).  The words of the 32
// tokens meet in shared memory (rows of nine words: the lanes' accesses then
// collide four ways at most) and value rows move as 16 bytes a thread.  Every
// byte moves once; reading and writing f32 rows is what bounds it.  The heads of
// the same rows are neighbours in the grid, so that what runs together is
// together in memory (reading 16383 rows x 32 heads: 117 us head by head, 107 to
// 110 so, 6.2 TB/s).  A write's registers are held to 64 a thread, four CTAs an SM:
// at three, 8505 rows x 8 heads took 21.4 us, at four 19.9, keys and values in CTAs
// of their own 24.3 (the same rows each time; other rows each time 20.9, 4.2 TB/s:
// a CTA's loads, rounding and stores follow one another, and nothing of the next
// quarter is under way meanwhile).
//
// Quarters of a ragged batch: sequence i's blocks start at row0[i] / 32 + 2 i,
// which leaves room for the two broken ends; a CTA searches its sequence, and the
// rows are on their way before its page is known.
template <uint32_t HD, bool READ>
__global__ void __launch_bounds__(256, READ ? (HD > 128u ? 6 : 8) : (HD > 128u ? 2 : 4)) kv_quarter_kernel(const KvCopyParams p) {
  constexpr uint32_t C = HD <= 128u ? 1u : HD / 128u;
  constexpr uint32_t PITCH = 9u;  // words per value row in shared memory
  __shared__ uint32_t vt[HD * PITCH];
  const uint32_t tid = threadIdx.x, lane = tid & 31u, g = tid >> 5;
  const uint32_t block = blockIdx.x / p.n_kv_head, h = blockIdx.x - block * p.n_kv_head;
  uint32_t r0, r1, first;
  const uint32_t i = kv_find(p.rows, p.pos, [&](uint32_t x, uint32_t start) { return start / 32u + 2u * x <= block; },
                             r0, r1, first);
  if (i >= p.rows.n_seq) return;  // (rows before the first sequence)
  const uint32_t n = r1 > r0 ? r1 - r0 : 0u;
  const uint64_t pos = first;
  const uint32_t b0 = r0 / 32u + 2u * i;
  const uint64_t t0 = (pos & ~(uint64_t)31u) + 32ull * (block - b0);  // the quarter's first position
  if (n == 0 || t0 >= pos + n) return;
  uint32_t page = 0xffffffffu;
  if (t0 < (uint64_t)p.table_stride * kKvPage) page = p.table[(size_t)i * p.table_stride + (uint32_t)(t0 / kKvPage)];
  const bool on = HD >= 128u || lane < HD / 4u;
  bool in[4];
  // the warp's first row (may lie before the call's, then it is not touched); the others are 8 rows on each
  const size_t at0 = (size_t)((uint64_t)r0 + t0 + g - pos) * p.row_stride + h * HD + lane * 4u, step = 8u * p.row_stride;
  float4 x[2][4][C];
#pragma unroll
  for (uint32_t j = 0; j < 4u; ++j) {
    const uint64_t t = t0 + g + 8u * j;
    in[j] = t >= pos && t < pos + n;
    if (!READ)  // the rows fly while the page is looked up
#pragma unroll
      for (uint32_t c = 0; c < C; ++c) {
        x[0][j][c] = x[1][j][c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (in[j] && on) {
          x[0][j][c] = __ldcs(reinterpret_cast<const float4*>(p.k + at0 + j * step + c * 128u));
          x[1][j][c] = __ldcs(reinterpret_cast<const float4*>(p.v + at0 + j * step + c * 128u));
        }
      }
  }
  if (page >= p.n_pages) {
    if (tid == 0) report(p.err, EOS_DEVERR_RANGE);
    return;
  }
  uint8_t* blk = p.pages + ((size_t)page * p.n_kv_head + h) * kv_block_bytes(HD);
  const uint32_t s0 = (uint32_t)(t0 % kKvPage);
  const bool whole = t0 >= pos && t0 + 32u <= pos + n;
  uint8_t* vq = blk + kKvPage * HD + (s0 / kKvQuarter) * (HD * kKvQuarter);
  // value rows of the quarter as 16-byte chunks: chunk x is element x / 2, half x % 2
  auto chunk = [&](uint32_t x) { return vq + (x >> 1) * 32u + (((x & 1u) ^ ((x >> 1) >> 2)) & 1u) * 16u; };
  // the bytes of word w of a value row (tokens w, w + 8, w + 16, w + 24) that this call writes
  auto keep = [&](uint32_t w) {
    uint32_t m = 0;
#pragma unroll
    for (uint32_t j = 0; j < 4u; ++j) m |= (t0 + w + 8u * j >= pos && t0 + w + 8u * j < pos + n) ? 0xffu << (8u * j) : 0u;
    return m;
  };
  if (READ) {
    for (uint32_t x = tid; x < 2u * HD; x += 256u) {
      const uint4 v = *reinterpret_cast<const uint4*>(chunk(x));
      uint32_t* dst = vt + (x >> 1) * PITCH + (x & 1u) * 4u;
      dst[0] = v.x;
      dst[1] = v.y;
      dst[2] = v.z;
      dst[3] = v.w;
    }
  }
  uint32_t kw[4][C], vw[4][C];
  float ks[4], vs[4];
  if (!READ) {
#pragma unroll
    for (uint32_t j = 0; j < 4u; ++j) {
      float ka = 0.0f, va = 0.0f;
#pragma unroll
      for (uint32_t c = 0; c < C; ++c) {
        ka = kv_absmax4(ka, x[0][j][c]);
        va = kv_absmax4(va, x[1][j][c]);
      }
      const KvRowScale sk = kv_row_scale(ka);
      const KvRowScale sv = kv_row_scale(va);
      ks[j] = sk.scale;
      vs[j] = sv.scale;
#pragma unroll
      for (uint32_t c = 0; c < C; ++c) {
        kw[j][c] = kv_quant4(x[0][j][c], sk);
        vw[j][c] = kv_quant4(x[1][j][c], sv);
      }
      if (!in[j]) continue;  // warp-uniform
      const uint32_t slot = s0 + g + 8u * j;
#pragma unroll
      for (uint32_t c = 0; c < C; ++c)
        if (on) *reinterpret_cast<uint32_t*>(blk + kv_k_offset<HD>(slot, lane * 4u + c * 128u)) = kw[j][c];
      if (lane < 2u) *reinterpret_cast<float*>(blk + kv_scale_offset<HD>(slot, lane)) = lane ? vs[j] : ks[j];
    }
#pragma unroll
    for (uint32_t c = 0; c < C; ++c)
      if (on)
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e)
          vt[(lane * 4u + c * 128u + e) * PITCH + g] = kv_pick_bytes(vw[0][c], vw[1][c], vw[2][c], vw[3][c], e);
  } else {
#pragma unroll
    for (uint32_t j = 0; j < 4u; ++j) {
      const uint32_t slot = s0 + g + 8u * j;
      ks[j] = vs[j] = 0.0f;
      if (!in[j]) continue;  // warp-uniform
#pragma unroll
      for (uint32_t c = 0; c < C; ++c)
        kw[j][c] = on ? *reinterpret_cast<const uint32_t*>(blk + kv_k_offset<HD>(slot, lane * 4u + c * 128u)) : 0u;
      ks[j] = *reinterpret_cast<const float*>(blk + kv_scale_offset<HD>(slot, 0));
      vs[j] = *reinterpret_cast<const float*>(blk + kv_scale_offset<HD>(slot, 1));
    }
  }
  __syncthreads();
  if constexpr (!READ) {
    for (uint32_t x = tid; x < 2u * HD; x += 256u) {
      const uint32_t* src = vt + (x >> 1) * PITCH + (x & 1u) * 4u;
      uint4 v = make_uint4(src[0], src[1], src[2], src[3]);
      if (!whole) {  // a broken end: the neighbours' bytes stay as they are
        const uint4 old = *reinterpret_cast<const uint4*>(chunk(x));
        v.x = (v.x & keep(4u * (x & 1u))) | (old.x & ~keep(4u * (x & 1u)));
        v.y = (v.y & keep(4u * (x & 1u) + 1u)) | (old.y & ~keep(4u * (x & 1u) + 1u));
        v.z = (v.z & keep(4u * (x & 1u) + 2u)) | (old.z & ~keep(4u * (x & 1u) + 2u));
        v.w = (v.w & keep(4u * (x & 1u) + 3u)) | (old.w & ~keep(4u * (x & 1u) + 3u));
      }
      *reinterpret_cast<uint4*>(chunk(x)) = v;
    }
  } else {
    uint32_t w[C][4];
#pragma unroll
    for (uint32_t c = 0; c < C; ++c)
#pragma unroll
      for (uint32_t e = 0; e < 4u; ++e) w[c][e] = on ? vt[(lane * 4u + c * 128u + e) * PITCH + g] : 0u;
#pragma unroll
    for (uint32_t j = 0; j < 4u; ++j) {
      if (!in[j] || !on) continue;
#pragma unroll
      for (uint32_t c = 0; c < C; ++c) {
        __stcs(reinterpret_cast<float4*>(p.k + at0 + j * step + c * 128u), kv_value4(kw[j][c], ks[j]));
        __stcs(reinterpret_cast<float4*>(p.v + at0 + j * step + c * 128u),
               kv_value4(kv_pick_bytes(w[c][0], w[c][1], w[c][2], w[c][3], j), vs[j]));
      }
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

// Rows or quarters: a quarter's CTA pays off from about eight rows of a sequence
// on (its launch covers up to two broken quarters per sequence).  Writing and
// reading 64 sequences of 8 heads, row by row and by quarters: two rows each 7.0
// and 12.7 us, four 9.4 and 12.4, eight 14.0 and 13.5, sixteen 23.6 and 14.6.
template <bool READ>
cudaError_t copy_launch(const KvPool& kv, const KvCopyParams& p, cudaStream_t st) {
  const KvRows& r = p.rows;
  const uint64_t blocks = (uint64_t)r.n_rows / 32u + 2ull * r.n_seq;
  if (r.n_rows >= 8ull * r.n_seq) {
    const uint32_t grid = (uint32_t)(blocks * kv.n_kv_head);
    if (kv.head_dim == 64) kv_quarter_kernel<64, READ><<<grid, 256, 0, st>>>(p);
    else if (kv.head_dim == 128) kv_quarter_kernel<128, READ><<<grid, 256, 0, st>>>(p);
    else kv_quarter_kernel<256, READ><<<grid, 256, 0, st>>>(p);
  } else {
    const uint32_t grid = (uint32_t)(((uint64_t)r.n_rows * kv.n_kv_head + 3u) / 4u);
    if (kv.head_dim == 64) kv_rows_kernel<64, READ><<<grid, 128, 0, st>>>(p);
    else if (kv.head_dim == 128) kv_rows_kernel<128, READ><<<grid, 128, 0, st>>>(p);
    else kv_rows_kernel<256, READ><<<grid, 128, 0, st>>>(p);
  }
  return cudaGetLastError();
}
}  // namespace

cudaError_t launch_kv_write(const KvPool& kv, const KvRowSet& rs, const float* k, const float* v, uint64_t row_stride,
                            uint32_t* err, cudaStream_t st) {
  if (rs.n_rows == 0 || rs.n_seq == 0) return cudaSuccess;
  return copy_launch<false>(kv, copy_params(kv, rs, k, v, row_stride, err), st);
}

cudaError_t launch_kv_read(const KvPool& kv, const KvRowSet& rs, float* k, float* v, uint64_t row_stride,
                           uint32_t* err, cudaStream_t st) {
  if (rs.n_rows == 0 || rs.n_seq == 0) return cudaSuccess;
  return copy_launch<true>(kv, copy_params(kv, rs, k, v, row_stride, err), st);
}

}  // namespace eos
