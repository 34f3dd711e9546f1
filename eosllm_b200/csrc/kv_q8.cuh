// kv_q8.cuh -- the 8-bit paged key/value cache: page layout, row geometry
// and the row quantizer shared by the cache kernels (kv_q8.cu) and the
// attention that reads the cache (kv_q8_attn.cu).
//
// A cache is a pool of pages of 128 tokens.  Page p holds, for kv head h, one
// block of kv_block_bytes(HD) bytes at ((p * n_kv_head) + h) blocks:
//   K      int8 [128 tokens][HD]    a matrix operand with HD contiguous
//   V      int8 [4][HD][32 tokens]  a matrix operand with tokens contiguous,
//                                   one 32-token quarter after the other
//   scales f32 [4][2][32]           per quarter: 32 key scales, 32 value scales
// value = int8 * scale, one scale per (token, head) row of HD elements.
//
// Both matrices are stored in the order in which the tensor core reads them
// from shared memory, so a block is copied there byte for byte (one bulk
// copy) and needs no conversion:
//   K rows are swizzled in 16-byte chunks: HD = 128 as 128-byte rows (chunk ^=
//   token % 8), HD = 256 as two such 128-dimension panels, HD = 64 as 64-byte
//   rows (chunk ^= token / 2 % 4);
//   V rows are 32 bytes (chunk ^= dim / 4 % 2), and token u = g + 8 j of a
//   quarter (g < 8, j < 4) sits at position 4 g + j: the accumulator fragment
//   of the score product leaves tokens g, g + 8, g + 16, g + 24 in one
//   thread, which then writes its four probabilities as one word.  The order
//   of the tokens inside a quarter does not matter to the sum over them.
#pragma once

#include "eos_common.cuh"

namespace eos {

constexpr uint32_t kKvPage = 128;  // tokens of a page
constexpr uint32_t kKvQuarter = 32;

__host__ __device__ constexpr uint32_t kv_block_bytes(uint32_t hd) { return 2u * kKvPage * hd + 1024u; }

// Byte offsets inside a block.
template <uint32_t HD>
__device__ __forceinline__ uint32_t kv_k_offset(uint32_t token, uint32_t dim) {
  if constexpr (HD == 64)
    return token * 64u + ((((dim >> 4) ^ (token >> 1)) & 3u) << 4) + (dim & 15u);
  return (dim >> 7) * (kKvPage * 128u) + token * 128u + ((((dim >> 4) ^ token) & 7u) << 4) + (dim & 15u);
}
__device__ __forceinline__ uint32_t kv_v_position(uint32_t token) {  // inside the token's quarter
  return 4u * (token & 7u) + ((token >> 3) & 3u);
}
template <uint32_t HD>
__device__ __forceinline__ uint32_t kv_v_offset(uint32_t token, uint32_t dim) {
  const uint32_t p = kv_v_position(token);
  return kKvPage * HD + (token >> 5) * (HD * kKvQuarter) + dim * 32u + (((p >> 4) ^ (dim >> 2)) & 1u) * 16u + (p & 15u);
}
template <uint32_t HD>
__device__ __forceinline__ uint32_t kv_scale_offset(uint32_t token, uint32_t value) {  // value: 0 key, 1 value scale
  return 2u * kKvPage * HD + (token >> 5) * 256u + value * 128u + (token & 31u) * 4u;
}

// Rows of a batch.  Row r of sequence i (row0[i] <= r < row0[i + 1]; row0 ==
// nullptr: n_rows / n_seq rows each) is the (r - row0[i])-th.  Device values
// outside [0, n_rows] are clamped.
struct KvRows {
  const uint32_t* row0;
  uint32_t n_seq, n_rows, per_seq;
};
__device__ __forceinline__ uint32_t kv_row_start(const KvRows& b, uint32_t i) {
  const uint32_t r = b.row0 != nullptr ? b.row0[i] : i * b.per_seq;
  return r < b.n_rows ? r : b.n_rows;
}
// The last sequence i for which before(i, its first row) holds -- sequences in
// order, so these are the first ones -- with its rows [r0, r1) and words[i]; n_seq
// where there is none.  Warp-uniform; 32 sequences are looked at at once, and
// what is needed of them comes along, so a batch of up to 31 takes one round trip.
template <typename F>
__device__ __forceinline__ uint32_t kv_find(const KvRows& b, const uint32_t* words, F before, uint32_t& r0, uint32_t& r1,
                                            uint32_t& word) {
  const uint32_t lane = threadIdx.x & 31u;
  uint32_t lo = 0, len = b.n_seq;
  while (len > 32u) {
    const uint32_t step = (len + 31u) / 32u, i = lo + lane * step;
    const uint32_t c = __popc(__ballot_sync(0xffffffffu, lane * step < len && before(i, kv_row_start(b, i))));
    if (c == 0) return b.n_seq;
    lo += (c - 1u) * step;
    len = len - (c - 1u) * step < step ? len - (c - 1u) * step : step;
  }
  const uint32_t i = lo + lane;
  const uint32_t start = i <= b.n_seq ? kv_row_start(b, i) : 0u, w = i < b.n_seq ? words[i] : 0u;
  const uint32_t c = __popc(__ballot_sync(0xffffffffu, lane < len && before(i, start)));
  if (c == 0) return b.n_seq;
  r0 = __shfl_sync(0xffffffffu, start, c - 1u);
  r1 = c < 32u ? __shfl_sync(0xffffffffu, start, c) : kv_row_start(b, lo + c);
  word = __shfl_sync(0xffffffffu, w, c - 1u);
  return lo + c - 1u;
}

// ---- the row quantizer ----------------------------------------------------
// scale = max|x| * fl32(1 / 127) in f32; q = the integer nearest to 127 x / max|x|
// (ties to even) of the real quotient.  The f32 estimate x * fl32(127 / max|x|)
// is off by at most 127 * 2^-24 < 1e-5, so wherever it lies 1e-4 away from a
// half it decides: it is rounded by adding 1.5 * 2^23, which leaves q in the
// sum's low byte, and its distance from q is exact.  Otherwise (about one
// element in 5000) 127 x is compared with h max|x|, h the half: products of
// at most 33 bits, each held exactly as a float and its remainder (fma), whose
// differences are exact too.  Rows below 2^-100 or above 2^120 are scaled by a
// power of two first, so that neither 127 / max|x| nor these products leave the
// range.  A row that holds a NaN or an infinity gets that as its scale and q = 0:
// it reads back as NaN.
//
// Elements go in pairs and maxima in threes: 17 million elements (a prompt batch's
// keys and values) took 22.7 us with single ones, when issuing bound it.
struct KvRowScale {
  float scale, amax, inv, factor;  // amax and inv of the row times factor; factor 0: not finite
};
// max(|a|, |b|, |c|), NaN if one is
__device__ __forceinline__ float kv_max3(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float kv_absmax4(float amax, float4 v) {
  return kv_max3(kv_max3(amax, v.x, v.y), v.z, v.w);
}
__device__ __forceinline__ float2 kv_fma2(float2 a, float2 b, float2 c) {
  uint64_t x, y, z, d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(z) : "f"(c.x), "f"(c.y));
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(x), "l"(y), "l"(z));
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(d));
  return r;
}
// From the row's maximum: a warp's lanes' (amax bits, NaN above all) joined.
__device__ __forceinline__ KvRowScale kv_row_scale(float lane_amax) {
  const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(lane_amax) & 0x7fffffffu);
  KvRowScale s;
  const float amax = __uint_as_float(bits);
  s.factor = bits >= 0x7f800000u ? 0.0f : (amax < 7.8886e-31f ? 1.2676506e30f : (amax > 1.329228e36f ? 5.421011e-20f : 1.0f));
  s.scale = __fmul_rn(amax, 1.0f / 127.0f);
  s.amax = s.factor > 0.0f ? amax * s.factor : 0.0f;
  s.inv = s.amax > 0.0f ? __fdiv_rn(127.0f, s.amax) : 0.0f;
  return s;
}
// r = 1.5 2^23 + q of the estimate, o its distance from the estimate: the other neighbour if that is nearer.
__device__ __forceinline__ float kv_near_half(float x, float r, float o, float amax) {
  const float sg = copysignf(0.5f, o), h = __fadd_rn(__fsub_rn(r, 12582912.0f), sg);
  const float a = __fmul_rn(127.0f, x), b = __fmul_rn(h, amax);
  const float d = __fadd_rn(__fsub_rn(a, b), __fsub_rn(__fmaf_rn(127.0f, x, -a), __fmaf_rn(h, amax, -b)));
  const bool over = sg > 0.0f ? d > 0.0f : d < 0.0f, odd = (__float_as_uint(r) & 1u) != 0u;
  return fabsf(o) > 0.4999f && (over || (d == 0.0f && odd)) ? r + 2.0f * sg : r;
}
// Four elements as the bytes of a word.
__device__ __forceinline__ uint32_t kv_quant4(float4 v, const KvRowScale& s) {
  constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23
  const float2 magic = make_float2(kMagic, kMagic), inv = make_float2(s.inv, s.inv), minus = make_float2(-1.0f, -1.0f);
  if (s.factor != 1.0f) {  // warp-uniform
    const bool on = s.factor > 0.0f;
    v = make_float4(on ? v.x * s.factor : 0.0f, on ? v.y * s.factor : 0.0f, on ? v.z * s.factor : 0.0f,
                    on ? v.w * s.factor : 0.0f);
  }
  const float2 x0 = make_float2(v.x, v.y), x1 = make_float2(v.z, v.w);
  float2 r0 = kv_fma2(x0, inv, magic), r1 = kv_fma2(x1, inv, magic);
  const float2 o0 = kv_fma2(x0, inv, kv_fma2(r0, minus, magic)), o1 = kv_fma2(x1, inv, kv_fma2(r1, minus, magic));
  if (kv_max3(kv_max3(o0.x, o0.y, o1.x), o1.y, o1.y) > 0.4999f) {
    r0 = make_float2(kv_near_half(x0.x, r0.x, o0.x, s.amax), kv_near_half(x0.y, r0.y, o0.y, s.amax));
    r1 = make_float2(kv_near_half(x1.x, r1.x, o1.x, s.amax), kv_near_half(x1.y, r1.y, o1.y, s.amax));
  }
  return __byte_perm(__byte_perm(__float_as_uint(r0.x), __float_as_uint(r0.y), 0x0040),
                     __byte_perm(__float_as_uint(r1.x), __float_as_uint(r1.y), 0x0040), 0x5410);
}

}  // namespace eos
