// kv_q8_attn.cu -- attention of a batch of sequences that share a prefix,
// over the 8-bit paged cache (layout: kv_q8.cuh), on the sm_100a tensor cores.
//
// Row t of the n_i rows of sequence i, head h, kv head g = h n_kv / n_head:
//   S_j = scale <q, k_j> over the prefix's tokens and the sequence's own
//   tokens 0 .. len_i - n_i + t;  out = sum_j softmax(S)_j v_j;  no token
//   visible: out = 0.
//
// A unit is (kv head, rows that see the same pages): the prefix with the rows of
// all sequences, and each sequence's own pages with its rows.  Units of up to
// kFewRows rows run as integer dot products on the CUDA cores
// (kv_attn_few_kernel), larger ones on the tensor cores (kv_attn_kernel);
// kv_attn_join_kernel joins what they leave of a row: maximum, sum,
// unnormalised output.  Lengths live on the device and every kernel reads them
// there, so a captured call follows them.
//
// Arithmetic.  Keys and values stay the integers they are in the cache: a
// query row is scaled to integers of 24 bits and split into three signed
// 8-bit digits, a tile's probabilities (times the value scales) become integers
// of 23 bits in three unsigned digits, and every product has exact s32 sums -- no
// conversion of the cache, no 16-bit rounding anywhere.  A probability p times
// weight w becomes an integer as the mantissa of the float 2^23 + p w, whose three
// low bytes are the digits.  Both integers are fixed-point: a query element is
// held to 2^-24 of its row's largest, a probability times a value scale to 2^-23
// (few rows: 2^-31) of the largest value scale that the row sees in the page times
// the page's largest probability.  So a query element, or a value row, far below
// its neighbours loses low bits (beside a visible value row 1e2 times larger, of
// whatever probability, an output is 1e-4 of its size off); with rows of like size
// the errors are those of 32-bit arithmetic.  What a row does not see takes no part.
//
// Scores are compared before the row's query scale c (which holds the softmax
// scale) is applied: z = sum * key scale, exponent (z - max z) c plus the exact
// rest max z c - reference, so a rounding of the reference is common to the row
// and cancels; where it is no longer small (scores of 1e7) the rest is left out.
// One pass with a running maximum and sum per row in f32; each tile's value sums
// are folded into f32 registers.
//
// On the tensor cores the products are tcgen05.mma kind::i8.  The digits are
// further columns of the same product (N = 3 rows), so a page of keys is one M
// = 128 (tokens) operand and a page of values one M = 128 (dimensions) operand
// whatever the number of rows, both as the cache holds them: a page is copied
// to shared memory and multiplied.  Sums become floats without a conversion: a
// product of constants first puts a bias on every sum, and a sum that is not
// negative is a subnormal float, see attn_join (with an integer addition per sum
// instead: 293 us where this took 261).  The units' tiles (pages) form one line,
// cut into equal pieces, one per CTA, whatever the mixture of lengths; every CTA
// computes the line's layout from the lengths.  Joining the digits and the
// softmax bound it (44 instructions per pair of score and output; 48 rows x 32
// heads over 65537 tokens of 8 heads: 245 us, memory alone 27; issue slots 55 %
// taken, the rest waits on the chain score - maximum - exponent); for few rows
// over a long prefix the page copies do (8 rows over 16384 tokens of 32 heads:
// 48 us, memory alone 21), and for small calls the chain launch - lengths -
// table - page.  Widening the cache to f16 and multiplying hi and lo halves needs
// no joining: as first built it took 340 and 112 us for these two, the digits then
// 346 and 54.  Most of what has sped the digits up since (sixteen softmax warps,
// maxima by halving, wider accumulator loads) would serve it too; it was not taken
// up again.
//
// A CTA: eight warps for every 16 rows score and fold -- half of them on the even
// tiles of a piece, half on the odd ones, so that one half's chain of waits is
// the other's work --, a warp copies pages, and one issues the products,
// whichever is ready first.  A tile's probabilities take the place of its keys in
// shared memory.
#include "eos_kernels.h"
#include "kv_q8.cuh"

namespace eos {

constexpr uint32_t kAttnMaxCtas = 320;    // bound on the grid (scratch is sized with it)
constexpr uint32_t kAttnMl = 8;           // floats per partial row: maximum, 3 unused, 4 partial sums
constexpr float kAttnLow = -3e38f;        // reference of tiles whose tokens are all hidden: finite, so that no difference is NaN
constexpr float kAttnFar = 1e6f;          // log2 scores beyond this are compared before they are scaled
constexpr float kAttnQMax = 8300000.0f;   // largest query integer (three balanced digits hold 127 * 65793)

// Division of x < 2^31 by a launch constant: a multiplication (error below
// 1 / d for these x, so the quotient is exact).
struct AttnDiv {
  uint32_t d, shift;
  uint64_t mul;
};
__device__ __forceinline__ uint32_t attn_div(uint32_t x, const AttnDiv& v) {
  return (uint32_t)(__umul64hi((uint64_t)x << 32, v.mul) >> v.shift);
}
inline AttnDiv attn_divisor(uint32_t d) {  // mul = ceil(2^(32 + s) / d), 2^(s - 1) < d <= 2^s
  AttnDiv v{d, 0, 0};
  while ((1ull << v.shift) < d) ++v.shift;
  v.mul = (uint64_t)((((unsigned __int128)1 << (32u + v.shift)) + d - 1u) / d);
  return v;
}

struct KvAttnParams {
  KvRows rows;
  const uint8_t* pages;         // the sequences' pool
  const uint8_t* prefix_pages;  // the prefix's (the same, or another of the same geometry)
  const uint32_t* prefix_table;
  const uint32_t* prefix_len;
  const uint32_t* table;
  const uint32_t* seq_len;
  uint32_t max_prefix, table_stride, max_len, max_rows;
  uint32_t n_pages, prefix_n_pages, n_head, n_kv_head, group;
  AttnDiv by_group, by_kv_head;
  const float* q;
  float* out;
  uint64_t q_stride, out_stride;
  float scale_log2;  // scale * log2(e)
  uint32_t* plan;    // quantum, prefix tiles, prefix row groups, prefix work, then the sequences' running work
  float *po, *pml;   // prefix partials: [unit + CTA][half][row][HD], [unit + CTA][half][row][kAttnMl]
  float *so, *sml;   // the sequences' partials, with seq_cap rows
  uint32_t rt;                   // rows of the line's groups
  uint32_t prefix_cap, seq_cap;  // rows of a partial
  uint32_t seq_groups;           // row groups reserved per sequence
  // clusters per unit and CTAs per cluster where the few-rows kernel has the prefix (the sequences), else 0: the
  // line has them
  uint32_t prefix_few, prefix_ctas, seq_few, seq_ctas;
  uint32_t* err;
};

__host__ __device__ constexpr uint32_t attn_ceil(uint32_t a, uint32_t b) { return (a + b - 1u) / b; }

// A unit's length on the line: its tiles behind kAttnStart places for what
// every unit costs besides (its queries, its partial).
constexpr uint32_t kAttnStart = 1;
__host__ __device__ constexpr uint32_t attn_cost(uint32_t tiles) { return tiles ? tiles + kAttnStart : 0u; }

// Rows and tokens of a sequence, cut to their bounds.
struct AttnSeq {
  uint32_t r0, n, len;
};
__device__ __forceinline__ AttnSeq attn_seq(const KvAttnParams& p, uint32_t i) {
  AttnSeq s;
  const uint32_t len = p.seq_len[i], r1 = kv_row_start(p.rows, i + 1u);
  s.r0 = kv_row_start(p.rows, i);
  s.n = r1 > s.r0 ? r1 - s.r0 : 0u;
  s.len = len < p.max_len ? len : p.max_len;
  return s;
}
// Places of a sequence on the line (rows beyond max_rows are left out).
template <uint32_t RT>
__device__ __forceinline__ uint32_t attn_seq_work(const KvAttnParams& p, const AttnSeq& s) {
  const uint32_t n = s.n < p.max_rows ? s.n : p.max_rows;
  return p.n_kv_head * attn_ceil(n * p.group, RT) * attn_cost(attn_ceil(s.len, kKvPage));
}

struct AttnPlan {
  uint32_t quantum, tp, rgp, wp, rows_p, prefix;
  AttnSeq mine;  // sequence `lane`
};

// One piece of a unit (the whole copy warp computes it).
struct AttnSeg {
  uint32_t head, rg;        // kv head, row group
  uint32_t step;            // places of the line that the piece takes
  uint32_t tile0, tiles;    // pages [tile0, tile0 + tiles) of the unit
  uint32_t seq;             // sequence, or n_seq for the prefix
  uint32_t row0, rows;      // first (query row * group + head in group) of the group, how many
  uint32_t base_row;        // query row of the unit's row 0
  uint32_t len, n;          // tokens of the unit; rows of the sequence
  uint32_t unit;            // partial index without the CTA
};

template <uint32_t RT>
__device__ __forceinline__ AttnSeg attn_segment(const KvAttnParams& p, const AttnPlan& pl, const uint32_t* cum,
                                                uint32_t w, uint32_t w1) {
  AttnSeg s;
  uint32_t tiles, x, u, at;
  if (w < pl.wp) {
    tiles = pl.tp;
    x = w;
    u = x / attn_cost(tiles);
    at = x - u * attn_cost(tiles);
    s.head = u / pl.rgp;
    s.rg = u - s.head * pl.rgp;
    s.seq = p.rows.n_seq;
    s.base_row = 0;
    s.len = pl.prefix;
    s.n = 0;
    s.row0 = s.rg * RT;
    s.rows = pl.rows_p * p.group - s.row0;
    s.unit = u;
  } else {
    x = w - pl.wp;
    uint32_t lo = 0, hi = p.rows.n_seq;  // cum[lo] <= x < cum[hi]
    while (hi - lo > 1u) {
      const uint32_t mid = (lo + hi) >> 1;
      if (cum[mid] <= x) lo = mid;
      else hi = mid;
    }
    x -= cum[lo];
    // the first 32 sequences sit in the lanes' registers
    AttnSeq q;
    if (lo < 32u) {
      q.r0 = __shfl_sync(0xffffffffu, pl.mine.r0, lo);
      q.n = __shfl_sync(0xffffffffu, pl.mine.n, lo);
      q.len = __shfl_sync(0xffffffffu, pl.mine.len, lo);
    } else {
      q = attn_seq(p, lo);
    }
    const uint32_t n = q.n < p.max_rows ? q.n : p.max_rows;
    tiles = attn_ceil(q.len, kKvPage);
    u = x / attn_cost(tiles);
    at = x - u * attn_cost(tiles);
    s.rg = attn_div(u, p.by_kv_head);
    s.head = u - s.rg * p.n_kv_head;
    s.seq = lo;
    s.base_row = q.r0;
    s.len = q.len;
    s.n = q.n;
    s.row0 = s.rg * RT;
    s.rows = n * p.group - s.row0;
    s.unit = lo * p.seq_groups * p.n_kv_head + u;
  }
  if (s.rows > RT) s.rows = RT;
  s.step = attn_cost(tiles) - at;
  if (s.step > w1 - w) s.step = w1 - w;
  s.tile0 = at > kAttnStart ? at - kAttnStart : 0u;
  s.tiles = at + s.step > kAttnStart ? at + s.step - kAttnStart - s.tile0 : 0u;
  return s;
}

// ---- tcgen05 --------------------------------------------------------------
// K-major shared-memory operand: start address >> 4, LBO 16 B (unused when
// swizzled), SBO = 8 rows, version 1, layout type (2: 128-byte swizzle, 4:
// 64-byte, 6: 32-byte).  Advancing K by 32 bytes adds 2 to the start field.
__device__ __forceinline__ uint64_t attn_desc(uint32_t addr, uint32_t row_bytes) {
  const uint64_t type = row_bytes == 128u ? 2u : (row_bytes == 64u ? 4u : 6u);
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)1u << 16) | ((uint64_t)((8u * row_bytes) >> 4) << 32) |
         ((uint64_t)1u << 46) | (type << 61);
}
// Instruction descriptor, kind::i8: D s32, A and B s8 or u8, both K-major.
__device__ constexpr uint32_t attn_idesc(bool a_signed, bool b_signed, uint32_t n) {
  return (2u << 4) | ((a_signed ? 1u : 0u) << 7) | ((b_signed ? 1u : 0u) << 10) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}
// An operand of bytes 255 throughout: cores of 8 rows x 16 bytes, no swizzle,
// neighbours 16 bytes apart, so that 128 rows of 32 bytes are kAttnOnes bytes.
// A product of two adds 32 * 255 * 255 = kAttnBias to every sum, one for every
// 128 dimensions at least the largest negative score sum (each element -128 *
// 127); two cover a value sum (128 tokens of 255 * -127).
constexpr uint32_t kAttnOnes = 384, kAttnBias = 32u * 255u * 255u;
__host__ __device__ constexpr uint32_t attn_score_biases(uint32_t hd) { return hd <= 128u ? 1u : hd / 128u; }
constexpr bool attn_bias_covers(uint32_t biases, uint64_t sum) {  // biased sums are not negative and below 2^23
  return (uint64_t)biases * kAttnBias >= sum && (uint64_t)biases * kAttnBias + sum < (1ull << 23);
}
static_assert(attn_bias_covers(attn_score_biases(64), 64u * 128u * 127u) &&
                  attn_bias_covers(attn_score_biases(128), 128u * 128u * 127u) &&
                  attn_bias_covers(attn_score_biases(256), 256u * 128u * 127u) &&
                  attn_bias_covers(2u, 128u * 255u * 127u),
              "a biased sum reads as a subnormal float");
__device__ __forceinline__ uint64_t attn_ones_desc(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)1u << 16) | ((uint64_t)1u << 32) | ((uint64_t)1u << 46);
}
__device__ __forceinline__ void attn_mma(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}\n" ::"r"(tmem_d),
      "l"(da), "l"(db), "r"(idesc), "r"(accumulate), "r"(0u), "r"(0u), "r"(0u), "r"(0u)
      : "memory");
}
__device__ __forceinline__ void attn_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void attn_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void attn_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void attn_fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// 16 TMEM lanes x 8 columns: thread t gets r[0..1] = lane t / 4, columns
// 2 (t % 4) + {0, 1}, and r[2..3] the same columns of lane t / 4 + 8.  Two: and
// r[4..7] the same of the 8 columns behind.
__device__ __forceinline__ void attn_ld(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void attn_ld_two(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void attn_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// use(y, j, d0, d1, d2) with the digit sums (digits RT columns apart) of 32 lanes
// and the first nact of two chunks of 8 columns: chunk y, lane g + 8 j.  Groups
// of 16 rows are read chunk by chunk, since often only one is in use; 32 rows by
// half the lanes, in half as many instructions.
template <uint32_t RT, typename F>
__device__ __forceinline__ void attn_sums(uint32_t taddr, uint32_t nact, F use) {
  if constexpr (RT == 16u) {
#pragma unroll
    for (uint32_t y = 0; y < 2u; ++y) {
      if (y >= nact) break;  // warp-uniform
      uint32_t r[3][8];
#pragma unroll
      for (uint32_t e = 0; e < 3u; ++e)
#pragma unroll
        for (uint32_t hh = 0; hh < 2u; ++hh) attn_ld(taddr + ((16u * hh) << 16) + e * RT + 8u * y, &r[e][4u * hh]);
      attn_ld_wait();
#pragma unroll
      for (uint32_t j = 0; j < 4u; ++j) use(y, j, &r[0][2u * j], &r[1][2u * j], &r[2][2u * j]);
    }
  } else if (nact > 0) {  // warp-uniform
#pragma unroll
    for (uint32_t hh = 0; hh < 2u; ++hh) {
      uint32_t r[3][8];
#pragma unroll
      for (uint32_t e = 0; e < 3u; ++e) attn_ld_two(taddr + ((16u * hh) << 16) + e * RT, r[e]);
      attn_ld_wait();
#pragma unroll
      for (uint32_t y = 0; y < 2u; ++y) {
        if (y >= nact) break;
#pragma unroll
        for (uint32_t j = 0; j < 2u; ++j)
          use(y, 2u * hh + j, &r[0][4u * y + 2u * j], &r[1][4u * y + 2u * j], &r[2][4u * y + 2u * j]);
      }
    }
  }
}
__device__ __forceinline__ void attn_bulk(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ float attn_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Pairs of f32 (the two columns of an accumulator fragment).
__device__ __forceinline__ uint64_t attn_pack(float2 a) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
  return r;
}
__device__ __forceinline__ float2 attn_unpack(uint64_t a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
  return r;
}
__device__ __forceinline__ float2 attn_fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(attn_pack(a)), "l"(attn_pack(b)), "l"(attn_pack(c)));
  return attn_unpack(d);
}
__device__ __forceinline__ float2 attn_add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(attn_pack(a)), "l"(attn_pack(b)));
  return attn_unpack(d);
}
__device__ __forceinline__ float2 attn_mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(attn_pack(a)), "l"(attn_pack(b)));
  return attn_unpack(d);
}
__device__ __forceinline__ float2 attn_two(float x) { return make_float2(x, x); }
// (256 D2 + D1 + D0 / 256) 2^-22 of three s32 sums d = D + BIAS, 0 <= d < 2^23:
// the bits of d, read as a float, are the subnormal d 2^-149, so fma(d, 2^127, c) =
// d 2^-22 + c takes the bias off, exactly and with no conversion; two roundings,
// of D1 + D0 / 256 (D0's bias goes with D1's: its 256th part has few bits) and of
// the sum.
template <uint32_t BIAS>
__device__ __forceinline__ float2 attn_join(const uint32_t* d0, const uint32_t* d1, const uint32_t* d2) {
  constexpr float two127 = 1.7014118346046923e38f, two119 = 6.646139978924579e35f, unit = 1.0f / 4194304.0f;
  static_assert(BIAS < (1u << 22) && BIAS % 32u == 0, "BIAS + BIAS / 256 has 24 bits");
  auto bits = [](const uint32_t* d) { return make_float2(__uint_as_float(d[0]), __uint_as_float(d[1])); };
  const float2 lo = attn_fma2(bits(d0), attn_two(two119),
                              attn_fma2(bits(d1), attn_two(two127), attn_two(-((float)BIAS + (float)BIAS / 256.0f) * unit)));
  return attn_fma2(attn_fma2(bits(d2), attn_two(two127), attn_two(-(float)BIAS * unit)), attn_two(256.0f), lo);
}
// Bytes 0, 1 and 2 of four words as three words.
__device__ __forceinline__ void attn_digits(const uint32_t* b, uint32_t* w) {
  const uint32_t lo01 = __byte_perm(b[0], b[1], 0x5140), lo23 = __byte_perm(b[2], b[3], 0x5140);
  w[0] = __byte_perm(lo01, lo23, 0x5410);
  w[1] = __byte_perm(lo01, lo23, 0x7632);
  w[2] = __byte_perm(__byte_perm(b[0], b[1], 0x0062), __byte_perm(b[2], b[3], 0x0062), 0x5410);
}

// A query row as integers: scale maps score integers (in units of 256) to log2
// scores; a negative softmax scale turns the integers' sign, so larger products
// are larger scores.
struct AttnQScale {
  float inv, scale;
  bool finite;
};
__device__ __forceinline__ uint32_t attn_absmax(uint32_t amax, float4 v) {
  amax = max(max(amax, __float_as_uint(v.x) & 0x7fffffffu), __float_as_uint(v.y) & 0x7fffffffu);
  return max(max(amax, __float_as_uint(v.z) & 0x7fffffffu), __float_as_uint(v.w) & 0x7fffffffu);
}
__device__ __forceinline__ AttnQScale attn_query_scale(uint32_t amax, float scale_log2) {
  AttnQScale s;
  s.finite = amax < 0x7f800000u;
  const float top = fmaxf(__uint_as_float(amax), 1e-30f);
  s.inv = s.finite ? __fdiv_rn(scale_log2 < 0.0f ? -kAttnQMax : kAttnQMax, top) : 0.0f;
  // (above 0, so that a hidden token's -infinity stays one when the softmax scale is 0; finite: a scale that large
  // parts any two scores all the same)
  s.scale = s.finite ? fminf(fmaxf(__fdiv_rn(top, kAttnQMax) * (256.0f * fabsf(scale_log2)), 1e-37f), 3e38f) : NAN;
  return s;
}
// Three balanced digits of four elements: bytes of (x + 0x808080) ^ 0x808080.
__device__ __forceinline__ void attn_query_digits(float4 v, const AttnQScale& s, uint32_t* d) {
  const float f[4] = {v.x, v.y, v.z, v.w};
  uint32_t b[4];
#pragma unroll
  for (uint32_t e = 0; e < 4u; ++e)
    b[e] = (uint32_t)((s.finite ? __float2int_rn(f[e] * s.inv) : 0) + 0x808080) ^ 0x808080u;
  attn_digits(b, d);
}
// Weights (probability times value scale) as integers: the largest value scale
// at hand becomes kAttnWeight -- 2^23 less what the roundings of the quotient may
// add --, whatever its mantissa: with powers of two only, the integers of a page
// were half as long at worst, and outputs 1.2e-6 off where 32-bit arithmetic was
// 0.5e-6.  The quotient is within 2 units in its last place, for all of a page.
constexpr float kAttnWeight = 8388604.0f;
__device__ __forceinline__ float attn_weight_top(float v) { return fmaxf(v, 4.930381e-32f); }  // 2^-104: a finite quotient
__device__ __forceinline__ float attn_weight_scale(float top) { return __fdividef(kAttnWeight, top); }
__device__ __forceinline__ float attn_weight_unit(float top) { return top * (4194304.0f / kAttnWeight); }  // sums in 2^22
__device__ __forceinline__ float attn_warp_max(float x) {
#pragma unroll
  for (uint32_t b = 16; b > 0; b >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, b));
  return x;
}

// ---- few rows: integer dot products on the CUDA cores -------------------------
// Up to kFewRows rows (query rows times heads of the kv head) against a unit's
// pages, dealt out to the CTAs (128 threads) of one or more clusters: whatever
// the length turns out to be, all of them have their share.  A cluster joins
// its CTAs' sums through shared memory, so a unit on one cluster is done with
// one launch.  Reading the cache is what bounds it: 2 HD + 8 bytes per token
// against 7 HD / 4 dp4a per token and row, so a few rows stay near the
// memory's time (one row over 16000 tokens of 32 heads: 26.2 us, 5.2 TB/s).  No
// barrier or tensor memory to set up and several CTAs per SM (four at 128
// dimensions, by launch bounds), each with a page's loads in flight: units of a
// page or two (a sequence's own tokens, a decode step) take one round trip to
// memory.
// Queries as in the tensor-core kernel, probabilities with 8 bits more; s32 sums
// over 16 dimensions (scores) and over a page (values) are exact.
// Measured both ways: 8 rows over 16384 tokens of 32 heads 131 us here, 48 on the
// tensor cores; four rows over 640 tokens of 8 heads 7.5 here, 10.4 there; 128
// units of four rows over 300 tokens 10.7 and 13.5; 384 of up to 700 tokens beside
// a prefix of 65537 246 and 247 in all; one row over 16000 tokens 26.1 and 37.0.
constexpr uint32_t kFewRows = 4;
constexpr uint32_t kFewThreads = 128;

// s8 x u8 (or s8 x s8) dot product of four.
__device__ __forceinline__ int32_t attn_dp4a(bool b_unsigned, uint32_t a, uint32_t b, int32_t c) {
  if (!b_unsigned) return __dp4a((int)a, (int)b, c);
  int32_t d;
  asm("dp4a.s32.u32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint4 attn_ld_stream(const void* src) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(src));
  return v;
}

__device__ __forceinline__ void attn_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A float of this CTA's shared memory as CTA `rank` of the cluster holds it.
__device__ __forceinline__ float attn_peer(const float* x, uint32_t rank) {
  uint32_t a;
  float v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(x)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

// Grid (clusters x CTAs, kv heads, sequences); prefix: one "sequence" of all
// rows.  direct: there is nothing to join the rows with, write them out.
template <uint32_t HD, uint32_t R>
__global__ void __launch_bounds__(kFewThreads, HD <= 128u ? 4 : (R == 1u ? 3 : 2))
    kv_attn_few_kernel(const KvAttnParams p, uint32_t prefix, uint32_t n_cta, uint32_t direct) {
  constexpr uint32_t CL = HD / 16u;                    // 16-byte chunks of a key row = lanes per token
  constexpr uint32_t DT = HD <= 128u ? 1u : HD / 128u; // dimensions per thread
  constexpr uint32_t QT = HD == 64u ? 2u : 4u;         // quarters of the values per thread
  __shared__ __align__(16) uint32_t qd[R][3][HD / 4u]; // query digits
  __shared__ float qscale[R];
  __shared__ __align__(16) uint8_t pd[R][4][kKvPage];  // probability digits by position
  __shared__ float red[2][4][2u * R];                  // per warp: maxima, largest value scales
  __shared__ float cl_o[R][HD], cl_ml[R][2];           // this CTA's sums, for the cluster
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const uint32_t g = blockIdx.y;
  AttnSeq s{0, 0, 0};
  const uint32_t* table = p.prefix_table;
  if (prefix) {
    s.len = p.prefix_len != nullptr ? *p.prefix_len : 0u;
    s.n = kv_row_start(p.rows, p.rows.n_seq);
    if (s.len > p.max_prefix) {
      s.len = p.max_prefix;
      if (blockIdx.x == 0 && g == 0 && tid == 0) report(p.err, EOS_DEVERR_RANGE);
    }
  } else {
    s = attn_seq(p, blockIdx.z);
    table = p.table + (size_t)blockIdx.z * p.table_stride;
    if (blockIdx.x == 0 && g == 0 && tid == 0 && (p.seq_len[blockIdx.z] > p.max_len || s.n > p.max_rows))
      report(p.err, EOS_DEVERR_RANGE);
  }
  const uint32_t pages = attn_ceil(s.len, kKvPage);
  uint32_t rows = (prefix || s.n < p.max_rows ? s.n : p.max_rows) * p.group;
  if (rows > R) rows = R;  // (the host chose R >= rows)
  pdl_trigger();
  if (rows == 0) return;  // the whole cluster
  const int32_t seen0 = (int32_t)s.len - (int32_t)s.n + 1;  // tokens a sequence's first row sees (may be negative)
  // the rows' digits, warp w those of rows w, w + 4
  for (uint32_t row = warp; row < R; row += 4u) {
    float scale = 0.0f;
    constexpr uint32_t QF = HD <= 128u ? 1u : HD / 128u;
    uint32_t d[QF][3];
#pragma unroll
    for (uint32_t c = 0; c < QF; ++c) d[c][0] = d[c][1] = d[c][2] = 0u;
    if (row < rows) {
      const uint32_t xr = attn_div(row, p.by_group);
      const float* src = p.q + (size_t)(s.r0 + xr) * p.q_stride + (size_t)(g * p.group + row - xr * p.group) * HD;
      float4 v[QF];
      uint32_t amax = 0;
#pragma unroll
      for (uint32_t c = 0; c < QF; ++c) {
        v[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (HD >= 128u || lane < HD / 4u) v[c] = *reinterpret_cast<const float4*>(src + c * 128u + lane * 4u);
        amax = attn_absmax(amax, v[c]);
      }
      amax = __reduce_max_sync(0xffffffffu, amax);
      const AttnQScale qsc = attn_query_scale(amax, p.scale_log2);
      scale = qsc.scale;
#pragma unroll
      for (uint32_t c = 0; c < QF; ++c) attn_query_digits(v[c], qsc, d[c]);
    }
#pragma unroll
    for (uint32_t c = 0; c < QF; ++c)
      if (HD >= 128u || lane < HD / 4u)
#pragma unroll
        for (uint32_t e = 0; e < 3u; ++e) qd[row][e][c * 32u + lane] = d[c][e];
    if (lane == 0) qscale[row] = scale;
  }
  __syncthreads();
  // score side: lane's chunk of the key rows, tokens 32 warp + i (32 / CL) + lane / CL
  const uint32_t lc = lane % CL, lt = lane / CL;
  // after the reduction over the CL lanes of a token, this lane holds token `own`
  const uint32_t own = warp * 32u + lc * (32u / CL) + lt;
  // value side: this thread's dimension(s) and quarters
  const uint32_t dim0 = HD == 64u ? (tid & 63u) : tid, q0 = HD == 64u ? (tid >> 6) * 2u : 0u;
  float o[R][DT], m[R], l[R];
#pragma unroll
  for (uint32_t r = 0; r < R; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.0f;
#pragma unroll
    for (uint32_t d = 0; d < DT; ++d) o[r][d] = 0.0f;
  }
  uint32_t par = 0;  // which red[]
  for (uint32_t pg = blockIdx.x; pg < pages; pg += gridDim.x, par ^= 1u) {
    const uint32_t page = table[pg];
    if (page >= (prefix ? p.prefix_n_pages : p.n_pages)) {  // hidden
      if (tid == 0) report(p.err, EOS_DEVERR_RANGE);
      continue;
    }
    const uint8_t* blk =
        (prefix ? p.prefix_pages : p.pages) + ((size_t)page * p.n_kv_head + g) * kv_block_bytes(HD);
    const uint32_t avail = s.len - pg * kKvPage;  // tokens (may exceed a page)
    uint4 kw[CL], vw[DT][QT][2];
#pragma unroll
    for (uint32_t i = 0; i < CL; ++i) {
      const uint32_t t = warp * 32u + i * (32u / CL) + lt;
      kw[i] = make_uint4(0u, 0u, 0u, 0u);
      if (t < avail) kw[i] = attn_ld_stream(blk + kv_k_offset<HD>(t, lc * 16u));
    }
    float ks = 0.0f, vs = 0.0f;
    if (own < avail) {
      ks = __ldg(reinterpret_cast<const float*>(blk + kv_scale_offset<HD>(own, 0)));
      vs = __ldg(reinterpret_cast<const float*>(blk + kv_scale_offset<HD>(own, 1)));
    }
#pragma unroll
    for (uint32_t d = 0; d < DT; ++d)
#pragma unroll
      for (uint32_t q = 0; q < QT; ++q)
#pragma unroll
        for (uint32_t c = 0; c < 2u; ++c) {
          const uint32_t dim = dim0 + d * 128u;
          vw[d][q][c] = make_uint4(0u, 0u, 0u, 0u);
          if ((q0 + q) * kKvQuarter < avail)
            vw[d][q][c] = attn_ld_stream(blk + kKvPage * HD + (q0 + q) * (HD * kKvQuarter) + dim * 32u +
                                         ((c ^ (dim >> 2)) & 1u) * 16u);
        }
    if (!(vs < INFINITY)) {  // a NaN or infinite value row: NaN score
      ks = NAN;
      vs = 0.0f;
    }
    // scores
    float z[R];
#pragma unroll
    for (uint32_t r = 0; r < R; ++r) {
      float part[CL];
      uint4 qw[3];
#pragma unroll
      for (uint32_t e = 0; e < 3u; ++e) qw[e] = *reinterpret_cast<const uint4*>(&qd[r][e][lc * 4u]);
#pragma unroll
      for (uint32_t i = 0; i < CL; ++i) {
        int32_t a[3];
#pragma unroll
        for (uint32_t e = 0; e < 3u; ++e) {
          a[e] = __dp4a((int)kw[i].x, (int)qw[e].x, 0);
          a[e] = __dp4a((int)kw[i].y, (int)qw[e].y, a[e]);
          a[e] = __dp4a((int)kw[i].z, (int)qw[e].z, a[e]);
          a[e] = __dp4a((int)kw[i].w, (int)qw[e].w, a[e]);
        }
        // below 2^18 each: (a2 2^8 + a1) is exact in s32; a0 / 256 joins as a float
        part[i] = fmaf((float)a[0], 1.0f / 256.0f, (float)(a[2] * 256 + a[1]));
      }
      // sums over the token's lanes, each lane ending with one token
#pragma unroll
      for (uint32_t b = CL / 2u; b > 0; b >>= 1) {
        const bool up = (lane & b) != 0u;
#pragma unroll
        for (uint32_t i = 0; i < CL; ++i) {
          if (i >= b) break;
          const float give = up ? part[i] : part[i + b], keep = up ? part[i + b] : part[i];
          part[i] = keep + __shfl_xor_sync(0xffffffffu, give, b);
        }
      }
      const int32_t seen = prefix ? (int32_t)s.len : seen0 + (int32_t)attn_div(r, p.by_group);
      const int32_t tok = (int32_t)(pg * kKvPage + own);
      z[r] = own < avail && tok < seen ? part[0] * ks : -INFINITY;
      const float mx = attn_warp_max(z[r]);
      if (lane == 0) red[par][warp][r] = mx;
    }
    // the largest value scale that a row sees: one for all, or one each where the page ends behind the first row's
    // tokens (what such a page hides has z = -infinity)
    const bool cut = !prefix && (int32_t)min(s.len, (pg + 1u) * kKvPage) > seen0;
#pragma unroll
    for (uint32_t r = 0; r < R; ++r) {
      if (r > 0 && !cut) break;
      const uint32_t top = __reduce_max_sync(0xffffffffu, cut && z[r] == -INFINITY ? 0u : __float_as_uint(vs));
      if (lane == 0) red[par][warp][R + r] = __uint_as_float(top);
    }
    __syncthreads();
    const float(*rd)[2u * R] = red[par];
    auto exponent = [&](uint32_t r) {
      const float most = fmaxf(fmaxf(rd[0][R + r], rd[1][R + r]), fmaxf(rd[2][R + r], rd[3][R + r]));
      return max(__float_as_uint(most) >> 23, 23u);
    };
    const uint32_t common = exponent(0);
    float f[R];
#pragma unroll
    for (uint32_t r = 0; r < R; ++r) {
      const float mt = fmaxf(fmaxf(rd[0][r], rd[1][r]), fmaxf(rd[2][r], rd[3][r]));
      const uint32_t top = r > 0 && cut ? exponent(r) : common;
      const float ref = mt == -INFINITY ? mt : __fmul_ru(mt, qscale[r]), nm = fmaxf(ref, m[r]);
      const float neg = nm == -INFINITY ? 0.0f : -nm;
      f[r] = attn_ex2(m[r] + neg);
      m[r] = nm;
      // (scores so large that a rounding of the reference is no common factor any more: relative to the page's largest)
      const float e = attn_ex2(fabsf(nm) > kAttnFar ? fmaf(z[r] - fmaxf(mt, kAttnLow), qscale[r], ref + neg)
                                                    : fmaf(z[r], qscale[r], neg));
      l[r] = fmaf(l[r], f[r], e);  // this token's share
      // e vs as 23 bits (the low bytes of 2^23 + ..) and a signed byte of what is left, in 1 / 256
      const float y = cut && z[r] == -INFINITY ? 0.0f : vs * __uint_as_float((276u - top) << 23);
      const float b = fmaf(e, y, 8388608.0f), rest = fmaf(e, y, 8388608.0f - b);
      const uint32_t w = __float_as_uint(b);
      uint8_t* at = &pd[r][0][warp * 32u + kv_v_position(own)];
      at[0] = (uint8_t)w;
      at[kKvPage] = (uint8_t)(w >> 8);
      at[2u * kKvPage] = (uint8_t)(w >> 16);
      at[3u * kKvPage] = (uint8_t)__float2int_rn(fminf(rest * 256.0f, 127.0f));
    }
    __syncthreads();
    // values
#pragma unroll
    for (uint32_t r = 0; r < R; ++r) {
      const float unit = __uint_as_float(((r > 0 && cut ? exponent(r) : common) - 22u) << 23);
      int32_t a[DT][4];
#pragma unroll
      for (uint32_t d = 0; d < DT; ++d) a[d][0] = a[d][1] = a[d][2] = a[d][3] = 0;
#pragma unroll
      for (uint32_t e = 0; e < 4u; ++e)
#pragma unroll
        for (uint32_t q = 0; q < QT; ++q)
#pragma unroll
          for (uint32_t c = 0; c < 2u; ++c) {
            const uint4 w = *reinterpret_cast<const uint4*>(&pd[r][e][(q0 + q) * kKvQuarter + c * 16u]);
#pragma unroll
            for (uint32_t d = 0; d < DT; ++d) {
              a[d][e] = attn_dp4a(e < 3u, vw[d][q][c].x, w.x, a[d][e]);
              a[d][e] = attn_dp4a(e < 3u, vw[d][q][c].y, w.y, a[d][e]);
              a[d][e] = attn_dp4a(e < 3u, vw[d][q][c].z, w.z, a[d][e]);
              a[d][e] = attn_dp4a(e < 3u, vw[d][q][c].w, w.w, a[d][e]);
            }
          }
#pragma unroll
      for (uint32_t d = 0; d < DT; ++d) {
        const float low = fmaf((float)a[d][1], 256.0f, fmaf((float)a[d][3], 1.0f / 256.0f, (float)a[d][0]));
        const float v = fmaf((float)a[d][2], 65536.0f, low);
        o[r][d] = fmaf(v, unit, o[r][d] * f[r]);
      }
    }
    // (the next page's red[] is the other buffer, and its pd[] follows a barrier that every warp reaches after these reads)
  }
  // this CTA's sums, then the cluster's: CTA 0 joins and writes them
#pragma unroll
  for (uint32_t r = 0; r < R; ++r) {
    float ls = l[r];
#pragma unroll
    for (uint32_t b = 16; b > 0; b >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, b);
    if (lane == 0) red[0][warp][r] = ls;
    if constexpr (HD == 64) {  // two threads hold the halves of a dimension's sum
      if (tid >= 64u) cl_o[r][tid & 63u] = o[r][0];
    } else {
#pragma unroll
      for (uint32_t d = 0; d < DT; ++d) cl_o[r][d * 128u + tid] = o[r][d];
    }
  }
  __syncthreads();
  if (tid < R) {
    cl_ml[tid][1] = (red[0][0][tid] + red[0][1][tid]) + (red[0][2][tid] + red[0][3][tid]);
#pragma unroll
    for (uint32_t r = 0; r < R; ++r)
      if (tid == r) cl_ml[r][0] = m[r];
  }
  if constexpr (HD == 64) {
    if (tid < 64u)
#pragma unroll
      for (uint32_t r = 0; r < R; ++r) cl_o[r][tid] += o[r][0];
  }
  attn_cluster_sync();
  const uint32_t rank = blockIdx.x % n_cta;
  if (rank == 0) {
    const uint32_t cap = prefix ? p.prefix_cap : p.seq_cap;
    const size_t id = ((size_t)(prefix ? 0u : blockIdx.z) * p.n_kv_head + g) * (gridDim.x / n_cta) + blockIdx.x / n_cta;
    float* po = (prefix ? p.po : p.so) + id * cap * HD;
    float* pml = (prefix ? p.pml : p.sml) + id * cap * kAttnMl;
    for (uint32_t r = 0; r < rows; ++r) {
      float mc[8], lc2[8], oc[8][DT], top = -INFINITY;
#pragma unroll
      for (uint32_t c = 0; c < 8u; ++c)
        if (c < n_cta) {
          mc[c] = attn_peer(&cl_ml[r][0], c);
          lc2[c] = attn_peer(&cl_ml[r][1], c);
#pragma unroll
          for (uint32_t d = 0; d < DT; ++d) oc[c][d] = attn_peer(&cl_o[r][(d * 128u + tid) % HD], c);
          top = fmaxf(top, mc[c]);
        }
      const float mu = top == -INFINITY ? 0.0f : top;
      float ls = 0.0f, acc[DT];
#pragma unroll
      for (uint32_t d = 0; d < DT; ++d) acc[d] = 0.0f;
#pragma unroll
      for (uint32_t c = 0; c < 8u; ++c)
        if (c < n_cta) {
          const float f = attn_ex2(mc[c] - mu);
          ls = fmaf(f, lc2[c], ls);
#pragma unroll
          for (uint32_t d = 0; d < DT; ++d) acc[d] = fmaf(f, oc[c][d], acc[d]);
        }
      if (tid >= HD) continue;
      if (direct) {
        const uint32_t xr = attn_div(r, p.by_group);
        const bool none = seen0 + (int32_t)xr <= 0;  // 0, also for a query that is not finite
        const float inv = ls == 0.0f ? 0.0f : __fdiv_rn(1.0f, ls);
        float* dst = p.out + (size_t)(s.r0 + xr) * p.out_stride + (size_t)(g * p.group + r - xr * p.group) * HD;
#pragma unroll
        for (uint32_t d = 0; d < DT; ++d) dst[d * 128u + tid] = none ? 0.0f : acc[d] * inv;
      } else {
#pragma unroll
        for (uint32_t d = 0; d < DT; ++d) po[(size_t)r * HD + d * 128u + tid] = acc[d];
        if (tid == 0) {
          pml[r * kAttnMl] = top;
          *reinterpret_cast<float4*>(pml + r * kAttnMl + 4u) = make_float4(ls, 0.0f, 0.0f, 0.0f);
        }
      }
    }
  }
  attn_cluster_sync();  // no CTA leaves while its sums are read
}

// mbar_wait whose polls may sleep up to 20 us each (until the phase completes)
// and which reads the clock only after sixteen: a warp that waits leaves the
// issue slots to the others.
__device__ __forceinline__ bool attn_try(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool attn_wait(uint64_t* bar, uint32_t parity) {
  for (uint32_t i = 0; i < 16u; ++i)
    if (attn_try(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  while (!attn_try(bar, parity))
    if (global_timer_ns() - t0 > EOS_WAIT_LIMIT_NS) return false;
  return true;
}

// One look at a barrier, without waiting.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// ---- geometry of a CTA ------------------------------------------------------
// Row groups of 16 (three digits each: N = 48), two CTAs per SM, for few rows: the
// page copies of four tiles in flight hide each other's latency.  Groups of 32,
// one CTA per SM, read a page half as often and share a tile's fixed work: 40
// rows over 65536 tokens of 8 heads 99 -> 95 us, 20 over 16384 of 32 74 -> 59, a
// prompt of 511 tokens 80 -> 69; with 16 rows half its columns would be empty.
// Their sixteen warps (two for the same 32 tokens, 16 rows each) took 293 us where
// eight with 32 rows each took 312 (48 rows over 65537 tokens, at the time).
// (Two CTAs of 32 do not fit the registers; 64 dimensions leave no room for 96
// rows of probabilities, 256 none for the value sums.)
template <uint32_t HD, uint32_t RT>
struct AttnGeo {
  static constexpr uint32_t kBlock = kv_block_bytes(HD);
  static constexpr uint32_t kQRow = HD < 128u ? HD : 128u;      // bytes of an operand row of K and Q
  static constexpr uint32_t kPanels = HD <= 128u ? 1u : HD / 128u;
  static constexpr uint32_t kQBytes = 3u * RT * HD;      // a job's query digits
  static constexpr uint32_t kCtas = HD <= 128u && RT == 16u ? 2u : 1u;  // per SM
  static constexpr uint32_t kCols = RT / 16u;           // a half's warps: four for every 16 rows
  static constexpr uint32_t kWarps = 8u * kCols;        // softmax warps
  static constexpr uint32_t kThreads = 32u * (kWarps + 2u);
  static constexpr uint32_t kStages = HD == 64u || RT == 32u ? 5u : 3u;  // blocks that shared memory holds
  static constexpr uint32_t kAcc = RT == 16u ? 64u : 128u;      // TMEM columns between accumulators (3 RT used)
  static constexpr uint32_t kTmem = HD <= 128u ? 4u * kAcc : 512u;  // scores of two tiles, values of two tiles
  static constexpr uint32_t kControl = RT == 16u ? 2048u : 4096u;  // barriers, scales, maxima; also what a 64-dimension value operand reads past its end
  static_assert(3u * RT * kKvPage <= kKvPage * HD, "a tile's probabilities take the place of its keys");
  static_assert(RT * HD * 4u <= kBlock, "a job's queries fit a stage");
  static constexpr uint32_t smem(uint32_t n_seq) {
    return kQBytes + kStages * kBlock + kControl + ((n_seq + 1u) * 4u + 15u) / 16u * 16u + 1024u;
  }
};

// A piece of a unit as the copy warp hands it to the others.
struct AttnJob {
  uint32_t tiles;           // 0: no further piece
  uint32_t rows, row0, unit, prefix;
  uint32_t left;            // tokens from the piece's first page on
  int32_t seen0;            // of which a sequence's first row sees so many (a prefix's rows: all)
};

struct AttnBars {
  uint64_t full[5], empty[5], q_ready, job_free, done;
  uint64_t s_full[2], s_free[2], p_ready[2], o_full[2], xmax[2][2];  // per half
  uint32_t tmem, ok[5];
  AttnJob job[2];
};

// CAUSAL: some unit's columns see different numbers of tokens (several rows of a sequence).  Without it the columns of
// a tile share one unit of the probabilities; a unit of their own costs them a product per pair of probabilities (seven
// sequences of up to 6 rows over 1537 tokens of 32 heads 26.5 us, 26.1 with a shared unit, a prompt of 511 tokens 68.8
// and 64.7; but a shared one let the value rows behind a row's last token coarsen its weights).
template <uint32_t HD, uint32_t RT, bool CAUSAL>
__global__ void __launch_bounds__((AttnGeo<HD, RT>::kThreads), (AttnGeo<HD, RT>::kCtas)) kv_attn_kernel(const KvAttnParams p) {
  using G = AttnGeo<HD, RT>;
  constexpr uint32_t S = G::kStages;
  constexpr uint32_t NC = 2;                                 // a warp's column chunks of 8
  constexpr uint32_t MH = HD <= 128u ? 1u : HD / 128u;       // value products of 128 dimensions
  extern __shared__ uint8_t attn_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(attn_smem_raw) + 1023u) & ~uintptr_t(1023));
  uint8_t* qop = smem;                                       // query digits
  uint8_t* stages = smem + G::kQBytes;
  uint8_t* control = stages + S * G::kBlock;
  AttnBars& bar = *reinterpret_cast<AttnBars*>(control);
  float* qs = reinterpret_cast<float*>(control + 512u);      // [2][RT] query scales
  float* xm = qs + 2u * RT;                                  // [half][2][4][RT] tile maxima per quarter
  uint32_t* xtop = reinterpret_cast<uint32_t*>(control + 384u);  // [half][2][cols][4] largest value scale per quarter
  uint8_t* ones = control + 512u + 72u * RT;
  static_assert(sizeof(AttnBars) <= 384u && 512u + 72u * RT + kAttnOnes <= G::kControl, "control words overlap");
  uint32_t* cum = reinterpret_cast<uint32_t*>(control + G::kControl);
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
  // the copy warp's first loads fly while the barriers are set up
  AttnSeq first{0, 0, 0};
  uint32_t prefix_len = 0, rows_end = 0;
  if (warp == G::kWarps) {
    if (p.prefix_len != nullptr) prefix_len = *p.prefix_len;
    rows_end = kv_row_start(p.rows, p.rows.n_seq);
    if (lane < p.rows.n_seq) first = attn_seq(p, lane);
  }
  if (tid == 0) {
    for (uint32_t s = 0; s < S; ++s) {
      mbar_init(&bar.full[s], 1);
      mbar_init(&bar.empty[s], 1);
    }
    mbar_init(&bar.q_ready, G::kWarps);
    mbar_init(&bar.job_free, G::kWarps);
    mbar_init(&bar.done, 1);
    for (uint32_t h = 0; h < 2u; ++h) {
      mbar_init(&bar.s_full[h], 1);
      mbar_init(&bar.s_free[h], 4u * G::kCols);
      mbar_init(&bar.p_ready[h], 4u * G::kCols);
      mbar_init(&bar.o_full[h], 1);
      for (uint32_t c = 0; c < G::kCols; ++c) mbar_init(&bar.xmax[h][c], 4);
    }
    fence_barrier_init();
  }
  if (warp == G::kWarps + 1u) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bar.tmem)),
                 "r"(G::kTmem)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid < kAttnOnes / 4u) {
    reinterpret_cast<uint32_t*>(ones)[tid] = 0xffffffffu;
    attn_fence_async();
  }
  attn_fence_before();
  __syncthreads();
  attn_fence_after();
  pdl_trigger();  // the joining kernel may start; it waits for this grid's completion
  const uint32_t tmem = bar.tmem;
  // TMEM: scores of half h at h kAcc, value sums at (2 + h MH + mh) kAcc

  if (warp == G::kWarps) {
    // ---- the line's layout: prefix units, then the sequences' (running work in cum) ----
    AttnPlan pl;
    pl.mine = first;
    pl.prefix = prefix_len < p.max_prefix ? prefix_len : p.max_prefix;
    if (p.prefix_few > 0) pl.prefix = 0;
    pl.rows_p = rows_end;
    pl.tp = attn_ceil(pl.prefix, kKvPage);
    pl.rgp = attn_ceil(pl.rows_p * p.group, RT);
    pl.wp = p.n_kv_head * pl.rgp * attn_cost(pl.tp);
    // (sequences that share rows -- a row0 that goes down -- could add up to more than the host's bound: the line ends there)
    const uint32_t most = 0x7fffffffu - pl.wp;
    uint32_t carry = 0;
    for (uint32_t i0 = 0; i0 < p.rows.n_seq; i0 += 32u) {
      uint32_t c = 0;
      const bool in = i0 + lane < p.rows.n_seq;
      if (in && p.seq_few == 0) c = attn_seq_work<RT>(p, i0 == 0 ? first : attn_seq(p, i0 + lane));
#pragma unroll
      for (uint32_t o = 1; o < 32u; o <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, c, o);
        if (lane >= o) c = min(c + t, most);
      }
      const uint32_t before = __shfl_up_sync(0xffffffffu, c, 1);
      if (in) cum[i0 + lane] = min(carry + (lane > 0 ? before : 0u), most);
      carry = min(carry + __shfl_sync(0xffffffffu, c, 31), most);
    }
    if (lane == 0) cum[p.rows.n_seq] = carry;
    __syncwarp();
    const uint32_t total = pl.wp + carry;
    pl.quantum = attn_ceil(total, gridDim.x);
    const uint64_t w_lo = (uint64_t)blockIdx.x * pl.quantum;
    uint32_t w = w_lo < total ? (uint32_t)w_lo : total;
    const uint32_t w1 = w_lo + pl.quantum < total ? (uint32_t)(w_lo + pl.quantum) : total;
    // ---- jobs: a stage with the piece's queries, then one per page ----
    uint32_t x = 0, nj = 0;  // stages used; jobs
    bool live = true;
    auto stage_free = [&]() {  // lane 0: stage x % S may be filled
      if (x >= S && !attn_wait(&bar.empty[x % S], (x / S - 1u) & 1u)) {
        report(p.err, EOS_DEVERR_WAIT_EMPTY);
        return false;
      }
      return true;
    };
    auto agree = [&](bool v) { return __shfl_sync(0xffffffffu, v ? 1u : 0u, 0) != 0u; };
    for (bool more = true; more && live; ++nj) {
      AttnSeg s{};
      while (w < w1) {  // the next piece that holds a tile
        s = attn_segment<RT>(p, pl, cum, w, w1);
        w += s.step;
        if (s.tiles > 0) break;
      }
      more = s.tiles > 0;
      const bool is_prefix = s.seq == p.rows.n_seq;
      const uint32_t* table = is_prefix ? p.prefix_table : p.table + (size_t)s.seq * p.table_stride;
      const uint8_t* pool = is_prefix ? p.prefix_pages : p.pages;
      const uint32_t pool_pages = is_prefix ? p.prefix_n_pages : p.n_pages;
      uint32_t mine = lane < s.tiles ? table[s.tile0 + lane] : 0u;
      if (lane == 0) {
        live = stage_free();
        if (live && nj > 0 && !attn_wait(&bar.job_free, (nj - 1u) & 1u)) {
          report(p.err, EOS_DEVERR_WAIT_EMPTY);
          live = false;
        }
        if (live) {
          const int32_t t0 = (int32_t)(s.tile0 * kKvPage);
          bar.job[nj & 1u] = AttnJob{s.tiles, s.rows, s.row0, s.unit, is_prefix ? 1u : 0u, s.len - (uint32_t)t0,
                                     is_prefix ? 0x40000000 : (int32_t)s.len - (int32_t)s.n + 1 - t0};
          if (more) mbar_arrive_expect_tx(&bar.full[x % S], s.rows * HD * 4u);
          else mbar_arrive(&bar.full[x % S]);
        }
      }
      live = agree(live);
      if (!live) break;
      if (more && lane < s.rows) {
        const uint32_t fr = s.row0 + lane, xr = attn_div(fr, p.by_group);
        attn_bulk(smem_u32(stages + (x % S) * G::kBlock + lane * HD * 4u),
                  p.q + (size_t)(s.base_row + xr) * p.q_stride + (size_t)(s.head * p.group + fr - xr * p.group) * HD,
                  HD * 4u, &bar.full[x % S]);
      }
      ++x;
      for (uint32_t j = 0; j < s.tiles; ++j) {
        if (j > 0 && j % 32u == 0) mine = j + lane < s.tiles ? table[s.tile0 + j + lane] : 0u;
        const uint32_t page = __shfl_sync(0xffffffffu, mine, j % 32u);
        if (lane == 0) {
          const uint32_t st = x % S;
          live = stage_free();
          if (!live) {
          } else if (page >= pool_pages) {
            report(p.err, EOS_DEVERR_RANGE);
            bar.ok[st] = 0u;
            mbar_arrive(&bar.full[st]);
          } else {
            bar.ok[st] = 1u;
            const uint8_t* src = pool + ((size_t)page * p.n_kv_head + s.head) * G::kBlock;
            const uint32_t dst = smem_u32(stages + st * G::kBlock);
            const uint32_t left = s.len - (s.tile0 + j) * kKvPage;
            if (left >= kKvPage) {
              mbar_arrive_expect_tx(&bar.full[st], G::kBlock);
            } else {  // the rows, quarters and scales that hold tokens
              const uint32_t kr = (left + 7u) / 8u * 8u * G::kQRow, nq = attn_ceil(left, kKvQuarter);
              const uint32_t vb = nq * HD * kKvQuarter, sb = nq * 256u;
              mbar_arrive_expect_tx(&bar.full[st], G::kPanels * kr + vb + sb);
              for (uint32_t pn = 0; pn < G::kPanels; ++pn)
                attn_bulk(dst + pn * kKvPage * 128u, src + pn * kKvPage * 128u, kr, &bar.full[st]);
              attn_bulk(dst + kKvPage * HD, src + kKvPage * HD, vb, &bar.full[st]);
              attn_bulk(dst + 2u * kKvPage * HD, src + 2u * kKvPage * HD, sb, &bar.full[st]);
            }
          }
        }
        live = agree(live);
        if (!live) break;
        // a whole page as eight copies side by side
        if (page < pool_pages && s.len - (s.tile0 + j) * kKvPage >= kKvPage && lane < 8u)
          attn_bulk(smem_u32(stages + (x % S) * G::kBlock) + lane * (G::kBlock / 8u),
                    pool + ((size_t)page * p.n_kv_head + s.head) * G::kBlock + lane * (G::kBlock / 8u), G::kBlock / 8u,
                    &bar.full[x % S]);
        ++x;
      }
    }
    if (blockIdx.x == 0) {  // the layout for the joining kernel; lengths and rows beyond their bounds
      if (lane == 0) {
        p.plan[0] = pl.quantum;
        p.plan[1] = pl.tp;
        p.plan[2] = pl.rgp;
        p.plan[3] = pl.wp;
        if (prefix_len > p.max_prefix) report(p.err, EOS_DEVERR_RANGE);
      }
      for (uint32_t i = lane; i <= p.rows.n_seq; i += 32u) {
        p.plan[4u + i] = cum[i];
        if (i < p.rows.n_seq && (p.seq_len[i] > p.max_len || attn_seq(p, i).n > p.max_rows))
          report(p.err, EOS_DEVERR_RANGE);
      }
    }
    // never leave copies in flight: every stage's last use has landed
    if (lane == 0)
      for (uint32_t y = x > S ? x - S : 0u; y < x; ++y)
        if (!attn_wait(&bar.full[y % S], (y / S) & 1u)) report(p.err, EOS_DEVERR_DRAIN);
  } else if (warp == G::kWarps + 1u) {
    // ---- products: tile j of a job belongs to half j % 2 ----
    if (lane == 0) {
      bool live = true;
      const uint64_t ones_desc = attn_ones_desc(smem_u32(ones));
      uint32_t x = 0;               // stages used before the job
      uint32_t ns0 = 0, ns1 = 0;    // score products issued, per half
      uint32_t nv0 = 0, nv1 = 0;    // value products issued
      for (uint32_t nj = 0; live; ++nj) {
        if (!attn_wait(&bar.q_ready, nj & 1u)) {
          report(p.err, EOS_DEVERR_WAIT_ACT);
          break;
        }
        const uint32_t tiles = bar.job[nj & 1u].tiles;
        if (tiles == 0) break;
        attn_fence_after();
        mbar_arrive(&bar.empty[x % S]);  // the queries have been read
        uint32_t js = 0, jv = 0, jo0 = 0, jo1 = 1, polls = 0;  // next score tile; values done; next value tile per half
        uint64_t t0 = 0;
        while (jv < tiles) {
          bool moved = false;
          {
            const uint32_t h = js & 1u, y = x + 1u + js;
            if (js < tiles && mbar_test(&bar.full[y % S], (y / S) & 1u) &&
                ((h ? ns1 : ns0) == 0 || mbar_test(&bar.s_free[h], ((h ? ns1 : ns0) - 1u) & 1u))) {
              attn_fence_after();
              const uint32_t ka = smem_u32(stages + (y % S) * G::kBlock), qa = smem_u32(qop);
              constexpr uint32_t id = attn_idesc(true, true, 3u * RT);
#pragma unroll
              for (uint32_t b = 0; b < attn_score_biases(HD); ++b)
                attn_mma(tmem + h * G::kAcc, ones_desc, ones_desc, attn_idesc(false, false, 3u * RT), b);
#pragma unroll
              for (uint32_t ks = 0; ks < HD / 32u; ++ks) {
                const uint32_t panel = ks / 4u, off = (ks % 4u) * 32u;
                attn_mma(tmem + h * G::kAcc, attn_desc(ka + panel * kKvPage * 128u + off, G::kQRow),
                         attn_desc(qa + panel * 3u * RT * 128u + off, G::kQRow), id, 1u);
              }
              attn_commit(&bar.s_full[h]);
              ++(h ? ns1 : ns0);
              ++js;
              moved = true;
            }
          }
#pragma unroll
          for (uint32_t h = 0; h < 2u; ++h) {
            uint32_t& jo = h ? jo1 : jo0;
            uint32_t& nv = h ? nv1 : nv0;
            if (jo < js && mbar_test(&bar.p_ready[h], nv & 1u)) {
              attn_fence_after();
              const uint32_t st = (x + 1u + jo) % S;
              const uint32_t sa = smem_u32(stages + st * G::kBlock);
              constexpr uint32_t id = attn_idesc(true, false, 3u * RT), bias = attn_idesc(false, false, 3u * RT);
#pragma unroll
              for (uint32_t mh = 0; mh < MH; ++mh) {
                const uint32_t acc = tmem + G::kAcc * (2u + h * MH + mh);
                attn_mma(acc, ones_desc, ones_desc, bias, 0u);
                attn_mma(acc, ones_desc, ones_desc, bias, 1u);
#pragma unroll
                for (uint32_t qd = 0; qd < 4u; ++qd)
                  attn_mma(acc, attn_desc(sa + kKvPage * HD + qd * HD * kKvQuarter + mh * 128u * kKvQuarter, 32u),
                           attn_desc(sa + qd * 32u, 128u), id, 1u);
              }
              attn_commit(&bar.o_full[h]);
              attn_commit(&bar.empty[st]);
              ++nv;
              jo += 2u;
              ++jv;
              moved = true;
            }
          }
          if (moved) {
            polls = 0;
            t0 = 0;
          } else if (__nanosleep(20), ++polls % 256u == 0) {  // bounded, like every wait
            const uint64_t now = global_timer_ns();
            if (t0 == 0) t0 = now;
            if (now - t0 > EOS_WAIT_LIMIT_NS) {
              report(p.err, EOS_DEVERR_WAIT_FULL);
              live = false;
              break;
            }
          }
        }
        x += 1u + tiles;
      }
      // TMEM is freed, and shared memory left, only after every product issued has completed
      attn_commit(&bar.done);
      if (!attn_wait(&bar.done, 0)) report(p.err, EOS_DEVERR_DRAIN);
    }
  } else {
    // ---- softmax and folding: warps 4 h + quarter work on the tiles of half h ----
    const uint32_t quad = warp & 3u, half = (warp >> 2) & 1u, grp = G::kCols == 1u ? 0u : warp >> 3, g = lane >> 2, cq = lane & 3u;
    const uint32_t c0 = 16u * grp;  // the warp's first column
    uint32_t x = 0;               // stages used before the job
    uint32_t n_own = 0, n_other = 0;  // tiles of this half and of the other before the job
    // job n's queries (in stage y) as three signed digits each, rows warp, warp + 8, ...
    auto prepare = [&](uint32_t n, uint32_t y) {
      if (!__all_sync(0xffffffffu, attn_wait(&bar.full[y % S], (y / S) & 1u))) return false;
      const uint32_t rows = bar.job[n & 1u].rows;
      const float* raw = reinterpret_cast<const float*>(stages + (y % S) * G::kBlock);
      if (bar.job[n & 1u].tiles > 0) {
#pragma unroll
        for (uint32_t r = warp; r < RT; r += G::kWarps) {
          float scale = 0.0f;
          if (r < rows) {
            float4 v[G::kPanels];
            uint32_t amax = 0;
#pragma unroll
            for (uint32_t pn = 0; pn < G::kPanels; ++pn) {
              v[pn] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
              if (HD >= 128u || lane < HD / 4u) v[pn] = *reinterpret_cast<const float4*>(raw + r * HD + pn * 128u + lane * 4u);
              amax = attn_absmax(amax, v[pn]);
            }
            amax = __reduce_max_sync(0xffffffffu, amax);
            const AttnQScale q = attn_query_scale(amax, p.scale_log2);
            // (times 2^17 of the scores' 2^22)
            scale = q.finite ? fminf(q.scale * 131072.0f, 3e38f) : NAN;
#pragma unroll
            for (uint32_t pn = 0; pn < G::kPanels; ++pn) {
              uint32_t d[3];
              attn_query_digits(v[pn], q, d);
              if (HD >= 128u || lane < HD / 4u) {
#pragma unroll
                for (uint32_t e = 0; e < 3u; ++e) {
                  const uint32_t row = e * RT + r;
                  const uint32_t sw = G::kQRow == 128u ? (row & 7u) : ((row >> 1) & 3u);
                  *reinterpret_cast<uint32_t*>(qop + pn * 3u * RT * 128u + row * G::kQRow +
                                               (((lane >> 2) ^ sw) << 4) + (lane & 3u) * 4u) = d[e];
                }
              }
            }
          }
          if (lane == 0) qs[(n & 1u) * RT + r] = scale;
        }
      }
      attn_fence_async();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bar.job_free);
        mbar_arrive(&bar.q_ready);
      }
      return true;
    };
    bool live = prepare(0, 0);
    for (uint32_t nj = 0; live; ++nj) {
      live = __all_sync(0xffffffffu, attn_wait(&bar.q_ready, nj & 1u)) != 0;
      if (!live) break;
      const AttnJob s = bar.job[nj & 1u];
      if (s.tiles == 0) break;
      const uint32_t nact = s.rows > c0 ? (s.rows - c0 + 7u) / 8u : 0u;  // chunks of 8 columns in use
      // this thread's columns c0 + 8 y + 2 cq + {0, 1}
      float2 m[NC], l[NC], f[NC], o[NC][MH][4];
#pragma unroll
      for (uint32_t y = 0; y < NC; ++y) {
        m[y] = attn_two(kAttnLow);
        l[y] = attn_two(0.0f);
        f[y] = attn_two(1.0f);
#pragma unroll
        for (uint32_t mh = 0; mh < MH; ++mh)
#pragma unroll
          for (uint32_t j = 0; j < 4u; ++j) o[y][mh][j] = attn_two(0.0f);
      }
      // tokens from the piece's first page on that column `col` sees; all columns see those below `common`
      auto limit = [&](uint32_t col) -> int32_t {
        const AttnJob& job = bar.job[nj & 1u];
        return min(job.seen0 + (int32_t)attn_div(job.row0 + col, p.by_group), (int32_t)job.left);
      };
      const int32_t common = limit(0), most = limit(s.rows - 1u);  // .. and none more than `most`
      float2 fold[NC];         // the last tile's probability unit, relative to the running reference
      uint32_t it = n_own;     // tiles of this half so far
      // o = o f + fold * (value product of the tile before)
      auto fold_tile = [&]() {
        if (!__all_sync(0xffffffffu, attn_wait(&bar.o_full[half], (it - 1u) & 1u))) return false;
        attn_fence_after();
        if (HD >= 128u || quad * 32u < HD) {
#pragma unroll
          for (uint32_t mh = 0; mh < MH; ++mh)
            attn_sums<RT>(tmem + G::kAcc * (2u + half * MH + mh) + ((quad * 32u) << 16) + c0, nact,
                          [&](uint32_t y, uint32_t j, const uint32_t* d0, const uint32_t* d1, const uint32_t* d2) {
                            o[y][mh][j] = attn_fma2(attn_join<2u * kAttnBias>(d0, d1, d2), fold[y],
                                                    attn_mul2(o[y][mh][j], f[y]));
                          });
        }
        attn_fence_before();
        return true;
      };
      for (uint32_t t = half; t < s.tiles && live; t += 2u) {
        const uint32_t pos = x + 1u + t, st = pos % S;
        // the scores, and (already complete) the page, whose scales are read here
        live = __all_sync(0xffffffffu, attn_wait(&bar.s_full[half], it & 1u) &&
                                           attn_wait(&bar.full[st], (pos / S) & 1u)) != 0;
        if (!live) break;
        attn_fence_after();
        const uint32_t tok0 = t * kKvPage;
        const uint8_t* sc = stages + st * G::kBlock + 2u * kKvPage * HD;
        const uint32_t avail = bar.ok[st] ? s.left - tok0 : 0u;  // tokens of the tile (may exceed a page)
        // the scales of quarter quad, token `lane`; this thread's four tokens are g + 8 j
        uint32_t vbits = *reinterpret_cast<const uint32_t*>(sc + quad * 256u + 128u + lane * 4u);
        uint32_t vown;  // .. its value scale; vbits: the same if every column sees the token
        float ks[4];
        // the tile's tokens, those that every column sees and those that one sees; between the two (a cut tile) a
        // column's largest value scale is its own, so that no row's rounding depends on tokens behind its last
        const int32_t held = (int32_t)min(avail, kKvPage), least = max(common - (int32_t)tok0, 0),
                      some = min(most - (int32_t)tok0, held);
        const bool cut = CAUSAL && least < some;
        {
          const bool in = quad * 32u + lane < avail, sound = vbits < 0x7f800000u;
          const float kv = *reinterpret_cast<const float*>(sc + quad * 256u + lane * 4u);
          const float k1 = in ? (sound ? 32.0f * kv : NAN) : 0.0f;      // a NaN or infinite value row: NaN score
          vbits = in && sound ? vbits : 0u;
          vown = vbits;
          if constexpr (CAUSAL)
            if (cut && (int32_t)(quad * 32u + lane) >= least) vbits = 0u;
#pragma unroll
          for (uint32_t j = 0; j < 4u; ++j) ks[j] = __shfl_sync(0xffffffffu, k1, g + 8u * j);
        }
        uint32_t* xt = xtop + ((half * 2u + (it & 1u)) * G::kCols + grp) * 4u;
        {
          const uint32_t top = __reduce_max_sync(0xffffffffu, vbits);
          if (lane == 0) xt[quad] = top;
        }
        const bool whole = avail >= kKvPage && (int32_t)(tok0 + kKvPage) <= common;  // nothing to mask
        float* xmt = xm + (half * 2u + (it & 1u)) * 4u * RT + c0 + 2u * cq;
        float2 sv[NC][4];
        attn_sums<RT>(tmem + half * G::kAcc + ((quad * 32u) << 16) + c0, nact,
                      [&](uint32_t y, uint32_t j, const uint32_t* d0, const uint32_t* d1, const uint32_t* d2) {
                        sv[y][j] = attn_mul2(attn_join<attn_score_biases(HD) * kAttnBias>(d0, d1, d2), attn_two(ks[j]));
                      });
        float2 mx[NC];
#pragma unroll
        for (uint32_t y = 0; y < NC; ++y) {
          mx[y] = attn_two(-INFINITY);
          if (y >= nact) continue;  // warp-uniform
          if (!whole) {
            const uint32_t col = c0 + 8u * y + 2u * cq;
            const int32_t lim0 = limit(col), lim1 = limit(col + 1u);
#pragma unroll
            for (uint32_t j = 0; j < 4u; ++j) {
              const uint32_t tok = quad * 32u + g + 8u * j;
              if (tok >= avail || (int32_t)(tok0 + tok) >= lim0) sv[y][j].x = -INFINITY;
              if (tok >= avail || (int32_t)(tok0 + tok) >= lim1) sv[y][j].y = -INFINITY;
            }
          }
          mx[y] = make_float2(fmaxf(fmaxf(sv[y][0].x, sv[y][1].x), fmaxf(sv[y][2].x, sv[y][3].x)),
                              fmaxf(fmaxf(sv[y][0].y, sv[y][1].y), fmaxf(sv[y][2].y, sv[y][3].y)));
        }
        // the four columns' maxima over the eight lanes that share them: each step
        // halves what a lane still holds, bit 2 of the lane its chunk, bit 3 its column
        {
          const bool hi = (lane & 4u) != 0u, odd = (lane & 8u) != 0u;
          const float2 keep = hi ? mx[1] : mx[0], send = hi ? mx[0] : mx[1];
          const float kx = fmaxf(keep.x, __shfl_xor_sync(0xffffffffu, send.x, 4));
          const float ky = fmaxf(keep.y, __shfl_xor_sync(0xffffffffu, send.y, 4));
          float k1 = fmaxf(odd ? ky : kx, __shfl_xor_sync(0xffffffffu, odd ? kx : ky, 8));
          k1 = fmaxf(k1, __shfl_xor_sync(0xffffffffu, k1, 16));
          if (lane < 16u) xmt[quad * RT + (lane & 4u) * 2u + ((lane >> 3) & 1u)] = k1;
        }
        attn_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bar.s_free[half]);
          mbar_arrive(&bar.xmax[half][grp]);
        }
        uint32_t tail[NC][2] = {};  // a cut tile: the largest value scale from `least` on that a column sees
        if constexpr (CAUSAL)
          if (cut) {  // lane l: the largest scale of the tokens from `least` to l behind it (a group's rows are at most 32)
            const uint32_t tok = (uint32_t)least + lane;
            uint32_t v = 0;
            if ((int32_t)tok < some) v = *reinterpret_cast<const uint32_t*>(sc + (tok >> 5) * 256u + 128u + (tok & 31u) * 4u);
            if (v >= 0x7f800000u) v = 0u;
#pragma unroll
            for (uint32_t o = 1; o < 32u; o <<= 1) v = max(v, __shfl_up_sync(0xffffffffu, v, o));
#pragma unroll
            for (uint32_t y = 0; y < NC; ++y)
#pragma unroll
              for (uint32_t z = 0; z < 2u; ++z) {
                const int32_t n = limit(c0 + 8u * y + 2u * cq + z) - (int32_t)tok0 - least;
                const uint32_t w = __shfl_sync(0xffffffffu, v, min(max(n - 1, 0), 31));
                tail[y][z] = n > 0 ? w : 0u;
              }
          }
        if (t > half) live = fold_tile();
        if (live) live = __all_sync(0xffffffffu, attn_wait(&bar.xmax[half][grp], it & 1u)) != 0;
        if (!live) break;
        // unit of the probabilities: from the largest value scale that a column sees in the tile (`top`), one for all
        // columns unless the tile is cut
        float top[NC][2], inv = 0.0f, vw[4];
        {
          const uint4 t4 = *reinterpret_cast<const uint4*>(xt);
          const float all = attn_weight_top(__uint_as_float(max(max(t4.x, t4.y), max(t4.z, t4.w))));
          if constexpr (!CAUSAL) inv = attn_weight_scale(all);
          const float v1 = CAUSAL ? __uint_as_float(vown) : __uint_as_float(vbits) * inv;
#pragma unroll
          for (uint32_t j = 0; j < 4u; ++j) vw[j] = __shfl_sync(0xffffffffu, v1, g + 8u * j);
#pragma unroll
          for (uint32_t y = 0; y < NC; ++y)
#pragma unroll
            for (uint32_t z = 0; z < 2u; ++z)
              top[y][z] = CAUSAL ? fmaxf(__uint_as_float(tail[y][z]), all) : all;
        }
        uint8_t* pop = stages + st * G::kBlock;  // the probabilities take the place of the keys
#pragma unroll
        for (uint32_t y = 0; y < NC; ++y) {
          if (y >= nact) break;  // warp-uniform
          const uint32_t col = c0 + 8u * y + 2u * cq;
          const float2 qsc = *reinterpret_cast<const float2*>(qs + (nj & 1u) * RT + col);
          const float2 m0 = *reinterpret_cast<const float2*>(xmt + 8u * y),
                       m1 = *reinterpret_cast<const float2*>(xmt + RT + 8u * y),
                       m2 = *reinterpret_cast<const float2*>(xmt + 2u * RT + 8u * y),
                       m3 = *reinterpret_cast<const float2*>(xmt + 3u * RT + 8u * y);
          // the tile's own reference, rounded up so that no probability exceeds 1
          // (its integers are relative to it: their rounding fades with the tile)
          const float t0 = fmaxf(fmaxf(m0.x, m1.x), fmaxf(m2.x, m3.x)), t1 = fmaxf(fmaxf(m0.y, m1.y), fmaxf(m2.y, m3.y));
          const float2 ref = make_float2(fmaxf(__fmul_ru(t0, qsc.x), kAttnLow), fmaxf(__fmul_ru(t1, qsc.y), kAttnLow));
          // z = (score - t) c + (t c - ref): the reference's rounding is a common factor as long as it is one
          const float2 t = make_float2(-fmaxf(t0, kAttnLow), -fmaxf(t1, kAttnLow));
          const float d0 = __fmaf_rn(-t.x, qsc.x, -ref.x), d1 = __fmaf_rn(-t.y, qsc.y, -ref.y);
          const float2 dl = make_float2(d0 > -0.5f ? d0 : 0.0f, d1 > -0.5f ? d1 : 0.0f);
          const float2 nm = make_float2(fmaxf(ref.x, m[y].x), fmaxf(ref.y, m[y].y));
          f[y] = make_float2(attn_ex2(m[y].x - nm.x), attn_ex2(m[y].y - nm.y));
          const float2 share = make_float2(attn_ex2(ref.x - nm.x), attn_ex2(ref.y - nm.y));
          const float2 un = make_float2(attn_weight_unit(top[y][0]), attn_weight_unit(top[y][1]));
          const float2 up = make_float2(attn_weight_scale(top[y][0]), attn_weight_scale(top[y][1]));
          fold[y] = attn_mul2(share, un);
          m[y] = nm;
          uint32_t b0[4], b1[4], d[3];
          float2 ls = attn_two(0.0f);
#pragma unroll
          for (uint32_t j = 0; j < 4u; ++j) {
            const float2 z = attn_fma2(attn_add2(sv[y][j], t), qsc, dl);
            const float2 e = make_float2(attn_ex2(z.x), attn_ex2(z.y));
            ls = attn_add2(ls, e);
            // (a hidden token's probability, 0, takes the unit first, so that the product is 0 too)
            const float2 w = attn_fma2(CAUSAL ? attn_mul2(e, up) : e, attn_two(vw[j]), attn_two(8388608.0f));
            b0[j] = __float_as_uint(w.x);
            b1[j] = __float_as_uint(w.y);
          }
          l[y] = attn_fma2(l[y], f[y], attn_mul2(ls, share));
          // row e RT + col of digit e, this thread's four tokens: one word
          uint8_t* at = pop + (g & 3u) * 4u;
          const uint32_t chunk = 2u * quad + (g >> 2);
          attn_digits(b0, d);
#pragma unroll
          for (uint32_t e = 0; e < 3u; ++e)
            *reinterpret_cast<uint32_t*>(at + (e * RT + col) * kKvPage + ((chunk ^ (col & 7u)) << 4)) = d[e];
          attn_digits(b1, d);
#pragma unroll
          for (uint32_t e = 0; e < 3u; ++e)
            *reinterpret_cast<uint32_t*>(at + (e * RT + col + 1u) * kKvPage + ((chunk ^ ((col + 1u) & 7u)) << 4)) = d[e];
        }
        ++it;
        attn_fence_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.p_ready[half]);
      }
      // the next job's queries, once both halves' score products have read
      // this one's; then this half's last value product
      const bool some = s.tiles > half;
      const uint32_t others = (s.tiles + half) / 2u;
      n_own += s.tiles - others;
      n_other += others;
      x += 1u + s.tiles;
      if (live && others > 0)
        live = __all_sync(0xffffffffu, attn_wait(&bar.s_full[half ^ 1u], (n_other - 1u) & 1u)) != 0;
      if (live) live = prepare(nj + 1u, x);
      if (live && some) live = fold_tile();
      if (!live) break;
      // the partial of this piece and half
      const size_t id = 2u * (size_t)(s.unit + blockIdx.x) + half;
      const uint32_t cap = s.prefix ? p.prefix_cap : p.seq_cap;
      float* po = (s.prefix ? p.po : p.so) + id * cap * HD;
      float* pml = (s.prefix ? p.pml : p.sml) + id * cap * kAttnMl;
#pragma unroll
      for (uint32_t y = 0; y < NC; ++y) {
        if (y >= nact) break;  // warp-uniform
        float2 ls = l[y];
#pragma unroll
        for (uint32_t o2 = 4; o2 < 32u; o2 <<= 1) {
          ls.x += __shfl_xor_sync(0xffffffffu, ls.x, o2);
          ls.y += __shfl_xor_sync(0xffffffffu, ls.y, o2);
        }
#pragma unroll
        for (uint32_t z = 0; z < 2u; ++z) {
          const uint32_t col = c0 + 8u * y + 2u * cq + z;
          if (col >= s.rows) continue;
          if (g == 0) {
            pml[col * kAttnMl + 4u + quad] = z ? ls.y : ls.x;
            if (quad == 0) pml[col * kAttnMl] = z ? m[y].y : m[y].x;
          }
          if (some && (HD >= 128u || quad * 32u < HD)) {
#pragma unroll
            for (uint32_t mh = 0; mh < MH; ++mh)
#pragma unroll
              for (uint32_t j = 0; j < 4u; ++j)
                po[(size_t)col * HD + mh * 128u + quad * 32u + g + 8u * j] =
                    256.0f * (z ? o[y][mh][j].y : o[y][mh][j].x);
          }
        }
      }
    }
    if (!live) report(p.err, EOS_DEVERR_WAIT_ACT);
  }
  attn_fence_before();
  __syncthreads();
  pdl_wait();  // the few-rows kernels before this one, see attn_line
  if (warp == G::kWarps + 1u)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(G::kTmem) : "memory");
}

// Joins a row's partials: one warp per (row, head), lane l holding HD / 32
// neighbouring elements.  Weights are relative to the largest maximum; the
// order of the sums is the line's, so results do not depend on timing.
template <uint32_t HD, bool LOOK>
__global__ void __launch_bounds__(64) kv_attn_join_kernel(const KvAttnParams p) {
  constexpr uint32_t E = HD / 32u;
  const uint32_t RT = p.rt;
  const uint32_t lane = threadIdx.x & 31u;
  const uint64_t x = (uint64_t)blockIdx.x * 2u + (threadIdx.x >> 5);
  if constexpr (LOOK)  // lengths and rows beyond their bounds, where no kernel before this one has looked at them
    if (x == 0)
      for (uint32_t i = lane; i < p.rows.n_seq; i += 32u)
        if (p.seq_len[i] > p.max_len || attn_seq(p, i).n > p.max_rows) report(p.err, EOS_DEVERR_RANGE);
  if (x >= (uint64_t)p.rows.n_rows * p.n_head) return;  // warp-uniform
  const uint32_t hw = attn_div((uint32_t)x, p.by_group);  // row * n_kv_head + kv head
  const uint32_t r = attn_div(hw, p.by_kv_head), g = hw - r * p.n_kv_head, hh = (uint32_t)x - hw * p.group;
  const uint32_t h = g * p.group + hh;
  // the row's sequence and the inputs' words: read while the attention still runs
  uint32_t i = 0, start, end;
  if (p.rows.row0 == nullptr) {
    i = r / p.rows.per_seq;
    start = kv_row_start(p.rows, i);
    end = kv_row_start(p.rows, i + 1u);
  } else {  // sequences that start at or before the row, 32 at a time
    uint32_t n = 0, c, first = 0, last = 0;
    for (;; n += 32u) {
      const bool in = n + lane <= p.rows.n_seq;
      first = in ? kv_row_start(p.rows, n + lane) : 0u;
      c = __popc(__ballot_sync(0xffffffffu, in && first <= r));
      if (c < 32u) break;
      last = __shfl_sync(0xffffffffu, first, 31);
    }
    i = n + c;
    if (i == 0 || i > p.rows.n_seq) return;  // before the first sequence or behind the last
    --i;
    start = c > 0 ? __shfl_sync(0xffffffffu, first, c - 1u) : last;
    end = __shfl_sync(0xffffffffu, first, c);
  }
  const uint32_t t = r - start;
  if (r < start || r >= end) return;  // (a row0 that goes down)
  if (t >= p.max_rows) return;        // (reported)
  const uint32_t seq_len = p.seq_len[i];
  // no token: 0, also for a query that is not finite
  const bool none = (int32_t)min(seq_len, p.max_len) - (int32_t)(end - r) + 1 <= 0 &&
                    (p.max_prefix == 0 || *p.prefix_len == 0);
  pdl_wait();
  // ids of the row's partials: [first, last] of the prefix and of its sequence
  struct Part {
    const float *o, *ml;
    uint32_t n, o_step, ml_step;
  } part[2] = {};
  // on the line: the CTAs that hold tiles of the unit, two halves each
  auto line = [&](Part& a, const float* o, const float* ml, uint32_t cap, uint32_t unit, uint32_t w, uint32_t tiles,
                  uint32_t row) {
    if (tiles == 0) return;
    const uint32_t quantum = max(__ldcg(p.plan), 1u);
    const uint32_t c0 = min((w + kAttnStart) / quantum, kAttnMaxCtas - 1u),
                   c1 = min((w + kAttnStart + tiles - 1u) / quantum, kAttnMaxCtas - 1u);
    if (c1 < c0) return;
    a.n = 2u * (c1 - c0 + 1u);
    a.o_step = cap * HD;
    a.ml_step = cap * kAttnMl;
    a.o = o + ((size_t)2u * (unit + c0) * cap + row) * HD;
    a.ml = ml + ((size_t)2u * (unit + c0) * cap + row) * kAttnMl;
  };
  // the few-rows kernel's clusters
  auto few = [&](Part& a, const float* o, const float* ml, uint32_t cap, uint32_t unit, uint32_t n, uint32_t row) {
    a.n = n;
    a.o_step = cap * HD;
    a.ml_step = cap * kAttnMl;
    a.o = o + ((size_t)unit * n * cap + row) * HD;
    a.ml = ml + ((size_t)unit * n * cap + row) * kAttnMl;
  };
  if (p.max_prefix > 0) {
    const uint32_t fr = r * p.group + hh;
    if (p.prefix_few > 0) {
      few(part[0], p.po, p.pml, p.prefix_cap, g, p.prefix_few, fr);
    } else {
      const uint32_t tp = __ldcg(p.plan + 1), rgp = __ldcg(p.plan + 2), rg = fr / RT, unit = g * rgp + rg;
      line(part[0], p.po, p.pml, p.prefix_cap, unit, unit * attn_cost(tp), tp, fr % RT);
    }
  }
  {
    const uint32_t len = seq_len < p.max_len ? seq_len : p.max_len;
    const uint32_t fr = t * p.group + hh, tiles = attn_ceil(len, kKvPage);
    if (p.seq_few > 0) {
      few(part[1], p.so, p.sml, p.seq_cap, i * p.n_kv_head + g, p.seq_few, fr);
    } else {
      const uint32_t rg = fr / RT, u = rg * p.n_kv_head + g;
      line(part[1], p.so, p.sml, p.seq_cap, i * p.seq_groups * p.n_kv_head + u,
           __ldcg(p.plan + 3) + __ldcg(p.plan + 4u + i) + u * attn_cost(tiles), tiles, fr % RT);
    }
  }
  // partial k of the row; lane k looks after its weight
  const uint32_t n = none ? 0u : part[0].n + part[1].n;
  auto ml_of = [&](uint32_t k) {
    return k < part[0].n ? part[0].ml + (size_t)k * part[0].ml_step
                         : part[1].ml + (size_t)(k - part[0].n) * part[1].ml_step;
  };
  auto o_of = [&](uint32_t k) {
    return (k < part[0].n ? part[0].o + (size_t)k * part[0].o_step
                          : part[1].o + (size_t)(k - part[0].n) * part[1].o_step) + lane * E;
  };
  float top = -INFINITY;
  for (uint32_t k = lane; k < n; k += 32u) top = fmaxf(top, __ldcg(ml_of(k)));
#pragma unroll
  for (uint32_t o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float mu = top == -INFINITY ? 0.0f : top;
  float l = 0.0f, acc[E];
#pragma unroll
  for (uint32_t e = 0; e < E; ++e) acc[e] = 0.0f;
  for (uint32_t k0 = 0; k0 < n; k0 += 32u) {
    float f = 0.0f, lk = 0.0f;
    if (k0 + lane < n) {
      const float4 ls = __ldcg(reinterpret_cast<const float4*>(ml_of(k0 + lane)) + 1);
      lk = (ls.x + ls.y) + (ls.z + ls.w);
      f = attn_ex2(__ldcg(ml_of(k0 + lane)) - mu);
      if (lk == 0.0f) f = 0.0f;  // no tile, or no visible token: its output may be unwritten
    }
    float lw = f * lk;
#pragma unroll
    for (uint32_t o = 16; o > 0; o >>= 1) lw += __shfl_xor_sync(0xffffffffu, lw, o);
    l += lw;
    const uint32_t m = n - k0 < 32u ? n - k0 : 32u;
    for (uint32_t b = 0; b < m; b += 8u) {  // eight partials' loads in flight
      float v[8][E];
#pragma unroll
      for (uint32_t z = 0; z < 8u; ++z)
        if (b + z < m) {
          const float* src = o_of(k0 + b + z);
#pragma unroll
          for (uint32_t e = 0; e < E; ++e) v[z][e] = __ldcg(src + e);
        }
#pragma unroll
      for (uint32_t z = 0; z < 8u; ++z) {
        const float w = __shfl_sync(0xffffffffu, f, b + z);
        if (b + z < m && w != 0.0f)
#pragma unroll
          for (uint32_t e = 0; e < E; ++e) acc[e] = fmaf(w, v[z][e], acc[e]);
      }
    }
  }
  const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
  float* dst = p.out + (size_t)r * p.out_stride + (size_t)h * HD + lane * E;
#pragma unroll
  for (uint32_t e = 0; e < E; ++e) dst[e] = acc[e] * inv;
}

namespace {

// How a call runs: the prefix and the sequences each on the tensor cores' line
// or, with at most kFewRows rows to a unit, on clusters of CTAs (see the two
// kernels); and where their partials sit.
struct AttnSplit {
  size_t plan, po, pml, so, sml, bytes;
  uint32_t rt, prefix_cap, seq_cap, seq_groups;
  uint32_t prefix_few, prefix_ctas, seq_few, seq_ctas;
  bool line;
};
// Clusters of up to eight CTAs for each of `units` units of up to `pages` pages.
// CTAs: as many as give the machine about five an SM (many units: one CTA
// each; 512 units of 3 pages on three CTAs each took 6 us longer).  Clusters:
// one, which needs no joining kernel, unless the units leave SMs idle (below
// about four CTAs each) and a CTA would still have four pages to read.
void attn_clusters(uint64_t units, uint32_t pages, uint32_t& clusters, uint32_t& ctas) {
  const uint64_t want = 5u * kSms / units;
  ctas = (uint32_t)(want < 1u ? 1u : (want > 8u ? 8u : want));
  if (ctas > pages) ctas = pages;
  const uint64_t most = 4u * kSms / (units * ctas), by_pages = pages / (ctas * 4u);
  clusters = (uint32_t)(most < by_pages ? most : by_pages);
  if (clusters < 1u) clusters = 1u;
}
// Rows of the line's groups: 32 where a unit has more than 16 (128 dimensions).
uint32_t attn_rt(const KvPool& kv, const KvAttnBatch& b, uint32_t group) {
  const uint64_t rows = (uint64_t)(b.max_prefix > 0 ? b.n_rows : b.max_rows) * group;
  return kv.head_dim == 128u && rows > 16u ? 32u : 16u;
}
AttnSplit attn_split(const KvPool& kv, const KvAttnBatch& b, uint32_t n_head) {
  const uint32_t group = n_head / kv.n_kv_head, rt = attn_rt(kv, b, group);
  AttnSplit s{};
  s.rt = rt;
  auto put = [&](uint64_t parts, uint32_t cap, size_t& o, size_t& ml) {
    o = s.bytes;
    s.bytes += (parts * cap * kv.head_dim * 4u + 255u) & ~(size_t)255u;
    ml = s.bytes;
    s.bytes += (parts * cap * kAttnMl * 4u + 255u) & ~(size_t)255u;
  };
  s.plan = 0;
  s.bytes = (4u * ((size_t)b.n_seq + 5u) + 255u) & ~(size_t)255u;
  const uint64_t rows = (uint64_t)b.n_rows * group, per_seq = (uint64_t)b.max_rows * group;
  if (b.max_prefix > 0) {
    const uint32_t pages = attn_ceil(b.max_prefix, kKvPage);
    s.prefix_cap = rows < rt ? (uint32_t)rows : rt;
    if (rows <= kFewRows) {
      attn_clusters(kv.n_kv_head, pages, s.prefix_few, s.prefix_ctas);
      put((uint64_t)kv.n_kv_head * s.prefix_few, s.prefix_cap, s.po, s.pml);
    } else {
      s.line = true;
      put(2u * ((uint64_t)kv.n_kv_head * ((rows + rt - 1u) / rt) + kAttnMaxCtas), s.prefix_cap, s.po, s.pml);
    }
  }
  if (b.max_len > 0) {
    const uint32_t pages = attn_ceil(b.max_len, kKvPage);
    s.seq_cap = per_seq < rt ? (uint32_t)per_seq : rt;
    s.seq_groups = (uint32_t)((per_seq + rt - 1u) / rt);
    if (per_seq <= kFewRows) {
      attn_clusters((uint64_t)b.n_seq * kv.n_kv_head, pages, s.seq_few, s.seq_ctas);
      put((uint64_t)b.n_seq * kv.n_kv_head * s.seq_few, s.seq_cap, s.so, s.sml);
    } else {
      s.line = true;
      put(2u * ((uint64_t)b.n_seq * s.seq_groups * kv.n_kv_head + kAttnMaxCtas), s.seq_cap, s.so, s.sml);
    }
  }
  return s;
}

template <uint32_t HD, uint32_t R>
cudaError_t attn_few(const KvAttnParams& p, uint32_t prefix, uint32_t direct, cudaStream_t st) {
  const uint32_t n = prefix ? p.prefix_few : p.seq_few, ctas = prefix ? p.prefix_ctas : p.seq_ctas;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(n * ctas, p.n_kv_head, prefix ? 1u : p.rows.n_seq);
  cfg.blockDim = dim3(kFewThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv_attn_few_kernel<HD, R>, p, prefix, ctas, direct);
}
template <uint32_t HD>
cudaError_t attn_few_rows(const KvAttnParams& p, uint32_t prefix, uint32_t rows, uint32_t direct, cudaStream_t st) {
  if (rows == 1) return attn_few<HD, 1>(p, prefix, direct, st);
  if (rows == 2) return attn_few<HD, 2>(p, prefix, direct, st);
  return attn_few<HD, 4>(p, prefix, direct, st);
}

template <uint32_t HD, uint32_t RT, bool CAUSAL>
cudaError_t attn_line_kernel(const KvAttnParams& p, int num_sms, uint64_t work, cudaStream_t st) {
  using G = AttnGeo<HD, RT>;
  static SmemAttr attr;
  cudaError_t e = ensure_smem_attr((const void*)kv_attn_kernel<HD, RT, CAUSAL>, (int)G::smem(EOS_ATTN_MAX_SEQ), attr);
  if (e != cudaSuccess) return e;
  uint64_t grid = (uint64_t)G::kCtas * (uint32_t)num_sms;
  if (grid > kAttnMaxCtas) grid = kAttnMaxCtas;
  if (grid > work) grid = work;
  if (grid == 0) grid = 1;
  // may start while the few-rows kernels of this call run (it reads nothing of
  // theirs) and waits for them at its end, so that the joining kernel, which
  // waits for this one, waits for all
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((uint32_t)grid);
  cfg.blockDim = dim3(G::kThreads);
  cfg.dynamicSmemBytes = G::smem(p.rows.n_seq);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = p.seq_few > 0 || p.prefix_few > 0 ? 1 : 0;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv_attn_kernel<HD, RT, CAUSAL>, p);
}

template <uint32_t HD, uint32_t RT>
cudaError_t attn_line(const KvAttnParams& p, int num_sms, uint64_t work, cudaStream_t st) {
  return p.max_len > 0 && p.seq_few == 0 && p.max_rows > 1u ? attn_line_kernel<HD, RT, true>(p, num_sms, work, st)
                                                            : attn_line_kernel<HD, RT, false>(p, num_sms, work, st);
}

template <uint32_t HD>
cudaError_t attn_launch(const KvAttnParams& p, bool line, int num_sms, uint64_t work, cudaStream_t st) {
  cudaError_t e = cudaSuccess;
  const bool first = !line && p.seq_few == 0 && p.prefix_few == 0;
  const bool alone = p.max_prefix == 0 && p.seq_few == 1u;  // nothing to join
  if (p.seq_few > 0) e = attn_few_rows<HD>(p, 0, p.seq_cap, alone ? 1u : 0u, st);
  if (alone || e != cudaSuccess) return e;
  if (p.prefix_few > 0) e = attn_few_rows<HD>(p, 1, p.prefix_cap, 0u, st);
  if (e != cudaSuccess) return e;
  if (line) {
    if constexpr (HD == 128) {
      e = p.rt == 32u ? attn_line<HD, 32>(p, num_sms, work, st) : attn_line<HD, 16>(p, num_sms, work, st);
    } else {
      e = attn_line<HD, 16>(p, num_sms, work, st);
    }
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((uint32_t)(((uint64_t)p.rows.n_rows * p.n_head + 1u) / 2u));
  cfg.blockDim = dim3(64);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  // it reads row0 and seq_len before it waits: early only behind this call's own
  // kernels, which started when the inputs were there
  at[0].val.programmaticStreamSerializationAllowed = first ? 0 : 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return p.seq_few == 0 && !line ? cudaLaunchKernelEx(&cfg, kv_attn_join_kernel<HD, true>, p)
                                 : cudaLaunchKernelEx(&cfg, kv_attn_join_kernel<HD, false>, p);
}

}  // namespace

size_t kv_attn_scratch_bytes(const KvPool& kv, const KvAttnBatch& b, uint32_t n_head) {
  return attn_split(kv, b, n_head).bytes;
}

// The line of tiles of the largest lengths (its words are 32-bit).
uint64_t kv_attn_work_bound(const KvPool& kv, const KvAttnBatch& b, uint32_t n_head) {
  const uint32_t group = n_head / kv.n_kv_head, rt = attn_rt(kv, b, group);
  const uint64_t tp = (b.max_prefix + kKvPage - 1u) / kKvPage, ts = (b.max_len + kKvPage - 1u) / kKvPage;
  const uint64_t rp = ((uint64_t)b.n_rows * group + rt - 1u) / rt;
  uint64_t rs = (uint64_t)b.n_seq * (((uint64_t)b.max_rows * group + rt - 1u) / rt);
  const uint64_t by_rows = rp + b.n_seq;  // sequences share n_rows
  if (rs > by_rows) rs = by_rows;
  return kv.n_kv_head * (rp * (tp + kAttnStart) + rs * (ts + kAttnStart));
}

cudaError_t launch_kv_attn(const KvPool& kv, const KvAttnBatch& b, const float* q, uint64_t q_stride, float* out,
                           uint64_t out_stride, uint32_t n_head, float scale, void* scratch, int num_sms,
                           uint32_t* err, cudaStream_t st) {
  if (kv.n_kv_head == 0 || n_head % kv.n_kv_head != 0) return cudaErrorNotSupported;  // whole groups of heads only
  if (b.n_rows == 0 || b.n_seq == 0) return cudaSuccess;
  const AttnSplit s = attn_split(kv, b, n_head);
  uint8_t* ws = static_cast<uint8_t*>(scratch);
  KvAttnParams p{};
  p.rows = KvRows{b.row0, b.n_seq, b.n_rows, b.row0 ? 0u : b.n_rows / b.n_seq};
  p.pages = kv.pages;
  p.prefix_pages = b.prefix_pool ? b.prefix_pool->pages : kv.pages;
  p.prefix_n_pages = b.prefix_pool ? b.prefix_pool->n_pages : kv.n_pages;
  p.prefix_table = b.prefix_table;
  p.prefix_len = b.prefix_len;
  p.table = b.table;
  p.seq_len = b.seq_len;
  p.max_prefix = b.max_prefix;
  p.table_stride = b.table_stride;
  p.max_len = b.max_len;
  p.max_rows = b.max_rows;
  p.n_pages = kv.n_pages;
  p.n_head = n_head;
  p.n_kv_head = kv.n_kv_head;
  p.group = n_head / kv.n_kv_head;
  p.by_group = attn_divisor(p.group);
  p.by_kv_head = attn_divisor(kv.n_kv_head);
  p.q = q;
  p.out = out;
  p.q_stride = q_stride;
  p.out_stride = out_stride;
  p.scale_log2 = (float)((double)scale * 1.4426950408889634);
  p.plan = reinterpret_cast<uint32_t*>(ws + s.plan);
  p.po = reinterpret_cast<float*>(ws + s.po);
  p.pml = reinterpret_cast<float*>(ws + s.pml);
  p.so = reinterpret_cast<float*>(ws + s.so);
  p.sml = reinterpret_cast<float*>(ws + s.sml);
  p.rt = s.rt;
  p.prefix_cap = s.prefix_cap;
  p.seq_cap = s.seq_cap;
  p.seq_groups = s.seq_groups;
  p.prefix_few = s.prefix_few;
  p.prefix_ctas = s.prefix_ctas;
  p.seq_few = s.seq_few;
  p.seq_ctas = s.seq_ctas;
  p.err = err;
  const uint64_t work = kv_attn_work_bound(kv, b, n_head);
  if (kv.head_dim == 64) return attn_launch<64>(p, s.line, num_sms, work, st);
  if (kv.head_dim == 128) return attn_launch<128>(p, s.line, num_sms, work, st);
  return attn_launch<256>(p, s.line, num_sms, work, st);
}

}  // namespace eos
