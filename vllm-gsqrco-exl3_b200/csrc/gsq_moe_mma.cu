// The experts' products on the tensor cores, for the four main types (Q4_K, Q6_K, IQ3_S, IQ4_XS in GGUF order) (sm_100a).
//
// The pairs of a token and one of its experts are gathered by expert, at most 8 or 16 to a group (gsq_moe.cu), so that an expert's
// weights are read and decoded once for them. A tile is 16 weight rows: 8 gate and the 8 up rows of the same channels, which
// leaves a channel's gate and up sums in one lane, or 16 rows of the down weights. The list of (group, tile) is cut into one
// contiguous range a block of equal estimated cost, one block an SM; a block takes as many groups of its range at a time as its columns of
// activations hold (a batch, mostly all of them), and cuts the batch's superblocks into 16 equal contiguous chunks, one a warp.
//
//   * Weights: each warp has a ring of asynchronous copies of its own (a stage is 16 rows x 2 superblocks, or 1; 16 lanes copy
//     consecutive 16-byte pieces of a row), filled ahead over tiles and batches, so the stream does not stop. Rows of 210- and 110-byte
//     blocks start at any even address: copies begin at the 16-byte boundary before, and the rows are read at their offset. (One bulk
//     copy a row was a loop over the 16 lanes that issue them: 95 of 427 instructions a superblock.)
//   * Activations: the block takes its batch's rows (X in 8 bits, or the activated products, which it quantises) into shared memory in
//     the order of the tensor-core instruction's B fragment. An instruction takes the 8 columns from its group's first on; what it finds
//     past the group's own only reaches sums that are not stored. A group of more than 8 takes two instructions on one decoding.
//   * Product: mma.sync m16n8k32 on bytes (m16n8k16 for Q6_K, whose sub-scales cover 16 values); a lane decodes exactly its share of
//     the A fragment. (tcgen05.mma has an 8-bit integer form, kind::i8, but 128 rows to an instruction and an accumulator that is read out of
//     TMEM once per slice, since every 32 values' sums are scaled on their own before they are added: gsq_gemm5.cuh does that for many
//     columns, and the linear path takes it from 33 rows on. Experts with more than 16 tokens could use it; here they decode their weights once
//     for every 16.) That scaling, not the instruction, is the cost: with a column for each of 8 tokens it is 14 instructions a slice and lane. A group of 1, 2 or 4 tokens therefore gives the free columns to other
//     slices: the instruction of slice j has the activations in the columns of slice j and zeros in the others, and the sums of 8, 4
//     or 2 slices come out side by side in one C fragment, scaled at once.
//   * Sums leave the instruction on the bit pattern of 1.5 * 2^23, so fma(sum, dA, -1.5 * 2^23 dA) is the exact integer times
//     d * sub-scale without a conversion; the second fma scales by the activations. Q4_K's high nibbles are multiplied where they
//     are, as unsigned bytes 16 times their value. Its minima, for 4 tokens and more, are a product of their own, min [16 rows x 8
//     slices] times d_x * sum of the quants [8 slices x 8 columns], in three tf32 parts that hold all 24 bits.
//   * A tile that several warps have parts of is added up by the warp that has its beginning, in the order of the warps.
//
// Measured, 64 experts of 4096 x 2048 with 1, 2, 4, 8, 16 tokens each, the whole layer (least time at the measured 6.54 TB/s in front): Q4_K 138:
// 173, 177, 185, 221, 308 us; IQ4_XS 131: 265, 268, 294, 334, 403; Q6_K 202: 276, 319, 335, 339, 427; IQ3_S 106: 346, 354, 374, 400, 480. Q4_K
// with one token an expert comes to 80 % of DRAM's rate, 93 % without the 25 us that a call takes besides. IQ4_XS and IQ3_S are bound by the logic pipe, which
// decodes them (look-ups of 8 nibbles, a codebook with signs): 72 to 81 % busy, the most frequent stall a full pipe, DRAM at 25 to 40 %. Q4_K and Q6_K
// in the layers captured (smaller ones with one token an expert, 8 tokens an expert) fill nothing (logic 37 to 57 %, issue slots 43 to 71 %): dependent instructions with four warps a scheduler, since one
// kernel with the forms for 1 to 16 tokens takes 126 to 128 registers.
// Many tokens an expert cost by sixteens: 64 experts of 5120 x 1280, top 8, Q4_K / Q6_K, 64, 256, 1024 tokens: 273, 670, 2278 us.
#include <type_traits>

#include "gsq_moe.cuh"
#include "gsq_tables.h"

namespace gsq {
namespace moe {

enum { Q4K = 0, Q6K = 1, IQ3S = 2, IQ4XS = 3 };
constexpr int WARPS = 16, THREADS = WARPS * 32;
constexpr int MAGIC = 0x4B400000;            // 1.5 * 2^23
constexpr float MAGIC_F = 12582912.0f;

__device__ const uint32_t g_iq3s[512] = GSQ_IQ3S_GRID_INIT;
__constant__ __align__(16) int8_t c_iq4[16] = GSQ_IQ4NL_VALUES_INIT;

__host__ __device__ constexpr int bs(int kind) { return kind == Q4K ? 144 : kind == Q6K ? 210 : kind == IQ3S ? 110 : 136; }
// Bytes between the rows of a stage: what a row's pieces may take (up to 14 bytes in front, 16-byte pieces), at distances that put what a
// warp reads at once on different banks.
__host__ __device__ constexpr int pitch(int kind, int sbs) {
  return kind == Q6K ? 240 : sbs == 1 ? 144 : kind == Q4K ? 288 : kind == IQ3S ? 240 : 304;
}
// Where row r of 16 is in a stage. Q4_K's 8-byte reads take rows 0 .. 3, then 4 .. 7 at once: at 144 bytes a row these have to be every
// second one.
template <int KIND, int SBS>
__host__ __device__ constexpr int row_place(int r) {
  return KIND == Q4K && SBS == 1 ? (r & 8) | (r & 3) << 1 | (r >> 2 & 1) : r;
}
constexpr int GRID_COPIES = 8;               // of IQ3_S's codebook in shared memory, one for lanes l, l + 8, ...
constexpr int WINDOW = 32;                   // groups of a block that are looked up at a time
__host__ __device__ constexpr size_t fixed_smem(int kind, int k, int cap) {   // all but the ring
  return (size_t)k * cap + (size_t)k / 32 * cap * 4 * (kind == Q4K ? 2 : 1) + (kind == IQ3S ? 512 * 4 * GRID_COPIES : 0) + WARPS * 64 * cap;
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the calling thread's last n groups of copies are done.
template <int N>
__device__ __forceinline__ void wait_all_but() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// C += A B, signed bytes (UA: A unsigned)
template <bool UA>
__device__ __forceinline__ void mma_k32(int (&c)[4], const uint32_t (&a)[4], uint2 b) {
  if constexpr (UA)
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
  else
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
}
__device__ __forceinline__ void mma_k16(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t b) {
  asm("mma.sync.aligned.m16n8k16.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5}, {%6}, {%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(b));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, float2 b) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(__float_as_uint(b.x)), "r"(__float_as_uint(b.y)));
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}
__device__ __forceinline__ uint32_t lds16(const uint8_t* p) { return *reinterpret_cast<const uint16_t*>(p); }
__device__ __forceinline__ uint32_t lds32(const uint8_t* p) { return *reinterpret_cast<const uint32_t*>(p); }
__device__ __forceinline__ uint32_t lds32h(const uint8_t* p) { return prmt(lds16(p), lds16(p + 2), 0x5410); }   // from an even address

// How a group of up to TT tokens (16: twice 8) uses the 8 columns of a C fragment: NJ parts (slices of 32 values; of 16 for Q6_K) times TT tokens,
// column j TT + token. A superblock is NC fragments. Lane (g, t) feeds column g, and has the sums of columns 2 t, 2 t + 1.
template <int KIND, int TT>
struct Columns {
  static constexpr int NJ = 8 / TT, PARTS = KIND == Q6K ? 16 : 8, NC = PARTS / NJ;
  static __device__ __forceinline__ int fed_part(int g) { return g / TT; }
  static __device__ __forceinline__ int fed_token(int g) { return g % TT; }
  static __device__ __forceinline__ int part(int t, int c) { return (2 * t + c) / TT; }   // (c: 0 or 1; the same for both unless TT is 1)
};

// What a lane reads of the staged activations of one superblock, CAP columns a slice.
template <int KIND, int CAP, int TT>
struct Act {
  static constexpr int TF = TT < 8 ? TT : 8;   // tokens of a fragment; of 16, fragment n has columns 8 n ..
  using Col = Columns<KIND, TF>;
  const uint8_t* q;        // [slice][column][32 bytes]
  const float* d;          // [slice][column]
  const float* sums;       // [slice][column]: d * sum of the quants (Q4_K); of column 2 t
  const float* mins;       // the same of slice t, column g
  // col: the group's first column
  __device__ __forceinline__ Act(const uint8_t* q_s, const float* d_s, const float* sum_s, int sb, int col, int g, int t) {
    const int j = Col::fed_part(g), i = Col::part(t, 0), s = KIND == Q6K ? i >> 1 : i;
    q = q_s + ((sb * 8 + (KIND == Q6K ? j >> 1 : j)) * CAP + col + Col::fed_token(g)) * 32 + 8 * t + (KIND == Q6K ? 4 * (j & 1) : 0);
    d = d_s + (sb * 8 + s) * CAP + col + 2 * t % TF;
    sums = sum_s + (sb * 8 + s) * CAP + col + 2 * t % TF;
    mins = sum_s + (sb * 8 + t) * CAP + col + g;
  }
  __device__ __forceinline__ void next() {
    q += CAP * 256;
    d += CAP * 8;
    sums += CAP * 8;
    mins += CAP * 8;
  }
  // this lane's words of the part that it feeds in fragment c (of the columns from 8 n on)
  __device__ __forceinline__ uint2 quants(int c, int n) const { return *reinterpret_cast<const uint2*>(q + CAP * 32 * Col::NJ * c + 256 * n); }
  __device__ __forceinline__ uint32_t quants16(int c, int n) const {
    return *reinterpret_cast<const uint32_t*>(q + (TF == 8 ? CAP * 32 * (c >> 1) + 4 * (c & 1) : CAP * 16 * Col::NJ * c) + 256 * n);
  }
  static __device__ __forceinline__ float2 two(const float* p, int c) {
    const int s = KIND != Q6K ? Col::NJ * c : TF == 8 ? c >> 1 : Col::NJ / 2 * c;
    if constexpr (TF > 1) return *reinterpret_cast<const float2*>(p + CAP * s);
    return make_float2(p[CAP * s], p[CAP * (s + (KIND != Q6K))]);   // (Q6_K: two halves of a slice)
  }
  __device__ __forceinline__ float2 scales(int c, int n) const { return two(d + 8 * n, c); }
  __device__ __forceinline__ float2 quant_sums(int c) const { return two(sums, c); }
  __device__ __forceinline__ float2 minima(int n) const { return make_float2(mins[8 * n], mins[CAP * 4 + 8 * n]); }   // slices t, t + 4
};

// Byte `at` (of 8 in two words) as a number on 2^23.
__device__ __forceinline__ float byte_on_2_23(const uint32_t (&w)[2], bool upper, uint32_t at) {
  return __uint_as_float(prmt(upper ? w[1] : w[0], 0x4B000000u, 0x7440u | at));
}

// One superblock of 16 rows: b0, b1 = the blocks of rows g and g + 8; acc: rows g, g + 8 by columns 2 t, 2 t + 1 of the C fragments (of the
// first 8 columns, then of the others).
template <int KIND, int CAP, int TT>
__device__ __forceinline__ void superblock(const uint8_t* b0, const uint8_t* b1, const Act<KIND, CAP, TT>& x, int g, int t, const uint32_t* grid,
                                           float (&acc)[CAP / 2]) {
  constexpr int TF = Act<KIND, CAP, TT>::TF, NT = TT > 8 ? 2 : 1;
  using Col = Columns<KIND, TF>;
  constexpr int NJ = Col::NJ, NC = Col::NC;
  const int fed = Col::fed_part(g), part0 = Col::part(t, 0), part1 = Col::part(t, 1);   // (parts within a fragment)
  // what the rows' scales come from
  uint32_t sc[2][2], mn[2][2];
  uint2 h0, h1;
  float d0, d1;
  if constexpr (KIND == Q4K) {
    const uint4 r0 = *reinterpret_cast<const uint4*>(b0), r1 = *reinterpret_cast<const uint4*>(b1);
    sc[0][0] = r0.y & 0x3F3F3F3Fu;
    sc[0][1] = (r0.w & 0x0F0F0F0Fu) | ((r0.y >> 2) & 0x30303030u);
    sc[1][0] = r1.y & 0x3F3F3F3Fu;
    sc[1][1] = (r1.w & 0x0F0F0F0Fu) | ((r1.y >> 2) & 0x30303030u);
    mn[0][0] = r0.z & 0x3F3F3F3Fu;
    mn[0][1] = ((r0.w >> 4) & 0x0F0F0F0Fu) | ((r0.z >> 2) & 0x30303030u);
    mn[1][0] = r1.z & 0x3F3F3F3Fu;
    mn[1][1] = ((r1.w >> 4) & 0x0F0F0F0Fu) | ((r1.z >> 2) & 0x30303030u);
    h0.x = r0.x;
    h1.x = r1.x;
    d0 = h2f(r0.x);
    d1 = h2f(r1.x);
  } else if constexpr (KIND == IQ4XS) {
    h0 = *reinterpret_cast<const uint2*>(b0);
    h1 = *reinterpret_cast<const uint2*>(b1);
    d0 = h2f(h0.x);
    d1 = h2f(h1.x);
  } else if constexpr (KIND == IQ3S) {
    h0.x = lds32h(b0 + 106);
    h1.x = lds32h(b1 + 106);
    d0 = h2f(lds16(b0));
    d1 = h2f(lds16(b1));
  } else {
    d0 = 0.25f * h2f(lds16(b0 + 208));
    d1 = 0.25f * h2f(lds16(b1 + 208));
  }
  // d * sub-scale of row 0 / 1 (of this lane's two) for column c (0 / 1) of fragment f: exact
  auto row_scale = [&](int row, int f, int c) {
    const int p = c ? part1 : part0;
    const float d = row ? d1 : d0;
    if constexpr (KIND == Q4K) {
      // (the parity of the slice says which nibble: odd ones are 16 times too large)
      const bool upper = TF == 1 ? p >= 4 : TF == 2 ? f : TF == 4 ? f >> 1 : f >> 2;
      const uint32_t at = TF == 1 ? p & 3 : TF == 2 ? p : TF == 4 ? (f & 1) * 2 + p : f & 3;
      const bool odd = TF == 8 ? f & 1 : TF == 1 ? c : p & 1;
      const float e = odd ? 0.0625f * d : d;
      return fmaf(byte_on_2_23(sc[row], upper, at), e, -8388608.0f * e);
    } else if constexpr (KIND == IQ4XS) {
      const uint2 h = row ? h1 : h0;
      const int s = f * NJ + p, l = (int)(((h.y >> (4 * s)) & 15u) | (((h.x >> (16 + 2 * s)) & 3u) << 4));
      return d * (__int_as_float(MAGIC + l) - (MAGIC_F + 32.0f));
    } else if constexpr (KIND == IQ3S) {
      const int s = f * NJ + p, l = 1 + 2 * (int)(((row ? h1.x : h0.x) >> (4 * s)) & 15u);
      return d * (__int_as_float(MAGIC + l) - MAGIC_F);
    } else {
      const int l = *reinterpret_cast<const int8_t*>((row ? b1 : b0) + 192 + f * NJ + p);
      return d * (__int_as_float(MAGIC + l) - MAGIC_F);
    }
  };
  // raw words that several slices share
  uint2 q4[2];
  uint32_t l6[2][2][2], h6[2][2];
  int half[4 * NT];
  float part[4 * NT] = {};
#pragma unroll
  for (int f = 0; f < NC; ++f) {
    constexpr int START = KIND == Q6K && TF == 8 ? 0 : MAGIC;
    int c[NT][4];
    uint2 fed_words[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      c[n][0] = c[n][1] = c[n][2] = c[n][3] = START;
      if constexpr (KIND == Q6K) fed_words[n] = make_uint2(x.quants16(f, n), 0);
      else fed_words[n] = x.quants(f, n);
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int s = f * NJ + j;        // part of the superblock
      auto fed_now = [&](int n) { return TF < 8 && fed != j ? make_uint2(0, 0) : fed_words[n]; };
      uint32_t a[4];
      if constexpr (KIND == Q4K) {
        if ((s & 1) == 0) {
          q4[0] = *reinterpret_cast<const uint2*>(b0 + 16 + 16 * s + 8 * t);
          q4[1] = *reinterpret_cast<const uint2*>(b1 + 16 + 16 * s + 8 * t);
        }
        const uint32_t m = s & 1 ? 0xF0F0F0F0u : 0x0F0F0F0Fu;
        a[0] = q4[0].x & m;
        a[1] = q4[1].x & m;
        a[2] = q4[0].y & m;
        a[3] = q4[1].y & m;
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_k32<true>(c[n], a, fed_now(n));
      } else if constexpr (KIND == IQ4XS) {
        const uint32_t t0 = reinterpret_cast<const uint32_t*>(c_iq4)[0], t1 = reinterpret_cast<const uint32_t*>(c_iq4)[1],
                       t2 = reinterpret_cast<const uint32_t*>(c_iq4)[2], t3 = reinterpret_cast<const uint32_t*>(c_iq4)[3];
        // 8 indices -> two words of values in the order of the nibbles: value 4 t, 16 + 4 t, 4 t + 1, ... (the activations have that order)
        auto look_up = [&](uint32_t v, uint32_t& lo, uint32_t& hi) {
          const uint32_t i = v & 0x77777777u, pick = ((v >> 1) & 0x44444444u) | 0x32103210u;
          lo = prmt(prmt(t0, t1, i), prmt(t2, t3, i), pick);
          hi = prmt(prmt(t0, t1, i >> 16), prmt(t2, t3, i >> 16), pick >> 16);
        };
        look_up(lds32(b0 + 8 + 16 * s + 4 * t), a[0], a[2]);
        look_up(lds32(b1 + 8 + 16 * s + 4 * t), a[1], a[3]);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_k32<false>(c[n], a, fed_now(n));
      } else if constexpr (KIND == IQ3S) {
        auto value = [&](uint32_t low, uint32_t high, uint32_t signs) {   // index low | high << 8, negated where a sign bit is set
          const uint32_t v = grid[(low | (high << 8)) * GRID_COPIES];
          const uint32_t ones = ((signs & 15u) * 0x00204081u) & 0x01010101u;
          return (v ^ (ones * 255u)) + ones;
        };
        const uint32_t q0 = lds16(b0 + 2 + 8 * s + 2 * t), q1 = lds16(b1 + 2 + 8 * s + 2 * t);
        const uint32_t e0 = b0[66 + s] >> (2 * t), e1 = b1[66 + s] >> (2 * t), g0 = b0[74 + 4 * s + t], g1 = b1[74 + 4 * s + t];
        a[0] = value(q0 & 255u, e0 & 1u, g0);
        a[1] = value(q1 & 255u, e1 & 1u, g1);
        a[2] = value(q0 >> 8, (e0 >> 1) & 1u, g0 >> 4);
        a[3] = value(q1 >> 8, (e1 >> 1) & 1u, g1 >> 4);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_k32<false>(c[n], a, fed_now(n));
      } else {
        // part s: half s % 2 of slice s / 2. A value less 32 (six bits) is taken as q << 2 with the top bit flipped: four times it, as
        // a signed byte
        const int n = s >> 3, q = (s >> 1) & 3, e = s & 1;
        if ((s & 7) == 0) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            h6[0][i] = lds32h(b0 + 128 + 32 * n + 16 * i + 4 * t);
            h6[1][i] = lds32h(b1 + 128 + 32 * n + 16 * i + 4 * t);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              l6[0][r][i] = lds32h(b0 + 64 * n + 32 * r + 16 * i + 4 * t);
              l6[1][r][i] = lds32h(b1 + 64 * n + 32 * r + 16 * i + 4 * t);
            }
          }
        }
        auto word = [&](int row) {     // nibble q / 2 of ql's half q % 2, bits 2 q of qh
          const uint32_t lo = q < 2 ? l6[row][q & 1][e] << 2 : l6[row][q & 1][e] >> 2;
          const uint32_t hi = q == 3 ? h6[row][e] : h6[row][e] << (6 - 2 * q);
          return (lo & 0x3C3C3C3Cu) | ((hi & 0xC0C0C0C0u) ^ 0x80808080u);
        };
        const uint32_t a0 = word(0), a1 = word(1);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_k16(c[n], a0, a1, fed_now(n).x);
      }
    }
    if constexpr (KIND == Q6K && TF == 8) {
      // halves of a slice: sum_a * scale_a + sum_b * scale_b as integers, converted once, scaled by d at the end
      const int u0 = *reinterpret_cast<const int8_t*>(b0 + 192 + f), u1 = *reinterpret_cast<const int8_t*>(b1 + 192 + f);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int n0 = u0 * c[n][0], n1 = u0 * c[n][1], n2 = u1 * c[n][2], n3 = u1 * c[n][3];
        int* h = half + 4 * n;
        float *p = part + 4 * n, *to = acc + 4 * n;
        if (f & 1) {
          const float2 d = x.scales(f, n);
          p[0] = fmaf((float)(h[0] + n0), d.x, p[0]);
          p[1] = fmaf((float)(h[1] + n1), d.y, p[1]);
          p[2] = fmaf((float)(h[2] + n2), d.x, p[2]);
          p[3] = fmaf((float)(h[3] + n3), d.y, p[3]);
        } else {
          h[0] = n0;
          h[1] = n1;
          h[2] = n2;
          h[3] = n3;
        }
        if (f == NC - 1) {
          to[0] = fmaf(d0, p[0], to[0]);
          to[1] = fmaf(d0, p[1], to[1]);
          to[2] = fmaf(d1, p[2], to[2]);
          to[3] = fmaf(d1, p[3], to[3]);
        }
      }
      continue;
    }
    const float a00 = row_scale(0, f, 0), a10 = row_scale(1, f, 0), a01 = TF == 1 ? row_scale(0, f, 1) : a00, a11 = TF == 1 ? row_scale(1, f, 1) : a10;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float2 d = x.scales(f, n);
      float* to = acc + 4 * n;
      to[0] = fmaf(fmaf(__int_as_float(c[n][0]), a00, -MAGIC_F * a00), d.x, to[0]);
      to[1] = fmaf(fmaf(__int_as_float(c[n][1]), a01, -MAGIC_F * a01), d.y, to[1]);
      to[2] = fmaf(fmaf(__int_as_float(c[n][2]), a10, -MAGIC_F * a10), d.x, to[2]);
      to[3] = fmaf(fmaf(__int_as_float(c[n][3]), a11, -MAGIC_F * a11), d.y, to[3]);
    }
    if constexpr (KIND == Q4K && TF <= 2) {
      const float n0 = -h2f(h0.x >> 16), n1 = -h2f(h1.x >> 16);
      const float2 xs = x.quant_sums(f);
      auto low = [&](int row, int p) {
        return (row ? n1 : n0) * (byte_on_2_23(mn[row], TF == 1 ? p >= 4 : f, TF == 1 ? p & 3 : p) - 8388608.0f);
      };
      const float m00 = low(0, part0), m10 = low(1, part0), m01 = TF == 1 ? low(0, part1) : m00, m11 = TF == 1 ? low(1, part1) : m10;
      acc[0] = fmaf(m00, xs.x, acc[0]);
      acc[1] = fmaf(m01, xs.y, acc[1]);
      acc[2] = fmaf(m10, xs.x, acc[2]);
      acc[3] = fmaf(m11, xs.y, acc[3]);
    }
  }
  if constexpr (KIND == Q4K && TF >= 4) {
    // rows g, g + 8 by slices t, t + 4; the sums' columns are the tokens (of 4 tokens, lanes t < 2 have them)
    auto low = [&](uint32_t w) { return __float_as_uint(__uint_as_float(prmt(w, 0x4B000000u, 0x7440u | t)) - 8388608.0f); };
    const uint32_t m0 = low(mn[0][0]), m1 = low(mn[1][0]), m2 = low(mn[0][1]), m3 = low(mn[1][1]);
    const float n0 = -h2f(h0.x >> 16), n1 = -h2f(h1.x >> 16);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      // in three parts of at most 11 bits, the smallest first
      const float2 xs = x.minima(n);
      auto upper = [](float v) { return __uint_as_float(__float_as_uint(v) & 0xFFFFE000u); };
      const float2 hi = make_float2(upper(xs.x), upper(xs.y)), r = make_float2(xs.x - hi.x, xs.y - hi.y), mid = make_float2(upper(r.x), upper(r.y));
      float c[4] = {0.0f, 0.0f, 0.0f, 0.0f}, *to = acc + 4 * n;
      mma_tf32(c, m0, m1, m2, m3, make_float2(r.x - mid.x, r.y - mid.y));
      mma_tf32(c, m0, m1, m2, m3, mid);
      mma_tf32(c, m0, m1, m2, m3, hi);
      if (TF == 8 || t < 2) {
        to[0] = fmaf(n0, c[0], to[0]);
        to[1] = fmaf(n0, c[1], to[1]);
        to[2] = fmaf(n1, c[2], to[2]);
        to[3] = fmaf(n1, c[3], to[3]);
      }
    }
  }
}

// A lane's sums over the parts that stood side by side: afterwards rows g, g + 8 by tokens 2 t, 2 t + 1.
template <int TT, int N>
__device__ __forceinline__ void fold(float (&acc)[N]) {
  if constexpr (TT == 1) {
    acc[0] += acc[1];
    acc[2] += acc[3];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (TT == 1 && (i & 1)) continue;
    if constexpr (TT <= 2) acc[i] += __shfl_xor_sync(0xFFFFFFFFu, acc[i], 1);
    if constexpr (TT <= 4) acc[i] += __shfl_xor_sync(0xFFFFFFFFu, acc[i], 2);
  }
}

// 8 quants of column `col` (words w0, w1; d: the scale of their 32, sum: the quants') into the staged activations. Whole warps call
// it: four lanes share a slice of 32 values.
template <int KIND, int CAP>
__device__ __forceinline__ void stage_piece(uint32_t w0, uint32_t w1, float d, int piece, int col, uint8_t* q_s, float* d_s, float* sum_s) {
  const int s = piece >> 2, p = piece & 3;
  uint8_t* to = q_s + (s * CAP + col) * 32;
  if constexpr (KIND == Q6K) {           // lane t's words t and 4 + t side by side
    *reinterpret_cast<uint32_t*>(to + 16 * (p & 1) + 4 * (p >> 1)) = w0;
    *reinterpret_cast<uint32_t*>(to + 16 * (p & 1) + 8 + 4 * (p >> 1)) = w1;
  } else if constexpr (KIND == IQ4XS) {  // values i and 16 + i side by side, as a byte of the block has them
    const uint32_t o0 = __shfl_xor_sync(0xFFFFFFFFu, w0, 2), o1 = __shfl_xor_sync(0xFFFFFFFFu, w1, 2);
    if (p < 2)
      *reinterpret_cast<uint4*>(to + 16 * p) = make_uint4(prmt(w0, o0, 0x5140), prmt(w0, o0, 0x7362), prmt(w1, o1, 0x5140), prmt(w1, o1, 0x7362));
  } else {
    *reinterpret_cast<uint2*>(to + 8 * p) = make_uint2(w0, w1);
  }
  if constexpr (KIND == Q4K) {
    int sum = dp4a((int)w0, 0x01010101, dp4a((int)w1, 0x01010101, 0));
    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
    if (p == 0) sum_s[s * CAP + col] = d * (float)sum;
  }
  if (p == 0) d_s[s * CAP + col] = d;
}

// Stores a tile's sums: rows g, g + 8 by columns 2 t, 2 t + 1 of the group (of its first 8 columns, then of the others).
template <bool DOWN, int N>
__device__ __forceinline__ void store_tile(const MoeArgs& a, const float (&acc)[N], int4 gr, int tile, const int* pair_s, const float* weight_s,
                                           int g, int t) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const int col = 8 * (i >> 1) + 2 * t + (i & 1), c = 4 * (i >> 1) + (i & 1);
    if (col < gr.z) {
      const int pair = pair_s[gr.w + col];
      if constexpr (DOWN) {
        float* to = a.part + (int64_t)pair * a.hidden + 16 * tile + g;
        const float wt = weight_s[gr.w + col];
        to[0] = wt * acc[c];
        to[8] = wt * acc[2 + c];
      } else {
        a.h[(int64_t)pair * a.inter + 8 * tile + g] = moe_act(a.act, acc[c]) * acc[2 + c];
      }
    }
  }
}

// A batch: units (group, tile) [u0, u1) of the block's list; first of its groups in the window, and how many.
struct Batch {
  int u0, u1, g0, n;
};
// The block's range of units, and the window of groups that it is at.
struct Window {
  int4 group[WINDOW];        // expert, first place in the list, pairs, first column of the batch's activations
  Batch batch[WINDOW];
  int first, batches, end;   // number of the window's first group; one past its last unit
};

// A batch's steps (a stage's superblocks of a tile) from chunk_begin(warp) to chunk_begin(warp + 1) are warp `warp`'s. steps: of a tile.
__device__ __forceinline__ int chunk_begin(const Batch& b, int steps, int warp) { return (b.u1 - b.u0) * steps * warp / WARPS; }

// A warp's way through the steps of its chunks, batch after batch of a window.
struct Place {
  int batch, left;           // steps left of the chunk
  int group, tile, step;     // group of the window, tile of the group, step of the tile
  bool live;
  __device__ __forceinline__ void enter(const Window& w, int tiles, int steps, int warp) {   // `batch`, or the next one with work for this warp
    for (live = false; !live && batch < w.batches; batch += !live) {
      const Batch b = w.batch[batch];
      const int s = chunk_begin(b, steps, warp);
      left = chunk_begin(b, steps, warp + 1) - s;
      if (left > 0) {
        live = true;
        const int u = s / steps, at = b.u0 + u;
        step = s - u * steps;
        group = at / tiles - w.first;
        tile = at - (group + w.first) * tiles;
      }
    }
  }
  // the step behind; true where it is another tile's (or there is none left)
  __device__ __forceinline__ bool next(const Window& w, int tiles, int steps, int warp) {
    if (--left == 0) {
      ++batch;
      enter(w, tiles, steps, warp);
      return true;
    }
    if (++step < steps) return false;
    step = 0;
    if (++tile == tiles) {
      tile = 0;
      ++group;
    }
    return true;
  }
};

// DOWN: rows of w2 on the activated products, else gate and up rows of w13 on X. SBS: superblocks of a stage; STAGES: of a warp's ring;
// CAP: columns of activations, and the most pairs of a group.
template <int KIND, bool DOWN, int SBS, int STAGES, int CAP>
__global__ void __launch_bounds__(THREADS, 1) moe_mma_kernel(const MoeArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Window win;
  __shared__ int pair_s[CAP];
  __shared__ float weight_s[CAP];                    // (down product)
  __shared__ int token_s[CAP];                       // (gate / up product)
  constexpr int PITCH = pitch(KIND, SBS), STAGE = 16 * PITCH, BS = bs(KIND), A = CAP / 2;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int k = DOWN ? a.inter : a.hidden, rows = DOWN ? a.hidden : 2 * a.inter, tiles = rows >> 4, nsb = k >> 8, steps = (nsb + SBS - 1) / SBS;
  const int64_t rb = DOWN ? a.rb2 : a.rb13;
  const uint8_t* const weights = DOWN ? a.w2 : a.w13;

  uint8_t* sp = smem;
  uint8_t* q_s = sp;
  sp += (size_t)k * CAP;
  float* d_s = reinterpret_cast<float*>(sp);
  sp += (size_t)k / 32 * CAP * 4;
  float* sum_s = reinterpret_cast<float*>(sp);       // d * sum of the quants (Q4_K)
  if (KIND == Q4K) sp += (size_t)k / 32 * CAP * 4;
  uint32_t* grid_s = reinterpret_cast<uint32_t*>(sp);
  if (KIND == IQ3S) sp += 512 * 4 * GRID_COPIES;
  float4* part_s = reinterpret_cast<float4*>(sp);    // [warps][CAP / 8][lanes]: sums of the tile that begins before the warp's chunk
  sp += WARPS * 64 * CAP;
  const uint8_t* ring = sp + (size_t)warp * STAGES * STAGE;
  // copies of a stage: copy i has pieces lane % 16 of rows 2 i and 2 i + 1, and where a row has more than 16 pieces one copy takes
  // pieces 16, 17 of all rows. Row r >= 8 of a gate / up tile is an up row.
  constexpr int PIECES = (SBS * BS + (KIND == Q4K ? 0 : KIND == IQ4XS ? 8 : 14) + 15) / 16;
  static_assert(PIECES <= 18 && 16 * PIECES <= PITCH, "");
  const uint32_t to_rows = smem_addr(ring) + row_place<KIND, SBS>(lane >> 4) * PITCH + 16 * (lane & 15);
  const uint32_t to_rest = smem_addr(ring) + (lane >> 1) * PITCH + 256 + 16 * (lane & 1);
  const uint8_t* const from_piece = weights + 16 * (lane & 15);
  const int64_t two_rows = 2 * rb, up_rows = DOWN ? 0 : (a.inter - 8) * rb;
  const int64_t from_rows = (lane >> 4) * rb, from_rest = (lane >> 1) * rb + (lane >= 16 ? up_rows : 0);

  // Launched while the kernel before runs (launch_kernel). The gate / up product waits for the plan; the down product has the plan from
  // before that product, and its first weights come in while that finishes.
  if (!DOWN) asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // the block's units: boundary b is a group and a share (of 65536) of its tiles
  auto boundary = [&](int b) {
    const int2 at = a.bounds[b];
    return at.x * tiles + (int)(((int64_t)at.y * tiles) >> 16);
  };
  const int block_u1 = boundary(blockIdx.x + 1);
  int u0 = boundary(blockIdx.x);
  if (KIND == IQ3S)
    for (int i = tid; i < 512 * GRID_COPIES; i += THREADS) grid_s[i] = g_iq3s[i / GRID_COPIES];

  for (; u0 < block_u1; u0 = win.end) {
    // the window's groups, their columns and batches: a group's first column is even (its scales are read in pairs), and 8 or 16
    // columns from there on exist
    __syncthreads();
    if (warp == 0) {
      const int first = u0 / tiles, n = min((block_u1 - 1) / tiles - first + 1, WINDOW);
      for (int i = lane; i < n; i += 32) win.group[i] = a.group[first + i];
      __syncwarp();
      if (lane == 0) {
        const int end = min(block_u1, (first + n) * tiles);
        int col = 0, b = 0;
        win.batch[0] = Batch{u0, end, 0, 0};
        for (int i = 0; i < n; ++i) {
          if (col + (win.group[i].z > 8 ? 16 : 8) > CAP) {
            win.batch[b].u1 = (first + i) * tiles;
            win.batch[++b] = Batch{(first + i) * tiles, end, i, 0};
            col = 0;
          }
          win.group[i].w = col;
          ++win.batch[b].n;
          col += (win.group[i].z + 1) & ~1;
        }
        win.first = first;
        win.batches = b + 1;
        win.end = end;
      }
    }
    __syncthreads();

    // the weights' stream
    Place in;
    in.batch = 0;
    in.enter(win, tiles, steps, warp);
    int64_t in_off = 0;                // of the tile's first row, at the next step
    auto row_offset = [&](const Place& p, int r) {
      const int row = DOWN ? 16 * p.tile + r : 8 * p.tile + (r & 7) + (r & 8 ? a.inter : 0);
      return ((int64_t)win.group[p.group].x * rows + row) * rb + p.step * (SBS * BS);
    };
    if (in.live) in_off = row_offset(in, 0);
    auto issue = [&](int slot) {       // one stage's copies; an empty group of copies where there is nothing left
      if (in.live) {
        const bool half = SBS == 2 && 2 * in.step + 1 == nsb;      // (an odd row length: its last step is one superblock)
        const int bytes = half ? BS : SBS * BS;
        // pieces that are always needed: of rows of 272 or 288 bytes 16 (and more, below), of 144 or 136 bytes (at 0 or 8) 9, of 210 bytes
        // (at any even place) 14
        constexpr bool ALL = KIND != IQ3S;
        const bool mine = KIND == IQ3S || (lane & 15) < (KIND == Q6K ? 14 : SBS == 1 ? 9 : 16);
        auto copy = [&](uint32_t to, const uint8_t* from, int64_t row, int piece, bool sure) {
          if (sure || 16 * piece < (KIND == Q4K ? 0 : (int)(row & 15)) + bytes) copy16(to + slot * STAGE, from + (KIND == Q4K ? row : row & ~(int64_t)15));
        };
        int64_t row = in_off + from_rows;
        if (ALL && !half) {
          if (mine) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              if (i == 4) row += up_rows;
              copy(to_rows + row_place<KIND, SBS>(2 * i) * PITCH, from_piece, row, 0, true);
              row += two_rows;
            }
          }
        } else {
#pragma unroll 2
          for (int i = 0; i < 8; ++i) {
            if (i == 4) row += up_rows;
            copy(to_rows + row_place<KIND, SBS>(2 * i) * PITCH, from_piece, row, lane & 15, false);
            row += two_rows;
          }
        }
        if (PIECES > 16) copy(to_rest, weights + 256 + 16 * (lane & 1), in_off + from_rest, 16 + (lane & 1), false);
        in_off += SBS * BS;
        if (in.next(win, tiles, steps, warp) && in.live) in_off = row_offset(in, 0);
      }
      commit();
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) issue(s);

    Place at;
    at.batch = 0;
    at.enter(win, tiles, steps, warp);
    int slot = 0;
    for (int batch = 0; batch < win.batches; ++batch) {
      const Batch bt = win.batch[batch];
      {
        // columns of the batch: pairs, then their rows' values (unused columns in between hold what was there)
        __syncthreads();                // the batch before is done with them
        if (DOWN) asm volatile("griddepcontrol.wait;" ::: "memory");
        if (tid < CAP) pair_s[tid] = -1;
        __syncthreads();
        if (tid < bt.n * CAP) {
          const int4 gr = win.group[bt.g0 + tid / CAP];
          const int i = tid % CAP;
          if (i < gr.z) {
            const int pair = a.list[gr.y + i];
            pair_s[gr.w + i] = pair;
            if (DOWN) weight_s[gr.w + i] = a.weights[pair];
            else token_s[gr.w + i] = pair / a.top_k;
          }
        }
        __syncthreads();
        // a warp takes a column's superblock at a time: 8 values a lane. X comes in quantised (by the blocks beside the plan's); the
        // activated products are quantised here.
        const int4 last = win.group[bt.g0 + bt.n - 1];
        const int columns = last.w + last.z;
        constexpr int U = 4;
        int col = warp / nsb, sb = warp - col * nsb;
        while (col < columns) {
          uint4 raw[U][DOWN ? 2 : 1];
          float d[U];
          int at_col[U], at_sb[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int row = col < columns ? pair_s[col] : -1;   // pair, or (gate / up) its token
            at_col[u] = row >= 0 ? col : -1;
            at_sb[u] = sb;
            if (row >= 0) {
              if constexpr (DOWN) {
                const uint4* p = reinterpret_cast<const uint4*>(a.h + (int64_t)row * k + 256 * sb + 8 * lane);
                raw[u][0] = __ldcg(p);
                raw[u][DOWN] = __ldcg(p + 1);
              } else {
                const uint2 q = __ldcg(reinterpret_cast<const uint2*>(a.xq + (int64_t)token_s[col] * k + 256 * sb + 8 * lane));
                raw[u][0] = make_uint4(q.x, q.y, 0, 0);
                d[u] = __ldcg(a.xd + (int64_t)token_s[col] * (k >> 5) + 8 * sb + (lane >> 2));
              }
            }
            for (sb += WARPS; sb >= nsb; sb -= nsb) ++col;
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (at_col[u] < 0) continue;
            uint32_t w0 = raw[u][0].x, w1 = raw[u][0].y;
            if constexpr (DOWN) {
              const float v[8] = {__uint_as_float(raw[u][0].x), __uint_as_float(raw[u][0].y), __uint_as_float(raw[u][0].z), __uint_as_float(raw[u][0].w),
                                  __uint_as_float(raw[u][1].x), __uint_as_float(raw[u][1].y), __uint_as_float(raw[u][1].z), __uint_as_float(raw[u][1].w)};
              int q[8];
              d[u] = moe_quant8(v, q);
              w0 = moe_pack4(q[0], q[1], q[2], q[3]);
              w1 = moe_pack4(q[4], q[5], q[6], q[7]);
            }
            stage_piece<KIND, CAP>(w0, w1, d[u], 32 * at_sb[u] + lane, at_col[u], q_s, d_s, sum_s);
          }
        }
        __syncthreads();
      }
      int open_unit = -1;               // the tile that this warp has the beginning of, but not the end, and its sums so far
      float open[A] = {};
      while (at.live && at.batch == batch) {
        // a tile, or this warp's part of one
        const int group = at.group, tile = at.tile, unit = (win.first + group) * tiles + tile;
        const bool begins = at.step == 0;
        const int4 gr = win.group[group];
        float acc[A] = {};
        uint32_t p0 = 0, p1 = 0;        // a row begins in its stage at what its offset is past a 16-byte boundary
        if (KIND != Q4K) {
          p0 = (uint32_t)row_offset(at, g);
          p1 = (uint32_t)row_offset(at, g + 8);
        }
        bool ends = false;
        auto run = [&](auto tokens) {
          constexpr int TT = decltype(tokens)::value;
          Act<KIND, CAP, TT> x(q_s, d_s, sum_s, at.step * SBS, gr.w, g, t);
          bool more = true;
          do {
            wait_all_but<STAGES - 2>();
            __syncwarp();               // every lane's pieces are there, and every lane is done with the stage before
            issue(slot == 0 ? STAGES - 1 : slot - 1);
            const uint8_t* b0 = ring + slot * STAGE + row_place<KIND, SBS>(g) * PITCH + (KIND == Q4K ? 0 : p0 & 15);
            const uint8_t* b1 = ring + slot * STAGE + row_place<KIND, SBS>(g + 8) * PITCH + (KIND == Q4K ? 0 : p1 & 15);
            ends = at.step == steps - 1;
            const int n = SBS == 2 && (!ends || (nsb & 1) == 0) ? 2 : 1;
#pragma unroll 1                        // (one copy of the code: a kernel starts with none of it in the instruction cache)
            for (int i = 0; i < n; ++i) {
              superblock<KIND, CAP, TT>(b0, b1, x, g, t, grid_s + (lane & (GRID_COPIES - 1)), acc);
              x.next();
              b0 += BS;
              b1 += BS;
            }
            p0 += SBS * BS;
            p1 += SBS * BS;
            if (++slot == STAGES) slot = 0;
            more = !at.next(win, tiles, steps, warp);
          } while (more);
          fold<TT>(acc);
        };
        if (gr.z == 1) run(std::integral_constant<int, 1>());
        else if (gr.z == 2) run(std::integral_constant<int, 2>());
        else if (KIND != Q6K && gr.z <= 4) run(std::integral_constant<int, 4>());   // (Q6_K, 4 tokens an expert: 347 us so, 337 in the form for 8)
        else if (CAP == 8 || gr.z <= 8) run(std::integral_constant<int, 8>());
        else if constexpr (CAP > 8) run(std::integral_constant<int, 16>());
        if (begins && ends) {
          store_tile<DOWN>(a, acc, win.group[group], tile, pair_s, weight_s, g, t);
        } else {
          if (begins) {
            open_unit = unit;
#pragma unroll
            for (int i = 0; i < A; ++i) open[i] = acc[i];
          } else {
#pragma unroll
            for (int i = 0; i < A / 4; ++i)
              part_s[(warp * (A / 4) + i) * 32 + lane] = make_float4(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
          }
        }
      }
      __syncthreads();                  // all parts are there, and nobody reads the activations any more
      if (open_unit >= 0) {
        const int tile_end = (open_unit - bt.u0 + 1) * steps;
        for (int o = warp + 1, from = chunk_begin(bt, steps, o); from < tile_end; ++o) {
          const int to = chunk_begin(bt, steps, o + 1);
          if (to > from) {
#pragma unroll
            for (int i = 0; i < A / 4; ++i) {
              const float4 q = part_s[(o * (A / 4) + i) * 32 + lane];
              open[4 * i] += q.x; open[4 * i + 1] += q.y; open[4 * i + 2] += q.z; open[4 * i + 3] += q.w;
            }
          }
          from = to;
        }
        store_tile<DOWN>(a, open, win.group[open_unit / tiles - win.first], open_unit % tiles, pair_s, weight_s, g, t);
      }
    }
  }
  if (DOWN) asm volatile("griddepcontrol.wait;" ::: "memory");   // (blocks without work, too: what comes next may reuse the workspace)
}

static int kind_of(int type) {
  return type == GSQ_TYPE_Q4_K ? Q4K : type == GSQ_TYPE_Q6_K ? Q6K : type == GSQ_TYPE_IQ3_S ? IQ3S : type == GSQ_TYPE_IQ4_XS ? IQ4XS : -1;
}

// Columns of activations, superblocks of a stage and stages of a warp's ring beside rows of k values. Where experts have more than 4 choices on
// average (`many`: MoeArgs), so that some have more than 8, 16 columns come before large stages: 16 tokens on one decoding of the weights (Q4_K,
// 64 experts of 4096 x 2048: 314 us, in groups of 8 430); else the other way round (a token an expert: 171 us, 187 with stages
// of one superblock). False: too long a row.
struct Plan {
  int cap, sbs, stages;
  size_t smem, room;         // of a block, and the most there is
};
static bool plan_of(int kind, int k, bool many, int max_smem, Plan* plan) {
  const size_t room = (size_t)max_smem - 2304;   // (2304: the window, the columns and the driver's own)
  static const int plans[2][4][3] = {{{16, 2, 2}, {8, 2, 2}, {8, 1, 3}, {8, 1, 2}}, {{16, 2, 2}, {16, 1, 3}, {8, 1, 3}, {8, 1, 2}}};
  static const int plans_q6k[3][3] = {{16, 1, 3}, {16, 1, 2}, {8, 1, 2}};
  for (int i = 0; i < (kind == Q6K ? 3 : 4); ++i) {
    const int* p = kind == Q6K ? plans_q6k[i] : plans[many][i];
    *plan = Plan{p[0], p[1], p[2], fixed_smem(kind, k, p[0]) + (size_t)p[2] * WARPS * 16 * pitch(kind, p[1]), room};
    if (plan->smem <= room) return true;
  }
  return false;
}

template <int KIND, bool DOWN, int SBS, int STAGES, int CAP>
static int launch_kernel(const MoeArgs& a, const Plan& p, cudaStream_t st) {
  static OncePerDevice smem;
  const int set = smem.set((const void*)moe_mma_kernel<KIND, DOWN, SBS, STAGES, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)p.room);
  if (set != GSQ_OK) return set;
  return moe_launch_behind(moe_mma_kernel<KIND, DOWN, SBS, STAGES, CAP>, a.blocks, THREADS, p.smem, st, a);
}

template <int KIND, bool DOWN>
static int launch(const MoeArgs& a, const Plan& p, cudaStream_t st) {
  if constexpr (KIND == Q6K) {
    if (p.cap == 8) return launch_kernel<KIND, DOWN, 1, 2, 8>(a, p, st);
    return p.stages == 3 ? launch_kernel<KIND, DOWN, 1, 3, 16>(a, p, st) : launch_kernel<KIND, DOWN, 1, 2, 16>(a, p, st);
  } else {
    if (p.cap == 8 && p.sbs == 2) return launch_kernel<KIND, DOWN, 2, 2, 8>(a, p, st);
    if (p.cap == 8) return p.stages == 3 ? launch_kernel<KIND, DOWN, 1, 3, 8>(a, p, st) : launch_kernel<KIND, DOWN, 1, 2, 8>(a, p, st);
    return p.sbs == 2 ? launch_kernel<KIND, DOWN, 2, 2, 16>(a, p, st) : launch_kernel<KIND, DOWN, 1, 3, 16>(a, p, st);
  }
}

}  // namespace moe

// The most pairs of a group that the tensor-core kernel takes for this type and row length; 0: it does not take it.
int moe_mma_serves(int type, int k, bool many) {
  const int kind = moe::kind_of(type);
  DeviceInfo di;
  moe::Plan p;
  return kind >= 0 && device_info(&di) == GSQ_OK && moe::plan_of(kind, k, many, di.max_smem_optin, &p) ? p.cap : 0;
}

// What a tile costs, in 256ths of one of a single token, as seen on the blocks of layers with groups of different sizes. In 16ths, the shares of few
// experts' blocks were as coarse as a share (27 tokens of 8 experts: 88 us, 74 in 256ths). Q6_K's form for two tokens is dear: with the
// others' rates the blocks of such groups were done at 33 us, those of single tokens at 28 (8 tokens, a rank's 64 of 128 experts: 56 us, 53 with its
// own).
void moe_mma_rates(int type, int (&rate)[5]) {
  static const int rates[2][5] = {{256, 272, 288, 320, 416}, {256, 320, 305, 305, 380}};
  for (int i = 0; i < 5; ++i) rate[i] = rates[type == GSQ_TYPE_Q6_K][i];
}

int moe_mma_product(const MoeArgs& a, int type, bool down, cudaStream_t st) {
  DeviceInfo di;
  const int rc = device_info(&di), kind = moe::kind_of(type);
  if (rc != GSQ_OK) return rc;
  moe::Plan p;
  if (!moe::plan_of(kind, down ? a.inter : a.hidden, a.many, di.max_smem_optin, &p)) return GSQ_ERR_UNSUPPORTED;
#define GSQ_MOE_KIND(K) \
  case moe::K: return down ? moe::launch<moe::K, true>(a, p, st) : moe::launch<moe::K, false>(a, p, st);
  switch (kind) {
    GSQ_MOE_KIND(Q4K)
    GSQ_MOE_KIND(Q6K)
    GSQ_MOE_KIND(IQ3S)
    GSQ_MOE_KIND(IQ4XS)
    default: return GSQ_ERR_UNSUPPORTED;
  }
#undef GSQ_MOE_KIND
}

}  // namespace gsq
