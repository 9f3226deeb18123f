// The experts' products on the tensor cores, for the four main types (Q4_K, Q6_K, IQ3_S, IQ4_XS in GGUF order) (sm_100a).
//
// The pairs of a token and one of its experts are gathered by expert, at most 8 to a group (gsq_moe.cu), so that an expert's
// weights are read and decoded once for 8 tokens. A tile is 16 weight rows: 8 gate and the 8 up rows of the same channels, which
// leaves a channel's gate and up sums in one lane, or 16 rows of the down weights. The list of (group, tile) is cut into one
// contiguous range a block, one block an SM.
//
//   * Weights: each warp has a ring of bulk copies of its own (16 rows x 1 or 2 superblocks a stage, one copy a row), filled ahead over
//     tiles and groups, so the stream does not stop where a group ends. Rows of 210- and 110-byte blocks start at any even address:
//     a copy begins at the 16-byte boundary before, and the rows are read at their offset.
//   * Activations: the block takes its group's rows (X, or the activated products), quantises them into shared memory in the order of
//     the tensor-core instruction's B fragment. Columns past the group's are left as they are: they only reach results that are not stored.
//   * Product: mma.sync m16n8k32 on bytes (m16n8k16 for Q6_K, whose sub-scales cover 16 values); a lane decodes exactly its share of
//     the A fragment. Sums leave the instruction on the bit pattern of 1.5 * 2^23, so fma(sum, dA, -1.5 * 2^23 dA) is the exact integer
//     times d * sub-scale without a conversion; the second fma scales by the activations. Q4_K's minima are a product of their
//     own, min [16 rows x 8 slices] times d_x * sum of the quants [8 slices x 8 columns], in three tf32 parts that hold all 24 bits.
//   * Few tiles a block: 2 to 16 warps share a tile along K and add their sums through shared memory in a fixed order.
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
__device__ int g_error = 0;                  // sticky: a wait on a copy gave up (gsq_device_error_flag)

__host__ __device__ constexpr int bs(int kind) { return kind == Q4K ? 144 : kind == Q6K ? 210 : kind == IQ3S ? 110 : 136; }
// Bytes between the rows of a stage: what a copy may take (14 bytes in front, the size to a multiple of 16), with 8 rows' 32 bytes on
// different banks where the row's own length does not do it.
__host__ __device__ constexpr int pitch(int kind, int sbs) {
  return kind == Q4K ? (sbs == 2 ? 288 : 160) : kind == Q6K ? (sbs == 2 ? 480 : 224) : kind == IQ3S ? (sbs == 2 ? 240 : 160) : (sbs == 2 ? 288 : 160);
}
constexpr int GRID_COPIES = 8;               // of IQ3_S's codebook in shared memory, one for lanes l, l + 8, ...
__host__ __device__ constexpr size_t fixed_smem(int kind, int k) {   // all but the ring
  return (size_t)k * 8 + (size_t)k / 32 * 32 + (kind == Q4K ? (size_t)k / 256 * 768 : 0) + (kind == IQ3S ? 512 * 4 * GRID_COPIES : 0) + 2 * WARPS * 512;
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t bar) { asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_row(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
// Gives up after about a second and raises the flag: the sums are then wrong, and nothing waits for ever.
__device__ __forceinline__ void bar_wait(uint32_t bar, uint32_t parity) {
  uint32_t done = 0;
  for (int spin = 0; spin < (1 << 22); ++spin) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return;
  }
  atomicExch(&g_error, 1);
}
__device__ __forceinline__ void warps_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

__device__ __forceinline__ void mma_k32(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint2 b, int init) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y), "r"(init));
}
__device__ __forceinline__ void mma_k16(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t b) {
  asm("mma.sync.aligned.m16n8k16.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5}, {%6}, {%7, %7, %7, %7};"
      : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
      : "r"(a0), "r"(a1), "r"(b), "r"(0));
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

// What a lane (g = lane / 4, t = lane % 4) reads of the staged activations of one superblock.
struct Act {
  const uint8_t* q;        // [slice][column][32 bytes], at this lane's 8 bytes of column g
  const float* d;          // [slice][column], at columns 2 t, 2 t + 1
  const float* mins;       // [part][t][column][2], at this lane's pair
};
__device__ __forceinline__ uint2 act_q(const Act& x, int s) { return *reinterpret_cast<const uint2*>(x.q + 256 * s); }
__device__ __forceinline__ float2 act_d(const Act& x, int s) { return *reinterpret_cast<const float2*>(x.d + 8 * s); }

// acc += (row scale) * (activation scale) * sum, for the four sums of a lane (rows g, g + 8; columns 2 t, 2 t + 1), sums on MAGIC.
__device__ __forceinline__ void scale_sums(float (&acc)[4], const int (&c)[4], float a0, float a1, float2 d) {
  const float m0 = -MAGIC_F * a0, m1 = -MAGIC_F * a1;
  acc[0] = fmaf(fmaf(__int_as_float(c[0]), a0, m0), d.x, acc[0]);
  acc[1] = fmaf(fmaf(__int_as_float(c[1]), a0, m0), d.y, acc[1]);
  acc[2] = fmaf(fmaf(__int_as_float(c[2]), a1, m1), d.x, acc[2]);
  acc[3] = fmaf(fmaf(__int_as_float(c[3]), a1, m1), d.y, acc[3]);
}

// One superblock of 16 rows: b0, b1 = the blocks of rows g and g + 8.
template <int KIND>
__device__ __forceinline__ void superblock(const uint8_t* b0, const uint8_t* b1, const Act& x, int t, const uint32_t* grid, float (&acc)[4]) {
  if constexpr (KIND == Q4K) {
    const uint4 h0 = *reinterpret_cast<const uint4*>(b0), h1 = *reinterpret_cast<const uint4*>(b1);
    const uint32_t sc[2][2] = {{h0.y & 0x3F3F3F3Fu, (h0.w & 0x0F0F0F0Fu) | ((h0.y >> 2) & 0x30303030u)},
                               {h1.y & 0x3F3F3F3Fu, (h1.w & 0x0F0F0F0Fu) | ((h1.y >> 2) & 0x30303030u)}};
    const uint32_t mn[2][2] = {{h0.z & 0x3F3F3F3Fu, ((h0.w >> 4) & 0x0F0F0F0Fu) | ((h0.z >> 2) & 0x30303030u)},
                               {h1.z & 0x3F3F3F3Fu, ((h1.w >> 4) & 0x0F0F0F0Fu) | ((h1.z >> 2) & 0x30303030u)}};
    const float d0 = h2f(h0.x), d1 = h2f(h1.x), n0 = -8388608.0f * d0, n1 = -8388608.0f * d1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint2 q0 = *reinterpret_cast<const uint2*>(b0 + 16 + 32 * j + 8 * t), q1 = *reinterpret_cast<const uint2*>(b1 + 16 + 32 * j + 8 * t);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int s = 2 * j + h;
        int c[4];
        mma_k32(c, (q0.x >> (4 * h)) & 0x0F0F0F0Fu, (q1.x >> (4 * h)) & 0x0F0F0F0Fu, (q0.y >> (4 * h)) & 0x0F0F0F0Fu,
                (q1.y >> (4 * h)) & 0x0F0F0F0Fu, act_q(x, s), MAGIC);
        // the sub-scale as the low byte of 2^23's bits, times d, less 2^23 d: exact
        const float a0 = fmaf(__uint_as_float(prmt(sc[0][s >> 2], 0x4B000000u, 0x7440 | (s & 3))), d0, n0);
        const float a1 = fmaf(__uint_as_float(prmt(sc[1][s >> 2], 0x4B000000u, 0x7440 | (s & 3))), d1, n1);
        scale_sums(acc, c, a0, a1, act_d(x, s));
      }
    }
    // minima: rows g, g + 8 by slices t, t + 4
    auto min_of = [&](uint32_t w) { return __float_as_uint(__uint_as_float(prmt(w, 0x4B000000u, 0x7440 | t)) - 8388608.0f); };
    const uint32_t m0 = min_of(mn[0][0]), m1 = min_of(mn[1][0]), m2 = min_of(mn[0][1]), m3 = min_of(mn[1][1]);
    float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int p = 2; p >= 0; --p) mma_tf32(c, m0, m1, m2, m3, *reinterpret_cast<const float2*>(x.mins + 64 * p));
    const float e0 = -h2f(h0.x >> 16), e1 = -h2f(h1.x >> 16);
    acc[0] = fmaf(e0, c[0], acc[0]);
    acc[1] = fmaf(e0, c[1], acc[1]);
    acc[2] = fmaf(e1, c[2], acc[2]);
    acc[3] = fmaf(e1, c[3], acc[3]);
  } else if constexpr (KIND == IQ4XS) {
    const uint2 h0 = *reinterpret_cast<const uint2*>(b0), h1 = *reinterpret_cast<const uint2*>(b1);
    const float d0 = h2f(h0.x), d1 = h2f(h1.x);
    const uint32_t t0 = reinterpret_cast<const uint32_t*>(c_iq4)[0], t1 = reinterpret_cast<const uint32_t*>(c_iq4)[1],
                   t2 = reinterpret_cast<const uint32_t*>(c_iq4)[2], t3 = reinterpret_cast<const uint32_t*>(c_iq4)[3];
    // 8 indices -> two words of values in the order of the nibbles: value 4 t, 16 + 4 t, 4 t + 1, ... (the activations have that order)
    auto look_up = [&](uint32_t v, uint32_t& lo, uint32_t& hi) {
      const uint32_t s = v & 0x77777777u, pick = ((v >> 1) & 0x44444444u) | 0x32103210u;
      lo = prmt(prmt(t0, t1, s), prmt(t2, t3, s), pick);
      hi = prmt(prmt(t0, t1, s >> 16), prmt(t2, t3, s >> 16), pick >> 16);
    };
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      uint32_t a0, a1, a2, a3;
      look_up(lds32(b0 + 8 + 16 * s + 4 * t), a0, a2);
      look_up(lds32(b1 + 8 + 16 * s + 4 * t), a1, a3);
      int c[4];
      mma_k32(c, a0, a1, a2, a3, act_q(x, s), MAGIC);
      const int l0 = (int)(((h0.y >> (4 * s)) & 15u) | (((h0.x >> (16 + 2 * s)) & 3u) << 4));
      const int l1 = (int)(((h1.y >> (4 * s)) & 15u) | (((h1.x >> (16 + 2 * s)) & 3u) << 4));
      scale_sums(acc, c, d0 * (__int_as_float(MAGIC + l0) - (MAGIC_F + 32.0f)), d1 * (__int_as_float(MAGIC + l1) - (MAGIC_F + 32.0f)), act_d(x, s));
    }
  } else if constexpr (KIND == IQ3S) {
    const float d0 = h2f(lds16(b0)), d1 = h2f(lds16(b1));
    const uint32_t ls0 = lds32h(b0 + 106), ls1 = lds32h(b1 + 106);
    auto value = [&](uint32_t low, uint32_t high, uint32_t signs) {   // index low | high << 8, negated where a sign bit is set
      const uint32_t v = grid[(low | (high << 8)) * GRID_COPIES];
      const uint32_t ones = ((signs & 15u) * 0x00204081u) & 0x01010101u;
      return (v ^ (ones * 255u)) + ones;
    };
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const uint32_t q0 = lds16(b0 + 2 + 8 * s + 2 * t), q1 = lds16(b1 + 2 + 8 * s + 2 * t);
      const uint32_t h0 = b0[66 + s] >> (2 * t), h1 = b1[66 + s] >> (2 * t), g0 = b0[74 + 4 * s + t], g1 = b1[74 + 4 * s + t];
      int c[4];
      mma_k32(c, value(q0 & 255u, h0 & 1u, g0), value(q1 & 255u, h1 & 1u, g1), value(q0 >> 8, (h0 >> 1) & 1u, g0 >> 4),
              value(q1 >> 8, (h1 >> 1) & 1u, g1 >> 4), act_q(x, s), MAGIC);
      const int l0 = 1 + 2 * (int)((ls0 >> (4 * s)) & 15u), l1 = 1 + 2 * (int)((ls1 >> (4 * s)) & 15u);
      scale_sums(acc, c, d0 * (__int_as_float(MAGIC + l0) - MAGIC_F), d1 * (__int_as_float(MAGIC + l1) - MAGIC_F), act_d(x, s));
    }
  } else {
    // value q - 32 (q six bits) as q << 2 with the top bit flipped: four times it, as a signed byte
    const float d0 = 0.25f * h2f(lds16(b0 + 208)), d1 = 0.25f * h2f(lds16(b1 + 208));
    float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      uint32_t h[2][2], l[2][2][2];   // [row][half of 16 bytes], ql: [row][64-value half][half of 16 bytes]
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        h[0][e] = lds32h(b0 + 128 + 32 * n + 16 * e + 4 * t);
        h[1][e] = lds32h(b1 + 128 + 32 * n + 16 * e + 4 * t);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          l[0][r][e] = lds32h(b0 + 64 * n + 32 * r + 16 * e + 4 * t);
          l[1][r][e] = lds32h(b1 + 64 * n + 32 * r + 16 * e + 4 * t);
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {   // slice 4 n + q: nibble q / 2 of ql's half q % 2, bits 2 q of qh
        const int s = 4 * n + q;
        auto word = [&](int row, int e) {
          const uint32_t lo = q < 2 ? l[row][q & 1][e] << 2 : l[row][q & 1][e] >> 2;
          const uint32_t hi = q == 3 ? h[row][e] : h[row][e] << (6 - 2 * q);
          return (lo & 0x3C3C3C3Cu) | ((hi & 0xC0C0C0C0u) ^ 0x80808080u);
        };
        const uint2 b = act_q(x, s);
        int ca[4], cb[4];
        mma_k16(ca, word(0, 0), word(1, 0), b.x);
        mma_k16(cb, word(0, 1), word(1, 1), b.y);
        const uint32_t s0 = lds16(b0 + 192 + 2 * s), s1 = lds16(b1 + 192 + 2 * s);
        const int u0 = (int)(int8_t)s0, v0 = (int)(int8_t)(s0 >> 8), u1 = (int)(int8_t)s1, v1 = (int)(int8_t)(s1 >> 8);
        const float2 d = act_d(x, s);
        part[0] = fmaf((float)(ca[0] * u0 + cb[0] * v0), d.x, part[0]);
        part[1] = fmaf((float)(ca[1] * u0 + cb[1] * v0), d.y, part[1]);
        part[2] = fmaf((float)(ca[2] * u1 + cb[2] * v1), d.x, part[2]);
        part[3] = fmaf((float)(ca[3] * u1 + cb[3] * v1), d.y, part[3]);
      }
    }
    acc[0] = fmaf(d0, part[0], acc[0]);
    acc[1] = fmaf(d0, part[1], acc[1]);
    acc[2] = fmaf(d1, part[2], acc[2]);
    acc[3] = fmaf(d1, part[3], acc[3]);
  }
}

// 8 consecutive activations of a row (piece `piece` of the row), in fp32.
template <bool DOWN>
__device__ __forceinline__ void load_act(const MoeArgs& a, int pair, int piece, float (&v)[8]) {
  if constexpr (DOWN) {
    load8<float, true>(a.h, (int64_t)pair * a.inter + 8 * piece, v);
  } else {
    const int64_t at = (int64_t)(pair / a.top_k) * a.x_stride + 8 * piece;
    if (a.x_dtype == GSQ_F32) {
      if (a.x_vec) load8<float, true>((const float*)a.x, at, v);
      else load8<float, false>((const float*)a.x, at, v);
    } else if (a.x_dtype == GSQ_F16) {
      if (a.x_vec) load8<__half, true>((const __half*)a.x, at, v);
      else load8<__half, false>((const __half*)a.x, at, v);
    } else {
      if (a.x_vec) load8<__nv_bfloat16, true>((const __nv_bfloat16*)a.x, at, v);
      else load8<__nv_bfloat16, false>((const __nv_bfloat16*)a.x, at, v);
    }
  }
}

// 8 values of column `col` into the staged activations. Whole warps call it: four lanes share a slice of 32 values.
template <int KIND>
__device__ __forceinline__ void stage_piece(const float (&v)[8], int piece, int col, uint8_t* q_s, float* d_s, float* min_s) {
  int q[8];
  const float d = moe_quant8(v, q);
  const int s = piece >> 2, p = piece & 3;
  const uint32_t w0 = moe_pack4(q[0], q[1], q[2], q[3]), w1 = moe_pack4(q[4], q[5], q[6], q[7]);
  uint8_t* to = q_s + 256 * s + 32 * col;
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
    int sum = q[0] + q[1] + q[2] + q[3] + q[4] + q[5] + q[6] + q[7];
    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
    if (p == 0) {                        // d * sum in three parts of at most 11 bits
      const float xs = d * (float)sum, hi = __uint_as_float(__float_as_uint(xs) & 0xFFFFE000u), r = xs - hi;
      const float mid = __uint_as_float(__float_as_uint(r) & 0xFFFFE000u);
      float* m = min_s + 192 * (s >> 3) + ((s & 3) * 8 + col) * 2 + ((s >> 2) & 1);
      m[0] = hi;
      m[64] = mid;
      m[128] = r - mid;
    }
  }
  if (p == 0) d_s[8 * s + col] = d;
}

// A block's work on one group: tiles [ta, tb), each by `ks` warps along K (k_of: this warp's superblocks).
struct Segment {
  int ta, tb, log_ks;
};

struct Work {
  int u0, u1, tiles, nsb;      // the block's units; tiles of an expert, superblocks of a row
  __device__ __forceinline__ int first_group() const { return u0 / tiles; }
  __device__ __forceinline__ int last_group() const { return (u1 - 1) / tiles; }
  __device__ __forceinline__ Segment segment(int group) const {
    Segment s;
    s.ta = max(u0 - group * tiles, 0);
    s.tb = min(u1 - group * tiles, tiles);
    // warps to a tile: rounds over the tiles times superblocks of a warp, and one for the sum where warps share a tile
    const int n = s.tb - s.ta;
    int best = 1 << 30;
    s.log_ks = 0;
#pragma unroll
    for (int l = 0; l < 5; ++l) {
      const int cost = ((n + (WARPS >> l) - 1) / (WARPS >> l)) * (((nsb + (1 << l) - 1) >> l) + (l > 0));
      if (cost < best) {
        best = cost;
        s.log_ks = l;
      }
    }
    return s;
  }
};

// Where a warp's stream of weights stands: superblocks sb .. of a tile of a group.
struct Stream {
  int group, expert, tile, sb, k0, k1, step, tb;
  bool live;
  __device__ __forceinline__ void enter(const Work& w, const int4* groups, int warp) {   // the first superblocks of `group` or of one behind it
    for (; group <= w.last_group(); ++group) {
      const Segment s = w.segment(group);
      const int kp = warp & ((1 << s.log_ks) - 1);
      tile = s.ta + (warp >> s.log_ks);
      k0 = (kp * w.nsb) >> s.log_ks;
      k1 = ((kp + 1) * w.nsb) >> s.log_ks;
      step = WARPS >> s.log_ks;
      tb = s.tb;
      sb = k0;
      if (tile < tb && k0 < k1) {
        live = true;
        expert = groups[group].x;
        return;
      }
    }
    live = false;
  }
  __device__ __forceinline__ void next(const Work& w, const int4* groups, int warp, int sbs) {
    sb += sbs;
    if (sb < k1) return;
    sb = k0;
    tile += step;
    if (tile < tb) return;
    ++group;
    enter(w, groups, warp);
  }
};

// DOWN: rows of w2 on the activated products, else gate and up rows of w13 on X. `sbs`: superblocks of a stage; `stages`: of a warp's ring.
template <int KIND, bool DOWN>
__global__ void __launch_bounds__(THREADS, 1) moe_mma_kernel(const MoeArgs a, int sbs, int stages) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int pair_s[8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int k = DOWN ? a.inter : a.hidden, rows = DOWN ? a.hidden : 2 * a.inter;
  const int64_t rb = DOWN ? a.rb2 : a.rb13;
  const uint8_t* const weights = DOWN ? a.w2 : a.w13;
  const int row_pitch = sbs == 2 ? pitch(KIND, 2) : pitch(KIND, 1), stage_bytes = 16 * row_pitch;

  uint8_t* sp = smem;
  uint8_t* q_s = sp;
  sp += (size_t)k * 8;
  float* d_s = reinterpret_cast<float*>(sp);
  sp += (size_t)k / 32 * 32;
  float* min_s = reinterpret_cast<float*>(sp);
  if (KIND == Q4K) sp += (size_t)k / 256 * 768;
  uint32_t* grid_s = reinterpret_cast<uint32_t*>(sp);
  if (KIND == IQ3S) sp += 512 * 4 * GRID_COPIES;
  float4* join_s = reinterpret_cast<float4*>(sp);    // [2][warps][lanes]
  sp += 2 * WARPS * 512;
  uint8_t* ring = sp + (size_t)warp * stages * stage_bytes;
  const uint32_t ring_at = smem_addr(ring), bars = smem_addr(sp + (size_t)WARPS * stages * stage_bytes) + 8 * stages * warp;

  if (lane == 0) {
    for (int s = 0; s < stages; ++s) bar_init(bars + 8 * s);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncwarp();

  const int groups = *a.groups;
  Work w;
  w.tiles = rows >> 4;
  w.nsb = k >> 8;
  const int64_t units = (int64_t)groups * w.tiles;
  w.u0 = (int)(units * blockIdx.x / gridDim.x);
  w.u1 = (int)(units * (blockIdx.x + 1) / gridDim.x);
  if (w.u0 == w.u1) return;

  // lane r < 16 copies row r of a stage
  Stream in{w.first_group(), 0, 0, 0, 0, 0, 0, 0, false};
  in.enter(w, a.group, warp);
  auto issue = [&](int slot) {
    const int n = min(sbs, in.k1 - in.sb);
    const int r = DOWN ? 16 * in.tile + (lane & 15) : 8 * in.tile + (lane & 7) + (lane & 8 ? a.inter : 0);
    const int64_t off = ((int64_t)in.expert * rows + r) * rb + in.sb * bs(KIND);
    const uint32_t bytes = ((uint32_t)(off & 15) + n * bs(KIND) + 15) & ~15u;
    uint32_t total = lane < 16 ? bytes : 0;
    total = __reduce_add_sync(0xFFFFFFFFu, total);
    if (lane == 0) bar_expect(bars + 8 * slot, total);
    __syncwarp();
    if (lane < 16) copy_row(ring_at + slot * stage_bytes + lane * row_pitch, weights + (off & ~(int64_t)15), bytes, bars + 8 * slot);
  };
  int issued = 0, used = 0;
  for (; issued < stages && in.live; ++issued) {
    issue(issued);
    in.next(w, a.group, warp, sbs);
  }
  if (KIND == IQ3S)
    for (int i = tid; i < 512 * GRID_COPIES; i += THREADS) grid_s[i] = g_iq3s[i / GRID_COPIES];

  for (int group = w.first_group(); group <= w.last_group(); ++group) {
    const int4 gr = a.group[group];     // expert, first place in the list, pairs
    const Segment seg = w.segment(group);
    __syncthreads();                    // the group before is done with the activations
    if (tid < gr.z) pair_s[tid] = a.list[gr.y + tid];
    __syncthreads();
    {
      const int per = k >> 3, total = gr.z * per;   // (whole warps: per is a multiple of 32)
      constexpr int U = 2;
      for (int i0 = tid; i0 < total; i0 += U * THREADS) {
        float v[U][8];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = i0 + u * THREADS;
          if (i < total) load_act<DOWN>(a, pair_s[i / per], i % per, v[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = i0 + u * THREADS;
          if (i < total) stage_piece<KIND>(v[u], i % per, i / per, q_s, d_s, min_s);
        }
      }
    }
    __syncthreads();
    const int ks = 1 << seg.log_ks, kp = warp & (ks - 1), slot0 = warp >> seg.log_ks;
    const int k0 = (kp * w.nsb) >> seg.log_ks, k1 = ((kp + 1) * w.nsb) >> seg.log_ks;
    int turn = 0;
    for (int tile = seg.ta + slot0; tile < seg.tb; tile += WARPS >> seg.log_ks) {
      float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int sb = k0; sb < k1; sb += sbs) {
        const int slot = used % stages;
        bar_wait(bars + 8 * slot, (used / stages) & 1);
        // this lane's rows in the stage, at the offset their copies began before them
        const int r0 = DOWN ? 16 * tile + g : 8 * tile + g, r1 = DOWN ? r0 + 8 : r0 + a.inter;
        const int64_t o0 = ((int64_t)gr.x * rows + r0) * rb + sb * bs(KIND), o1 = ((int64_t)gr.x * rows + r1) * rb + sb * bs(KIND);
        const uint8_t* b0 = ring + slot * stage_bytes + g * row_pitch + (KIND == Q4K ? 0 : (int)(o0 & 15));
        const uint8_t* b1 = ring + slot * stage_bytes + (g + 8) * row_pitch + (KIND == Q4K ? 0 : (int)(o1 & 15));
        const int n = min(sbs, k1 - sb);
        for (int i = 0; i < n; ++i) {
          const Act x{q_s + (sb + i) * 2048 + 32 * g + 8 * t, d_s + (sb + i) * 64 + 2 * t, min_s + (sb + i) * 192 + (t * 8 + g) * 2};
          superblock<KIND>(b0 + i * bs(KIND), b1 + i * bs(KIND), x, t, grid_s + (lane & (GRID_COPIES - 1)), acc);
        }
        ++used;
        __syncwarp();                   // all lanes have read the stage
        if (in.live) {
          issue(slot);
          ++issued;
          in.next(w, a.group, warp, sbs);
        }
      }
      if (ks > 1) {
        float4* buf = join_s + turn * WARPS * 32;
        turn ^= 1;                      // (the other buffer's readers have passed this tile's barrier by the next but one)
        buf[warp * 32 + lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        warps_sync(1 + slot0, 32 * ks);
        if (kp == 0) {
          for (int i = 1; i < ks; ++i) {
            const float4 o = buf[(warp + i) * 32 + lane];
            acc[0] += o.x; acc[1] += o.y; acc[2] += o.z; acc[3] += o.w;
          }
        }
      }
      if (kp == 0) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int col = 2 * t + c;
          if (col < gr.z) {
            const int pair = pair_s[col];
            if constexpr (DOWN) {
              float* to = a.part + (int64_t)pair * a.hidden + 16 * tile + g;
              const float wt = a.weights[pair];
              to[0] = wt * acc[c];
              to[8] = wt * acc[2 + c];
            } else {
              a.h[(int64_t)pair * a.inter + 8 * tile + g] = moe_act(a.act, acc[c]) * acc[2 + c];
            }
          }
        }
      }
    }
  }
}

static int kind_of(int type) {
  return type == GSQ_TYPE_Q4_K ? Q4K : type == GSQ_TYPE_Q6_K ? Q6K : type == GSQ_TYPE_IQ3_S ? IQ3S : type == GSQ_TYPE_IQ4_XS ? IQ4XS : -1;
}

// Superblocks of a stage and stages of a warp's ring that fit beside a row length of k: two superblocks a copy where that leaves two
// stages or more, at most four stages. False: too long a row.
static bool ring_of(int kind, int k, int max_smem, int* sbs, int* stages, size_t* smem) {
  const size_t fixed = fixed_smem(kind, k);
  for (int s = kind == Q6K ? 1 : 2; s >= 1; --s) {
    const size_t stage = (size_t)WARPS * (16 * pitch(kind, s) + 8);
    if (fixed + 2 * stage > (size_t)max_smem - 1024) continue;
    const size_t n = ((size_t)max_smem - 1024 - fixed) / stage;
    *sbs = s;
    *stages = (int)(n < 4 ? n : 4);
    *smem = fixed + *stages * stage;
    return true;
  }
  return false;
}

template <int KIND, bool DOWN>
static int launch(const MoeArgs& a, const DeviceInfo& di, cudaStream_t st) {
  int sbs, stages;
  size_t smem;
  if (!ring_of(KIND, DOWN ? a.inter : a.hidden, di.max_smem_optin, &sbs, &stages, &smem)) return GSQ_ERR_UNSUPPORTED;
  GSQ_CUDA_TRY(cudaFuncSetAttribute(moe_mma_kernel<KIND, DOWN>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  moe_mma_kernel<KIND, DOWN><<<di.sm_count, THREADS, smem, st>>>(a, sbs, stages);
  GSQ_CUDA_TRY(cudaGetLastError());
  return GSQ_OK;
}

}  // namespace moe

// Whether the tensor-core kernel takes a product of this type and row length.
bool moe_mma_serves(int type, int k) {
  const int kind = moe::kind_of(type);
  DeviceInfo di;
  int sbs, stages;
  size_t smem;
  return kind >= 0 && device_info(&di) == GSQ_OK && moe::ring_of(kind, k, di.max_smem_optin, &sbs, &stages, &smem);
}

int moe_mma_product(const MoeArgs& a, int type, bool down, cudaStream_t st) {
  DeviceInfo di;
  const int rc = device_info(&di);
  if (rc != GSQ_OK) return rc;
#define GSQ_MOE_KIND(K) \
  case moe::K: return down ? moe::launch<moe::K, true>(a, di, st) : moe::launch<moe::K, false>(a, di, st);
  switch (moe::kind_of(type)) {
    GSQ_MOE_KIND(Q4K)
    GSQ_MOE_KIND(Q6K)
    GSQ_MOE_KIND(IQ3S)
    GSQ_MOE_KIND(IQ4XS)
    default: return GSQ_ERR_UNSUPPORTED;
  }
#undef GSQ_MOE_KIND
}

int moe_error_flag(int* flag) {
  GSQ_CUDA_TRY(cudaMemcpyFromSymbol(flag, moe::g_error, sizeof(int)));
  return GSQ_OK;
}

}  // namespace gsq
