// What the kernels of the mixture-of-experts layer share (gsq_moe.cu, gsq_moe_dot.cu): their arguments, the layout of the
// workspace, the 8-bit form of activations and the gated activations.
#pragma once
#include "gsq_common.cuh"
#include "gsq_quant.cuh"

namespace gsq {

struct MoeArgs {
  const uint8_t *w13, *w2;     // [experts][2 inter][row bytes], [experts][hidden][row bytes], GGUF order
  int64_t rb13, rb2;           // bytes of a row
  int experts, hidden, inter;
  int act;                     // GSQ_ACT_*
  int m, top_k;                // tokens, choices of each; a "pair" is token * top_k + choice
  const void* x;
  int x_dtype, x_vec;          // x_vec: rows 16-byte aligned
  int64_t x_stride;
  const float* weights;        // [m][top_k]
  const void* ids;             // [m][top_k], int32 or int64
  int ids64;
  void* y;                     // [m][hidden] in x_dtype
  int64_t y_stride;
  // workspace
  int8_t *xq, *hq;             // 8-bit activations: [m][hidden], [pairs][inter]
  float *xd, *hd;              // their scales, one per 32 values
  float* h;                    // [pairs][inter]: act(gate) * up
  float* part;                 // [pairs][hidden]: weight times down product
  // pairs by expert, at most 8 to a group
  int* groups;                 // how many
  int4* group;                 // expert, first place in the list, pairs
  int* list;                   // pairs
};

// Expert of a pair, -1 for one that is not here (negative or past the last).
__device__ __forceinline__ int moe_expert(const MoeArgs& a, int pair) {
  const int64_t e = a.ids64 ? __ldg(reinterpret_cast<const long long*>(a.ids) + pair) : (int64_t)__ldg(reinterpret_cast<const int*>(a.ids) + pair);
  return e >= 0 && e < a.experts ? (int)e : -1;
}

// q = round(127 x / amax), ties away from zero, of 8 of the 32 values that 4 adjacent lanes share; returns the scale amax / 127.
// The product 127 x is exact for 16-bit x, so that a quotient that is half an integer is recognised (x / (amax / 127) rounds
// twice before it rounds to an integer). NaN or an infinity in the block makes the scale NaN or infinite, and so the product NaN.
// Whole warps call it.
__device__ __forceinline__ float moe_quant8(const float (&v)[8], int (&q)[8]) {
  float amax = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) asm("max.NaN.f32 %0, %1, %2;" : "=f"(amax) : "f"(amax), "f"(fabsf(v[e])));
#pragma unroll
  for (int o = 2; o > 0; o >>= 1) asm("max.NaN.f32 %0, %1, %2;" : "=f"(amax) : "f"(amax), "f"(__shfl_xor_sync(0xFFFFFFFFu, amax, o)));
  const float s = amax > 1e36f ? 0x1p-10f : 1.0f, den = amax * s;   // 127 x stays finite
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float t = amax > 0.0f ? __fdiv_rn(127.0f * (v[e] * s), den) : 0.0f;
    q[e] = (int)roundf(t);                                          // (NaN becomes 0)
  }
  return __fdiv_rn(amax, 127.0f);
}

__device__ __forceinline__ uint32_t moe_pack4(int a, int b, int c, int d) {
  return (uint32_t)(a & 0xFF) | ((uint32_t)(b & 0xFF) << 8) | ((uint32_t)(c & 0xFF) << 16) | ((uint32_t)(d & 0xFF) << 24);
}

__device__ __forceinline__ float moe_act(int act, float g) {
  return act == GSQ_ACT_SILU ? __fdividef(g, 1.0f + expf(-g)) : 0.5f * g * (1.0f + erff(g * 0.70710678118654752f));
}

// gsq_moe_dot.cu: the two products for every pair, from xq / xd to h, from hq / hd to part
int moe_dot_gate_up(const MoeArgs& a, int type, cudaStream_t st);
int moe_dot_down(const MoeArgs& a, int type, cudaStream_t st);
// gsq_moe_mma.cu: the same by groups, from x to h, from h to part
bool moe_mma_serves(int type, int k);
int moe_mma_product(const MoeArgs& a, int type, bool down, cudaStream_t st);

}  // namespace gsq
