// What the kernels of the mixture-of-experts layer share (gsq_moe.cu, gsq_moe_dot.cu): their arguments, the layout of the
// workspace, the 8-bit form of activations and the gated activations.
#pragma once
#include "gsq_common.cuh"
#include "gsq_quant.cuh"

namespace gsq {

constexpr int MOE_BLOCKS = 256;   // most blocks of a product (one an SM)

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
  // pairs by expert, at most group_max (8 or 16) to a group
  int group_max;
  // more than 4 choices an expert on average, another rank's among them (the host does not see the ids). 64 experts, top 8, with and without: Q4_K
  // 4096 x 2048 40 tokens 226, 204 us, 64 tokens 266, 284, 128 tokens 391, 493; IQ4_XS / Q6_K 5120 x 1280 64 tokens 329, 383. Where they are a quarter of all
  // experts, and the layout comes at a quarter of the tokens: Q4_K 64 tokens 177, 166, 128 tokens 223, 189; IQ4_XS / Q6_K the same within 1 %.
  bool many;
  int rate[5];                 // cost of a tile of a group of 1, 2, up to 4, 8, 16 pairs
  int2* bounds;                // [blocks + 1]: where a block's share of (group, tile) begins: a group, and 65536ths of its tiles
  int blocks;                  // of the products
  int4* group;                 // expert, first place in the list, pairs
  int* list;                   // pairs
};

// Expert of a pair, -1 for one that is not here (negative or past the last).
__device__ __forceinline__ int moe_expert(const MoeArgs& a, int pair) {
  // (not the read-only path: the block that plans may have made the choice itself)
  const int64_t e = a.ids64 ? reinterpret_cast<const long long*>(a.ids)[pair] : (int64_t) reinterpret_cast<const int*>(a.ids)[pair];
  return e >= 0 && e < a.experts ? (int)e : -1;
}

// q = round(127 x / amax), ties away from zero, of 8 of the 32 values that 4 adjacent lanes share; returns the scale amax / 127.
// The quotient is formed with an approximate reciprocal, and whether it reaches the half-integer that it is next to is decided by
// the sign of 127 |x| - half * amax in one fused step, which is exact for 16-bit x (127 x is then exact): the result is that of
// the correctly rounded quotient. (Eight divisions a lane took three times as long: 10 of 16 us of a block's 8 x 5120 activations.)
// NaN or an infinity in the block makes the scale NaN or infinite, and so every product with the block NaN or infinite. Whole warps call it.
__device__ __forceinline__ float moe_quant8(const float (&v)[8], int (&q)[8]) {
  float amax = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) asm("max.NaN.f32 %0, %1, %2;" : "=f"(amax) : "f"(amax), "f"(fabsf(v[e])));
#pragma unroll
  for (int o = 2; o > 0; o >>= 1) asm("max.NaN.f32 %0, %1, %2;" : "=f"(amax) : "f"(amax), "f"(__shfl_xor_sync(0xFFFFFFFFu, amax, o)));
  // 127 x and the reciprocal far from overflow and from 0 (a block of zeros stays zeros: 0 < half * amax)
  float s = 1.0f;
  if (!(amax > 1e-30f && amax < 1e36f)) s = amax >= 1e36f ? 0x1p-20f : 0x1p100f;
  const float top = fmaxf(amax * s, 1e-30f), inv = rcp_approx(top);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float a = 127.0f * fabsf(v[e] * s), on = __fadd_rd(a * inv, 8388608.0f);   // the quotient's floor on 2^23
    const float half = (on - 8388608.0f) + 0.5f;
    const int n = (__float_as_int(on) & 0xFF) + (fmaf(-half, top, a) >= 0.0f);       // (NaN: whatever, the scale is NaN)
    q[e] = v[e] < 0.0f ? -n : n;
  }
  return amax * 0.007874015748f;
}

__device__ __forceinline__ uint32_t moe_pack4(int a, int b, int c, int d) {
  return (uint32_t)(a & 0xFF) | ((uint32_t)(b & 0xFF) << 8) | ((uint32_t)(c & 0xFF) << 16) | ((uint32_t)(d & 0xFF) << 24);
}

// gelu by the complement: 1 + erf(g / sqrt 2) cancels for negative g (a thousandth of the value at -4, all of it from -6 on), and where the
// gates of all 32 values of a block are such, nothing else hides it.
// silu by a rounded division: the approximate one gives 0 for divisors past 2^126, gates from -87.4 to -88.7.
__device__ __forceinline__ float moe_act(int act, float g) {
  return act == GSQ_ACT_SILU ? __fdiv_rn(g, 1.0f + expf(-g)) : 0.5f * g * erfcf(g * -0.70710678118654752f);
}

// A launch that may begin while the kernel before it in the stream still runs: it waits (griddepcontrol.wait) before it reads what that
// kernel writes. What came before that kernel is over by then.
template <typename K, typename... A>
static int moe_launch_behind(K kern, unsigned blocks, unsigned threads, size_t smem, cudaStream_t st, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  GSQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, args...));
  return GSQ_OK;
}

// gsq_moe_dot.cu: the two products for every pair, from xq / xd to h, from hq / hd to part
int moe_dot_gate_up(const MoeArgs& a, int type, cudaStream_t st);
int moe_dot_down(const MoeArgs& a, int type, cudaStream_t st);
// gsq_moe_mma.cu: the same by groups, from xq / xd to h, from h to part
int moe_mma_serves(int type, int k, bool many);
int moe_mma_product(const MoeArgs& a, int type, bool down, cudaStream_t st);
void moe_mma_rates(int type, int (&rate)[5]);   // MoeArgs::rate

}  // namespace gsq
