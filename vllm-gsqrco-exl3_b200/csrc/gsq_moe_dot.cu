// The experts' products, one pair of a token and one of its experts at a time: dp4a over GGUF blocks of all ten types (sm_100a).
//
// Not in the reference's Route L; its stock path for MoE layers runs ggml_moe_a8 / ggml_moe_a8_vec
// (plugin/vllm_gguf_plugin/csrc/gguf/moe.cuh, moe_vec.cuh).
//
// A warp owns one channel of a pair: the gate and the up row of that channel (gate / up product), or two rows of the down
// product. Lane l takes slices l, l + 32, ... of 32 values, decodes them and dots them with the 8-bit activations of its pair:
// integer sums per sub-scale, scaled in fp32.
#include "gsq_f1_codec.cuh"
#include "gsq_moe.cuh"
#include "gsq_tables.h"

namespace gsq {

enum { MD_Q4K = 10, MD_Q6K = 11, MD_IQ3S = 12, MD_IQ4XS = 13 };   // beside the F1_* kinds of gsq_f1_codec.cuh

static __device__ const uint32_t g_md_iq3s_grid[512] = GSQ_IQ3S_GRID_INIT;
static __constant__ __align__(16) int8_t c_md_iq4nl[16] = GSQ_IQ4NL_VALUES_INIT;

__host__ __device__ constexpr int md_block_bytes(int kind) {
  return kind == MD_Q4K ? 144 : kind == MD_Q6K ? 210 : kind == MD_IQ3S ? 110 : kind == MD_IQ4XS ? 136 : f1_block_bytes(kind);
}

__device__ __forceinline__ uint32_t md_u32(const uint8_t* p) { return ldg_stream_u16(p) | (ldg_stream_u16(p + 2) << 16); }

// The product of slice s of the superblock at b with 32 activations: words u, scale d8.
template <int KIND>
__device__ __forceinline__ float md_dot(const uint8_t* b, int s, const int (&u)[8], float d8) {
  if constexpr (KIND < 10) {
    Raw<KIND> raw;
    raw.fetch(b, s);
    Slice<KIND> sl;
    sl.decode(raw, s);
    int grp[2];
    return sl.template dot<false>(u, d8, grp);
  } else {
    int w[8], s0 = 0, s1 = 0;
    if constexpr (KIND == MD_Q4K) {
      const uint32_t dd = md_u32(b);
      const int j = s & 3;
      uint32_t sc = ldg_stream_u8(b + 4 + j), mn = ldg_stream_u8(b + 8 + j);
      if (s < 4) {
        sc &= 63u;
        mn &= 63u;
      } else {
        const uint32_t t = ldg_stream_u8(b + 12 + j);
        sc = (t & 15u) | ((sc >> 6) << 4);
        mn = (t >> 4) | ((mn >> 6) << 4);
      }
      int sum = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        w[e] = (int)((ldg_stream_u32(b + 16 + 32 * (s >> 1) + 4 * e) >> (4 * (s & 1))) & 0x0F0F0F0Fu);
        s0 = dp4a(w[e], u[e], s0);
        sum = dp4a(0x01010101, u[e], sum);
      }
      return d8 * (h2f(dd) * (float)(s0 * (int)sc) - h2f(dd >> 16) * (float)(sum * (int)mn));
    } else if constexpr (KIND == MD_Q6K) {
      const int n = s >> 2, r = s & 3;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t lo = (md_u32(b + 64 * n + 32 * (r & 1) + 4 * e) >> (4 * (r >> 1))) & 0x0F0F0F0Fu;
        const uint32_t hi = (md_u32(b + 128 + 32 * n + 4 * e) >> (2 * r)) & 0x03030303u;
        w[e] = (int)((((lo | (hi << 4)) | 0x80808080u) - 0x20202020u) ^ 0x80808080u);   // each byte less 32
        if (e < 4) s0 = dp4a(w[e], u[e], s0);
        else s1 = dp4a(w[e], u[e], s1);
      }
      const uint32_t sc = ldg_stream_u16(b + 192 + 2 * s);
      return d8 * h2f(ldg_stream_u16(b + 208)) * (float)(s0 * (int)(int8_t)sc + s1 * (int)(int8_t)(sc >> 8));
    } else if constexpr (KIND == MD_IQ4XS) {
      const uint32_t ls = ((ldg_stream_u8(b + 4 + (s >> 1)) >> (4 * (s & 1))) & 15u) | (((ldg_stream_u16(b + 2) >> (2 * s)) & 3u) << 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t v = ldg_stream_u32(b + 8 + 16 * s + 4 * e);
        uint32_t lo = 0, hi = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          lo |= (uint32_t)(uint8_t)c_md_iq4nl[(v >> (8 * c)) & 15u] << (8 * c);
          hi |= (uint32_t)(uint8_t)c_md_iq4nl[(v >> (8 * c + 4)) & 15u] << (8 * c);
        }
        s0 = dp4a((int)lo, u[e], s0);
        s0 = dp4a((int)hi, u[4 + e], s0);
      }
      return d8 * h2f(ldg_stream_u16(b)) * (float)(s0 * ((int)ls - 32));
    } else {
      const uint32_t qh = ldg_stream_u8(b + 66 + s), ls = (ldg_stream_u8(b + 106 + (s >> 1)) >> (4 * (s & 1))) & 15u;
      const uint32_t sg = md_u32(b + 74 + 4 * s);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t g = g_md_iq3s_grid[ldg_stream_u8(b + 2 + 8 * s + e) | (((qh >> e) & 1u) << 8)];
        s0 = dp4a(apply_signs4(g, sg >> (4 * e)), u[e], s0);
      }
      return d8 * h2f(ldg_stream_u16(b)) * (float)(s0 * (1 + 2 * (int)ls));
    }
  }
}

// Products of two rows with one 8-bit vector of k values, summed over the warp.
template <int KIND>
__device__ __forceinline__ float2 md_two_rows(const uint8_t* r0, const uint8_t* r1, int k, const int8_t* q, const float* d, int lane) {
  float2 acc = make_float2(0.0f, 0.0f);
  for (int sl = lane; sl < k >> 5; sl += 32) {
    const int4 ua = __ldg(reinterpret_cast<const int4*>(q + 32 * sl)), ub = __ldg(reinterpret_cast<const int4*>(q + 32 * sl + 16));
    const int u[8] = {ua.x, ua.y, ua.z, ua.w, ub.x, ub.y, ub.z, ub.w};
    const float d8 = __ldg(d + sl);
    const int64_t at = (int64_t)(sl >> 3) * md_block_bytes(KIND);
    acc.x += md_dot<KIND>(r0 + at, sl & 7, u, d8);
    acc.y += md_dot<KIND>(r1 + at, sl & 7, u, d8);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    acc.x += __shfl_xor_sync(0xFFFFFFFFu, acc.x, o);
    acc.y += __shfl_xor_sync(0xFFFFFFFFu, acc.y, o);
  }
  return acc;
}

constexpr int MD_WARPS = 8;

template <int KIND>
__global__ void __launch_bounds__(MD_WARPS * 32) moe_dot_gate_up_kernel(const MoeArgs a) {
  const int lane = threadIdx.x & 31, c = blockIdx.x * MD_WARPS + (threadIdx.x >> 5);
  for (int pair = blockIdx.y; pair < a.m * a.top_k; pair += gridDim.y) {
    const int e = moe_expert(a, pair), t = pair / a.top_k;
    if (e < 0) continue;
    const uint8_t* g = a.w13 + ((int64_t)e * 2 * a.inter + c) * a.rb13;
    const float2 p = md_two_rows<KIND>(g, g + a.inter * a.rb13, a.hidden, a.xq + (int64_t)t * a.hidden, a.xd + (int64_t)t * (a.hidden >> 5), lane);
    if (lane == 0) a.h[(int64_t)pair * a.inter + c] = moe_act(a.act, p.x) * p.y;
  }
}

template <int KIND>
__global__ void __launch_bounds__(MD_WARPS * 32) moe_dot_down_kernel(const MoeArgs a) {
  const int lane = threadIdx.x & 31, r = 2 * (blockIdx.x * MD_WARPS + (threadIdx.x >> 5));
  for (int pair = blockIdx.y; pair < a.m * a.top_k; pair += gridDim.y) {
    const int e = moe_expert(a, pair);
    if (e < 0) continue;
    const uint8_t* w = a.w2 + ((int64_t)e * a.hidden + r) * a.rb2;
    const float2 p = md_two_rows<KIND>(w, w + a.rb2, a.inter, a.hq + (int64_t)pair * a.inter, a.hd + (int64_t)pair * (a.inter >> 5), lane);
    const float wt = a.weights[pair];
    if (lane == 0) *reinterpret_cast<float2*>(a.part + (int64_t)pair * a.hidden + r) = make_float2(wt * p.x, wt * p.y);
  }
}

#define GSQ_MD_TYPES(CASE)                                                                                              \
  CASE(GSQ_TYPE_Q4_K, MD_Q4K) CASE(GSQ_TYPE_Q6_K, MD_Q6K) CASE(GSQ_TYPE_IQ3_S, MD_IQ3S) CASE(GSQ_TYPE_IQ4_XS, MD_IQ4XS) \
  CASE(GSQ_TYPE_Q2_K, F1_Q2K) CASE(GSQ_TYPE_IQ2_XXS, F1_IQ2XXS) CASE(GSQ_TYPE_IQ2_XS, F1_IQ2XS)                          \
  CASE(GSQ_TYPE_IQ2_S, F1_IQ2S) CASE(GSQ_TYPE_IQ3_XXS, F1_IQ3XXS) CASE(GSQ_TYPE_IQ1_M, F1_IQ1M)

int moe_dot_gate_up(const MoeArgs& a, int type, cudaStream_t st) {
  const dim3 grid(a.inter / MD_WARPS, (unsigned)(a.m * a.top_k < 65535 ? a.m * a.top_k : 65535));
  switch (type) {
#define CASE(T, K) \
  case T: moe_dot_gate_up_kernel<K><<<grid, MD_WARPS * 32, 0, st>>>(a); break;
    GSQ_MD_TYPES(CASE)
#undef CASE
    default: return GSQ_ERR_UNSUPPORTED;
  }
  GSQ_CUDA_TRY(cudaGetLastError());
  return GSQ_OK;
}

int moe_dot_down(const MoeArgs& a, int type, cudaStream_t st) {
  const dim3 grid(a.hidden / (2 * MD_WARPS), (unsigned)(a.m * a.top_k < 65535 ? a.m * a.top_k : 65535));
  switch (type) {
#define CASE(T, K) \
  case T: moe_dot_down_kernel<K><<<grid, MD_WARPS * 32, 0, st>>>(a); break;
    GSQ_MD_TYPES(CASE)
#undef CASE
    default: return GSQ_ERR_UNSUPPORTED;
  }
  GSQ_CUDA_TRY(cudaGetLastError());
  return GSQ_OK;
}

}  // namespace gsq
