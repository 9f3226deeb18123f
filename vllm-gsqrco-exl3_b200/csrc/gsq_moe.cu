// Mixture-of-experts layer over GGUF-quantised experts for a few tokens (sm_100a): the router's choice, the pairs of a token and
// an expert gathered by expert, the weighted sum, the host side. The products are in gsq_moe_mma.cu (the four main types) and
// gsq_moe_dot.cu (the others).
//
//   choice   s = softmax(logits) or sigmoid(logits); the top_k experts of largest logit (of largest s + bias where there is a
//            bias), ties to the lowest number; weights s (/ their sum) * scale
//   layer    y = sum over the choices of weight * W2[e] q8(act(W13[e][gate] q8(x)) * (W13[e][up] q8(x)))
//
// q8: 32 values to a 32-bit scale (moe_quant8). Sums in fp32; the activated product is rounded once, to its 8 bits, the result
// once, to X's type. An expert whose logit is -inf or NaN is never chosen, and a choice that is not there (-1) adds nothing:
// a token without experts gets zeros.
#include "gsq_moe.cuh"

namespace gsq {

// Larger key = larger score; 0 = not to be chosen.
__device__ __forceinline__ uint32_t score_key(float v) {
  if (!(v > -INFINITY)) return 0;
  const uint32_t b = __float_as_uint(v + 0.0f);   // (-0 and 0 are the same score)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

constexpr int ROUTE_PER_LANE = GSQ_MOE_MAX_EXPERTS / 32;

struct RouteArgs {
  const void* logits;
  int dtype;
  int64_t stride;
  int m, experts, top_k, scoring, renormalize;
  const float* bias;
  float scale;
  float* weights;
  int32_t* ids;
};

// Scores and keys of a token, one warp: lane l holds experts l, l + 32, ...
template <int PER_LANE>
__device__ __forceinline__ void route_scores(const RouteArgs& a, int token, int lane, float (&s)[PER_LANE], uint32_t (&key)[PER_LANE]) {
  float top = -INFINITY;
  // (one branch on the type around all loads: they are under way together)
  const int64_t row = token * a.stride;
  if (a.dtype == GSQ_F32) {
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) s[i] = lane + 32 * i < a.experts ? reinterpret_cast<const float*>(a.logits)[row + lane + 32 * i] : -INFINITY;
  } else {
    uint16_t raw[PER_LANE];
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) raw[i] = lane + 32 * i < a.experts ? reinterpret_cast<const uint16_t*>(a.logits)[row + lane + 32 * i] : 0;
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i)
      s[i] = lane + 32 * i >= a.experts ? -INFINITY
             : a.dtype == GSQ_F16       ? __half2float(__ushort_as_half(raw[i]))
                                        : __uint_as_float((uint32_t)raw[i] << 16);
  }
#pragma unroll
  for (int i = 0; i < PER_LANE; ++i) {
    const float z = s[i];
    s[i] = isnan(z) ? -INFINITY : fminf(z, 3.402823466e38f);   // experts at +inf share the weight
    key[i] = score_key(s[i]);
    top = fmaxf(top, s[i]);
  }
  float sum = 1.0f;
  if (a.scoring == GSQ_MOE_SOFTMAX) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) {
      s[i] = key[i] ? expf(s[i] - top) : 0.0f;
      sum += s[i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  } else {
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) s[i] = key[i] ? __fdiv_rn(1.0f, 1.0f + expf(-s[i])) : 0.0f;
  }
  if (sum > 0.0f) {
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) s[i] = __fdiv_rn(s[i], sum);
  }
  if (a.bias) {
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i)
      if (key[i]) key[i] = score_key(s[i] + a.bias[lane + 32 * i]);
  }
}

// One warp, one token. Each lane puts its experts in order (larger key first, lower number first among equals); each round takes the
// largest of the lanes' first ones, the lowest number among equals, and its lane goes on to its next.
template <int PER_LANE>
__device__ __forceinline__ void route_token(const RouteArgs& a, int token, int lane) {
  float s[PER_LANE];
  uint32_t key[PER_LANE];
  route_scores<PER_LANE>(a, token, lane, s, key);
  uint32_t first[PER_LANE];
  int at[PER_LANE];
#pragma unroll
  for (int i = 0; i < PER_LANE; ++i) {
    first[i] = key[i];
    at[i] = i;
  }
  if constexpr (PER_LANE <= 8) {
#pragma unroll
    for (int i = 1; i < PER_LANE; ++i)
#pragma unroll
      for (int j = i; j > 0; --j)
        if (first[j] > first[j - 1]) {             // (insertion: equal ones stay in order)
          const uint32_t k = first[j];
          first[j] = first[j - 1];
          first[j - 1] = k;
          const int n = at[j];
          at[j] = at[j - 1];
          at[j - 1] = n;
        }
  }
  int id = -1;                                     // lane r keeps round r's choice
  for (int r = 0; r < a.top_k; ++r) {
    if constexpr (PER_LANE > 8) {                  // (too many to put in order: the largest left to the front each time)
#pragma unroll
      for (int i = PER_LANE - 1; i > 0; --i)
        if (first[i] > first[i - 1] || (first[i] == first[i - 1] && at[i] < at[i - 1])) {
          const uint32_t k = first[i];
          first[i] = first[i - 1];
          first[i - 1] = k;
          const int n = at[i];
          at[i] = at[i - 1];
          at[i - 1] = n;
        }
    }
    const uint32_t best = __reduce_max_sync(0xFFFFFFFFu, first[0]);
    if (best == 0) break;
    const uint32_t e = __reduce_min_sync(0xFFFFFFFFu, first[0] == best ? (uint32_t)(lane + 32 * at[0]) : 0xFFFFFFFFu);
    if ((e & 31) == (uint32_t)lane) {
#pragma unroll
      for (int i = 1; i < PER_LANE; ++i) {
        first[i - 1] = first[i];
        at[i - 1] = at[i];
      }
      first[PER_LANE - 1] = 0;
    }
    if (lane == r) id = (int)e;
  }
  float mine = 0.0f, total = 0.0f;
#pragma unroll
  for (int i = 0; i < PER_LANE; ++i) {
    const float v = __shfl_sync(0xFFFFFFFFu, s[i], id & 31);
    if (id >= 0 && (id >> 5) == i) mine = v;
  }
  for (int r = 0; r < a.top_k; ++r) total += __shfl_sync(0xFFFFFFFFu, mine, r);
  if (lane < a.top_k) {
    if (a.renormalize) mine = total > 0.0f ? __fdiv_rn(mine, total) : 0.0f;
    a.weights[(int64_t)token * a.top_k + lane] = mine * a.scale;
    a.ids[(int64_t)token * a.top_k + lane] = id;
  }
}

template <int PER_LANE>
__global__ void __launch_bounds__(128) moe_route_kernel(const RouteArgs a) {
  const int token = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (token < a.m) route_token<PER_LANE>(a, token, threadIdx.x & 31);
}

static int launch_route(const RouteArgs& a, cudaStream_t st) {
  const unsigned grid = (unsigned)(((int64_t)a.m + 3) / 4);
  if (a.experts <= 64) moe_route_kernel<2><<<grid, 128, 0, st>>>(a);
  else if (a.experts <= 256) moe_route_kernel<8><<<grid, 128, 0, st>>>(a);
  else moe_route_kernel<ROUTE_PER_LANE><<<grid, 128, 0, st>>>(a);
  GSQ_CUDA_TRY(cudaGetLastError());
  return GSQ_OK;
}

// Rows of k values -> 8-bit form. One thread takes 8 values; `i`: which.
template <typename T, bool VEC>
__device__ __forceinline__ void quant_piece(const void* x, int64_t stride, int64_t rows, int k, int8_t* q8, float* d8, int64_t i) {
  const int per_row = k >> 3;
  const int64_t row = i / per_row;
  const int c = (int)(i - row * per_row);
  float v[8] = {};
  if (row < rows) load8<T, VEC>(reinterpret_cast<const T*>(x), row * stride + 8 * c, v);
  int q[8];
  const float d = moe_quant8(v, q);
  if (row < rows) {
    *reinterpret_cast<uint2*>(q8 + row * k + 8 * c) = make_uint2(moe_pack4(q[0], q[1], q[2], q[3]), moe_pack4(q[4], q[5], q[6], q[7]));
    if ((c & 3) == 0) d8[row * (k >> 5) + (c >> 2)] = d;
  }
}
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) moe_quant_kernel(const void* x, int64_t stride, int64_t rows, int k, int8_t* q8, float* d8) {
  quant_piece<T, VEC>(x, stride, rows, k, q8, d8, (int64_t)blockIdx.x * 256 + threadIdx.x);
}

static int launch_quant(const void* x, int dtype, int vec, int64_t stride, int64_t rows, int k, int8_t* q8, float* d8, cudaStream_t st) {
  const unsigned grid = (unsigned)((rows * (k >> 3) + 255) / 256);
  if (dtype == GSQ_F32) {
    if (vec) moe_quant_kernel<float, true><<<grid, 256, 0, st>>>(x, stride, rows, k, q8, d8);
    else moe_quant_kernel<float, false><<<grid, 256, 0, st>>>(x, stride, rows, k, q8, d8);
  } else if (dtype == GSQ_F16) {
    if (vec) moe_quant_kernel<__half, true><<<grid, 256, 0, st>>>(x, stride, rows, k, q8, d8);
    else moe_quant_kernel<__half, false><<<grid, 256, 0, st>>>(x, stride, rows, k, q8, d8);
  } else {
    if (vec) moe_quant_kernel<__nv_bfloat16, true><<<grid, 256, 0, st>>>(x, stride, rows, k, q8, d8);
    else moe_quant_kernel<__nv_bfloat16, false><<<grid, 256, 0, st>>>(x, stride, rows, k, q8, d8);
  }
  GSQ_CUDA_TRY(cudaGetLastError());
  return GSQ_OK;
}

// y = sum of a token's parts, in the order of its choices.
constexpr int COMBINE_THREADS = 64;               // (a token's 2048 values on 8 SMs)
__global__ void __launch_bounds__(COMBINE_THREADS) moe_combine_kernel(const MoeArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int per_row = a.hidden >> 2;
  const int64_t i = (int64_t)blockIdx.x * COMBINE_THREADS + threadIdx.x, t = i / per_row;
  if (t >= a.m) return;
  const int c = 4 * (int)(i - t * per_row);
  float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  constexpr int U = 8;                            // parts under way together
  for (int r0 = 0; r0 < a.top_k; r0 += U) {
    bool here[U];
    float4 p[U];
#pragma unroll
    for (int u = 0; u < U; ++u) here[u] = r0 + u < a.top_k && moe_expert(a, (int)(t * a.top_k) + r0 + u) >= 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
      p[u] = here[u] ? __ldcg(reinterpret_cast<const float4*>(a.part + (t * a.top_k + r0 + u) * a.hidden + c)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (here[u]) {
        s.x += p[u].x; s.y += p[u].y; s.z += p[u].z; s.w += p[u].w;
      }
  }
  const int64_t at = t * a.y_stride + c;
  store_out_dyn(a.y, a.x_dtype, at, s.x);
  store_out_dyn(a.y, a.x_dtype, at + 1, s.y);
  store_out_dyn(a.y, a.x_dtype, at + 2, s.z);
  store_out_dyn(a.y, a.x_dtype, at + 3, s.w);
}

// What a group costs: its tiles, at moe_mma_rates' rates.
// A block that goes on to another group stages its columns first and starts its pipelines anew: counted as `lead` tiles in front of the
// group's own, one for each pair. (8 experts with 7 tokens on average, 148 blocks: the few that have the end of one group and the
// beginning of the next were done at 47 us, the others at 39. The layer with no lead, a quarter, a half, one tile a pair: 72.2, 70.8, 67.2,
// 62.5 us; 64 tokens of 64 experts: 275, 271, 270, 273.)
struct GroupCost {
  const int* rate;
  int tiles;                                      // of a group: the mean of the two products'
  __device__ __forceinline__ int of_tiles(int n) const { return rate[n <= 2 ? n - 1 : n <= 4 ? 2 : n <= 8 ? 3 : 4]; }
  __device__ __forceinline__ int lead(int n) const { return of_tiles(n) * n / tiles; }
  __device__ __forceinline__ int of(int n) const { return of_tiles(n) + lead(n); }
};

// Pairs by expert: group, list, bounds. Block 0; PER_LANE > 0: it makes the choice first (few tokens). An expert's pairs stay in
// their order, so that the same ones share a group every time (a group's size decides the order of its sums). Everything behind it
// waits for it, so it is kept short: per warp of pairs the equal ones are found by matching, and the rest are sums over the
// warps, the experts, and a search per block of the products.
constexpr int PLAN_THREADS = 1024, PLAN_WARPS = PLAN_THREADS / 32;
template <int PER_LANE>
__global__ void __launch_bounds__(PLAN_THREADS) moe_plan_kernel(const MoeArgs a, const RouteArgs r) {
  __shared__ uint8_t of_warp[PLAN_WARPS][GSQ_MOE_MAX_EXPERTS];   // an expert's pairs among a warp's 32
  __shared__ int place[GSQ_MOE_MAX_EXPERTS], cost_upto[GSQ_MOE_MAX_EXPERTS], group_upto[GSQ_MOE_MAX_EXPERTS];
  __shared__ uint8_t last_of[GSQ_MOE_MAX_EXPERTS];               // pairs of an expert's last group, where it is not a full one
  __shared__ int3 warp_sum[PLAN_WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, pairs = a.m * a.top_k, experts = a.experts;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (blockIdx.x > 0) {                                          // the other blocks quantise X meanwhile
    const int64_t i = (int64_t)(blockIdx.x - 1) * PLAN_THREADS + tid;
    if (a.x_dtype == GSQ_F32) {
      if (a.x_vec) quant_piece<float, true>(a.x, a.x_stride, a.m, a.hidden, a.xq, a.xd, i);
      else quant_piece<float, false>(a.x, a.x_stride, a.m, a.hidden, a.xq, a.xd, i);
    } else if (a.x_dtype == GSQ_F16) {
      if (a.x_vec) quant_piece<__half, true>(a.x, a.x_stride, a.m, a.hidden, a.xq, a.xd, i);
      else quant_piece<__half, false>(a.x, a.x_stride, a.m, a.hidden, a.xq, a.xd, i);
    } else {
      if (a.x_vec) quant_piece<__nv_bfloat16, true>(a.x, a.x_stride, a.m, a.hidden, a.xq, a.xd, i);
      else quant_piece<__nv_bfloat16, false>(a.x, a.x_stride, a.m, a.hidden, a.xq, a.xd, i);
    }
    return;
  }
  const int warps = min((pairs + 31) >> 5, PLAN_WARPS);           // that have pairs
  for (int w = 0; w < warps; ++w)
    if (tid < experts) of_warp[w][tid] = 0;
  if constexpr (PER_LANE > 0)
    for (int t = warp; t < a.m; t += PLAN_WARPS) route_token<PER_LANE>(r, t, lane);
  __syncthreads();

  const bool once = pairs <= PLAN_THREADS;
  int expert = -1, rank = 0, n = 0;
  if (once) {
    if (warp < warps) {
      expert = tid < pairs ? moe_expert(a, tid) : -1;
      const uint32_t same = __match_any_sync(0xFFFFFFFFu, expert);
      rank = __popc(same & ((1u << lane) - 1));
      if (expert >= 0 && rank == 0) of_warp[warp][expert] = (uint8_t)__popc(same);
    }
    __syncthreads();
    if (tid < experts)
      for (int w = 0; w < warps; ++w) n += of_warp[w][tid];
  } else {
    place[tid] = 0;
    __syncthreads();
    for (int p = tid; p < pairs; p += PLAN_THREADS) {
      const int e = moe_expert(a, p);
      if (e >= 0) atomicAdd(&place[e], 1);
    }
    __syncthreads();
    n = place[tid];
    __syncthreads();
  }
  // sums over the experts before: pairs, groups, cost
  const int most = a.group_max, most_bits = most == 8 ? 3 : 4, g = (n + most - 1) >> most_bits;
  const GroupCost group_cost{a.rate, (a.inter >> 4) + (a.hidden >> 5)};
  const int full = group_cost.of(most), last = n & (most - 1), cost = (n >> most_bits) * full + (last ? group_cost.of(last) : 0);
  int3 upto = make_int3(n, g, cost);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xFFFFFFFFu, upto.x, o), y = __shfl_up_sync(0xFFFFFFFFu, upto.y, o), z = __shfl_up_sync(0xFFFFFFFFu, upto.z, o);
    if (lane >= o) {
      upto.x += x;
      upto.y += y;
      upto.z += z;
    }
  }
  if (lane == 31) warp_sum[warp] = upto;
  __syncthreads();
  const int3 other = warp_sum[lane];
  const uint32_t mine = 0xFFFFFFFFu;
  upto.x += __reduce_add_sync(mine, lane < warp ? other.x : 0);
  upto.y += __reduce_add_sync(mine, lane < warp ? other.y : 0);
  upto.z += __reduce_add_sync(mine, lane < warp ? other.z : 0);
  const int groups = __reduce_add_sync(mine, other.y), total = __reduce_add_sync(mine, other.z);
  place[tid] = upto.x - n;
  cost_upto[tid] = upto.z;
  group_upto[tid] = upto.y;
  last_of[tid] = (uint8_t)last;
  for (int i = 0; i < g; ++i) a.group[upto.y - g + i] = make_int4(tid, upto.x - n + most * i, min(most, n - most * i), 0);
  __syncthreads();

  // block b of the products begins at cost total * b / blocks: in the first expert whose groups end behind that
  for (int b = tid; b <= a.blocks; b += PLAN_THREADS) {
    int2 at = make_int2(groups, 0);
    if (b < a.blocks && total > 0) {
      const int target = (int)((uint32_t)total * b / a.blocks);   // (total: below 2^22, 5120 groups; b up to 2^8)
      int lo = 0, hi = experts - 1;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (cost_upto[mid] > target) hi = mid;
        else lo = mid + 1;
      }
      // its groups: full ones, then the rest
      const int first = lo ? group_upto[lo - 1] : 0, before = lo ? cost_upto[lo - 1] : 0, in = target - before;
      const int i = min(in / full, group_upto[lo] - first - 1), rest = in - i * full;
      const int size = first + i + 1 < group_upto[lo] || !last_of[lo] ? most : last_of[lo];
      // rest < group_cost.of(size): below 65536, so that the boundary lies in the group
      at = make_int2(first + i, (max(rest - group_cost.lead(size), 0) << 16) / group_cost.of_tiles(size));
    }
    a.bounds[b] = at;
  }
  if (once) {
    if (expert >= 0) {
      for (int w = 0; w < warp; ++w) rank += of_warp[w][expert];
      a.list[place[expert] + rank] = tid;
    }
    return;
  }
  for (int p0 = 0; p0 < pairs; p0 += PLAN_THREADS) {
    const int p = p0 + tid, e = p < pairs ? moe_expert(a, p) : -1;
    for (int i = lane; i < experts; i += 32) of_warp[warp][i] = 0;
    __syncwarp();
    const uint32_t same = __match_any_sync(0xFFFFFFFFu, e);
    if (e >= 0 && lane == __ffs(same) - 1) of_warp[warp][e] = (uint8_t)__popc(same);
    __syncthreads();
    if (e >= 0) {
      int at = place[e] + __popc(same & ((1u << lane) - 1));
      for (int w = 0; w < warp; ++w) at += of_warp[w][e];
      a.list[at] = p;
    }
    __syncthreads();
    if (tid < experts)
      for (int w = 0; w < PLAN_WARPS; ++w) place[tid] += of_warp[w][tid];
    __syncthreads();
  }
}
static_assert(PLAN_THREADS == GSQ_MOE_MAX_EXPERTS, "a thread an expert");

// Tokens of one pass: the workspace holds that many, and the numbers of groups and tiles stay far from 2^31.
constexpr int64_t PASS_TOKENS = 1024;

// Workspace: pieces in the order of `next`, each 256-byte aligned.
struct Pieces {
  size_t at = 0;
  size_t next(size_t bytes) {
    const size_t p = at;
    at += (bytes + 255) & ~(size_t)255;
    return p;
  }
};
struct MoeLayout {
  size_t weights, ids, bounds, group, list, xq, xd, h, hq, hd, part, total;
  MoeLayout(int64_t m, int64_t hidden, int64_t inter, int top_k) {
    Pieces p;
    weights = p.next((size_t)m * top_k * 4);
    ids = p.next((size_t)m * top_k * 4);
    m = m < PASS_TOKENS ? m : PASS_TOKENS;
    const size_t pairs = (size_t)m * top_k;
    bounds = p.next((MOE_BLOCKS + 1) * 8);
    group = p.next(pairs * 16);
    list = p.next(pairs * 4);
    xq = p.next((size_t)m * hidden);
    xd = p.next((size_t)m * hidden / 8);
    h = p.next(pairs * inter * 4);
    hq = p.next(pairs * inter);
    hd = p.next(pairs * inter / 8);
    part = p.next(pairs * hidden * 4);
    total = p.at;
  }
};

static bool at_multiple(const void* p, size_t bytes) { return (uintptr_t)p % bytes == 0; }
static size_t element_bytes(int dtype) { return dtype == GSQ_F32 ? 4 : 2; }

static int check_router(const gsq_moe_router* r, int64_t m, int64_t experts, int top_k) {
  if (!r || !r->logits || m < 0 || experts <= 0 || top_k <= 0 || top_k > experts || r->row_stride < 0) return GSQ_ERR_UNSUPPORTED;
  if (experts > GSQ_MOE_MAX_EXPERTS || top_k > GSQ_MOE_MAX_TOP_K || m > INT32_MAX) return GSQ_ERR_TOO_LARGE;
  if (r->dtype != GSQ_F32 && r->dtype != GSQ_F16 && r->dtype != GSQ_BF16) return GSQ_ERR_UNSUPPORTED;
  if (r->scoring != GSQ_MOE_SOFTMAX && r->scoring != GSQ_MOE_SIGMOID) return GSQ_ERR_UNSUPPORTED;
  if (!at_multiple(r->logits, element_bytes(r->dtype)) || !at_multiple(r->bias, 4)) return GSQ_ERR_UNSUPPORTED;
  return GSQ_OK;
}

static RouteArgs route_args(const gsq_moe_router* r, int64_t m, int64_t experts, int top_k, float* weights, int32_t* ids) {
  return RouteArgs{r->logits, r->dtype, r->row_stride, (int)m, (int)experts, top_k, r->scoring, r->renormalize, r->bias, r->scale, weights, ids};
}

static int check_moe(const gsq_moe* w, const void* x, int x_dtype, int64_t m, int64_t x_row_stride, int top_k, const void* y,
                     int64_t y_row_stride, const void* ws, size_t ws_bytes) {
  if (!w || m < 0 || top_k <= 0 || w->experts <= 0) return GSQ_ERR_UNSUPPORTED;
  const int b13 = block_bytes(w->w13_type), b2 = block_bytes(w->w2_type);
  if (!b13 || !b2 || w->hidden <= 0 || w->inter <= 0 || w->hidden % 256 || w->inter % 256) return GSQ_ERR_UNSUPPORTED;
  if (w->activation != GSQ_ACT_SILU && w->activation != GSQ_ACT_GELU) return GSQ_ERR_UNSUPPORTED;
  if (x_dtype != GSQ_F32 && x_dtype != GSQ_F16 && x_dtype != GSQ_BF16) return GSQ_ERR_UNSUPPORTED;
  if (m == 0) return GSQ_OK;
  if (!w->w13 || !w->w2 || !x || !y || !at_multiple(w->w13, 16) || !at_multiple(w->w2, 16)) return GSQ_ERR_UNSUPPORTED;
  if (!at_multiple(x, element_bytes(x_dtype)) || !at_multiple(y, element_bytes(x_dtype))) return GSQ_ERR_UNSUPPORTED;
  if (x_row_stride < 0 || (m > 1 && y_row_stride < w->hidden)) return GSQ_ERR_UNSUPPORTED;
  if (w->hidden > (1 << 17) || w->inter > (1 << 17) || w->experts > GSQ_MOE_MAX_EXPERTS || top_k > GSQ_MOE_MAX_TOP_K || m > GSQ_MOE_MAX_TOKENS)
    return GSQ_ERR_TOO_LARGE;
  if (!ws || ws_bytes < gsq_moe_workspace_bytes(m, w->hidden, w->inter, top_k) || !at_multiple(ws, 256)) return GSQ_ERR_SCRATCH;
  return GSQ_OK;
}

// Up to this many tokens and experts the plan's one block makes the choice as well (a warp takes two tokens; more experts than 8 a lane
// do not fit its registers), which saves a launch. The layer, in the plan and apart, 128 experts of 2048 x 768 (256 of 2048 x 512): 1 token 23.4, 25.4 us
// (21.6, 22.6), 16 tokens 66.3, 72.4 (57.7, 62.2), 48 tokens 107, 110 (108, 108), 64 tokens 113, 116 (114, 113), 80 tokens 123, 123 (126, 121), 128 tokens 147, 142 (150, 137).
constexpr int64_t PLAN_ROUTES = 64, PLAN_EXPERTS = 256;

static int launch_plan(const MoeArgs& a, const RouteArgs* r, cudaStream_t st) {
  const unsigned grid = 1 + (unsigned)(((int64_t)a.m * (a.hidden >> 3) + PLAN_THREADS - 1) / PLAN_THREADS);
  if (!r) return moe_launch_behind(moe_plan_kernel<0>, grid, PLAN_THREADS, 0, st, a, RouteArgs{});
  if (a.experts <= 64) return moe_launch_behind(moe_plan_kernel<2>, grid, PLAN_THREADS, 0, st, a, *r);
  if (a.experts <= 128) return moe_launch_behind(moe_plan_kernel<4>, grid, PLAN_THREADS, 0, st, a, *r);
  return moe_launch_behind(moe_plan_kernel<8>, grid, PLAN_THREADS, 0, st, a, *r);
}

// route: the choice to be made here, or NULL where ids and weights are there.
static int run_experts(const gsq_moe* w, const void* x, int x_dtype, int64_t m, int64_t x_row_stride, const float* weights, const void* ids,
                       int ids64, int top_k, void* y, int64_t y_row_stride, uint8_t* ws, const RouteArgs* route, cudaStream_t st) {
  const MoeLayout l(m, w->hidden, w->inter, top_k);
  MoeArgs a;
  a.w13 = (const uint8_t*)w->w13;
  a.w2 = (const uint8_t*)w->w2;
  a.rb13 = w->hidden / 256 * block_bytes(w->w13_type);
  a.rb2 = w->inter / 256 * block_bytes(w->w2_type);
  a.experts = (int)w->experts;
  a.hidden = (int)w->hidden;
  a.inter = (int)w->inter;
  a.act = w->activation;
  a.top_k = top_k;
  a.x_dtype = x_dtype;
  a.x_stride = x_row_stride;
  const int64_t es = (int64_t)element_bytes(x_dtype), id_bytes = ids64 ? 8 : 4;
  a.x_vec = (uintptr_t)x % 16 == 0 && (m == 1 || x_row_stride * es % 16 == 0);
  a.ids64 = ids64;
  a.y_stride = y_row_stride;
  a.bounds = (int2*)(ws + l.bounds);
  DeviceInfo di;
  const int rc0 = device_info(&di);
  if (rc0 != GSQ_OK) return rc0;
  a.blocks = di.sm_count < MOE_BLOCKS ? di.sm_count : MOE_BLOCKS;
  a.group = (int4*)(ws + l.group);
  a.list = (int*)(ws + l.list);
  a.xq = (int8_t*)(ws + l.xq);
  a.xd = (float*)(ws + l.xd);
  a.h = (float*)(ws + l.h);
  a.hq = (int8_t*)(ws + l.hq);
  a.hd = (float*)(ws + l.hd);
  a.part = (float*)(ws + l.part);
  a.many = m * top_k > 4 * w->experts;
  const int up_mma = moe_mma_serves(w->w13_type, a.hidden, a.many), down_mma = moe_mma_serves(w->w2_type, a.inter, a.many);
  moe_mma_rates(up_mma ? w->w13_type : w->w2_type, a.rate);
  a.group_max = up_mma == 8 || down_mma == 8 ? 8 : 16;
  for (int64_t t0 = 0; t0 < m; t0 += PASS_TOKENS) {
    a.m = (int)(m - t0 < PASS_TOKENS ? m - t0 : PASS_TOKENS);
    a.x = (const uint8_t*)x + t0 * x_row_stride * es;
    a.y = (uint8_t*)y + t0 * y_row_stride * es;
    a.weights = weights + t0 * top_k;
    a.ids = (const uint8_t*)ids + t0 * top_k * id_bytes;
    int rc = GSQ_OK;
    const bool plan = up_mma || down_mma;
    const bool plan_routes = route && plan && m <= PLAN_ROUTES && a.experts <= PLAN_EXPERTS;
    if (route && t0 == 0 && !plan_routes) rc = launch_route(*route, st);
    if (rc == GSQ_OK && plan) rc = launch_plan(a, plan_routes ? route : nullptr, st);
    if (rc != GSQ_OK) return rc;
    if (up_mma) {
      rc = moe_mma_product(a, w->w13_type, false, st);
    } else {
      if (!plan) rc = launch_quant(a.x, x_dtype, a.x_vec, x_row_stride, a.m, a.hidden, a.xq, a.xd, st);
      if (rc == GSQ_OK) rc = moe_dot_gate_up(a, w->w13_type, st);
    }
    if (rc != GSQ_OK) return rc;
    if (down_mma) {
      rc = moe_mma_product(a, w->w2_type, true, st);
    } else {
      rc = launch_quant(a.h, GSQ_F32, 1, a.inter, (int64_t)a.m * top_k, a.inter, a.hq, a.hd, st);
      if (rc == GSQ_OK) rc = moe_dot_down(a, w->w2_type, st);
    }
    if (rc != GSQ_OK) return rc;
    const int64_t sums = (int64_t)a.m * (a.hidden >> 2);
    rc = moe_launch_behind(moe_combine_kernel, (unsigned)((sums + COMBINE_THREADS - 1) / COMBINE_THREADS), COMBINE_THREADS, 0, st, a);
    if (rc != GSQ_OK) return rc;
  }
  return GSQ_OK;
}

}  // namespace gsq

extern "C" size_t gsq_moe_workspace_bytes(int64_t m, int64_t hidden, int64_t inter, int top_k) {
  if (m <= 0 || hidden <= 0 || inter <= 0 || top_k <= 0) return 0;
  return gsq::MoeLayout(m, hidden, inter, top_k).total;
}

extern "C" int gsq_moe_route(const gsq_moe_router* r, int64_t m, int64_t experts, int top_k, float* topk_weights, int32_t* topk_ids,
                             void* stream) {
  if (m == 0) return GSQ_OK;
  const int rc = gsq::check_router(r, m, experts, top_k);
  if (rc != GSQ_OK) return rc;
  if (!topk_weights || !topk_ids || !gsq::at_multiple(topk_weights, 4) || !gsq::at_multiple(topk_ids, 4)) return GSQ_ERR_UNSUPPORTED;
  return gsq::launch_route(gsq::route_args(r, m, experts, top_k, topk_weights, topk_ids), (cudaStream_t)stream);
}

extern "C" int gsq_moe_experts(const gsq_moe* w, const void* x, int x_dtype, int64_t m, int64_t x_row_stride, const float* topk_weights,
                               const void* topk_ids, int ids_64, int top_k, void* y, int64_t y_row_stride, void* workspace,
                               size_t workspace_bytes, void* stream) {
  const int rc = gsq::check_moe(w, x, x_dtype, m, x_row_stride, top_k, y, y_row_stride, workspace, workspace_bytes);
  if (rc != GSQ_OK || m == 0) return rc;
  if (!topk_weights || !topk_ids || !gsq::at_multiple(topk_weights, 4) || !gsq::at_multiple(topk_ids, ids_64 ? 8 : 4)) return GSQ_ERR_UNSUPPORTED;
  return gsq::run_experts(w, x, x_dtype, m, x_row_stride, topk_weights, topk_ids, ids_64, top_k, y, y_row_stride, (uint8_t*)workspace,
                          nullptr, (cudaStream_t)stream);
}

extern "C" int gsq_moe_layer(const gsq_moe* w, const void* x, int x_dtype, int64_t m, int64_t x_row_stride, const gsq_moe_router* r, int top_k,
                             void* y, int64_t y_row_stride, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = gsq::check_moe(w, x, x_dtype, m, x_row_stride, top_k, y, y_row_stride, workspace, workspace_bytes);
  if (rc != GSQ_OK || m == 0) return rc;
  rc = gsq::check_router(r, m, w->experts, top_k);
  if (rc != GSQ_OK) return rc;
  const gsq::MoeLayout l(m, w->hidden, w->inter, top_k);
  uint8_t* ws = (uint8_t*)workspace;
  float* weights = (float*)(ws + l.weights);
  int32_t* ids = (int32_t*)(ws + l.ids);
  const gsq::RouteArgs route = gsq::route_args(r, m, w->experts, top_k, weights, ids);
  return gsq::run_experts(w, x, x_dtype, m, x_row_stride, weights, ids, 0, top_k, y, y_row_stride, ws, &route, (cudaStream_t)stream);
}
