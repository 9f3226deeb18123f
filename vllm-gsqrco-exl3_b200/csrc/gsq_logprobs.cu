// Log probabilities of given tokens with rank, entropy and the most probable alternatives, from rows of logits (sm_100a).
//
//   m = max x, S = sum e^(x - m), log p_i = x_i - m - log S, H = log S - (sum e^(x - m) (x - m)) / S
//
// One block a row: a pass for the maximum, one for the sums and the rank, one for each alternative (the largest key below the
// last one).
#include "gsq_common.cuh"

namespace gsq {

struct LogprobArgs {
  const void* x;
  int dtype;
  int64_t stride;
  int vocab, top_n;
  const int64_t* ids;
  float* logprobs;
  int64_t* ranks;
  float* entropy;
  float* top_logprobs;
  int64_t* top_ids;
};

// Order of a row: larger key first. High half: the value (NaN 0, then -inf up); low half: lower index, larger key.
__device__ __forceinline__ uint32_t lp_value_key(float v) {
  if (isnan(v)) return 0;
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t lp_key(float v, int i) { return ((uint64_t)lp_value_key(v) << 32) | (uint32_t)(0x7FFFFFFF - i); }

template <typename T>
__device__ __forceinline__ float lp_f32(T v);
template <>
__device__ __forceinline__ float lp_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float lp_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float lp_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

constexpr int LP_THREADS = 512;

template <typename V, typename F>
__device__ __forceinline__ V lp_reduce(V v, V* buf, F op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  v = buf[0];
  for (int i = 1; i < LP_THREADS / 32; ++i) v = op(v, buf[i]);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(LP_THREADS) logprobs_kernel(const LogprobArgs a) {
  __shared__ unsigned long long buf[LP_THREADS / 32];
  const int64_t row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.stride;
  auto add = [](float p, float q) { return p + q; };
  float top = -INFINITY;
  for (int i = threadIdx.x; i < a.vocab; i += LP_THREADS) top = fmaxf(top, lp_f32(x[i]));
  top = lp_reduce(top, reinterpret_cast<float*>(buf), [](float p, float q) { return fmaxf(p, q); });
  const float base = top == -INFINITY ? 0.0f : top;
  const int64_t id = a.ids[row];
  const bool has = id >= 0 && id < a.vocab;
  const float given = has ? lp_f32(x[id]) : 0.0f;
  const uint64_t given_key = lp_key(given, (int)id);
  float s = 0.0f, t = 0.0f;
  int before = 0;
  for (int i = threadIdx.x; i < a.vocab; i += LP_THREADS) {
    const float v = lp_f32(x[i]), y = v - base, e = expf(y);
    s += e;
    t += v == -INFINITY ? 0.0f : e * y;
    before += lp_key(v, i) > given_key;
  }
  s = lp_reduce(s, reinterpret_cast<float*>(buf), add);
  t = lp_reduce(t, reinterpret_cast<float*>(buf), add);
  before = lp_reduce(before, reinterpret_cast<int*>(buf), [](int p, int q) { return p + q; });
  const float lse = logf(s);
  auto logprob = [&](float v) { return v == -INFINITY && !isnan(lse) ? -INFINITY : (v - base) - lse; };
  if (threadIdx.x == 0) {
    a.logprobs[row] = has ? logprob(given) : id < 0 ? 0.0f : NAN;
    a.ranks[row] = has ? before + 1 : 0;
    a.entropy[row] = s == 0.0f ? 0.0f : lse - t / s;
  }
  uint64_t last = ~0ull;
  for (int n = 0; n < a.top_n; ++n) {
    uint64_t best = 0;
    for (int i = threadIdx.x; i < a.vocab; i += LP_THREADS) {
      const uint64_t k = lp_key(lp_f32(x[i]), i);
      if (k < last && k > best) best = k;
    }
    best = lp_reduce((unsigned long long)best, buf, [](unsigned long long p, unsigned long long q) { return p > q ? p : q; });
    if (threadIdx.x == 0) {
      const int i = 0x7FFFFFFF - (int)(uint32_t)best;
      a.top_logprobs[row * a.top_n + n] = best ? logprob(lp_f32(x[i])) : -INFINITY;
      a.top_ids[row * a.top_n + n] = best ? i : -1;
    }
    last = best;
  }
}

}  // namespace gsq

extern "C" int gsq_token_logprobs(const void* logits, int dtype, int64_t m, int64_t vocab, int64_t row_stride, const int64_t* token_ids,
                                  int top_n, float* logprobs, int64_t* ranks, float* entropy, float* top_logprobs, int64_t* top_ids,
                                  void* stream) {
  using namespace gsq;
  if (m < 0 || vocab <= 0 || top_n < 0 || row_stride < 0) return GSQ_ERR_UNSUPPORTED;
  if (dtype != GSQ_F32 && dtype != GSQ_F16 && dtype != GSQ_BF16) return GSQ_ERR_UNSUPPORTED;
  if (m == 0) return GSQ_OK;
  if (m > INT32_MAX || vocab > (1 << 30) || top_n > GSQ_LOGPROBS_MAX_TOP_N) return GSQ_ERR_TOO_LARGE;
  if (!logits || !token_ids || !logprobs || !ranks || !entropy || (top_n && (!top_logprobs || !top_ids))) return GSQ_ERR_UNSUPPORTED;
  LogprobArgs a{logits, dtype, row_stride, (int)vocab, top_n, token_ids, logprobs, ranks, entropy, top_logprobs, top_ids};
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == GSQ_F32) logprobs_kernel<float><<<(unsigned)m, LP_THREADS, 0, st>>>(a);
  else if (dtype == GSQ_F16) logprobs_kernel<__half><<<(unsigned)m, LP_THREADS, 0, st>>>(a);
  else logprobs_kernel<__nv_bfloat16><<<(unsigned)m, LP_THREADS, 0, st>>>(a);
  GSQ_CUDA_TRY(cudaGetLastError());
  return GSQ_OK;
}
