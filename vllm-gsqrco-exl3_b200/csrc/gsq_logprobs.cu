// Log probabilities of given tokens with rank, entropy and the most probable alternatives, from rows of logits (sm_100a).
//
//   m = max x, S = sum e^(x - m), log p_i = x_i - m - log S, H = log S - (sum e^(x - m) (x - m)) / S
//
// The logits are read once. Every thread keeps the running maximum, S and sum e^(x - m) (x - m) of its values (rescaled when the maximum
// grows) and counts the values in front of the given token; the parts are joined over the block and the cluster in a fixed order.
// A row is cut over a cluster of 1 .. 16 blocks, so that a few rows use the whole GPU, and the parts meet in shared memory:
// no workspace, one launch.
//
// Alternatives: the threads' maxima, gathered to 32 groups, give a value that at least top_n values of the block's part reach
// (the top_n-th largest of the 32). Only threads whose maximum reaches it can hold candidates: their values are read again
// (from L2) and the candidates, a few more than top_n, ordered by counting. Where more than the list's room reach that value
// (rows of equal logits), the larger ones are collected alone and the equal ones taken by a scan in index order that ends as
// soon as it has enough.
#include <cooperative_groups.h>

#include "gsq_common.cuh"

namespace cg = cooperative_groups;

namespace gsq {

struct LogprobArgs {
  const void* x;
  int64_t stride;
  int vocab, top_n;
  const int64_t* ids;
  float* logprobs;
  int64_t* ranks;
  float* entropy;
  float* top_logprobs;
  int64_t* top_ids;
};

constexpr int LP_THREADS = 256;
constexpr int LP_WARPS = LP_THREADS / 32;
constexpr int LP_UNROLL = 4;      // 16-byte loads of a thread in flight, twice
constexpr int LP_ROOM = 1024;     // candidates of a block
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.69314718055994531f;

// Order of a row: larger key first. High half: the value (NaN 0, then -inf up); low half: lower index, larger key.
__device__ __forceinline__ uint32_t lp_value_key(float v) {
  if (isnan(v)) return 0;
  const uint32_t b = __float_as_uint(v + 0.0f);   // (-0 and 0 are equal)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long lp_key(float v, int i) { return ((unsigned long long)lp_value_key(v) << 32) | (uint32_t)(0x7FFFFFFF - i); }
__device__ __forceinline__ float lp_key_value(unsigned long long k) {
  const uint32_t b = (uint32_t)(k >> 32);
  return b == 0 ? NAN : __uint_as_float(b & 0x80000000u ? b ^ 0x80000000u : ~b);
}

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Sixteen bytes of logits.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float most(const uint4& r) {
    return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
  }
  static __device__ __forceinline__ void get(const uint4& r, float (&f)[N]) {
    f[0] = __uint_as_float(r.x); f[1] = __uint_as_float(r.y); f[2] = __uint_as_float(r.z); f[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float most(const uint4& r) {   // (the packed maximum returns the number where one side is NaN)
    const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&r);
    const __nv_bfloat162 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ void get(const uint4& r, float (&f)[N]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
};
template <>
struct Vec<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float most(const uint4& r) {
    const __half2* p = reinterpret_cast<const __half2*>(&r);
    const __half2 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ void get(const uint4& r, float (&f)[N]) {
    const __half2* p = reinterpret_cast<const __half2*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(p[i]);
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
  static __device__ __forceinline__ float one(const __half* p) { return __half2float(*p); }
};

// Maximum, sum of 2^y and sum of 2^y y over some values, y = (x - m) log2 e. A NaN in s stays there.
struct Stat {
  float m, s, t;
};
// `a` to the larger maximum m. (The distance of two maxima may be infinite: 2^-10000 is 0 as well, and 0 times it stays 0.)
__device__ __forceinline__ void raise(Stat& a, float m) {
  if (m > a.m) {
    const float d = fmaxf((a.m - m) * LOG2E, -1e4f), f = ex2(d);
    a.t = f * fmaf(a.s, d, a.t);
    a.s *= f;
    a.m = m;
  }
}
__device__ __forceinline__ Stat join(Stat a, Stat b) {
  const float m = fmaxf(a.m, b.m);
  raise(a, m);
  raise(b, m);
  return Stat{m, a.s + b.s, a.t + b.t};
}

// The values of one thread's vectors go through here. `most`: their maximum.
template <int N>
__device__ __forceinline__ void add_values(Stat& a, const float (&f)[N], float most) {
  if (most > -INFINITY) {
    raise(a, most);
#pragma unroll
    for (int i = 0; i < N; ++i) {              // (x log2 e - m log2 e in one step would overflow at the types' lowest values)
      const float y = (f[i] - a.m) * LOG2E, e = ex2(y);
      a.s += e;
      a.t = fmaf(e, fmaxf(y, -1e4f), a.t);     // (0 times -inf of a masked value)
    }
  } else {                                     // -inf and NaN only
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (isnan(f[i])) a.s = NAN;
  }
}

struct LogprobShared {
  unsigned long long cand[LP_ROOM];
  unsigned long long best[GSQ_LOGPROBS_MAX_TOP_N];   // this block's alternatives in order; 0 past the last
  Stat stat[LP_WARPS];
  int before[LP_WARPS];
  Stat part;                                         // the block's: read by the cluster's first block
  int part_before;
  float group[32];
  float limit;
  int found, hot_found, scan[LP_WARPS];
  uint16_t hot[LP_THREADS];
};

// The part of a row that a block has: `head` single values, whole vectors [v0, v1), `tail` single values, in index order.
template <typename T>
struct Part {
  const T* row;
  const T* body;       // the first whole vector of the row
  int head, tail, tail_at, body_at, v0, v1;
  // Values of unit u (0: head, 1 .. v1 - v0: vectors, after them the tail); returns how many and the index of the first.
  __device__ __forceinline__ int unit(int u, float (&f)[Vec<T>::N], int& at) const {
    const int nv = v1 - v0;
    if (u >= 1 && u <= nv) {
      Vec<T>::get(ldg_stream_v4(body + (int64_t)(v0 + u - 1) * Vec<T>::N), f);
      at = body_at + (v0 + u - 1) * Vec<T>::N;
      return Vec<T>::N;
    }
    const int n = u == 0 ? head : tail;
    at = u == 0 ? 0 : tail_at;
#pragma unroll
    for (int i = 0; i < Vec<T>::N; ++i) f[i] = i < n ? Vec<T>::one(row + at + i) : NAN;
    return n;
  }
};

// Values that hold pred(value), from unit 0 on in index order, until `need` are in the list. Whole blocks call it.
template <typename T, typename P>
__device__ void take_in_order(LogprobShared& sh, const Part<T>& p, int need, P pred) {
  const int tid = threadIdx.x, lane = tid & 31, units = p.v1 - p.v0 + 2;
  int taken = 0;
  for (int u0 = 0; u0 < units && taken < need; u0 += LP_THREADS) {
    float f[Vec<T>::N];
    int at = 0, n = 0, mine = 0;
    if (u0 + tid < units) n = p.unit(u0 + tid, f, at);
#pragma unroll
    for (int i = 0; i < Vec<T>::N; ++i) mine += i < n && pred(f[i]);
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) sh.scan[tid >> 5] = upto;
    __syncthreads();
    int before = taken + upto - mine, all = 0;
    for (int w = 0; w < LP_WARPS; ++w) {
      if (w < (tid >> 5)) before += sh.scan[w];
      all += sh.scan[w];
    }
#pragma unroll
    for (int i = 0; i < Vec<T>::N; ++i)
      if (i < n && pred(f[i]) && before < need) {
        sh.cand[sh.found + before] = lp_key(f[i], at + i);
        ++before;
      }
    taken += all;
    __syncthreads();
  }
  if (tid == 0) sh.found += min(taken, need);
  __syncthreads();
}

// The block's values that are larger than `limit` (or equal: `equal`) into the list; returns how many there are, of which the
// first LP_ROOM are in it. `mine`: the calling thread's maximum.
template <typename T>
__device__ int collect(LogprobShared& sh, const Part<T>& p, float mine, float limit, bool equal) {
  const int tid = threadIdx.x;
  if (tid == 0) sh.found = sh.hot_found = 0;
  __syncthreads();
  if (equal ? mine >= limit : mine > limit) sh.hot[atomicAdd(&sh.hot_found, 1)] = (uint16_t)tid;
  __syncthreads();
  const int per = (p.v1 - p.v0 + LP_THREADS - 1) / LP_THREADS, tasks = sh.hot_found * per + 2;
  for (int j = tid; j < tasks; j += LP_THREADS) {
    int u;                                        // the edges, then every vector of the hot threads
    if (j < 2) {
      u = j == 0 ? 0 : p.v1 - p.v0 + 1;
    } else {
      const int h = (j - 2) / per;
      u = 1 + sh.hot[h] + ((j - 2) - h * per) * LP_THREADS;
      if (u > p.v1 - p.v0) continue;
    }
    float f[Vec<T>::N];
    int at;
    const int n = p.unit(u, f, at);
#pragma unroll
    for (int i = 0; i < Vec<T>::N; ++i)
      if (i < n && (equal ? f[i] >= limit : f[i] > limit)) {
        const int slot = atomicAdd(&sh.found, 1);
        if (slot < LP_ROOM) sh.cand[slot] = lp_key(f[i], at + i);
      }
  }
  __syncthreads();
  const int n = sh.found;
  __syncthreads();                                // (the next call starts by clearing it)
  return n;
}

// The list's `n` largest keys in order into best[] (0 past the last). Every key's place is the number of larger ones.
__device__ __forceinline__ void order_list(LogprobShared& sh, const unsigned long long* list, int count, unsigned long long* best, int n) {
  if (threadIdx.x < GSQ_LOGPROBS_MAX_TOP_N) best[threadIdx.x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < count; i += LP_THREADS) {
    const unsigned long long k = list[i];
    int place = 0;
    for (int j = 0; j < count; ++j) place += list[j] > k;
    if (place < n) best[place] = k;
  }
  __syncthreads();
}

// The block's top_n alternatives, in order, into sh.best.
template <typename T>
__device__ void alternatives(LogprobShared& sh, const Part<T>& p, float mine, int top_n) {
  const int tid = threadIdx.x, lane = tid & 31;
  float g = mine;
#pragma unroll
  for (int o = LP_THREADS / 64; o > 0; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xFFFFFFFFu, g, o));
  if (tid % (LP_THREADS / 32) == 0) sh.group[tid / (LP_THREADS / 32)] = g;
  __syncthreads();
  if (tid < 32) {
    g = sh.group[lane];
    int place = 0;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const float v = __shfl_sync(0xFFFFFFFFu, g, j);
      place += v > g || (v == g && j < lane);
    }
    if (place == top_n - 1) sh.limit = g;
  }
  __syncthreads();
  float limit = sh.limit;
  int found = collect(sh, p, mine, limit, true);
  if (found > LP_ROOM) {
    // more than the list takes reach the limit: the larger ones, with a limit that rises to the top_n-th of those seen until
    // they fit (it rises to a value that is larger than the last one), then the equal ones of lowest index
    found = collect(sh, p, mine, limit, false);
    while (found > LP_ROOM) {
      order_list(sh, sh.cand, LP_ROOM, sh.best, top_n);
      limit = lp_key_value(sh.best[top_n - 1]);
      found = collect(sh, p, mine, limit, false);
    }
    if (found < top_n) take_in_order(sh, p, top_n - found, [limit](float v) { return v == limit; });
  }
  // fewer numbers than alternatives: NaN in index order
  const int all = p.head + p.tail + (p.v1 - p.v0) * Vec<T>::N;
  found = sh.found;
  if (found < top_n && found < all) {
    __syncthreads();
    take_in_order(sh, p, top_n - found, [](float v) { return isnan(v); });
  }
  order_list(sh, sh.cand, sh.found, sh.best, top_n);
}

template <typename T>
__global__ void __launch_bounds__(LP_THREADS, 4) logprobs_kernel(const LogprobArgs a) {
  __shared__ LogprobShared sh;
  constexpr int N = Vec<T>::N;
  cg::cluster_group cluster = cg::this_cluster();
  const int cs = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t row = blockIdx.x / cs;
  const int tid = threadIdx.x, lane = tid & 31;

  Part<T> p;
  p.row = reinterpret_cast<const T*>(a.x) + row * a.stride;
  const int head = min(a.vocab, (int)((16 - ((uintptr_t)p.row & 15)) & 15) / (int)sizeof(T));
  const int vectors = (a.vocab - head) / N;
  p.body = p.row + head;
  p.body_at = head;
  p.head = rank == 0 ? head : 0;
  p.tail_at = head + vectors * N;
  p.tail = rank == cs - 1 ? a.vocab - p.tail_at : 0;
  p.v0 = (int)((int64_t)vectors * rank / cs);
  p.v1 = (int)((int64_t)vectors * (rank + 1) / cs);

  // the first loads are on their way before the given token is looked up
  uint4 next[LP_UNROLL];
  auto fetch = [&](int v) {
#pragma unroll
    for (int u = 0; u < LP_UNROLL; ++u)
      if (v + u * LP_THREADS < p.v1) next[u] = ldg_stream_v4(p.body + (int64_t)(v + u * LP_THREADS) * N);
  };
  fetch(p.v0 + tid);
  const int64_t id64 = a.ids[row];
  const bool has = id64 >= 0 && id64 < a.vocab;
  const int id = has ? (int)id64 : -1;
  const float given = has ? Vec<T>::one(p.row + id) : INFINITY;
  const bool odd = isnan(given);                              // its place is behind every number
  const unsigned long long given_key = lp_key(given, id);

  Stat st{-INFINITY, 0.0f, 0.0f};
  int before = 0;
  // values in front of the given one: those of a vector that lies before it count when equal too
  auto count = [&](const float (&f)[N], int at) {
    if (odd || (at <= id && id < at + N)) {
#pragma unroll
      for (int i = 0; i < N; ++i) before += lp_key(f[i], at + i) > given_key;
    } else if (at < id) {
#pragma unroll
      for (int i = 0; i < N; ++i) before += f[i] >= given;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) before += f[i] > given;
    }
  };
  for (int v = p.v0 + tid; v < p.v1; v += LP_UNROLL * LP_THREADS) {
    uint4 now[LP_UNROLL];
#pragma unroll
    for (int u = 0; u < LP_UNROLL; ++u) now[u] = next[u];
    fetch(v + LP_UNROLL * LP_THREADS);
#pragma unroll
    for (int u = 0; u < LP_UNROLL; ++u) {
      if (v + u * LP_THREADS < p.v1) {
        const float most = Vec<T>::most(now[u]);
        float f[N];
        Vec<T>::get(now[u], f);
        add_values<N>(st, f, most);
        if (has && (most >= given || odd)) count(f, p.body_at + (v + u * LP_THREADS) * N);
      }
    }
  }
  if ((tid < p.head) || (tid >= 32 && tid - 32 < p.tail)) {   // single values at the row's ends
    const int i = tid < 32 ? tid : p.tail_at + tid - 32;
    const float f[1] = {Vec<T>::one(p.row + i)};
    add_values<1>(st, f, isnan(f[0]) ? -INFINITY : f[0]);
    before += has && lp_key(f[0], i) > given_key;
  }
  const float mine = st.m;

#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Stat b{__shfl_xor_sync(0xFFFFFFFFu, st.m, o), __shfl_xor_sync(0xFFFFFFFFu, st.s, o), __shfl_xor_sync(0xFFFFFFFFu, st.t, o)};
    st = lane & o ? join(b, st) : join(st, b);                // (the same order on both sides)
    before += __shfl_xor_sync(0xFFFFFFFFu, before, o);
  }
  if (lane == 0) {
    sh.stat[tid >> 5] = st;
    sh.before[tid >> 5] = before;
  }
  if (a.top_n) alternatives(sh, p, mine, a.top_n);
  else __syncthreads();
  if (tid == 0) {
    st = sh.stat[0];
    before = sh.before[0];
    for (int w = 1; w < LP_WARPS; ++w) {
      st = join(st, sh.stat[w]);
      before += sh.before[w];
    }
    sh.part = st;
    sh.part_before = before;
  }
  if (cs > 1) cluster.sync();
  else __syncthreads();
  if (rank == 0) {
    st = sh.part;
    before = sh.part_before;
    for (int r = 1; r < cs; ++r) {
      const LogprobShared* q = cluster.map_shared_rank(&sh, r);
      st = join(st, q->part);
      before += q->part_before;
    }
    const float base = st.m == -INFINITY ? 0.0f : st.m, lse = logf(st.s);
    auto logprob = [&](float v) { return v == -INFINITY && !isnan(lse) ? -INFINITY : (v - base) - lse; };
    if (tid == 0) {
      a.logprobs[row] = has ? logprob(given) : id64 < 0 ? 0.0f : NAN;
      a.ranks[row] = has ? before + 1 : 0;
      a.entropy[row] = st.s == 0.0f ? 0.0f : lse - st.t * LN2 / st.s;
    }
    if (a.top_n) {
      const unsigned long long* best = sh.best;
      if (cs > 1) {                               // the blocks' lists, joined
        for (int i = tid; i < cs * a.top_n; i += LP_THREADS) sh.cand[i] = cluster.map_shared_rank(&sh, i / a.top_n)->best[i % a.top_n];
        __syncthreads();
        unsigned long long* joined = sh.cand + 16 * GSQ_LOGPROBS_MAX_TOP_N;
        order_list(sh, sh.cand, cs * a.top_n, joined, a.top_n);
        best = joined;
      }
      if (tid < a.top_n) {
        const unsigned long long k = best[tid];
        a.top_logprobs[row * a.top_n + tid] = k ? logprob(lp_key_value(k)) : -INFINITY;
        a.top_ids[row * a.top_n + tid] = k ? 0x7FFFFFFF - (int)(uint32_t)k : -1;
      }
    }
  }
  if (cs > 1) cluster.sync();                     // no block leaves while its part may be read
}

template <typename T>
static int launch_logprobs(const LogprobArgs& a, int64_t m, cudaStream_t st) {
  DeviceInfo di;
  const int rc = device_info(&di);
  if (rc != GSQ_OK) return rc;
  const void* kern = (const void*)logprobs_kernel<T>;
  // blocks of a row: as many as leave every block at least one round of loads, while the grid stays within two blocks an SM
  const int64_t rounds = (a.vocab / Vec<T>::N) / (LP_THREADS * LP_UNROLL);
  int cs = 1;
  while (cs < 16 && 2 * cs * m <= 2 * di.sm_count && cs <= rounds) cs *= 2;
  if (cs > 8) GSQ_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(m * cs));
  cfg.blockDim = dim3(LP_THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cs;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  GSQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, logprobs_kernel<T>, a));
  return GSQ_OK;
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
  if ((uintptr_t)logits % (dtype == GSQ_F32 ? 4 : 2)) return GSQ_ERR_UNSUPPORTED;
  const LogprobArgs a{logits, row_stride, (int)vocab, top_n, token_ids, logprobs, ranks, entropy, top_logprobs, top_ids};
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == GSQ_F32 ? launch_logprobs<float>(a, m, st) : dtype == GSQ_F16 ? launch_logprobs<__half>(a, m, st) : launch_logprobs<__nv_bfloat16>(a, m, st);
}
