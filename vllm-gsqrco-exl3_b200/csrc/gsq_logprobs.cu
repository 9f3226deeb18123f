// Log probabilities of given tokens with rank, entropy and the most probable alternatives, from rows of logits (sm_100a).
//
//   m = max x, S = sum e^(x - m), log p_i = x_i - m - log S, H = log S - (sum e^(x - m) (x - m)) / S
//
// The logits are read once. Every thread keeps the running maximum, S and sum e^(x - m) (x - m) of its values (rescaled when the maximum
// grows) and counts the values in front of the given token; the parts are joined over the block and the cluster in a fixed order.
// A row is cut over a cluster of 1 .. 16 blocks, so that a few rows use the whole GPU, and the parts meet in shared memory:
// no workspace, one launch. Rows of at most 256 whole vectors take a warp each.
//
// Measured (bf16): 2048 rows of 248320 values with 5 alternatives 187 us in the first 20 ms, 5.4 TB/s (0.83 of the measured 6.54), and 207 in the long run, 4.9 TB/s, when the
// card holds its power limit;
// 512 rows of 151936 37 us: some SMs have four rows, others three, and an SM goes through its rows at 32 B/ns at most; one row of 248320, 20 alternatives, 9.4 us, all of it latency: loads 1.5, alternatives 2.5, joining the cluster 3.5, launch 2.
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
constexpr int LP_AGAIN = 512;     // rounds of one thread to be read again
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

// Two fp32 numbers as one operand: half the issue slots of the scalar forms.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void halves(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// Sixteen bytes of logits. most(): the larger of two words' values, kept packed (the number where one side is NaN); floor():
// values of at least LOWEST, NaN kept; larger(): `n` with the values > g counted in, to be read by total(); below(): the next
// value under g.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static constexpr float LOWEST = -1e38f, SMALL = -1e37f, LARGE = 1e37f;
  static constexpr uint32_t MASKED = 0xFF800000u;     // -inf
  static __device__ __forceinline__ uint32_t most(uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
  static __device__ __forceinline__ float most(uint32_t a) { return __uint_as_float(a); }
  static __device__ __forceinline__ uint32_t floor(uint32_t a) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(a)), "f"(LOWEST));
    return __float_as_uint(r);
  }
  static __device__ __forceinline__ void get(const uint4& r, float (&f)[N]) {
    f[0] = __uint_as_float(r.x); f[1] = __uint_as_float(r.y); f[2] = __uint_as_float(r.z); f[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint32_t larger(uint32_t n, const uint4& r, float g) {
    float f[N];
    get(r, f);
#pragma unroll
    for (int i = 0; i < N; ++i) n += f[i] > g;
    return n;
  }
  static __device__ __forceinline__ int total(uint32_t n) { return (int)n; }
  static __device__ __forceinline__ float below(float g) { return nextafterf(g, -INFINITY); }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
};
// The packed comparisons set all bits of a half. Subtracted from a 32-bit sum, such words leave the count L of the low halves in the
// sum's low half and H - L in its high half, H the count of the high ones.
__device__ __forceinline__ int packed_count(uint32_t n) { return (int)((2 * (n & 0xFFFFu) + (n >> 16)) & 0xFFFFu); }
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static constexpr float LOWEST = -1e38f, SMALL = -1e37f, LARGE = 1e37f;
  static constexpr uint32_t MASKED = 0xFF80FF80u;
  static __device__ __forceinline__ uint32_t most(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ float most(uint32_t a) { return fmaxf(__uint_as_float(a << 16), __uint_as_float(a & 0xFFFF0000u)); }
  static __device__ __forceinline__ uint32_t floor(uint32_t a) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(0xFE96FE96u));   // -9.97e37
    return r;
  }
  static __device__ __forceinline__ void get(const uint4& r, float (&f)[N]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ uint32_t larger(uint32_t n, const uint4& r, float g) {
    const __nv_bfloat162 gg = __float2bfloat162_rn(g);
    const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) n -= __hgt2_mask(p[i], gg);
    return n;
  }
  static __device__ __forceinline__ int total(uint32_t n) { return packed_count(n); }
  static __device__ __forceinline__ float below(float g) {   // (of 0 and -0: the largest negative one)
    const unsigned short b = __bfloat16_as_ushort(__float2bfloat16_rn(g));
    return __bfloat162float(__ushort_as_bfloat16(g == 0.0f ? 0x8001 : g > 0.0f ? b - 1 : b + 1));
  }
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
};
template <>
struct Vec<__half> {
  static constexpr int N = 8;
  static constexpr float LOWEST = -65504.0f, SMALL = -6e4f, LARGE = 1e37f;
  static constexpr uint32_t MASKED = 0xFC00FC00u;
  static __device__ __forceinline__ uint32_t most(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ float most(uint32_t a) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&a));
    return fmaxf(v.x, v.y);
  }
  static __device__ __forceinline__ uint32_t floor(uint32_t a) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(0xFBFFFBFFu));   // -65504
    return r;
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
  static __device__ __forceinline__ uint32_t larger(uint32_t n, const uint4& r, float g) {
    const __half2 gg = __float2half2_rn(g);
    const __half2* p = reinterpret_cast<const __half2*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) n -= __hgt2_mask(p[i], gg);
    return n;
  }
  static __device__ __forceinline__ int total(uint32_t n) { return packed_count(n); }
  static __device__ __forceinline__ float below(float g) {   // (of 0 and -0: the largest negative one)
    const unsigned short b = __half_as_ushort(__float2half_rn(g));
    return __half2float(__ushort_as_half(g == 0.0f ? 0x8001 : g > 0.0f ? b - 1 : b + 1));
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

// The parts of n lanes (a power of two; lanes n, n + 1, ... hold lane 0's, 1's, ... again) in one order.
__device__ __forceinline__ void join_parts(Stat st, int before, int n, Stat* to, int* to_before) {
  const int lane = threadIdx.x & 31;
  for (int o = n >> 1; o > 0; o >>= 1) {
    const Stat b{__shfl_xor_sync(0xFFFFFFFFu, st.m, o), __shfl_xor_sync(0xFFFFFFFFu, st.s, o), __shfl_xor_sync(0xFFFFFFFFu, st.t, o)};
    st = lane & o ? join(b, st) : join(st, b);
    before += __shfl_xor_sync(0xFFFFFFFFu, before, o);
  }
  if (lane == 0) {
    *to = st;
    *to_before = before;
  }
}

// One value.
__device__ __forceinline__ void add_value(Stat& a, float f) {
  if (f > -INFINITY) {
    raise(a, f);
    const float y = (f - a.m) * LOG2E, e = ex2(y);
    a.s += e;
    a.t = fmaf(e, fmaxf(y, -1e4f), a.t);       // (0 times -inf)
  } else if (isnan(f)) {
    a.s = NAN;
  }
}

// U vectors of one thread; returns their maximum. One comparison decides for all of them whether the sums are rescaled. A masked
// value (-inf) is taken as LOWEST, whose exponential is 0 as well and 0 times whose distance stays 0, as long as the maximum is
// far from LOWEST and from overflow; where it is not, the values go one by one.
template <typename T, int U>
__device__ __forceinline__ float add_vectors(Stat& a, const uint4 (&r)[U]) {
  using V = Vec<T>;
  uint32_t top = r[0].x;
#pragma unroll
  for (int u = 0; u < U; ++u) top = V::most(top, V::most(V::most(r[u].x, r[u].y), V::most(r[u].z, r[u].w)));
  const float most = V::most(top);
  if (most > -INFINITY) raise(a, most);
  if (a.m > V::SMALL && a.m < V::LARGE) {
    const uint64_t shift = pair(-a.m, -a.m), scale = pair(LOG2E, LOG2E);
    uint64_t s[2] = {0, 0}, t[2] = {0, 0};     // (two chains each)
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint4 w = make_uint4(V::floor(r[u].x), V::floor(r[u].y), V::floor(r[u].z), V::floor(r[u].w));
      float f[V::N];
      V::get(w, f);
#pragma unroll
      for (int i = 0; i < V::N; i += 2) {      // (x log2 e - m log2 e in one step would be off by more where both are large)
        const uint64_t y = mul2(add2(pair(f[i], f[i + 1]), shift), scale);
        float y0, y1;
        halves(y, y0, y1);
        const uint64_t e = pair(ex2(y0), ex2(y1));
        s[(i >> 1) & 1] = add2(s[(i >> 1) & 1], e);
        t[(i >> 1) & 1] = fma2(e, y, t[(i >> 1) & 1]);
      }
    }
    float s0, s1, t0, t1;
    halves(add2(s[0], s[1]), s0, s1);
    halves(add2(t[0], t[1]), t0, t1);
    a.s += s0 + s1;
    a.t += t0 + t1;
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[V::N];
      V::get(r[u], f);
#pragma unroll
      for (int i = 0; i < V::N; ++i) add_value(a, f[i]);
    }
  }
  return most;
}

struct LogprobShared {
  unsigned long long cand[LP_ROOM];
  unsigned long long best[GSQ_LOGPROBS_MAX_TOP_N];   // this block's alternatives in order; 0 past the last
  Stat stat[LP_WARPS];
  int before[LP_WARPS];
  Stat part;                                         // the block's: read by the cluster's first block; there, then the row's
  int part_before;
  float group[32];
  unsigned long long least;
  int found, again_found, scan[LP_WARPS];
  uint32_t again[LP_AGAIN];                          // vectors (of the part) at which a thread's round to be read again begins
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
      Vec<T>::get(ld_stream_v4(body + (int64_t)(v0 + u - 1) * Vec<T>::N), f);
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

// What a thread remembers of its rounds of loads: the largest maximum of one, which it was, and the largest of the others.
struct Rounds {
  float most, second;
  int at;
};

// The block's values that are larger than `limit` (or equal: `equal`) into the list; returns how many there are, of which the
// first LP_ROOM are in it. Only rounds whose maximum reaches the limit are read again: mostly one of a few threads each.
template <typename T>
__device__ int collect(LogprobShared& sh, const Part<T>& p, const Rounds& mine, int rounds, float limit, bool equal) {
  const int tid = threadIdx.x;
  if (tid == 0) sh.found = sh.again_found = 0;
  __syncthreads();
  auto reaches = [&](float v) { return equal ? v >= limit : v > limit; };
  if (reaches(mine.most)) {
    const int n = reaches(mine.second) ? rounds : 1, at = atomicAdd(&sh.again_found, n);
    for (int i = 0; i < n; ++i)
      if (at + i < LP_AGAIN) sh.again[at + i] = (n == 1 ? mine.at : i) * (LP_UNROLL * LP_THREADS) + tid;
  }
  __syncthreads();
  const int again = sh.again_found, vectors = p.v1 - p.v0;
  const bool all = again > LP_AGAIN;              // every vector of the part
  const int tasks = 2 + (all ? vectors : again * LP_UNROLL);
  for (int j = tid; j < tasks; j += LP_THREADS) {
    int u = j == 0 ? 0 : vectors + 1;             // the edges first
    if (j >= 2) {
      const int v = all ? j - 2 : (int)sh.again[(j - 2) / LP_UNROLL] + (j - 2) % LP_UNROLL * LP_THREADS;
      if (v >= vectors) continue;
      u = v + 1;
    }
    float f[Vec<T>::N];
    int at;
    const int n = p.unit(u, f, at);
#pragma unroll
    for (int i = 0; i < Vec<T>::N; ++i)
      if (i < n && reaches(f[i])) {
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
__device__ void alternatives(LogprobShared& sh, const Part<T>& p, float mine, const Rounds& mine_by_round, int rounds, int top_n) {
  const int tid = threadIdx.x, lane = tid & 31;
  float g = mine;
#pragma unroll
  for (int o = LP_THREADS / 64; o > 0; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xFFFFFFFFu, g, o));
  if (tid % (LP_THREADS / 32) == 0) sh.group[tid / (LP_THREADS / 32)] = g;
  __syncthreads();
  g = sh.group[lane];
  int place = 0;
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    const float v = __shfl_sync(0xFFFFFFFFu, g, j);
    place += v > g || (v == g && j < lane);
  }
  const uint32_t at = __ballot_sync(0xFFFFFFFFu, place == top_n - 1);
  float limit = __shfl_sync(0xFFFFFFFFu, g, __ffs(at) - 1);
  int found = collect(sh, p, mine_by_round, rounds, limit, true);
  if (found > LP_ROOM) {
    // more than the list takes reach the limit: the larger ones, with a limit that rises to the top_n-th of those seen until
    // they fit (it rises to a value that is larger than the last one), then the equal ones of lowest index
    found = collect(sh, p, mine_by_round, rounds, limit, false);
    while (found > LP_ROOM) {
      order_list(sh, sh.cand, LP_ROOM, sh.best, top_n);
      limit = lp_key_value(sh.best[top_n - 1]);
      found = collect(sh, p, mine_by_round, rounds, limit, false);
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

// The blocks' lists (each in order) into sh.cand, but for what cannot be among the first top_n: 32 keys, the first 32 / cs of
// every list, have a top_n-th largest; smaller ones are left out.
__device__ __forceinline__ void join_lists(LogprobShared& sh, cg::cluster_group& cluster, int cs, int top_n) {
  const int tid = threadIdx.x;
  unsigned long long k[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {                   // cs * top_n <= 512
    const int i = tid + j * LP_THREADS;
    k[j] = i < cs * top_n ? cluster.map_shared_rank(&sh, i / top_n)->best[i % top_n] : 0;
  }
  if (tid < 32) {
    const int per = 32 / cs;
    const unsigned long long g = tid % per < top_n ? cluster.map_shared_rank(&sh, tid / per)->best[tid % per] : 0;
    int place = 0;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const unsigned long long v = __shfl_sync(0xFFFFFFFFu, g, j);
      place += v > g || (v == g && j < tid);
    }
    if (place == top_n - 1) sh.least = g;
    if (tid == 0) sh.found = 0;
  }
  __syncthreads();
  const unsigned long long least = sh.least;
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (k[j] && k[j] >= least) sh.cand[atomicAdd(&sh.found, 1)] = k[j];
  __syncthreads();
}

// These kernels are launched while the one before still runs (the head's product lets them), and wait for it before they read anything;
// theirs follow in the same way. (One row, calls in a chain: 12.3 -> 10.1 us a call.)
__device__ __forceinline__ void behind_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
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

  behind_previous();
  // the first loads are on their way before the given token is looked up
  constexpr int U = LP_UNROLL;
  uint4 next[U];
  auto fetch = [&](int v) {
    if (v + (U - 1) * LP_THREADS < p.v1) {
#pragma unroll
      for (int u = 0; u < U; ++u) next[u] = ld_stream_v4(p.body + (int64_t)(v + u * LP_THREADS) * N);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        next[u] = make_uint4(Vec<T>::MASKED, Vec<T>::MASKED, Vec<T>::MASKED, Vec<T>::MASKED);
        if (v + u * LP_THREADS < p.v1) next[u] = ld_stream_v4(p.body + (int64_t)(v + u * LP_THREADS) * N);
      }
    }
  };
  fetch(p.v0 + tid);
  const int64_t id64 = a.ids[row];
  const bool has = id64 >= 0 && id64 < a.vocab;
  const int id = has ? (int)id64 : -1;
  const float given = has ? Vec<T>::one(p.row + id) : INFINITY;
  const unsigned long long given_key = lp_key(given, id);
  // values in front of the given one: larger ones, and equal ones of vectors that end before it (those of its own vector are added
  // below). A masked or NaN one has no value under it: keys are compared one by one.
  const bool odd = has && !(given > -INFINITY);
  const float under = Vec<T>::below(given);
  const int own = has && id >= p.body_at ? (id - p.body_at) / N : -1;   // the given token's vector
  Stat st{-INFINITY, 0.0f, 0.0f};
  int before = 0;
  const int rounds = (p.v1 - p.v0 + U * LP_THREADS - 1) / (U * LP_THREADS);
  Rounds by_round{-INFINITY, -INFINITY, 0};
  for (int round = 0, v = p.v0 + tid; v < p.v1; ++round, v += U * LP_THREADS) {
    uint4 now[U];
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = next[u];
    fetch(v + U * LP_THREADS);
    const float most = add_vectors<T, U>(st, now);
    by_round.second = fmaxf(by_round.second, fminf(most, by_round.most));
    if (most > by_round.most) {
      by_round.most = most;
      by_round.at = round;
    }
    if (has && !odd && most >= given) {
      uint32_t n = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) n = Vec<T>::larger(n, now[u], v + u * LP_THREADS < own ? under : given);
      before += Vec<T>::total(n);
    } else if (odd) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[N];
        Vec<T>::get(now[u], f);
#pragma unroll
        for (int i = 0; i < N; ++i)
          before += v + u * LP_THREADS < p.v1 && lp_key(f[i], p.body_at + (v + u * LP_THREADS) * N + i) > given_key;
      }
    }
  }
  if (!odd && has && own >= p.v0 && own < p.v1 && tid < N) {
    const int i = p.body_at + own * N + tid;
    before += i < id && Vec<T>::one(p.row + i) == given;
  }
  if ((tid < p.head) || (tid >= 32 && tid - 32 < p.tail)) {   // single values at the row's ends
    const int i = tid < 32 ? tid : p.tail_at + tid - 32;
    const float f = Vec<T>::one(p.row + i);
    add_value(st, f);
    before += has && lp_key(f, i) > given_key;
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
  if (a.top_n) alternatives(sh, p, mine, by_round, rounds, a.top_n);
  else __syncthreads();
  if (tid < 32) join_parts(sh.stat[lane & (LP_WARPS - 1)], sh.before[lane & (LP_WARPS - 1)], LP_WARPS, &sh.part, &sh.part_before);
  if (cs > 1) {
    cluster.sync();
    if (rank == 0 && tid < 32) {
      const LogprobShared* q = cluster.map_shared_rank(&sh, lane & (cs - 1));
      const Stat part = q->part;
      const int part_before = q->part_before;
      __syncwarp();
      join_parts(part, part_before, cs, &sh.part, &sh.part_before);
    }
  }
  if (rank == 0) {
    __syncthreads();
    st = sh.part;
    before = sh.part_before;
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
        join_lists(sh, cluster, cs, a.top_n);
        unsigned long long* joined = sh.cand + 16 * GSQ_LOGPROBS_MAX_TOP_N;
        order_list(sh, sh.cand, sh.found, joined, a.top_n);
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

// Rows of at most 256 whole vectors: a warp a row, the row in registers, no barrier. With a block a row, 4096 rows of 1000 fp32 logits
// took 46 us: a row's fixed steps outweigh its 4 KB. Here 11.7 us (2048 rows 8.5): 80 registers leave three blocks an SM, so that 512 blocks go in two
// waves. In bf16 (160 registers, one block an SM) 18.8. Longer rows pay the block's steps: 1028 values 45.4, 4096 values 48.1.
constexpr int LPW_WARPS = 8, LPW_VECTORS = 8, LPW_ROOM = 128;

template <typename T>
__global__ void __launch_bounds__(LPW_WARPS * 32) logprobs_rows_kernel(const LogprobArgs a, int rows) {
  constexpr int N = Vec<T>::N, H = LPW_VECTORS / 2;
  __shared__ unsigned long long cand_all[LPW_WARPS][LPW_ROOM], best_all[LPW_WARPS][GSQ_LOGPROBS_MAX_TOP_N];
  __shared__ int found_all[LPW_WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = (int64_t)blockIdx.x * LPW_WARPS + warp;
  behind_previous();
  if (row >= rows) return;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.stride;
  const int head = min(a.vocab, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T));
  const int vectors = (a.vocab - head) / N, tail_at = head + vectors * N;
  uint4 r[2][H];
#pragma unroll
  for (int u = 0; u < LPW_VECTORS; ++u) {
    r[u / H][u % H] = make_uint4(Vec<T>::MASKED, Vec<T>::MASKED, Vec<T>::MASKED, Vec<T>::MASKED);
    if (lane + 32 * u < vectors) r[u / H][u % H] = ld_stream_v4(x + head + (lane + 32 * u) * N);
  }
  const int64_t id64 = a.ids[row];
  // a lane's single value: of the head (lanes 0 ..) or of the tail (lanes 16 ..)
  const int single = lane < head ? lane : lane >= 16 && tail_at + lane - 16 < a.vocab ? tail_at + lane - 16 : -1;
  const float edge = single >= 0 ? Vec<T>::one(x + single) : 0.0f;
  const bool has = id64 >= 0 && id64 < a.vocab;
  const int id = has ? (int)id64 : -1;
  const float given = has ? Vec<T>::one(x + id) : INFINITY;
  const unsigned long long given_key = lp_key(given, id);
  // every value of the lane and its index
  auto each = [&](auto f) {
#pragma unroll
    for (int u = 0; u < LPW_VECTORS; ++u) {
      if (lane + 32 * u < vectors) {
        float v[N];
        Vec<T>::get(r[u / H][u % H], v);
#pragma unroll
        for (int i = 0; i < N; ++i) f(v[i], head + (lane + 32 * u) * N + i);
      }
    }
    if (single >= 0) f(edge, single);
  };
  Stat st{-INFINITY, 0.0f, 0.0f};
  add_vectors<T, H>(st, r[0]);
  if (vectors > 32 * H) add_vectors<T, H>(st, r[1]);
  if (single >= 0) add_value(st, edge);
  const float mine = st.m;
  int before = 0;
  if (has && !(mine < given)) each([&](float v, int i) { before += lp_key(v, i) > given_key; });
  // (the maximum of a lane of NaN alone is -inf: not under a given value of NaN or -inf)
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Stat b{__shfl_xor_sync(0xFFFFFFFFu, st.m, o), __shfl_xor_sync(0xFFFFFFFFu, st.s, o), __shfl_xor_sync(0xFFFFFFFFu, st.t, o)};
    st = lane & o ? join(b, st) : join(st, b);
    before += __shfl_xor_sync(0xFFFFFFFFu, before, o);
  }
  const float base = st.m == -INFINITY ? 0.0f : st.m, lse = logf(st.s);
  auto logprob = [&](float v) { return v == -INFINITY && !isnan(lse) ? -INFINITY : (v - base) - lse; };
  if (lane == 0) {
    a.logprobs[row] = has ? logprob(given) : id64 < 0 ? 0.0f : NAN;
    a.ranks[row] = has ? before + 1 : 0;
    a.entropy[row] = st.s == 0.0f ? 0.0f : lse - st.t * LN2 / st.s;
  }
  if (!a.top_n) return;
  unsigned long long *cand = cand_all[warp], *best = best_all[warp];
  int& found_at = found_all[warp];
  if (lane == 0) found_at = 0;
  best[lane] = 0;
  int place = 0;
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    const float v = __shfl_sync(0xFFFFFFFFu, mine, j);
    place += v > mine || (v == mine && j < lane);
  }
  const float limit = __shfl_sync(0xFFFFFFFFu, mine, __ffs(__ballot_sync(0xFFFFFFFFu, place == a.top_n - 1)) - 1);
  __syncwarp();
  if (mine >= limit)
    each([&](float v, int i) {
      if (v >= limit) {
        const int slot = atomicAdd(&found_at, 1);
        if (slot < LPW_ROOM) cand[slot] = lp_key(v, i);
      }
    });
  __syncwarp();
  const int found = found_at;
  if (found <= LPW_ROOM && found >= min(a.top_n, a.vocab)) {
    for (int i = lane; i < found; i += 32) {
      const unsigned long long k = cand[i];
      int at = 0;
      for (int j = 0; j < found; ++j) at += cand[j] > k;
      if (at < a.top_n) best[at] = k;
    }
  } else {                                        // many equal ones, or fewer numbers than alternatives: the next key of the row each time
    unsigned long long last = ~0ull;
    for (int n = 0; n < a.top_n && last; ++n) {
      unsigned long long k = 0;
      each([&](float v, int i) {
        const unsigned long long q = lp_key(v, i);
        if (q < last && q > k) k = q;
      });
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long q = __shfl_xor_sync(0xFFFFFFFFu, k, o);
        if (q > k) k = q;
      }
      if (lane == 0) best[n] = k;
      last = k;
    }
  }
  __syncwarp();
  if (lane < a.top_n) {
    const unsigned long long k = best[lane];
    a.top_logprobs[row * a.top_n + lane] = k ? logprob(lp_key_value(k)) : -INFINITY;
    a.top_ids[row * a.top_n + lane] = k ? 0x7FFFFFFF - (int)(uint32_t)k : -1;
  }
}

template <typename T>
static int launch_logprobs(const LogprobArgs& a, int64_t m, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // (behind_previous)
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (a.vocab <= LPW_VECTORS * 32 * Vec<T>::N) {
    cfg.gridDim = dim3((unsigned)((m + LPW_WARPS - 1) / LPW_WARPS));
    cfg.blockDim = dim3(LPW_WARPS * 32);
    GSQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, logprobs_rows_kernel<T>, a, (int)m));
    return GSQ_OK;
  }
  DeviceInfo di;
  const int rc = device_info(&di);
  if (rc != GSQ_OK) return rc;
  const void* kern = (const void*)logprobs_kernel<T>;
  // blocks of a row: doubled while that leaves every block half a round of loads or more and the grid within two blocks an SM. One row with 0 (20) alternatives, so and with
  // a whole round at least: 16400 values 4.5, 4.9 us (8.2, 8.6), 64000 4.6, 5.1 (8.5, 8.9), 151936 5.4, 5.5 (9.5, 9.4); of a single round the other is the better, 8193 values 4.4, 3.7 (8.2, 6.1)
  const int64_t rounds = (a.vocab / Vec<T>::N) / (LP_THREADS * LP_UNROLL);
  int cs = 1;
  while (cs < 16 && 2 * cs * m <= 2 * di.sm_count && cs <= rounds) cs *= 2;
  if (cs > 8) {
    static OncePerDevice large;
    const int set = large.set(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (set != GSQ_OK) return set;
  }
  cfg.gridDim = dim3((unsigned)(m * cs));
  cfg.blockDim = dim3(LP_THREADS);
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cs;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.numAttrs = 2;
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
  if ((uintptr_t)logits % (dtype == GSQ_F32 ? 4 : 2) || ((uintptr_t)logprobs | (uintptr_t)entropy | (uintptr_t)top_logprobs) % 4 ||
      ((uintptr_t)token_ids | (uintptr_t)ranks | (uintptr_t)top_ids) % 8)
    return GSQ_ERR_UNSUPPORTED;
  const LogprobArgs a{logits, row_stride, (int)vocab, top_n, token_ids, logprobs, ranks, entropy, top_logprobs, top_ids};
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == GSQ_F32) return launch_logprobs<float>(a, m, st);
  return dtype == GSQ_F16 ? launch_logprobs<__half>(a, m, st) : launch_logprobs<__nv_bfloat16>(a, m, st);
}
