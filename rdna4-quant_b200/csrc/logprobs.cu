// Likelihoods of given tokens: log softmax at the token, its rank, the entropy
// of the row and its k most likely ids, in one pass over the logits.
//
//   m = max x,  S = sum e^(x - m),  A = sum e^(x - m) (x - m)
//   logprob = (x_t - m) - log S,    entropy = log S - A / S
//
// (m, S, A) of parts join like a softmax's: with M = max m and f = e^(m - M),
// S <- sum f S and A <- sum f (A + S (m - M)).  Ids are ordered by one 64-bit
// key (value, lowest id first), so every selection has one right answer.
//
// Bound: HBM, each logit read once.  A cluster of C CTAs shares a row (C = 1 for
// many rows; up to 8 for few, so that a single row of a large vocabulary is
// spread over the SMs); a thread keeps four 16-byte loads in flight, takes their
// maximum on packed pairs, and rescales its running sums only when that moved.
//
// Top k.  While it streams, every thread keeps its largest value and the place
// of the chunk that had it, i.e. an upper and a lower bound of its largest key.
// The k-th largest of the lower bounds of disjoint groups of elements is a lower
// bound tau of the k-th largest key, and a close one: of 128 groups of four
// threads, about k (1 + k / 256) elements reach it.  Only groups whose upper
// bound reaches tau are read again (k of 128, from L2, unless values tie), and
// what reaches tau, some k elements, goes into sorted warp lists of 32 that bound
// the count whatever the values are (ties, masks, sorted rows).  Ranks among
// the lists' keys then give the CTA's order, and sorted lists of CTAs merge.
#include <cuda_bf16.h>

#include "r4q_common.cuh"

namespace r4q {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 32;
constexpr int kGroups = kThreads / 4;     // of four neighbouring threads
constexpr int kMaxCluster = 8;
constexpr int kUnroll = 4;                // 16-byte loads in flight per thread
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// order of floats as unsigned integers; NaN is the lowest, -0 equals +0
__device__ __forceinline__ uint32_t ordered(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(float x, int i) {
  return ((uint64_t)ordered(x) << 32) | (0xffffffffu - (uint32_t)i);
}
__device__ __forceinline__ int id_of(uint64_t key) { return (int)(0xffffffffu - (uint32_t)key); }
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return o == 0u ? __int_as_float(0x7fc00000) : __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}

// A type's 16-byte word: its floats, the largest of four words (NaN if there
// is one; `skip` passes over NaN), and the word of single elements.
template <typename X> struct Vec;
template <> struct Vec<__half> {
  static constexpr int n = 8;
  static __device__ __forceinline__ void get(const uint4 u, float (&x)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(u32_as_h2(w[j]));
      x[2 * j] = f.x;
      x[2 * j + 1] = f.y;
    }
  }
  static __device__ __forceinline__ float most(const uint4 u) {
    const __half2 m = __hmax2_nan(__hmax2_nan(u32_as_h2(u.x), u32_as_h2(u.y)),
                                  __hmax2_nan(u32_as_h2(u.z), u32_as_h2(u.w)));
    return __half2float(__hmax_nan(__low2half(m), __high2half(m)));
  }
  static __device__ __forceinline__ float most4(const uint4 (&u)[4]) {
    auto mx = [](uint32_t a, uint32_t b) { return h2_as_u32(__hmax2_nan(u32_as_h2(a), u32_as_h2(b))); };
    uint4 m;
    m.x = mx(mx(u[0].x, u[1].x), mx(u[2].x, u[3].x));
    m.y = mx(mx(u[0].y, u[1].y), mx(u[2].y, u[3].y));
    m.z = mx(mx(u[0].z, u[1].z), mx(u[2].z, u[3].z));
    m.w = mx(mx(u[0].w, u[1].w), mx(u[2].w, u[3].w));
    return most(m);
  }
  static __device__ __forceinline__ float one(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ uint32_t bits(const __half* p) { return __half_as_ushort(*p); }
  static constexpr uint32_t kNegInf = 0xfc00u;
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int n = 8;
  static __device__ __forceinline__ void get(const uint4 u, float (&x)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[2 * j] = __uint_as_float(w[j] << 16);
      x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint32_t mx(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  static __device__ __forceinline__ float most(const uint4 u) {
    const uint32_t m = mx(mx(u.x, u.y), mx(u.z, u.w));
    return __uint_as_float(mx(m, m << 16) & 0xffff0000u);
  }
  static __device__ __forceinline__ float most4(const uint4 (&u)[4]) {
    uint4 m;
    m.x = mx(mx(u[0].x, u[1].x), mx(u[2].x, u[3].x));
    m.y = mx(mx(u[0].y, u[1].y), mx(u[2].y, u[3].y));
    m.z = mx(mx(u[0].z, u[1].z), mx(u[2].z, u[3].z));
    m.w = mx(mx(u[0].w, u[1].w), mx(u[2].w, u[3].w));
    return most(m);
  }
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ uint32_t bits(const __nv_bfloat16* p) { return __bfloat16_as_ushort(*p); }
  static constexpr uint32_t kNegInf = 0xff80u;
};
template <> struct Vec<float> {
  static constexpr int n = 4;
  static __device__ __forceinline__ void get(const uint4 u, float (&x)[4]) {
    x[0] = __uint_as_float(u.x);
    x[1] = __uint_as_float(u.y);
    x[2] = __uint_as_float(u.z);
    x[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ float mx(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
  }
  static __device__ __forceinline__ float most(const uint4 u) {
    return mx(mx(__uint_as_float(u.x), __uint_as_float(u.y)), mx(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
  static __device__ __forceinline__ float most4(const uint4 (&u)[4]) {
    return mx(mx(most(u[0]), most(u[1])), mx(most(u[2]), most(u[3])));
  }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ uint32_t bits(const float* p) { return __float_as_uint(*p); }
  static constexpr uint32_t kNegInf = 0xff800000u;
};

// A row as 16-byte words of the memory it lies in: word i holds elements
// i n - head .. of the row; of the first and the last one perhaps only some are
// the row's, and those alone are read.  What is outside the row counts as -inf.
template <typename X>
struct Row {
  const X* x;
  int V, head, words;
  __device__ __forceinline__ Row(const X* p, int V_) : x(p), V(V_) {
    head = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(X));
    words = (head + V + Vec<X>::n - 1) / Vec<X>::n;
  }
  __device__ __forceinline__ int first(int i) const { return i * Vec<X>::n - head; }   // element
  __device__ __forceinline__ uint4 load(int i) const {
    const int e = first(i);
    if (i < words && e >= 0 && e + Vec<X>::n <= V) return *reinterpret_cast<const uint4*>(x + e);
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < Vec<X>::n; ++j) {
      const uint32_t b = i < words && e + j >= 0 && e + j < V ? Vec<X>::bits(x + e + j) : Vec<X>::kNegInf;
      if (Vec<X>::n == 8) w[j / 2] |= b << (16 * (j & 1)); else w[j & 3] = b;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

struct Sums {
  float m = -INFINITY, S = 0.f, A = 0.f;
  __device__ __forceinline__ void join(float m2, float S2, float A2) {
    const float M = fmaxf(m, m2);
    if (M == -INFINITY) return;
    const float d = fmaxf(m - M, -1e4f), d2 = fmaxf(m2 - M, -1e4f), f = ex2(d * kLog2e), f2 = ex2(d2 * kLog2e);
    A = f * (A + S * d) + f2 * (A2 + S2 * d2);
    S = f * S + f2 * S2;
    m = M;
  }
};

struct Shared {
  alignas(16) uint64_t group[kGroups];   // lower bound of the largest key of each group of this CTA
  uint64_t list[kWarps * kMaxTop];       // collected keys
  uint64_t top[kMaxTop];                 // this CTA's k best
  float m[kWarps], S[kWarps], A[kWarps];
  int before[kWarps], nan[kWarps];
  uint64_t tau;
  int n_list;
  float cm, cS, cA;                      // this CTA's sums
  int cbefore, cnan;
};

__device__ __forceinline__ uint32_t peer(const void* p, int rank) {
  uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(p)), r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
__device__ __forceinline__ float peer_f(const float* p, int rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ int peer_i(const int* p, int rank) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(peer(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t peer_u(const uint64_t* p, int rank) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(peer(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Keeps the warp's 32 best keys, lane i the i-th best: takes lane `from`'s key.
__device__ __forceinline__ void insert(uint64_t& best, uint64_t key, int lane) {
  const unsigned better = __ballot_sync(0xffffffffu, best > key);   // a prefix: the list is sorted
  const uint64_t up = __shfl_up_sync(0xffffffffu, best, 1);
  const int at = __popc(better);
  if (lane == at) best = key;
  if (lane > at) best = up;
}

// The 32 best of two sorted lists (lane i: the i-th best), sorted: the larger of
// a[i] and b[31 - i] are those, a bitonic sequence, which five steps sort.
__device__ __forceinline__ uint64_t merge(uint64_t a, uint64_t b, int lane) {
  const uint64_t o = __shfl_xor_sync(0xffffffffu, b, 31);
  uint64_t v = a > o ? a : o;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const uint64_t p = __shfl_xor_sync(0xffffffffu, v, d);
    v = ((lane & d) == 0) == (v > p) ? v : p;
  }
  return v;
}

template <typename X>
__global__ void __launch_bounds__(kThreads, 2)
    logprobs_kernel(const X* __restrict__ logits, long ld, const long long* __restrict__ tokens, int V, int k,
                    float* logprob, long long* rank_out, float* entropy, long long* top_ids, float* top_lp) {
  constexpr int n = Vec<X>::n;
  __shared__ Shared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, C = gridDim.x, cta = blockIdx.x;
  const long row = blockIdx.y;
  pdl_wait_trigger();
  const Row<X> r(logits + row * ld, V);
  const long long tok = tokens ? tokens[row] : -1;
  const bool has_t = tok >= 0 && tok < V;
  const int t = has_t ? (int)tok : -1;
  const float xt = has_t ? Vec<X>::one(r.x + t) : INFINITY;

  // ---- one pass: this CTA's words cta * kThreads + tid, strided by C * kThreads
  Sums s;
  float best = -INFINITY;
  int best_w = -1, before = 0, nan = 0;      // best_w: first word of the chunk with the thread's largest value
  const int stride = C * kThreads;
  for (int i = cta * kThreads + tid; i < r.words; i += kUnroll * stride) {
    uint4 u[kUnroll];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) u[j] = r.load(i + j * stride);
    float c = Vec<X>::most4(u);
    if (c != c) {                            // NaN: the row is none; the order goes on without it
      nan = 1;
      c = -INFINITY;
#pragma unroll
      for (int j = 0; j < kUnroll; ++j) {
        float x[n];
        Vec<X>::get(u[j], x);
#pragma unroll
        for (int q = 0; q < n; ++q) c = fmaxf(c, x[q]);
      }
    }
    if (c > best || best_w < 0) {
      best = c;
      best_w = i;
    }
    if (c > s.m) {
      const float d = fmaxf(s.m - c, -1e4f), f = ex2(d * kLog2e);
      s.A = f * (s.A + s.S * d);
      s.S *= f;
      s.m = c;
    }
    const float m = s.m == -INFINITY ? 0.f : s.m;
    const bool count = c >= xt || xt != xt;
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      float x[n];
      Vec<X>::get(u[j], x);
#pragma unroll
      for (int q = 0; q < n; ++q) {
        const float d = fmaxf(x[q] - m, -1e4f), e = ex2(d * kLog2e);   // -inf: no 0 * inf
        s.S += e;
        s.A = fmaf(e, d, s.A);
      }
      if (count) {                           // what precedes the token
        const int e0 = r.first(i + j * stride);
#pragma unroll
        for (int q = 0; q < n; ++q) {
          const unsigned e = (unsigned)(e0 + q);
          if (xt == xt) before += x[q] > xt || (x[q] == xt && e < (unsigned)t);
          else before += e < (unsigned)V && (x[q] == x[q] || e < (unsigned)t);
        }
      }
    }
  }

  // ---- the CTA's sums, and bounds of the largest key of each group of four threads
  uint64_t upper = 0, lower = 0;
  if (best_w >= 0) {
    upper = key_of(best, max(0, r.first(best_w)));
    // of its chunk, the last element of the row
    const int w = best_w + min(kUnroll - 1, (r.words - 1 - best_w) / stride) * stride;
    lower = key_of(best, min(V - 1, r.first(w) + n - 1));
  }
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) {
    const uint64_t o = __shfl_xor_sync(0xffffffffu, upper, d), p = __shfl_xor_sync(0xffffffffu, lower, d);
    upper = o > upper ? o : upper;
    lower = p > lower ? p : lower;
  }
  // -inf may stand for NaN alone, which comes after it: no bound
  if (lane % 4 == 0) sh.group[tid >> 2] = (uint32_t)(lower >> 32) > ordered(-INFINITY) ? lower : 0ull;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    s.join(__shfl_xor_sync(0xffffffffu, s.m, d), __shfl_xor_sync(0xffffffffu, s.S, d),
           __shfl_xor_sync(0xffffffffu, s.A, d));
    before += __shfl_xor_sync(0xffffffffu, before, d);
    nan |= __shfl_xor_sync(0xffffffffu, nan, d);
  }
  if (lane == 0) {
    sh.m[warp] = s.m;
    sh.S[warp] = s.S;
    sh.A[warp] = s.A;
    sh.before[warp] = before;
    sh.nan[warp] = nan;
  }
  if (tid == 0) {
    sh.n_list = 0;
    sh.tau = 0;
  }
  if (tid < kMaxTop) sh.top[tid] = 0;
  __syncthreads();
  if (warp == kWarps - 1) {
    Sums c;
    int b = 0, bad = 0;
    if (lane < kWarps) {
      c.m = sh.m[lane];
      c.S = sh.S[lane];
      c.A = sh.A[lane];
      b = sh.before[lane];
      bad = sh.nan[lane];
    }
#pragma unroll
    for (int d = kWarps / 2; d > 0; d >>= 1) {
      c.join(__shfl_xor_sync(0xffffffffu, c.m, d), __shfl_xor_sync(0xffffffffu, c.S, d),
             __shfl_xor_sync(0xffffffffu, c.A, d));
      b += __shfl_xor_sync(0xffffffffu, b, d);
      bad |= __shfl_xor_sync(0xffffffffu, bad, d);
    }
    if (lane == 0) {
      sh.cm = c.m;
      sh.cS = c.S;
      sh.cA = c.A;
      sh.cbefore = b;
      sh.cnan = bad;
    }
  }

  // ---- the CTA's k best
  if (k > 0) {
    if (tid < kGroups) {                               // tau: the k-th largest lower bound, or 0
      const uint64_t mine = sh.group[tid];
      int above = 0;
#pragma unroll 8
      for (int q = 0; q < kGroups; q += 2) {
        const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(&sh.group[q]);
        above += (two.x > mine) + (two.y > mine);
      }
      if (above == k - 1 && mine) sh.tau = mine;
    }
    __syncthreads();
    const uint64_t tau = sh.tau;
    const float tau_value = value_of(tau);
    uint64_t mine = 0;                                 // the warp's best so far, lane i the i-th
    unsigned open = __ballot_sync(0xffffffffu, lane % 4 == 0 && upper >= tau);   // no bound: every group
    for (; open; open &= open - 1) {                   // a group's words: four neighbours in each stride
      const int first = cta * kThreads + warp * 32 + __ffs(open) - 1;
      for (int base = 0; first + base * stride < r.words; base += 8) {   // 8 strides x 4 words at once
        const int w = first + lane % 4 + (base + lane / 4) * stride;
        const uint4 u = r.load(w);
        if (tau && !__any_sync(0xffffffffu, !(Vec<X>::most(u) < tau_value))) continue;
        float x[n];
        Vec<X>::get(u, x);
#pragma unroll
        for (int q = 0; q < n; ++q) {
          const int e = r.first(w) + q;
          const uint64_t key = w < r.words && e >= 0 && e < V ? key_of(x[q], e) : 0ull;
          const uint64_t floor = __shfl_sync(0xffffffffu, mine, k - 1);
          unsigned in = __ballot_sync(0xffffffffu, key >= tau && key > floor);
          for (; in; in &= in - 1) insert(mine, __shfl_sync(0xffffffffu, key, __ffs(in) - 1), lane);
        }
      }
    }
    const unsigned have = __ballot_sync(0xffffffffu, lane < k && mine);
    int at = 0;
    if (lane == 0 && have) at = atomicAdd(&sh.n_list, __popc(have));   // in any order: the keys are ranked below
    at = __shfl_sync(0xffffffffu, at, 0);
    if (have >> lane & 1) sh.list[at + lane] = mine;
    __syncthreads();
    const int total = sh.n_list;
    for (int i = tid; i < total; i += kThreads) {
      const uint64_t key = sh.list[i];
      int above = 0;
#pragma unroll 4
      for (int q = 0; q < total; ++q) above += sh.list[q] > key;
      if (above < k) sh.top[above] = key;
    }
  }
  if (C > 1) cluster_sync(); else __syncthreads();

  // ---- CTA 0 of the cluster joins the others and writes the row
  if (cta == 0 && warp == 0) {
    Sums c;
    int b = 0, bad = 0;
    if (lane < C) {
      c.m = peer_f(&sh.cm, lane);
      c.S = peer_f(&sh.cS, lane);
      c.A = peer_f(&sh.cA, lane);
      b = peer_i(&sh.cbefore, lane);
      bad = peer_i(&sh.cnan, lane);
    }
    uint64_t list[kMaxCluster];                        // sorted lists of the CTAs, lane i the i-th key
    if (k > 0)
#pragma unroll
      for (int q = 0; q < kMaxCluster; ++q) list[q] = q < C ? peer_u(&sh.top[lane], q) : 0ull;
#pragma unroll
    for (int d = kMaxCluster / 2; d > 0; d >>= 1) {
      c.join(__shfl_xor_sync(0xffffffffu, c.m, d), __shfl_xor_sync(0xffffffffu, c.S, d),
             __shfl_xor_sync(0xffffffffu, c.A, d));
      b += __shfl_xor_sync(0xffffffffu, b, d);
      bad |= __shfl_xor_sync(0xffffffffu, bad, d);
    }
    const float m = __shfl_sync(0xffffffffu, c.m, 0), S = __shfl_sync(0xffffffffu, c.S, 0);
    const bool none = __shfl_sync(0xffffffffu, bad, 0) || isinf(m);
    const float quiet = __int_as_float(0x7fc00000), logS = logf(S);
    if (lane == 0) {
      if (logprob) logprob[row] = none || !has_t ? quiet : xt - m - logS;
      if (rank_out) rank_out[row] = has_t ? b + 1 : 0;
      if (entropy) entropy[row] = none ? quiet : logS - c.A / S;
    }
    if (k > 0) {
      if (C > 1)
#pragma unroll
        for (int d = kMaxCluster / 2; d > 0; d >>= 1)
#pragma unroll
          for (int q = 0; q < d; ++q) list[q] = merge(list[q], list[q + d], lane);
      if (lane < k) {
        if (top_ids) top_ids[row * k + lane] = id_of(list[0]);
        if (top_lp) top_lp[row * k + lane] = none ? quiet : value_of(list[0]) - m - logS;
      }
    }
  }
  if (C > 1) cluster_sync();                           // shared memory stays until CTA 0 has read it
}

template <typename X>
int launch(const void* logits, long ld, const long long* tokens, int M, int V, int k, float* logprob, long long* rank,
           float* entropy, long long* top_ids, float* top_lp, cudaStream_t st) {
  // CTAs per row: as many as keep one word per thread and the grid within two CTAs an SM
  int C = kMaxCluster;
  while (C > 1 && ((long)M * C > 2L * num_sms() || (long)(C / 2) * kThreads * Vec<X>::n >= V)) C >>= 1;
  for (int at = 0; at < M; at += 65535) {
    const int rows = M - at < 65535 ? M - at : 65535;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(C, rows);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim.x = C;
    attrs[0].val.clusterDim.y = 1;
    attrs[0].val.clusterDim.z = 1;
    attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = 2;
    const long long o = at;
    const cudaError_t e = cudaLaunchKernelEx(
        &cfg, logprobs_kernel<X>, (const X*)logits + o * ld, ld, tokens ? tokens + o : nullptr, V, k,
        logprob ? logprob + o : nullptr, rank ? rank + o : nullptr, entropy ? entropy + o : nullptr,
        top_ids ? top_ids + o * k : nullptr, top_lp ? top_lp + o * k : nullptr);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return set_error(R4Q_ERR_CUDA, "logprobs_kernel (cluster %d): %s", C, cudaGetErrorString(e));
    }
  }
  return R4Q_OK;
}

}  // namespace
}  // namespace r4q

using namespace r4q;

extern "C" int r4q_token_logprobs(const void* logits, int type, long ld, const long long* tokens, int M, int V, int k,
                                  float* logprob, long long* rank, float* entropy, long long* top_ids,
                                  float* top_logprobs, void* stream) {
  if (M < 0 || V < 1 || V > 0x3fffffff || k < 0 || k > kMaxTop || k > V)
    return set_error(R4Q_ERR_ARG, "token_logprobs: bad shape (rows %d, vocabulary %d, k %d of at most %d)", M, V, k,
                     kMaxTop);
  if (type != R4Q_T_F16 && type != R4Q_T_BF16 && type != R4Q_T_F32)
    return set_error(R4Q_ERR_ARG, "token_logprobs: unknown type %d", type);
  if (M == 0) return R4Q_OK;
  if (!logits || (M > 1 && ld < V))
    return set_error(R4Q_ERR_ARG, "token_logprobs: null logits or row stride %ld < %d", ld, V);
  if (!tokens && (logprob || rank)) return set_error(R4Q_ERR_ARG, "token_logprobs: logprob and rank need tokens");
  if (!aligned(logits, type == R4Q_T_F32 ? 4 : 2)) return set_error(R4Q_ERR_ALIGN, "token_logprobs: logits misaligned");
  const auto go = type == R4Q_T_F16 ? launch<__half> : type == R4Q_T_BF16 ? launch<__nv_bfloat16> : launch<float>;
  return go(logits, ld, tokens, M, V, k, logprob, rank, entropy, top_ids, top_logprobs, (cudaStream_t)stream);
}
