// Likelihoods of given tokens: log softmax at the token, its rank, the entropy
// of the row and its k most likely ids, in one pass over the logits.
//
//   m = max x,  t = (x - m) log2(e),  S = sum 2^t,  A = sum 2^t t
//   logprob = (x_t - m) - ln2 log2 S,    entropy = ln2 (log2 S - A / S)
//
// (m, S, A) of parts join like a softmax's: with M = max m, d = (m - M) log2(e)
// and f = 2^d, S <- sum f S and A <- sum f (A + S d).  Ids are ordered by one
// 64-bit key (value, lowest id first), so every selection has one right answer.
//
// Bound: HBM, each logit read once, if the issue slots allow: 11.6 logits a clock
// and SM at the measured bandwidth, of some five instructions each.  So maxima
// are taken on packed pairs, the sums with two-wide fp32 instructions, the
// running sums are rescaled only when the maximum moved, and f16 logits need one
// multiply-add for t: 2^t is taken from x log2(e) - M with M the rounded
// m log2(e), whose rounding (at most 2^-8) the thread takes out of its sums once.
// (bf16 and fp32 logits may be so large that it would not be small: subtract first.)
// A cluster of C CTAs shares a row (C = 1 for many rows; up to 8 for few, so that
// a single row of a large vocabulary is spread over the SMs); CTAs are small, so
// that others stream while one selects.  Every warp streams its own 2 KB chunks
// through a ring in shared memory by bulk copies, two ahead: loads ahead in
// registers cost occupancy or spills (2048 x 151936 f16, top 5: 294 us with a chunk
// ahead in registers, 199 us without).
//
// Top k.  While it streams, every thread keeps its largest value and the place
// of the chunk that had it, i.e. an upper and a lower bound of its largest key.
// The k-th largest of the lower bounds of disjoint groups of elements is a lower
// bound tau of the k-th largest key, and a close one: of 128 groups of threads,
// about k (1 + k / 256) elements reach it.  Only the elements of threads whose
// upper bound reaches tau are read again (some k threads, from L2, unless values
// tie), by the whole CTA at once, and what reaches tau is put into a list.  Should
// that overflow (ties, masks, sorted rows), every warp goes through its own
// threads' elements with a sorted list of its 32 best, which bounds the count
// whatever the values are.  Ranks among the lists' keys then give the CTA's
// order, and sorted lists of CTAs merge.
#include <cuda_bf16.h>

#include <mutex>
#include <type_traits>

#include "f32x2.cuh"
#include "paged.cuh"
#include "r4q_common.cuh"
#include "tma_dev.cuh"

namespace r4q {
namespace {

constexpr int kThreads = 256;
constexpr int kResident = 4;              // CTAs per SM that the registers allow
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 32;
constexpr int kGroups = 128;              // of neighbouring threads
constexpr int kGroupLanes = kThreads / kGroups;
constexpr int kList = kWarps * kMaxTop;   // collected keys of a CTA
constexpr int kMaxCluster = 8;
constexpr int kUnroll = 4;                // 16-byte words of a lane in a chunk
constexpr int kChunk = 32 * kUnroll;      // words of a warp's chunk, 2 KB
constexpr int kStages = 2;                // chunks of a warp's ring
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kTiny = -150.f;           // 2^kTiny is 0 in fp32: also stands for log2 0, where 0 * -inf would be NaN

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

// A type's 16-byte word: its floats, its largest and the largest of four words
// (NaN if there is one), and how single elements are read.
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
  // how many elements of four words exceed the words' thresholds (a pair of one value each)
  static __device__ __forceinline__ int above(const uint4 (&u)[4], const uint32_t (&th)[4]) {
    __half2 a = __float2half2_rn(0.f);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2 h = u32_as_h2(th[j]);
      a = __hadd2(a, __hadd2(__hadd2(__hgt2(u32_as_h2(u[j].x), h), __hgt2(u32_as_h2(u[j].y), h)),
                             __hadd2(__hgt2(u32_as_h2(u[j].z), h), __hgt2(u32_as_h2(u[j].w), h))));
    }
    return __half2int_rn(__hadd(__low2half(a), __high2half(a)));
  }
  static __device__ __forceinline__ float one(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ uint32_t bits(const __half* p) { return __half_as_ushort(*p); }
  static constexpr uint32_t kNegInf = 0xfc00u, kSign = 0x8000u, kPair = 0x10001u;
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
  static __device__ __forceinline__ int above(const uint4 (&u)[4], const uint32_t (&th)[4]) {
    auto b2 = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
    __nv_bfloat162 a = __float2bfloat162_rn(0.f);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __nv_bfloat162 h = b2(th[j]);
      a = __hadd2(a, __hadd2(__hadd2(__hgt2(b2(u[j].x), h), __hgt2(b2(u[j].y), h)),
                             __hadd2(__hgt2(b2(u[j].z), h), __hgt2(b2(u[j].w), h))));
    }
    return (int)(__low2float(a) + __high2float(a));
  }
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ uint32_t bits(const __nv_bfloat16* p) { return __bfloat16_as_ushort(*p); }
  static constexpr uint32_t kNegInf = 0xff80u, kSign = 0x8000u, kPair = 0x10001u;
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
  static __device__ __forceinline__ int above(const uint4 (&u)[4], const uint32_t (&th)[4]) {
    int a = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float h = __uint_as_float(th[j]);
      a += (__uint_as_float(u[j].x) > h) + (__uint_as_float(u[j].y) > h) + (__uint_as_float(u[j].z) > h) +
           (__uint_as_float(u[j].w) > h);
    }
    return a;
  }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ uint32_t bits(const float* p) { return __float_as_uint(*p); }
  static constexpr uint32_t kNegInf = 0xff800000u, kSign = 0x80000000u, kPair = 1u;
};

// A row as 16-byte words of the memory it lies in: word i holds elements
// i n - head .. of the row; of the first and the last one perhaps only some are
// the row's, and those alone are read.  What is outside the row counts as -inf.
template <typename X>
struct Row {
  const X* x;
  int V, head, words, lo, hi;              // words lo .. hi are the row's entirely
  __device__ __forceinline__ Row(const X* p, int V_) : x(p), V(V_) {
    head = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(X));
    words = (head + V + Vec<X>::n - 1) / Vec<X>::n;
    lo = head ? 1 : 0;
    hi = (head + V) / Vec<X>::n - 1;
  }
  __device__ __forceinline__ int first(int i) const { return i * Vec<X>::n - head; }   // element
  __device__ __forceinline__ uint4 load(int i) const {
    const int e = first(i);
    if (i >= lo && i <= hi) return *reinterpret_cast<const uint4*>(x + e);
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < Vec<X>::n; ++j) {
      const uint32_t b = i < words && e + j >= 0 && e + j < V ? Vec<X>::bits(x + e + j) : Vec<X>::kNegInf;
      if (Vec<X>::n == 8) w[j / 2] |= b << (16 * (j & 1)); else w[j & 3] = b;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // whether the chunk of words from i on is the row's entirely, i.e. may be copied in bulk
  __device__ __forceinline__ bool bulk(int i) const { return i >= lo && i + kChunk - 1 <= hi; }
  __device__ __forceinline__ const void* at(int i) const { return x - head + (long)i * Vec<X>::n; }
};

struct Sums {
  float m = -INFINITY, S = 0.f, A = 0.f;
  __device__ __forceinline__ void join(float m2, float S2, float A2) {
    const float M = fmaxf(m, m2);
    if (M == -INFINITY) return;
    const float d = fmaxf((m - M) * kLog2e, kTiny), d2 = fmaxf((m2 - M) * kLog2e, kTiny), f = ex2(d), f2 = ex2(d2);
    A = f * (A + S * d) + f2 * (A2 + S2 * d2);
    S = f * S + f2 * S2;
    m = M;
  }
};

struct Shared {
  alignas(16) uint64_t group[kGroups];   // lower bound of the largest key of each group of this CTA
  uint64_t list[kList];                  // collected keys
  uint64_t top[kMaxTop];                 // this CTA's k best
  uint64_t bars[kWarps * kStages];
  float m[kWarps], S[kWarps], A[kWarps];
  int before[kWarps], nan[kWarps];
  unsigned char open[kThreads];          // threads whose elements are read again
  uint64_t tau;
  int n_open, n_list;
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

__device__ int g_logprob_status;         // a bounded wait gave up

__device__ __forceinline__ void copy_chunk(void* dst, const void* src, uint64_t* bar) {
  mbar_expect_tx(bar, kChunk * 16);
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)), "l"(src), "r"(kChunk * 16), "r"(smem_u32(bar)) : "memory");
}

template <typename X>
__global__ void __launch_bounds__(kThreads, kResident)
    logprobs_kernel(const X* __restrict__ logits, long ld, const long long* __restrict__ tokens, int V, int k,
                    float* logprob, long long* rank_out, float* entropy, long long* top_ids, float* top_lp, int polls) {
  constexpr int n = Vec<X>::n;
  __shared__ Shared sh;
  extern __shared__ __align__(16) uint4 ring_mem[];    // [warp][stage][kChunk]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, C = gridDim.x, cta = blockIdx.x;
  const long row = blockIdx.y;
  const Row<X> r(logits + row * ld, V);
  if (lane == 0) {
#pragma unroll
    for (int j = 0; j < kStages; ++j) mbar_init(&sh.bars[warp * kStages + j], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  pdl_wait_trigger();
  // ---- one pass: chunks of the row, dealt to the warps of the cluster in turn
  constexpr bool kFused = std::is_same<X, __half>::value;    // t in one multiply-add
  const F2 l2e(kLog2e, kLog2e);
  F2 SA(0.f, 0.f), low(0.f, 0.f), shift(0.f, 0.f);   // S and A, and what their additions rounded away
  float most = -INFINITY, M = 0.f;           // running maximum; what t is relative to: m, or m log2(e) rounded
  float best = -INFINITY;
  int best_w = -1, before = 0, nan = 0;      // best_w: first word of the chunk with the thread's largest value
  const int stride = C * kWarps * kChunk, begin = (cta * kWarps + warp) * kChunk;
  uint4* ring = ring_mem + warp * kStages * kChunk;
  uint64_t* bars = sh.bars + warp * kStages;
  if (lane == 0)
#pragma unroll
    for (int j = 0; j < kStages; ++j)
      if (begin + j * stride < r.words && r.bulk(begin + j * stride))
        copy_chunk(ring + j * kChunk, r.at(begin + j * stride), &bars[j]);
  const long long tok = tokens ? tokens[row] : -1;
  const bool has_t = tok >= 0 && tok < V;
  const int t = has_t ? (int)tok : -1;
  const float xt = has_t ? Vec<X>::one(r.x + t) : INFINITY;
  // what precedes the token: values above xt, and with a lower id those equal to
  // it, i.e. above the next lower value
  const uint32_t tb = has_t ? Vec<X>::bits(r.x + t) : 0u;
  const uint32_t above_t = tb * Vec<X>::kPair;
  const uint32_t from_t = ((tb & ~Vec<X>::kSign) == 0 ? Vec<X>::kSign | 1u : tb & Vec<X>::kSign ? tb + 1 : tb - 1) *
                          Vec<X>::kPair;
  const bool plain_t = fabsf(xt) < INFINITY;

  int stage = 0;
  unsigned parity = 0;                       // bit j: of stage j
  for (int base = begin; base < r.words; base += stride) {
    const int i = base + lane;               // this lane's words: i, i + 32, ..
    uint4* mine = ring + stage * kChunk + lane;
    if (r.bulk(base)) {
      if (!mbar_wait_warp(&bars[stage], parity >> stage & 1, polls)) {
        // the copies in flight get their time once more; the row's results are void
        for (int j = 0; j < kStages; ++j) {
          const int s2 = (stage + j) % kStages, at = base + j * stride;
          if (at < r.words && r.bulk(at)) mbar_wait_warp(&bars[s2], parity >> s2 & 1, kWaitPolls);
        }
        if (lane == 0) atomicOr(&g_logprob_status, kPagedTimeout);
        nan = 1;
        break;
      }
      parity ^= 1u << stage;
    } else {                                 // a chunk at the row's ends: every lane puts its own words there
#pragma unroll 1
      for (int j = 0; j < kUnroll; ++j) mine[32 * j] = r.load(i + 32 * j);
    }
    // words are read from shared memory again where they are used: held in registers
    // throughout, they and what is made of them exceed the 64 of four CTAs an SM
    const uint32_t words = smem_u32(mine);
    float c;
    {
      uint4 u[kUnroll];
#pragma unroll
      for (int j = 0; j < kUnroll; ++j) u[j] = lds128(words + 512 * j);
      c = Vec<X>::most4(u);
    }
    if (c != c) {                            // NaN: the row is none; the order goes on without it
      nan = 1;
      c = -INFINITY;
#pragma unroll 1
      for (int j = 0; j < kUnroll; ++j) {
        float x[n];
        Vec<X>::get(lds128(words + 512 * j), x);
#pragma unroll
        for (int q = 0; q < n; ++q) c = fmaxf(c, x[q]);
      }
    }
    if (c > best || best_w < 0) {
      best = c;
      best_w = i;
    }
    if (c > most) {
      const float to = kFused ? c * kLog2e : c;
      const float d = most == -INFINITY ? kTiny : fmaxf(kFused ? M - to : (M - to) * kLog2e, kTiny), f = ex2(d);
      const float2 a = SA.get(), b = low.get();
      SA = F2(f * a.x, f * fmaf(a.x, d, a.y));
      low = F2(f * b.x, f * fmaf(b.x, d, b.y));
      most = c;
      M = to;
      shift = F2(-to, -to);
    }
    // the chunk's sums; -inf gives 0 * -inf in A, and only then t is bounded below
    F2 Sc(0.f, 0.f), Ac(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      float x[n];
      Vec<X>::get(lds128(words + 512 * j), x);
#pragma unroll
      for (int q = 0; q < n; q += 2) {
        const F2 two(x[q], x[q + 1]), t = kFused ? fma(two, l2e, shift) : mul(add(two, shift), l2e);
        const float2 f = t.get();
        const F2 e(ex2(f.x), ex2(f.y));
        Sc = add(Sc, e);
        Ac = fma(e, t, Ac);
      }
    }
    float2 sum = Ac.get();
    if (sum.x + sum.y != sum.x + sum.y) {
      Ac = F2(0.f, 0.f);
#pragma unroll 1
      for (int j = 0; j < kUnroll; ++j) {
        float x[n];
        Vec<X>::get(lds128(words + 512 * j), x);
#pragma unroll
        for (int q = 0; q < n; q += 2) {
          const F2 two(x[q], x[q + 1]);
          const float2 f = (kFused ? fma(two, l2e, shift) : mul(add(two, shift), l2e)).get();
          const F2 t(fmaxf(f.x, kTiny), fmaxf(f.y, kTiny));
          Ac = fma(F2(ex2(fmaxf(f.x, kTiny)), ex2(fmaxf(f.y, kTiny))), t, Ac);
        }
      }
      sum = Ac.get();
    }
    {   // to the thread's sums, whose rounding errors go along (Kahan 1965): a long row's would add up
      const float2 s = Sc.get();
      const F2 y = sub(F2(s.x + s.y, sum.x + sum.y), low), t = add(SA, y);
      low = sub(sub(t, SA), y);
      SA = t;
    }
    if (has_t && (c >= xt || xt != xt)) {    // what precedes the token
      uint32_t th[kUnroll];
      bool has = !plain_t;
#pragma unroll
      for (int j = 0; j < kUnroll; ++j) {
        const int e0 = r.first(i + 32 * j);
        th[j] = e0 < t ? from_t : above_t;
        has |= (unsigned)(t - e0) < (unsigned)n;
      }
      if (!has) {
        uint4 u[kUnroll];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) u[j] = lds128(words + 512 * j);
        before += Vec<X>::above(u, th);
      } else {                               // the token's own chunk; a token of no finite value
#pragma unroll 1
        for (int j = 0; j < kUnroll; ++j) {
          const int e0 = r.first(i + 32 * j);
          float x[n];
          Vec<X>::get(lds128(words + 512 * j), x);
#pragma unroll
          for (int q = 0; q < n; ++q) {
            const unsigned e = (unsigned)(e0 + q);
            before += xt == xt ? x[q] > xt || (x[q] == xt && e < (unsigned)t)
                               : e < (unsigned)V && (x[q] == x[q] || e < (unsigned)t);
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0) {                         // the stage is read: its next chunk may come
      const int at = base + kStages * stride;
      if (at < r.words && r.bulk(at)) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        copy_chunk(ring + stage * kChunk, r.at(at), &bars[stage]);
      }
    }
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  Sums s;
  s.m = most;
  {
    const float2 a = SA.get();
    const float off = kFused && most > -INFINITY && most < INFINITY ? fmaf(most, kLog2e, -M) : 0.f, f = ex2(-off);
    s.S = a.x * f;
    s.A = (a.y - off * a.x) * f;
  }

  // ---- bounds of the largest key of the thread, and the CTA's sums
  uint64_t upper = 0, lower = 0;
  if (best_w >= 0) {
    upper = key_of(best, max(0, r.first(best_w)));
    lower = key_of(best, min(V - 1, r.first(best_w + 32 * (kUnroll - 1)) + n - 1));   // the chunk's last, or a later one
  }
  // of the group; a value of -inf may stand for NaN alone, which comes after it: no bound
  uint64_t bound = (uint32_t)(lower >> 32) > ordered(-INFINITY) ? lower : 0ull;
#pragma unroll
  for (int d = 1; d < kGroupLanes; d <<= 1) {
    const uint64_t o = __shfl_xor_sync(0xffffffffu, bound, d);
    bound = o > bound ? o : bound;
  }
  if (lane % kGroupLanes == 0) sh.group[tid / kGroupLanes] = bound;
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
    sh.n_list = sh.n_open = 0;
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
    const bool again = upper >= tau && begin + lane < r.words;           // no bound: every thread's elements
    const unsigned who = __ballot_sync(0xffffffffu, again);
    int at = 0;
    if (lane == 0 && who) at = atomicAdd(&sh.n_open, __popc(who));       // in any order, like the list:
    at = __shfl_sync(0xffffffffu, at, 0);                                // its keys are ranked in the end
    if (again) sh.open[at + __popc(who & ((1u << lane) - 1))] = (unsigned char)tid;
    __syncthreads();
    const int per = ((r.words - cta * kWarps * kChunk + stride - 1) / stride) * kUnroll;   // words of a thread
    const long work = (long)sh.n_open * per;
    const bool few = tau && work <= 1 << 16;                             // exact in the division below
    if (few) {
      const float inv = 1.0f / (float)per;
      constexpr int kAhead = 4;
      for (int f = tid; f < (int)work; f += kAhead * kThreads) {
        uint4 u[kAhead];
        int w[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          const int g = min(f + j * kThreads, (int)work - 1), q = (int)(((float)g + 0.5f) * inv), c = g - q * per;
          const int o = sh.open[q];
          w[j] = (cta * kWarps + (o >> 5)) * kChunk + (o & 31) + (c / kUnroll) * stride + 32 * (c % kUnroll);
          if (f + j * kThreads >= (int)work) w[j] = r.words;
          u[j] = r.load(w[j]);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          if (Vec<X>::most(u[j]) < tau_value) continue;                  // NaN: goes on
          float x[n];
          Vec<X>::get(u[j], x);
#pragma unroll
          for (int i = 0; i < n; ++i)
            if (x[i] >= tau_value && w[j] < r.words) {                   // finite: not what stands for outside the row
              const uint64_t key = key_of(x[i], r.first(w[j]) + i);
              if (key >= tau) {
                const int to = atomicAdd(&sh.n_list, 1);
                if (to < kList) sh.list[to] = key;
              }
            }
        }
      }
      __syncthreads();
    }
    if (!few || sh.n_list > kList) {
      __syncthreads();
      if (tid == 0) sh.n_list = 0;
      __syncthreads();
      uint64_t mine = 0;                               // the warp's best so far, lane i the i-th
      for (unsigned open = who; open; open &= open - 1) {   // a thread's words, a chunk per four lanes
        const int first = begin + __ffs(open) - 1;
        for (int base = 0; first + base * stride < r.words; base += 32 / kUnroll) {
          const int w = first + (base + lane / kUnroll) * stride + 32 * (lane % kUnroll);
          const uint4 u = r.load(w);
          if (tau && !__any_sync(0xffffffffu, !(Vec<X>::most(u) < tau_value))) continue;
          float x[n];
          Vec<X>::get(u, x);
#pragma unroll 1
          for (int i = 0; i < n; ++i) {
            const int e = r.first(w) + i;
            float v = x[0];
#pragma unroll
            for (int q = 1; q < n; ++q) v = i == q ? x[q] : v;
            const uint64_t key = w < r.words && e >= 0 && e < V ? key_of(v, e) : 0ull;
            const uint64_t floor = __shfl_sync(0xffffffffu, mine, k - 1);
            unsigned in = __ballot_sync(0xffffffffu, key >= tau && key > floor);
            for (; in; in &= in - 1) insert(mine, __shfl_sync(0xffffffffu, key, __ffs(in) - 1), lane);
          }
        }
      }
      const unsigned have = __ballot_sync(0xffffffffu, lane < k && mine);
      if (lane == 0 && have) at = atomicAdd(&sh.n_list, __popc(have));
      at = __shfl_sync(0xffffffffu, at, 0);
      if (have >> lane & 1) sh.list[at + lane] = mine;
      __syncthreads();
    }
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
    const float quiet = __int_as_float(0x7fc00000), logS = log2f(S);
    if (lane == 0) {
      if (logprob) logprob[row] = none || !has_t ? quiet : xt - m - kLn2 * logS;
      if (rank_out) rank_out[row] = has_t ? b + 1 : 0;
      if (entropy) entropy[row] = none ? quiet : kLn2 * (logS - c.A / S);
    }
    if (k > 0) {
      if (C > 1)
#pragma unroll
        for (int d = kMaxCluster / 2; d > 0; d >>= 1)
#pragma unroll
          for (int q = 0; q < d; ++q) list[q] = merge(list[q], list[q + d], lane);
      if (lane < k) {
        if (top_ids) top_ids[row * k + lane] = id_of(list[0]);
        if (top_lp) top_lp[row * k + lane] = none ? quiet : value_of(list[0]) - m - kLn2 * logS;
      }
    }
  }
  if (C > 1) cluster_sync();                           // shared memory stays until CTA 0 has read it
}

template <typename X>
int launch(const void* logits, long ld, const long long* tokens, int M, int V, int k, float* logprob, long long* rank,
           float* entropy, long long* top_ids, float* top_lp, cudaStream_t st) {
  constexpr int kRing = kWarps * kStages * kChunk * 16;
  static std::mutex mu;
  static bool attr_done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lk(mu);
    if (dev >= 64 || !attr_done[dev]) {
      const cudaError_t e =
          cudaFuncSetAttribute(logprobs_kernel<X>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing);
      if (e != cudaSuccess) {
        cudaGetLastError();
        return set_error(R4Q_ERR_CUDA, "logprobs_kernel: %s", cudaGetErrorString(e));
      }
      if (dev < 64) attr_done[dev] = true;
    }
  }
  // CTAs per row: as many as keep one chunk per warp and the grid within one wave
  int C = kMaxCluster;
  while (C > 1 && ((long)M * C > (long)kResident * num_sms() || (long)(C / 2) * kWarps * kChunk * Vec<X>::n >= V)) C >>= 1;
  for (int at = 0; at < M; at += 65535) {
    const int rows = M - at < 65535 ? M - at : 65535;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(C, rows);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kRing;
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
        top_ids ? top_ids + o * k : nullptr, top_lp ? top_lp + o * k : nullptr, wait_polls());
    if (e != cudaSuccess) {
      cudaGetLastError();
      return set_error(R4Q_ERR_CUDA, "logprobs_kernel (cluster %d): %s", C, cudaGetErrorString(e));
    }
  }
  return R4Q_OK;
}

}  // namespace

cudaError_t logprob_status_word(int** word) { return cudaGetSymbolAddress((void**)word, g_logprob_status); }

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
