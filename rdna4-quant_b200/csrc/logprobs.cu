// Likelihoods of given tokens: log softmax at the token, its rank, the entropy
// of the row and its k most likely ids.
//
// lse = m + log S with S = sum e^(x - m); entropy = log S - sum e^(x - m) (x - m) / S.
// The order of ids is by (value, lowest id first), as one 64-bit key.
#include <cuda_bf16.h>

#include "r4q_common.cuh"

namespace r4q {
namespace {

constexpr int kThreads = 512;
constexpr int kMaxTop = 32;

__device__ __forceinline__ float load_f(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float load_f(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_f(const float* p) { return *p; }

// order of floats as unsigned integers; NaN is the lowest, -0 equals +0
__device__ __forceinline__ uint32_t ordered(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ unsigned long long key_of(float x, int i) {
  return ((unsigned long long)ordered(x) << 32) | (0xffffffffu - (uint32_t)i);
}
__device__ __forceinline__ float value_of(unsigned long long key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return o == 0u ? __int_as_float(0x7fc00000) : __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}

template <typename F, typename T>
__device__ __forceinline__ T block_reduce(T v, T* buf, F f) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, s));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  T r = buf[0];
  for (int w = 1; w < kThreads / 32; ++w) r = f(r, buf[w]);
  return r;
}

template <typename X>
__global__ void __launch_bounds__(kThreads)
    logprobs_kernel(const X* __restrict__ logits, long ld, const long long* __restrict__ tokens, int V, int k,
                    float* logprob, long long* rank, float* entropy, long long* top_ids, float* top_lp) {
  __shared__ unsigned long long kbuf[kThreads / 32];
  __shared__ float fbuf[kThreads / 32];
  __shared__ int ibuf[kThreads / 32];
  const long row = blockIdx.x;
  const X* x = logits + row * ld;
  const long long t = tokens ? tokens[row] : -1;
  const bool has_t = t >= 0 && t < V;
  const unsigned long long tkey = has_t ? key_of(load_f(x + t), (int)t) : ~0ull;
  float m = -INFINITY;
  int before = 0, nan = 0;
  for (int i = threadIdx.x; i < V; i += kThreads) {
    const float v = load_f(x + i);
    m = fmaxf(m, v);
    nan |= v != v;
    before += key_of(v, i) > tkey;
  }
  m = block_reduce(m, fbuf, [](float a, float b) { return fmaxf(a, b); });
  nan = block_reduce(nan, ibuf, [](int a, int b) { return a | b; });
  before = block_reduce(before, ibuf, [](int a, int b) { return a + b; });
  float S = 0.f, A = 0.f;
  for (int i = threadIdx.x; i < V; i += kThreads) {
    const float d = fmaxf(load_f(x + i) - m, -1e4f), e = expf(d);
    S += e;
    A += e * d;
  }
  S = block_reduce(S, fbuf, [](float a, float b) { return a + b; });
  A = block_reduce(A, fbuf, [](float a, float b) { return a + b; });
  const bool bad = nan || isinf(m);
  const float none = __int_as_float(0x7fc00000);
  const float logS = logf(S);
  if (threadIdx.x == 0) {
    if (logprob) logprob[row] = bad || !has_t ? none : load_f(x + t) - m - logS;
    if (rank) rank[row] = has_t ? before + 1 : 0;
    if (entropy) entropy[row] = bad ? none : logS - A / S;
  }
  unsigned long long last = ~0ull;
  for (int j = 0; j < k; ++j) {
    unsigned long long best = 0;
    for (int i = threadIdx.x; i < V; i += kThreads) {
      const unsigned long long key = key_of(load_f(x + i), i);
      if (key < last && key > best) best = key;
    }
    last = block_reduce(best, kbuf, [](unsigned long long a, unsigned long long b) { return a > b ? a : b; });
    if (threadIdx.x == 0) {
      if (top_ids) top_ids[row * k + j] = (long long)(0xffffffffu - (uint32_t)last);
      if (top_lp) top_lp[row * k + j] = bad ? none : value_of(last) - m - logS;
    }
  }
}

template <typename X>
void launch(const void* logits, long ld, const long long* tokens, int M, int V, int k, float* logprob, long long* rank,
            float* entropy, long long* top_ids, float* top_lp, cudaStream_t st) {
  logprobs_kernel<X><<<M, kThreads, 0, st>>>((const X*)logits, ld, tokens, V, k, logprob, rank, entropy, top_ids,
                                             top_lp);
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
  if (!logits || (M > 1 && ld < V)) return set_error(R4Q_ERR_ARG, "token_logprobs: null logits or row stride %ld < %d", ld, V);
  if (!tokens && (logprob || rank)) return set_error(R4Q_ERR_ARG, "token_logprobs: logprob and rank need tokens");
  if (!aligned(logits, type == R4Q_T_F32 ? 4 : 2)) return set_error(R4Q_ERR_ALIGN, "token_logprobs: logits misaligned");
  cudaStream_t st = (cudaStream_t)stream;
  if (type == R4Q_T_F16) launch<__half>(logits, ld, tokens, M, V, k, logprob, rank, entropy, top_ids, top_logprobs, st);
  else if (type == R4Q_T_BF16) launch<__nv_bfloat16>(logits, ld, tokens, M, V, k, logprob, rank, entropy, top_ids, top_logprobs, st);
  else launch<float>(logits, ld, tokens, M, V, k, logprob, rank, entropy, top_ids, top_logprobs, st);
  return check_launch("logprobs_kernel");
}
