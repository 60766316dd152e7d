// Attention of one new token over the paged FP8 KV cache.
//
// o = sum_j p_j V_j / sum_j p_j with p_j = exp2(s_j - m), s_j the score in the
// log2 domain and m the running maximum: one pass over K and V.
//
// One CTA per (sequence, query head), positions strided over its 8 warps, a
// lane holds 4 of the 128 elements; the warps join through shared memory.
#include "paged.cuh"
#include "r4q_common.cuh"

namespace r4q {
namespace {

__device__ int g_attn_status;
constexpr int kWarps = 8;

__global__ void __launch_bounds__(kWarps * 32)
    paged_attn_kernel(const __half* q, long ldq, const PagedView c, const long long* seq_lens, __half* o, long ldo,
                      int Hg, int fwht) {
  __shared__ float part[kWarps][130];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.x, b = blockIdx.y, kh = h / Hg;
  const long long cap = (long long)c.max_blocks * c.page;
  long long seq = seq_lens[b];
  if (seq > cap || seq < 0) {
    if (threadIdx.x == 0) atomicOr(&g_attn_status, kPagedBadPage);
    seq = seq < 0 ? 0 : cap;
  }
  float qv[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, m = -1e30f, l = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) qv[i] = seq ? __half2float(q[(long)b * ldq + (long)h * kHeadDim + 4 * lane + i]) : 0.f;
  const float scale = (c.k_scale ? c.k_scale[kh] : 1.f) * rsqrtf((float)kHeadDim) * 1.4426950408889634f;
  for (int p = warp; p < (int)seq; p += kWarps) {
    const int pg = c.table[(long)b * c.ld_table + p / c.page];
    const bool ok = pg >= 0 && pg < c.n_pages;
    if (!ok && lane == 0) atomicOr(&g_attn_status, kPagedBadPage);
    const long off = ((long)kh * c.page + p % c.page) * kHeadDim + 4 * lane;
    const uint32_t kw = ok ? *reinterpret_cast<const uint32_t*>(c.k + pg * c.k_stride + off) : 0u;
    const uint32_t vw = ok ? *reinterpret_cast<const uint32_t*>(c.v + pg * c.v_stride + off) : 0u;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) s += qv[i] * fp8_decode((kw >> (8 * i)) & 0xff);
    s = warp_sum(s) * scale;
    const float mn = fmaxf(m, s), f = exp2f(m - mn), e = exp2f(s - mn);
    m = mn;
    l = l * f + e;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = acc[i] * f + e * fp8_decode((vw >> (8 * i)) & 0xff);
  }
  if (lane == 0) part[warp][128] = m, part[warp][129] = l;
#pragma unroll
  for (int i = 0; i < 4; ++i) part[warp][4 * lane + i] = acc[i];
  __syncthreads();
  if (threadIdx.x >= kHeadDim) return;
  float M = -1e30f, L = 0.f, O = 0.f;
  for (int w = 0; w < kWarps; ++w) M = fmaxf(M, part[w][128]);
  for (int w = 0; w < kWarps; ++w) {
    const float f = exp2f(part[w][128] - M);
    L += part[w][129] * f;
    O += part[w][threadIdx.x] * f;
  }
  float r = L > 0.f ? O * ((c.v_scale ? c.v_scale[kh] : 1.f) / L) : 0.f;
  if (fwht) r = fwht32_lane(r, lane);
  o[(long)b * ldo + (long)h * kHeadDim + threadIdx.x] = __float2half(r);
}

}  // namespace

cudaError_t paged_attn_status(int clear, int* word) {
  const int zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(word, g_attn_status, sizeof(int));
  if (e == cudaSuccess && *word && clear) e = cudaMemcpyToSymbol(g_attn_status, &zero, sizeof(int));
  return e;
}

}  // namespace r4q

using namespace r4q;

extern "C" size_t r4q_paged_flash_decode_workspace_bytes(int B, int H, int Hk, int page, int max_blocks) {
  (void)B; (void)H; (void)Hk; (void)page; (void)max_blocks;
  return 0;
}

extern "C" int r4q_paged_flash_decode(const void* q, long ldq, const r4q_paged_cache* cache,
                                      const long long* seq_lens, void* o, long ldo, int B, int H, int flags,
                                      void* workspace, size_t ws_bytes, void* stream) {
  PagedView c;
  int st = paged_view("paged_flash_decode", cache, &c);
  if (st) return st;
  if (B < 0 || B > 4096 || B > c.seqs)
    return set_error(R4Q_ERR_ARG, "paged_flash_decode: batch %d (at most 4096 and the table's %d rows)", B, c.seqs);
  if (H < c.Hk || H % c.Hk || H > 65535) return set_error(R4Q_ERR_ARG, "paged_flash_decode: bad heads H=%d Hk=%d", H, c.Hk);
  if (flags & ~R4Q_ATTN_FWHT) return set_error(R4Q_ERR_ARG, "paged_flash_decode: unknown flags %d", flags);
  if (B == 0) return R4Q_OK;
  if (!q || !o || !seq_lens) return set_error(R4Q_ERR_ARG, "paged_flash_decode: null pointer");
  if (B > 1 && (ldq < (long)H * kHeadDim || ldo < (long)H * kHeadDim))
    return set_error(R4Q_ERR_ARG, "paged_flash_decode: row strides below H * 128");
  if (!aligned(q, 16) || (B > 1 && ldq % 8) || !aligned(o, 16) || (B > 1 && ldo % 8))
    return set_error(R4Q_ERR_ALIGN, "paged_flash_decode: q and o must be 16-byte aligned, strides multiples of 8");
  const size_t need = r4q_paged_flash_decode_workspace_bytes(B, H, c.Hk, c.page, c.max_blocks);
  if (need && (!workspace || ws_bytes < need))
    return set_error(R4Q_ERR_CAPACITY, "paged_flash_decode: workspace %zu < %zu bytes", ws_bytes, need);
  paged_attn_kernel<<<dim3(H, B), kWarps * 32, 0, (cudaStream_t)stream>>>(
      (const __half*)q, ldq, c, seq_lens, (__half*)o, ldo, H / c.Hk, flags & R4Q_ATTN_FWHT);
  return check_launch("paged_attn_kernel");
}
