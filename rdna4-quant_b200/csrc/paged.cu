// Paged FP8 KV cache: new tokens into pages (with the per-head RMSNorm + RoPE
// of q and k), page copies over all layers, block-table updates, and the
// status of the kernels that keep their status words in the library.
#include <algorithm>
#include <atomic>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <mutex>

#include "f32x2.cuh"
#include "paged.cuh"
#include "r4q_common.cuh"

namespace r4q {
namespace {

__device__ int g_write_status;

// ---------------------------------------------------------------- KV write
// A warp takes up to four heads of one kind (q, k or v) of one token, a half-warp
// per head: what differs between the kinds is uniform in the warp, the token's
// position, page and rotation row are looked up once, and eight loads a lane are
// in flight together.  Lane s of a half holds elements 2s, 2s + 1 of each
// 32-block: the RoPE partners i, i + 64 and the terms that head_kernel
// (r4q_head_norm_rope) adds in one lane are in one lane here too, and a butterfly
// over the half finishes the sum of squares in its order.  Norm and rotation equal
// that kernel's to the bit, and K is encoded from fp32 as by its KV write: below 248
// (and, without R4Q_KV_FULL_RANGE, from there on too) a decode step stores the bytes
// that it would.  A contiguous prefill rounds K to fp16 first, so that its codes may
// be a step away from these.  Bound: issue slots, so the arithmetic is two-wide fp32: 8192 tokens
// of 40/8 heads 60 us, 3.6 TB/s (72 us with scalar fp32 and comparisons per value;
// a warp per head, 4 bytes a lane, 92).
constexpr int kPairs = 2;
constexpr int kWriteThreads = 128;
constexpr int kHeads = 2 * kPairs;
struct WriteArgs {
  const __half *q, *k, *v;
  long ldq, ldk, ldv;
  const __half *qw, *kw, *cos_tab, *sin_tab;
  long tab_stride, tab_rows;
  __half *q_out, *k_out;
  long ldqo, ldko;
  PagedView c;
  const int* rows;
  const long long* pos;
  int M, H, groups, q_groups, k_groups;   // groups of kHeads heads per token: q's, then k's, then v's
  FastDiv by_groups, by_page;
  float eps;
  int flags;
};

// The codes of four values.  The cache codec (fp8_encode) keeps three mantissa
// bits, ties away from zero; below 2^-6 it keeps the sign alone, and from 256 on
// (with `full`: from 448 on) it stores 448, which it also stores for NaN.  Here the
// rounding is done on the float, so that the hardware's conversion in pairs is
// exact; 2^-6 is the smallest normal number at a scale of 2^-120, below which the
// fp32 pipe flushes to a signed zero; and the top binade is set to 448 on four
// bytes at once.  Five integer instructions a value: that pipe is what bounds a
// plain write (a dozen with comparisons and selections on each float).
__device__ __forceinline__ float rounded(float x) {
  const uint32_t u = __float_as_uint(fminf(x, 448.0f));                 // NaN: 448; the conversion bounds the other side
  float r = __uint_as_float((u + 0x80000u) & 0xfff00000u);
  asm("mul.rn.ftz.f32 %0, %0, 0f03800000;" : "+f"(r));                  // 2^-120
  return r * 0x1p120f;
}
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, bool full) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(rounded(b)), "f"(rounded(a)));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(rounded(d)), "f"(rounded(c)));
  uint32_t w = (uint32_t)lo | (uint32_t)hi << 16;
  if (!full) {
    const uint32_t top = ((w & 0x78787878u) + 0x08080808u) & 0x80808080u, one = top >> 7;   // exponent field 15
    w = (w | (top - one)) & ~one;
  }
  return w;
}

__device__ __forceinline__ F2 pair_of(uint32_t u) {
  const float2 f = __half22float2(u32_as_h2(u));
  return F2(f.x, f.y);
}

__global__ void __launch_bounds__(kWriteThreads) paged_write_kernel(const WriteArgs a) {
  const int lane = threadIdx.x & 31, sl = lane & 15, half = lane >> 4;
  const int w = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int m = a.by_groups.div(w);
  if (m >= a.M) return;
  pdl_wait_trigger();
  int g = w - m * a.groups;
  const bool is_q = g < a.q_groups, is_v = g >= a.q_groups + a.k_groups;
  g -= is_q ? 0 : is_v ? a.q_groups + a.k_groups : a.q_groups;
  const int h0 = g * kHeads, n = (is_q ? a.H : a.c.Hk) - h0;        // this warp: heads h0 .. of the kind, n left
  const long long pos = a.pos[m];
  const int row = a.rows ? a.rows[m] : m;
  const int at = (h0 + half) * kHeadDim + 2 * sl;                   // this lane's first element in the token's row
  const uint32_t* src = reinterpret_cast<const uint32_t*>(
      (is_q ? a.q + m * a.ldq : is_v ? a.v + m * a.ldv : a.k + m * a.ldk) + at);
  uint32_t x32[kPairs][4];                           // before the position's lookups: independent of them
#pragma unroll
  for (int i = 0; i < kPairs; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) x32[i][j] = 2 * i + half < n ? src[i * kHeadDim + 16 * j] : 0u;
  if (pos < 0) return;
  const bool norm = (a.flags & R4Q_HEAD_NORM) && !is_v, rope = (a.flags & R4Q_HEAD_ROPE) && !is_v;
  const bool full = a.flags & R4Q_KV_FULL_RANGE;
  bool ok = row >= 0 && row < a.c.seqs && pos < (long long)a.c.max_blocks * a.c.page;
  if (ok && (a.flags & R4Q_HEAD_ROPE)) ok = pos < a.tab_rows;   // of a token, all heads or none
  int pg = 0, in_page = 0;
  uint32_t c32[2] = {0u, 0u}, s32[2] = {0u, 0u};
  if (ok) {
    const int blk = a.by_page.div((int)pos);
    in_page = (int)pos - blk * a.c.page;
    pg = a.c.table[row * a.c.ld_table + blk];
    if (rope)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        c32[j] = reinterpret_cast<const uint32_t*>(a.cos_tab + pos * a.tab_stride)[sl + 16 * j];
        s32[j] = reinterpret_cast<const uint32_t*>(a.sin_tab + pos * a.tab_stride)[sl + 16 * j];
      }
    ok = pg >= 0 && pg < a.c.n_pages;
  }
  if (!ok) {
    if (lane == 0) atomicOr(&g_write_status, kPagedBadPage);
    return;
  }
  uint32_t w32[4];
  if (norm)
#pragma unroll
    for (int j = 0; j < 4; ++j) w32[j] = reinterpret_cast<const uint32_t*>(is_q ? a.qw : a.kw)[sl + 16 * j];
  __half* out = is_q ? a.q_out + m * a.ldqo : !is_v && a.k_out ? a.k_out + m * a.ldko : nullptr;
  uint32_t* o32 = reinterpret_cast<uint32_t*>(out + at);
  const long head_bytes = (long)a.c.page * kHeadDim;
  uint8_t* page = (is_v ? a.c.v + pg * a.c.v_stride : a.c.k + pg * a.c.k_stride) + (h0 + half) * head_bytes +
                  in_page * kHeadDim;
  const float* scale = is_v ? a.c.v_scale : a.c.k_scale;
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    if (2 * i >= n) break;                           // uniform
    const bool in = 2 * i + half < n;
    F2 v[4] = {pair_of(x32[i][0]), pair_of(x32[i][1]), pair_of(x32[i][2]), pair_of(x32[i][3])};
    if (norm) {
      F2 ss(0.f, 0.f);
#pragma unroll
      for (int j = 0; j < 4; ++j) ss = fma(v[j], v[j], ss);
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) {
        const float2 f = ss.get();
        ss = add(ss, F2(__shfl_xor_sync(0xffffffffu, f.x, d), __shfl_xor_sync(0xffffffffu, f.y, d)));
      }
      const float2 f = ss.get();
      const float rrms = rsqrtf((f.x + f.y) / (float)kHeadDim + a.eps);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = mul(mul(v[j], F2(rrms, rrms)), pair_of(w32[j]));
    }
    if (rope)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const F2 e = v[j], o = v[j + 2], c = pair_of(c32[j]);
        const F2 s = pair_of(s32[j]), minus_s = pair_of(s32[j] ^ 0x80008000u);
        v[j] = fma(e, c, mul(o, minus_s));
        v[j + 2] = fma(o, c, mul(e, s));
      }
    float2 f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = v[j].get();
    if (out && in)
#pragma unroll
      for (int j = 0; j < 4; ++j) o32[i * kHeadDim + 16 * j] = h2_as_u32(__floats2half2_rn(f[j].x, f[j].y));
    if (is_q) continue;
    // a lane has the codes of elements 2s, 2s + 1 of four 32-blocks: even lanes
    // store four bytes of blocks 0 and 1 with their neighbour's, odd lanes of 2 and 3
    if (scale) {
      const float s = scale[min(h0 + 2 * i + half, a.c.Hk - 1)];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f[j].x = f[j].x / s;
        f[j].y = f[j].y / s;
      }
    }
    const uint32_t e01 = encode4(f[0].x, f[0].y, f[1].x, f[1].y, full);
    const uint32_t e23 = encode4(f[2].x, f[2].y, f[3].x, f[3].y, full);
    const bool even = !(lane & 1);
    const uint32_t own = even ? e01 : e23, got = __shfl_xor_sync(0xffffffffu, even ? e23 : e01, 1);
    if (in) {
      uint32_t* d32 = reinterpret_cast<uint32_t*>(page + 2 * i * head_bytes) + (even ? 0 : 16) + (sl >> 1);
      const uint32_t lo = even ? own : got, hi = even ? got : own;      // of lanes 2n, 2n + 1
      d32[0] = prmt(lo, hi, 0x5410u);
      d32[8] = prmt(lo, hi, 0x7632u);
    }
  }
}

// ------------------------------------------------------------- page copies
// Bound: HBM, every byte read and written once.  A CTA copies 16 KB of a page,
// four 16-byte loads a thread in flight: a fork's few pages over all layers
// (tens of MB) then still fill the SMs.  The moves travel in the launch's
// parameters: no copy to the device, and nothing to keep alive behind the call.
constexpr int kMaxMoves = 448;          // (src, dst) pairs in one launch's parameters (3.5 KB)
constexpr int kCopyVecs = 4, kCopyChunk = 256 * kCopyVecs;   // 16-byte words of a CTA
struct Moves {
  int src[kMaxMoves], dst[kMaxMoves];
};

__global__ void __launch_bounds__(256)
    copy_pages_kernel(uint8_t* pool, long outer_stride, long page_stride, long words,
                      const __grid_constant__ Moves mv) {
  pdl_wait_trigger();
  uint8_t* base = pool + (long)blockIdx.z * outer_stride;
  const uint4* s = reinterpret_cast<const uint4*>(base + (long)mv.src[blockIdx.y] * page_stride);
  uint4* d = reinterpret_cast<uint4*>(base + (long)mv.dst[blockIdx.y] * page_stride);
  const long at = (long)blockIdx.x * kCopyChunk + threadIdx.x;
  uint4 v[kCopyVecs];
#pragma unroll
  for (int j = 0; j < kCopyVecs; ++j)
    if (at + 256 * j < words) v[j] = s[at + 256 * j];
#pragma unroll
  for (int j = 0; j < kCopyVecs; ++j)
    if (at + 256 * j < words) d[at + 256 * j] = v[j];
}

constexpr int kMaxCells = 320;
struct Cells {
  int r[kMaxCells], c[kMaxCells], v[kMaxCells];
};
__global__ void table_set_kernel(int* table, long ld, int n, const __grid_constant__ Cells cells) {
  pdl_wait_trigger();
  for (int i = threadIdx.x; i < n; i += blockDim.x) table[cells.r[i] * ld + cells.c[i]] = cells.v[i];
}

}  // namespace

static std::atomic<int> g_wait_polls{kWaitPolls};
int wait_polls() { return g_wait_polls.load(std::memory_order_relaxed); }

// The status words as they are, cleared in the same step: what a kernel that another
// thread launches meanwhile sets is either taken here or left for the next call.
static __device__ int g_taken[3];
static __global__ void take_status_kernel(int* write, int* attn, int* likelihood, int clear) {
  int* const word[3] = {write, attn, likelihood};
  for (int i = 0; i < 3; ++i) g_taken[i] = clear ? atomicExch(word[i], 0) : atomicOr(word[i], 0);
}

// What the status words say.  A wait that gave up voids a whole call's outputs, a bad
// page those of its row: the first gives the code, and the message names both.
static int status_of(int write, int attn, int likelihood) {
  const bool aw = attn & kPagedTimeout, lw = likelihood & kPagedTimeout;
  const bool wp = write & kPagedBadPage, ap = attn & kPagedBadPage;
  char wait[160] = "", page[160] = "";
  if (aw || lw)
    snprintf(wait, sizeof(wait), "a bounded wait of %s%s%s gave up since the last check: those outputs are not valid",
             aw ? "the paged attention" : "", aw && lw ? " and " : "", lw ? "the likelihood kernel" : "");
  if (wp || ap)
    snprintf(page, sizeof(page), "%s%s%s met a row, position, length or page id outside the cache since the last check",
             wp ? "a paged write" : "", wp && ap ? " and " : "", ap ? "a paged attention" : "");
  if (!*wait && !*page) return R4Q_OK;
  return set_error(*wait ? R4Q_ERR_TIMEOUT : R4Q_ERR_PAGE, "%s%s%s", wait, *wait && *page ? "; " : "", page);
}

int paged_view(const char* what, const r4q_paged_cache* c, PagedView* out) {
  if (!c || !c->k_pages || !c->v_pages || !c->table) return set_error(R4Q_ERR_ARG, "%s: null cache pointer", what);
  if (c->page < 16 || c->page % 16 || c->page > 4096)
    return set_error(R4Q_ERR_ARG, "%s: page of %d positions (a multiple of 16, at most 4096)", what, c->page);
  if (c->n_pages < 1 || c->Hk < 1 || c->Hk > 65535 || c->seqs < 1 || c->max_blocks < 1 || c->ld_table < c->max_blocks)
    return set_error(R4Q_ERR_ARG, "%s: bad cache (pages %d, kv heads %d, table %d x %d)", what, c->n_pages, c->Hk,
                     c->seqs, c->max_blocks);
  if ((long)c->Hk * c->page > (1L << 24) || (long)c->max_blocks * c->page > (1L << 30))
    return set_error(R4Q_ERR_ARG, "%s: Hk * page above 2^24 or max_blocks * page above 2^30", what);
  const long bytes = (long)c->Hk * c->page * kHeadDim;
  const long ks = c->k_stride ? c->k_stride : bytes, vs = c->v_stride ? c->v_stride : bytes;
  if (ks < bytes || vs < bytes) return set_error(R4Q_ERR_ARG, "%s: page strides below a page's %ld bytes", what, bytes);
  if (!aligned(c->k_pages, 16) || !aligned(c->v_pages, 16) || ks % 16 || vs % 16)
    return set_error(R4Q_ERR_ALIGN, "%s: pages must be 16-byte aligned", what);
  *out = PagedView{(uint8_t*)c->k_pages, (uint8_t*)c->v_pages, ks, vs, c->n_pages, c->page, c->Hk, c->table,
                   c->ld_table, c->seqs, c->max_blocks, c->k_scale, c->v_scale};
  return R4Q_OK;
}

}  // namespace r4q

using namespace r4q;

extern "C" int r4q_paged_kv_write(const void* q, long ldq, const void* k, long ldk, const void* v, long ldv,
                                  const void* q_norm_w, const void* k_norm_w, const void* cos_tab,
                                  const void* sin_tab, long tab_stride, long tab_rows, void* q_out, long ldqo,
                                  void* k_out, long ldko, const r4q_paged_cache* cache, const int* rows,
                                  const long long* pos, int M, int H, float eps, int flags, void* stream) {
  WriteArgs a{};
  int st = paged_view("paged_kv_write", cache, &a.c);
  if (st) return st;
  const bool has_q = q && H > 0;
  if (M < 0 || H < 0) return set_error(R4Q_ERR_ARG, "paged_kv_write: bad shape M=%d H=%d", M, H);
  if (M == 0) return R4Q_OK;
  if (!k || !v || !pos) return set_error(R4Q_ERR_ARG, "paged_kv_write: null k, v or pos");
  if (has_q && !q_out) return set_error(R4Q_ERR_ARG, "paged_kv_write: q without q_out");
  if (!rows && M > a.c.seqs)
    return set_error(R4Q_ERR_ARG, "paged_kv_write: %d tokens for %d sequences need rows", M, a.c.seqs);
  if (flags & ~(R4Q_HEAD_NORM | R4Q_HEAD_ROPE | R4Q_KV_FULL_RANGE))
    return set_error(R4Q_ERR_ARG, "paged_kv_write: unknown flags %d", flags);
  if ((flags & R4Q_HEAD_NORM) && ((has_q && !q_norm_w) || !k_norm_w))
    return set_error(R4Q_ERR_ARG, "paged_kv_write: norm weights required");
  if ((flags & R4Q_HEAD_ROPE) && (!cos_tab || !sin_tab || tab_rows < 1 || tab_stride < kHeadDim / 2))
    return set_error(R4Q_ERR_ARG, "paged_kv_write: rope tables required (rows %ld, stride %ld)", tab_rows, tab_stride);
  const long kd = (long)a.c.Hk * kHeadDim, qd = (long)H * kHeadDim;
  if (M > 1 && (ldk < kd || ldv < kd || (k_out && ldko < kd) || (has_q && (ldq < qd || ldqo < qd))))
    return set_error(R4Q_ERR_ARG, "paged_kv_write: row strides below the heads of a token");
  const bool rope = flags & R4Q_HEAD_ROPE, norm = flags & R4Q_HEAD_NORM;
  if (!aligned(k, 16) || !aligned(v, 16) || ldk % 8 || ldv % 8 || (k_out && (!aligned(k_out, 16) || ldko % 8)) ||
      (has_q && (!aligned(q, 16) || !aligned(q_out, 16) || ldq % 8 || ldqo % 8)) ||
      (rope && (!aligned(cos_tab, 16) || !aligned(sin_tab, 16) || tab_stride % 8)) ||
      (norm && (!aligned(k_norm_w, 16) || (has_q && !aligned(q_norm_w, 16)))))
    return set_error(R4Q_ERR_ALIGN, "paged_kv_write: 16-byte aligned pointers and strides in multiples of 8 needed");
  a.q = (const __half*)q; a.k = (const __half*)k; a.v = (const __half*)v;
  a.ldq = ldq; a.ldk = ldk; a.ldv = ldv;
  a.qw = (const __half*)q_norm_w; a.kw = (const __half*)k_norm_w;
  a.cos_tab = (const __half*)cos_tab; a.sin_tab = (const __half*)sin_tab;
  a.tab_stride = tab_stride; a.tab_rows = tab_rows;
  a.q_out = (__half*)q_out; a.k_out = (__half*)k_out; a.ldqo = ldqo; a.ldko = ldko;
  a.rows = rows; a.pos = pos;
  a.M = M; a.H = has_q ? H : 0; a.eps = eps; a.flags = flags;
  a.q_groups = (a.H + kHeads - 1) / kHeads;
  a.k_groups = (a.c.Hk + kHeads - 1) / kHeads;
  a.groups = a.q_groups + 2 * a.k_groups;
  a.by_groups = fast_div(a.groups);
  a.by_page = fast_div(a.c.page);
  const long warps = (long)M * a.groups;
  if (warps > 0x7ffffff0L) return set_error(R4Q_ERR_ARG, "paged_kv_write: %d tokens of %d heads are too many", M, H);
  const cudaError_t e =
      launch_pdl(paged_write_kernel, dim3((unsigned)((warps * 32 + kWriteThreads - 1) / kWriteThreads)),
                 dim3(kWriteThreads), 0, (cudaStream_t)stream, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(R4Q_ERR_CUDA, "paged_write_kernel: %s", cudaGetErrorString(e));
  }
  return R4Q_OK;
}

extern "C" int r4q_kv_copy_pages(void* pool, long outer, long outer_stride, long page_stride, long page_bytes,
                                 int n_pages, const int* src, const int* dst, int n, void* stream) {
  if (n < 0 || outer < 0 || (n && (!pool || !src || !dst)) || n_pages < 1 || page_bytes < 16)
    return set_error(R4Q_ERR_ARG, "kv_copy_pages: bad arguments (n %d, pools %ld, pages %d)", n, outer, n_pages);
  if (page_stride < page_bytes || (outer > 1 && outer_stride < page_bytes))
    return set_error(R4Q_ERR_ARG, "kv_copy_pages: strides below a page's %ld bytes", page_bytes);
  if (!aligned(pool, 16) || page_bytes % 16 || page_stride % 16 || outer_stride % 16)
    return set_error(R4Q_ERR_ALIGN, "kv_copy_pages: pool, page size and strides must be multiples of 16 bytes");
  const long chunks = (page_bytes / 16 + kCopyChunk - 1) / kCopyChunk;
  if (outer > 65535 || chunks > 0x7fffffffL)
    return set_error(R4Q_ERR_ARG, "kv_copy_pages: %ld pools (at most 65535) of %ld-byte pages", outer, page_bytes);
  if (n == 0 || outer == 0) return R4Q_OK;
  for (int i = 0; i < n; ++i)
    if (src[i] < 0 || src[i] >= n_pages || dst[i] < 0 || dst[i] >= n_pages)
      return set_error(R4Q_ERR_ARG, "kv_copy_pages: move %d (%d -> %d) outside the pool of %d pages", i, src[i],
                       dst[i], n_pages);
  uint8_t* seen = (uint8_t*)calloc(n_pages, 1);      // per page, 1: read, 2: written
  if (!seen) return set_error(R4Q_ERR_CAPACITY, "kv_copy_pages: no host memory for %d pages", n_pages);
  int twice = -1, both = -1;
  for (int i = 0; i < n; ++i) {
    if (seen[dst[i]] & 2) twice = dst[i];
    seen[src[i]] |= 1;
    seen[dst[i]] |= 2;
  }
  for (int i = 0; i < n; ++i)
    if (seen[src[i]] == 3) both = src[i];
  free(seen);
  if (twice >= 0) return set_error(R4Q_ERR_ARG, "kv_copy_pages: page %d is written twice", twice);
  if (both >= 0) return set_error(R4Q_ERR_ARG, "kv_copy_pages: page %d is both read and written", both);
  for (int at = 0; at < n; at += kMaxMoves) {
    const int part = n - at < kMaxMoves ? n - at : kMaxMoves;
    Moves mv;
    memcpy(mv.src, src + at, part * sizeof(int));
    memcpy(mv.dst, dst + at, part * sizeof(int));
    const cudaError_t e =
        launch_pdl(copy_pages_kernel, dim3((unsigned)chunks, part, (unsigned)outer), dim3(256), 0,
                   (cudaStream_t)stream, (uint8_t*)pool, outer_stride, page_stride, page_bytes / 16, mv);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return set_error(R4Q_ERR_CUDA, "copy_pages_kernel: %s", cudaGetErrorString(e));
    }
  }
  return R4Q_OK;
}

extern "C" int r4q_kv_table_set(int* table, long ld, int rows, int cols, const int* r, const int* c, const int* v,
                                int n, void* stream) {
  if (n < 0 || rows < 0 || cols < 0 || ld < cols || (n && (!table || !r || !c || !v)))
    return set_error(R4Q_ERR_ARG, "kv_table_set: bad arguments (n %d, table %d x %d)", n, rows, cols);
  for (int i = 0; i < n; ++i)
    if (r[i] < 0 || r[i] >= rows || c[i] < 0 || c[i] >= cols)
      return set_error(R4Q_ERR_ARG, "kv_table_set: cell %d (%d, %d) outside the table of %d x %d", i, r[i], c[i], rows,
                       cols);
  if (n > 1) {                                       // threads write in any order: a cell twice has no one value
    long* cell = (long*)malloc(n * sizeof(long));
    if (!cell) return set_error(R4Q_ERR_CAPACITY, "kv_table_set: no host memory for %d cells", n);
    for (int i = 0; i < n; ++i) cell[i] = (long)r[i] * cols + c[i];
    std::sort(cell, cell + n);
    const long* twice = std::adjacent_find(cell, cell + n);
    const long bad = twice == cell + n ? -1 : *twice;
    free(cell);
    if (bad >= 0)
      return set_error(R4Q_ERR_ARG, "kv_table_set: cell (%ld, %ld) is written twice", bad / cols, bad % cols);
  }
  for (int at = 0; at < n; at += kMaxCells) {
    const int part = n - at < kMaxCells ? n - at : kMaxCells;
    Cells cells;
    memcpy(cells.r, r + at, part * sizeof(int));
    memcpy(cells.c, c + at, part * sizeof(int));
    memcpy(cells.v, v + at, part * sizeof(int));
    const cudaError_t e = launch_pdl(table_set_kernel, dim3(1), dim3(256), 0, (cudaStream_t)stream, table, ld, part, cells);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return set_error(R4Q_ERR_CUDA, "table_set_kernel: %s", cudaGetErrorString(e));
    }
  }
  return R4Q_OK;
}

extern "C" int r4q_kernel_status(int clear) {
  static std::mutex mu;                              // g_taken is one per device
  std::lock_guard<std::mutex> lk(mu);
  int *write = nullptr, *attn = nullptr, *likelihood = nullptr, word[3] = {0, 0, 0};
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaGetSymbolAddress((void**)&write, g_write_status);
  if (e == cudaSuccess) e = paged_attn_status_word(&attn);
  if (e == cudaSuccess) e = logprob_status_word(&likelihood);
  if (e == cudaSuccess) {
    take_status_kernel<<<1, 1>>>(write, attn, likelihood, clear);
    e = cudaGetLastError();
  }
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(word, g_taken, sizeof(word));
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(R4Q_ERR_CUDA, "kernel_status: %s", cudaGetErrorString(e));
  }
  return status_of(word[0], word[1], word[2]);
}

extern "C" long r4q_debug_wait_limit(long polls) {
  return g_wait_polls.exchange(polls < 0 || polls > kWaitPolls ? kWaitPolls : (int)polls);
}

extern "C" int r4q_debug_status_of(int write, int attention, int likelihoods) {
  return status_of(write, attention, likelihoods);
}
