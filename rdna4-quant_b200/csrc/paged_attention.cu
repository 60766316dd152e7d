// Attention of one new token per sequence over the paged FP8 KV cache, split
// over the cache's length and joined.
//
//   o = sum_j p_j V_j / sum_j p_j,   p_j = 2^(s_j - m),   s_j = q.K_j ks log2(e) / sqrt(128)
//
// in one pass over K and V with the running maximum m; parts of a sequence join
// as (m, l, O): M = max m, weights 2^(m - M), any m that l and O were taken from.
//
// Bound: HBM, 256 bytes per position and kv head; the arithmetic (tensor cores
// through m16n8k16, FP8 -> f16 by the hardware pair conversion) has to hide
// under it.
//
// Split.  The work is one list of 32-position tiles, ordered by (sequence, kv
// head, group of 8 query heads, tile); its length comes from the lengths on the
// device.  Every CTA takes an equal run of it and every warp of the CTA an equal
// run of that, whatever the lengths are: a batch of one long and many short
// sequences loads the SMs as evenly as an even one.  A (sequence, head) that lies
// inside one warp's run is finished by that warp; parts join in shared memory
// within a CTA, and through the workspace across CTAs, in a second small
// kernel (programmatic dependent launch) that reads them in list order: no
// atomics and no state between calls, so results repeat bit for bit and nothing
// is shared by calls that run at once.
//
// Per warp.  A ring of K/V tiles filled by TMA (128-byte swizzle, one box per
// tile, or two of 16 positions when the page is no multiple of 32); lane 0
// issues, the coordinates of the next 32 tiles are worked out by the 32 lanes
// together, so that the block-table reads do not wait for one another.  Pages
// that do not exist are loaded from behind the pool, i.e. as zeros.
//
// Precision.  q, K and V enter the products exactly (f16); a weight enters as
// two f16 numbers, its rounding and what that left, which takes no extra
// instruction: query heads fill 8 of the 16 rows of a product, the remainders the
// other 8.  Weights are carried times 2^15 (l too, so that it cancels): f16 then
// holds them to 2^-22 of themselves down to 2^-18 of the largest, and to 2^-40 of
// that below.  Scores, maxima, sums and O are fp32.  One rounding to f16 at the end.
#include <cuda.h>

#include <mutex>

#include "paged.cuh"
#include "r4q_common.cuh"
#include "tma_dev.cuh"

namespace r4q {
namespace {

__device__ int g_attn_status;

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kSlots = 2;
constexpr int kTile = 32;                         // positions per tile
constexpr int kTileBytes = kTile * kHeadDim;      // of K, and of V
constexpr int kGroup = 8;                         // query heads per pass over K and V
constexpr int kPitch = 132;                       // floats of a part's head: O[128], m, l, padding
constexpr int kPartFloats = kGroup * kPitch;
constexpr int kMaxBatch = 2048;
constexpr int kJoinWarps = 4;
constexpr float kWeightBits = 15.f;               // weights are carried times 2^15
constexpr float kLowest = -3e38f;                 // a maximum before the first score: no finite score is below it

struct AttnArgs {
  const __half* q;
  long ldq;
  PagedView c;
  const long long* seq_lens;
  __half* o;
  long ldo;
  int B, H, Hg, Hc, chunks, fwht;  // Hc: kv heads x groups of 8 query heads
  FastDiv by_page, by_Hc, by_chunks, by_ctas;
  int per_seg;       // a CTA per (sequence, head, group) instead of equal runs
  int two_boxes;     // 16-position boxes
  int polls;         // of the wait for a tile
  int* header;       // workspace: tiles per CTA, then the prefix sums of tiles [B + 1]
  float* parts;      // workspace: [CTA][2][kPartFloats]
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int row, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row),
      "r"(page), "r"(smem_u32(bar)) : "memory");
}

// H32 of the 32-element blocks of a head that a warp holds 4 per lane (4 lane ..).
__device__ __forceinline__ void fwht32_x4(float (&v)[4], int lane) {
  float a = v[0] + v[1], b = v[0] - v[1], c = v[2] + v[3], d = v[2] - v[3];
  v[0] = a + c; v[1] = b + d; v[2] = a - c; v[3] = b - d;
#pragma unroll
  for (int s = 1; s < 8; s <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float o = __shfl_xor_sync(0xffffffffu, v[i], s);
      v[i] = (lane & s) ? o - v[i] : v[i] + o;
    }
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] *= kInvSqrt32;
}

// The running join of parts of a head, O 4 elements per lane.
struct Joined {
  float M = kLowest, L = 0.f, O[4] = {0.f, 0.f, 0.f, 0.f};
  // parts i = first, first + step, .. < n at part(i), four at a time: their loads go out
  // together, and so do their weights, relative to the maximum of the four (eight at a
  // time is 1-3 % slower over the whole: this runs once, and its code has to be fetched)
  template <typename F>
  __device__ __forceinline__ void add_all(int first, int step, int n, int lane, F part) {
    constexpr int k = 4;
    for (int i = first; i < n; i += k * step) {
      float4 v[k];
      float m[k], l[k];
#pragma unroll
      for (int j = 0; j < k; ++j) {
        m[j] = kLowest;
        l[j] = 0.f;
        v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i + j * step < n) {
          const float* p = part(i + j * step);
          v[j] = *reinterpret_cast<const float4*>(p + 4 * lane);
          m[j] = p[kHeadDim];
          l[j] = p[kHeadDim + 1];
        }
      }
      float mn = M;
#pragma unroll
      for (int j = 0; j < k; ++j) mn = fmaxf(mn, m[j]);
      const float f = ex2(M - mn);
      M = mn;
      L *= f;
#pragma unroll
      for (int q = 0; q < 4; ++q) O[q] *= f;
#pragma unroll
      for (int j = 0; j < k; ++j) {
        const float e = ex2(m[j] - mn);
        L += l[j] * e;
        O[0] += v[j].x * e;
        O[1] += v[j].y * e;
        O[2] += v[j].z * e;
        O[3] += v[j].w * e;
      }
    }
  }
  __device__ __forceinline__ void put(float* p, int lane) const {
    *reinterpret_cast<float4*>(p + 4 * lane) = make_float4(O[0], O[1], O[2], O[3]);
    if (lane == 0) {
      p[kHeadDim] = M;
      p[kHeadDim + 1] = L;
    }
  }
};
__device__ __forceinline__ __half* out_head(const AttnArgs& a, int b, int head) {
  return a.o + (long)b * a.ldo + (long)head * kHeadDim;
}
__device__ __forceinline__ void store_head(const AttnArgs& a, __half* o, int kh, float L, float (&O)[4], int lane) {
  const float inv = L > 0.f ? (a.c.v_scale ? a.c.v_scale[kh] : 1.f) / L : 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) O[i] *= inv;
  if (a.fwht) fwht32_x4(O, lane);
  reinterpret_cast<uint2*>(o)[lane] =
      make_uint2(h2_as_u32(__floats2half2_rn(O[0], O[1])), h2_as_u32(__floats2half2_rn(O[2], O[3])));
}

struct Place {                 // of a tile in the list
  int b, hc, t, T;             // sequence, kv head * chunks + chunk, tile and tiles of the sequence
};
__device__ __forceinline__ Place place_of(const int* prefix, const AttnArgs& a, int x) {
  const int y = a.by_Hc.div(x);
  int lo = 0, hi = a.B;                               // prefix[lo] <= y < prefix[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= y) lo = mid; else hi = mid;
  }
  const int T = prefix[lo + 1] - prefix[lo], rem = x - prefix[lo] * a.Hc;
  int hc = (int)__fdividef((float)rem, (float)T);     // below 2^16: off by one at most
  hc -= hc * T > rem;
  hc += (hc + 1) * T <= rem;
  return Place{lo, hc, rem - hc * T, T};
}

__global__ void __launch_bounds__(kThreads, 1)
    paged_attn_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                      const AttnArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * (kSlots * 2 * kTileBytes);
  float* part0 = reinterpret_cast<float*>(smem + kWarps * kSlots * 2 * kTileBytes);   // [warp][head, tail][..]
  uint64_t* bars = reinterpret_cast<uint64_t*>(part0 + kWarps * 2 * kPartFloats);
  int* meta = reinterpret_cast<int*>(bars + kWarps * kSlots);                          // [warp][head, tail] segment
  int* wsum = meta + 2 * kWarps;
  int* prefix = wsum + kWarps;                                                        // [B + 1] tiles before
  int* seqs = prefix + a.B + 1;                                                       // [B] lengths
  uint64_t* wbars = bars + warp * kSlots;
  const int Hc = a.Hc;

  if (lane == 0) {
    for (int s = 0; s < kSlots; ++s) mbar_init(&wbars[s], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    meta[2 * warp] = meta[2 * warp + 1] = -1;
  }
  if (tid == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmk)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmv)) : "memory");
  }
  pdl_wait_trigger();

  // lengths, and the prefix sums of their tiles
  {
    const int each = (a.B + kWarps * 32 - 1) / (kWarps * 32), b0 = tid * each;
    const long long cap = (long long)a.c.max_blocks * a.c.page;
    int own = 0;
    bool bad = false;
    for (int b = b0; b < min(a.B, b0 + each); ++b) {
      const long long n = a.seq_lens[b];
      bad |= n < 0 || n > cap;
      const int len = (int)(n < 0 ? 0 : n > cap ? cap : n);
      seqs[b] = len;
      own += (len + kTile - 1) / kTile;
    }
    if (bad && blockIdx.x == 0) atomicOr(&g_attn_status, kPagedBadPage);
    int inc = own;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, inc, s);
      if (lane >= s) inc += o;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    int at = inc - own;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) at += w < warp ? wsum[w] : 0;
    if (tid == 0) prefix[0] = 0;
    for (int b = b0; b < min(a.B, b0 + each); ++b) prefix[b + 1] = at += (seqs[b] + kTile - 1) / kTile;
    __syncthreads();
  }
  const int N = prefix[a.B] * Hc;
  // four tiles at least: fewer parts to join (8 against 4: 1 x 2048 8.0 against 7.0 us, 1 x 8192 11.8 against 11.2)
  const int per_cta = a.per_seg ? 0 : max(4, a.by_ctas.div(N + (int)gridDim.x - 1));
  if (blockIdx.x == 0 && a.header)
    for (int i = tid; i < a.B + 2; i += kThreads) a.header[i] = i ? prefix[i - 1] : per_cta;

  for (int b = blockIdx.x; b < a.B; b += gridDim.x)
    if (prefix[b + 1] == prefix[b])                           // a sequence without a position
      for (int i = tid; i < a.H * (kHeadDim / 8); i += kThreads)
        reinterpret_cast<uint4*>(a.o + (long)b * a.ldo)[i] = make_uint4(0, 0, 0, 0);

  // this CTA's run of the list, and this warp's
  int R0, R1;
  if (a.per_seg) {
    const int b = a.by_Hc.div(blockIdx.x), T = prefix[b + 1] - prefix[b];
    R0 = prefix[b] * Hc + ((int)blockIdx.x - b * Hc) * T;
    R1 = R0 + T;
  } else {
    R0 = min(N, (int)blockIdx.x * per_cta);
    R1 = min(N, R0 + per_cta);
  }
  const int pw = (R1 - R0 + kWarps - 1) / kWarps;
  const int beg = min(R1, R0 + warp * pw), end = min(R1, beg + pw);

  if (beg < end) {
    Place at;
    int win = beg, pg0 = 0, pg1 = 0, row0 = 0, row1 = 0;      // coordinates of tile win + lane
    auto look_up = [&](int first) {
      win = first;
      const Place p = place_of(prefix, a, min(first + lane, end - 1));
      if (first == beg)                                       // where the warp begins
        at = Place{__shfl_sync(0xffffffffu, p.b, 0), __shfl_sync(0xffffffffu, p.hc, 0),
                   __shfl_sync(0xffffffffu, p.t, 0), __shfl_sync(0xffffffffu, p.T, 0)};
      if (first + lane < end) {
        const int pos = p.t * kTile, kh = a.by_chunks.div(p.hc), blk = a.by_page.div(pos);
        const int* tab = a.c.table + (long)p.b * a.c.ld_table;
        pg0 = tab[blk];
        row0 = (kh - blk) * a.c.page + pos;
        bool bad = false;
        if (a.two_boxes) {
          const int p1 = pos + kTile / 2, blk1 = a.by_page.div(p1);
          pg1 = p1 < seqs[p.b] ? tab[blk1] : 0;
          row1 = (kh - blk1) * a.c.page + p1;
          if (pg1 < 0 || pg1 >= a.c.n_pages) pg1 = a.c.n_pages, bad = true;
        }
        if (pg0 < 0 || pg0 >= a.c.n_pages) pg0 = a.c.n_pages, bad = true;
        if (bad) atomicOr(&g_attn_status, kPagedBadPage);
      }
    };
    auto issue = [&](int x, int slot) {                       // whole warp; x < end
      if (x >= win + 32) look_up(x);
      const int s = x - win;
      const int p0 = __shfl_sync(0xffffffffu, pg0, s), r0 = __shfl_sync(0xffffffffu, row0, s);
      const int p1 = __shfl_sync(0xffffffffu, pg1, s), r1 = __shfl_sync(0xffffffffu, row1, s);
      if (lane == 0) {
        const uint32_t k = smem_u32(ring + slot * 2 * kTileBytes), v = k + kTileBytes;
        mbar_expect_tx(&wbars[slot], 2 * kTileBytes);
        load_box(k, &tmk, r0, p0, &wbars[slot]);
        load_box(v, &tmv, r0, p0, &wbars[slot]);
        if (a.two_boxes) {
          load_box(k + kTileBytes / 2, &tmk, r1, p1, &wbars[slot]);
          load_box(v + kTileBytes / 2, &tmv, r1, p1, &wbars[slot]);
        }
      }
    };
    look_up(beg);
    uint32_t qa[8], qb[8];
    // the maximum, and what scores are taken from: m - 15, or m itself where fp32 cannot tell them apart
    float m = kLowest, base = kLowest, l = 0.f, scale = 0.f, oacc[16][4];
    int seq = 0;
    bool first = at.t == 0;                                   // the segment began in this warp
    auto start_segment = [&]() {
      const int kh = a.by_chunks.div(at.hc), head = (at.hc - kh * a.chunks) * kGroup + g;
      seq = seqs[at.b];
      scale = (a.c.k_scale ? a.c.k_scale[kh] : 1.f) * rsqrtf((float)kHeadDim) * 1.4426950408889634f;
      const uint4* qp = reinterpret_cast<const uint4*>(a.q + (long)at.b * a.ldq +
                                                       ((long)kh * a.Hg + head) * kHeadDim + 32 * t);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 v = head < a.Hg ? qp[i] : make_uint4(0, 0, 0, 0);
        qa[2 * i] = v.x; qb[2 * i] = v.y; qa[2 * i + 1] = v.z; qb[2 * i + 1] = v.w;
      }
      m = base = kLowest;
      l = 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) oacc[j][i] = 0.f;
    };
    start_segment();
#pragma unroll
    for (int s = 0; s < kSlots; ++s)
      if (beg + s < end) issue(beg + s, s);
    int slot = 0;
    unsigned parity = 0;
    for (int x = beg; x < end; ++x) {
      if (!mbar_wait_warp(&wbars[slot], parity, a.polls)) {   // drain what is in flight and stop
        if (lane == 0) atomicOr(&g_attn_status, kPagedTimeout);
        for (int y = x; y < min(end, x + kSlots); ++y) {
          mbar_wait_warp(&wbars[slot], parity, kWaitPolls);
          slot = slot + 1 == kSlots ? 0 : slot + 1;
          if (slot == 0) parity ^= 1;
        }
        break;
      }
      const uint32_t kb = smem_u32(ring + slot * 2 * kTileBytes), vb = kb + kTileBytes;
      const int nvalid = min(kTile, seq - at.t * kTile);
      if (nvalid < kTile) {                                   // rows behind the sequence may hold anything
        for (int i = lane; i < (kTile - nvalid) * 8; i += 32)
          reinterpret_cast<uint4*>(ring + slot * 2 * kTileBytes + kTileBytes)[nvalid * 8 + i] = make_uint4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the slot's next load comes after these writes
        __syncwarp();
      }
      // ---- S = Q K^T, 4 x 8 positions
      float sc[4][2];
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) {
        const int pr = nt * 8 + g;
        const uint4 k0 = lds128(kb + pr * 128 + (((2 * t) ^ (pr & 7)) << 4));
        const uint4 k1 = lds128(kb + pr * 128 + (((2 * t + 1) ^ (pr & 7)) << 4));
        const uint32_t kw[8] = {k0.x, k0.y, k0.z, k0.w, k1.x, k1.y, k1.z, k1.w};
        float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          mma16816(c, qa[j], 0u, qb[j], 0u, fp8x2_to_h2((uint16_t)(kw[j] & 0xFFFFu)),
                   fp8x2_to_h2((uint16_t)(kw[j] >> 16)));
        const int p0 = nt * 8 + 2 * t;
        sc[nt][0] = p0 < nvalid ? c[0] * scale : -INFINITY;
        sc[nt][1] = p0 + 1 < nvalid ? c[1] * scale : -INFINITY;
      }
      // ---- running maximum and weights
      float mx = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[1][0], sc[1][1])),
                       fmaxf(fmaxf(sc[2][0], sc[2][1]), fmaxf(sc[3][0], sc[3][1])));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      if (__any_sync(0xffffffffu, mx > m)) {
        m = fmaxf(m, mx);
        float to = m - kWeightBits;
        to = m - to > kWeightBits ? m : to;                   // from 2^24 on m - 15 may round to m - 16: 2^16 is no f16
        const float f = ex2(base - to);
        base = to;
        l *= f;
#pragma unroll
        for (int j = 0; j < 16; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) oacc[j][i] *= f;
      }
      uint32_t ph[4], pl[4];                                  // rounded weights and remainders
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) {
        const float e0 = ex2(sc[nt][0] - base), e1 = ex2(sc[nt][1] - base);
        l += e0 + e1;
        const __half2 h = __floats2half2_rn(e0, e1);
        const float2 r = __half22float2(h);
        ph[nt] = h2_as_u32(h);
        pl[nt] = h2_as_u32(__floats2half2_rn(e0 - r.x, e1 - r.y));
      }
      // ---- O += P V, 2 x 16 positions
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const int r0 = kk * 16 + 2 * t, r1 = r0 + 1, r2 = r0 + 8, r3 = r0 + 9;
        const uint4 v0 = lds128(vb + r0 * 128 + ((g ^ (r0 & 7)) << 4));
        const uint4 v1 = lds128(vb + r1 * 128 + ((g ^ (r1 & 7)) << 4));
        const uint4 v2 = lds128(vb + r2 * 128 + ((g ^ (r2 & 7)) << 4));
        const uint4 v3 = lds128(vb + r3 * 128 + ((g ^ (r3 & 7)) << 4));
        const uint32_t w0[4] = {v0.x, v0.y, v0.z, v0.w}, w1[4] = {v1.x, v1.y, v1.z, v1.w};
        const uint32_t w2[4] = {v2.x, v2.y, v2.z, v2.w}, w3[4] = {v3.x, v3.y, v3.z, v3.w};
#pragma unroll
        for (int wi = 0; wi < 4; ++wi) {
          // bytes of rows (r0, r1) and (r2, r3) side by side
          const uint32_t lo01 = prmt(w0[wi], w1[wi], 0x5140u), hi01 = prmt(w0[wi], w1[wi], 0x7362u);
          const uint32_t lo23 = prmt(w2[wi], w3[wi], 0x5140u), hi23 = prmt(w2[wi], w3[wi], 0x7362u);
          const uint32_t p01[4] = {lo01 & 0xFFFFu, lo01 >> 16, hi01 & 0xFFFFu, hi01 >> 16};
          const uint32_t p23[4] = {lo23 & 0xFFFFu, lo23 >> 16, hi23 & 0xFFFFu, hi23 >> 16};
#pragma unroll
          for (int k = 0; k < 4; ++k)                         // element 16 g + 4 wi + k of the head
            mma16816(oacc[4 * wi + k], ph[2 * kk], pl[2 * kk], ph[2 * kk + 1], pl[2 * kk + 1],
                     fp8x2_to_h2((uint16_t)p01[k]), fp8x2_to_h2((uint16_t)p23[k]));
        }
      }
      __syncwarp();                                           // the slot is read; the next load may overwrite it
      if (x + kSlots < end) {
        if (lane == 0) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        issue(x + kSlots, slot);
      }
      slot = slot + 1 == kSlots ? 0 : slot + 1;
      if (slot == 0) parity ^= 1;

      // ---- end of the segment, or of this warp's run
      const bool last = at.t + 1 == at.T;
      if (last || x + 1 == end) {
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const int kh = a.by_chunks.div(at.hc), hg = (at.hc - kh * a.chunks) * kGroup + g;
        // head: began before, ends here; tail: goes on in the next warp; a whole one passes through the tail's place
        const int which = last && !first ? 0 : 1;
        float* p = part0 + (2 * warp + which) * kPartFloats + g * kPitch;
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          *reinterpret_cast<float4*>(p + 32 * t + j) =
              make_float4(oacc[j][0] + oacc[j][2], oacc[j + 1][0] + oacc[j + 1][2], oacc[j + 2][0] + oacc[j + 2][2],
                          oacc[j + 3][0] + oacc[j + 3][2]);
          *reinterpret_cast<float4*>(p + 32 * t + 16 + j) =
              make_float4(oacc[j][1] + oacc[j][3], oacc[j + 1][1] + oacc[j + 1][3], oacc[j + 2][1] + oacc[j + 2][3],
                          oacc[j + 3][1] + oacc[j + 3][3]);
        }
        if (t == 0) {
          p[kHeadDim] = base;
          p[kHeadDim + 1] = l;
        }
        if (first && last) {
          __syncwarp();
          const float* part = part0 + (2 * warp + 1) * kPartFloats;
#pragma unroll 1
          for (int h = 0; h < kGroup && hg - g + h < a.Hg; ++h) {
            const float4 v = *reinterpret_cast<const float4*>(part + h * kPitch + 4 * lane);
            float O[4] = {v.x, v.y, v.z, v.w};
            store_head(a, out_head(a, at.b, kh * a.Hg + hg - g + h), kh, part[h * kPitch + kHeadDim + 1], O, lane);
          }
          __syncwarp();
        } else if (lane == 0) {
          meta[2 * warp + which] = at.b * Hc + at.hc;
        }
        if (x + 1 < end) {                                    // the next segment
          at.t = 0;
          if (++at.hc == Hc) {
            at.hc = 0;
            do { ++at.b; } while (prefix[at.b + 1] == prefix[at.b]);
            at.T = prefix[at.b + 1] - prefix[at.b];
          }
          first = true;
          start_segment();
        }
      } else {
        ++at.t;
      }
    }
  }
  __syncthreads();

  // ---- join the parts of this CTA, segment by segment; a warp per head.
  // Lane 2 w + which looks at part (w, which): it opens a segment of this CTA if it
  // is the head of the first warp, or a tail that does not go on from the warp
  // before; then come the tails of the next warps, up to the head that closes it.
  const int mine = lane < 2 * kWarps ? meta[lane] : -1, before = __shfl_up_sync(0xffffffffu, mine, 2);
  const bool opens = mine >= 0 && ((lane & 1) ? lane < 2 || before != mine : lane == 0);
  for (unsigned open = __ballot_sync(0xffffffffu, opens); open; open &= open - 1) {
    const int from = __ffs(open) - 1, seg = __shfl_sync(0xffffffffu, mine, from), w = from >> 1;
    const unsigned of = __ballot_sync(0xffffffffu, mine == seg), heads = of & 0x55555555u;
    const int b = a.by_Hc.div(seg), hc = seg - b * Hc, T = prefix[b + 1] - prefix[b], s0 = prefix[b] * Hc + hc * T;
    const int kh = a.by_chunks.div(hc), hg = (hc - kh * a.chunks) * kGroup + warp;
    if (hg >= a.Hg) continue;
    Joined j;
    j.add_all(0, 1, __popc(of), lane, [&](int i) {
      return part0 + (2 * (w + i) + (heads >> (2 * (w + i)) & 1 ? 0 : 1)) * kPartFloats + warp * kPitch;
    });
    if (s0 >= R0 && s0 + T <= R1)
      store_head(a, out_head(a, b, kh * a.Hg + hg), kh, j.L, j.O, lane);
    else
      j.put(a.parts + ((long)blockIdx.x * 2 + (s0 < R0 ? 0 : 1)) * kPartFloats + warp * kPitch, lane);
  }
}

// Joins the (sequence, head) parts that lie in several CTAs: a CTA per query
// head, its warps take every fourth part.
__global__ void __launch_bounds__(kJoinWarps * 32) paged_join_kernel(const AttnArgs a) {
  __shared__ float part[kJoinWarps][kPitch];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head = blockIdx.x, b = blockIdx.y, kh = head / a.Hg, hg = head - kh * a.Hg;
  const int hc = kh * a.chunks + hg / kGroup;
  pdl_wait_trigger();
  const int per_cta = a.header[0], p0 = a.header[1 + b], T = a.header[2 + b] - p0;
  const int s0 = p0 * a.Hc + hc * T, c0 = s0 / per_cta, c1 = (s0 + T - 1) / per_cta;
  if (T == 0 || c0 == c1) return;
  Joined j;
  j.add_all(warp, kJoinWarps, c1 - c0 + 1, lane, [&](int i) {
    return a.parts + ((long)(c0 + i) * 2 + (i == 0 ? 1 : 0)) * kPartFloats + (hg % kGroup) * kPitch;
  });
  j.put(part[warp], lane);
  __syncthreads();
  if (warp) return;
  Joined all;
  all.add_all(0, 1, kJoinWarps, lane, [&](int i) { return part[i]; });
  store_head(a, out_head(a, b, head), kh, all.L, all.O, lane);
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int page_map(CUtensorMap* m, const void* base, const PagedView& c, long stride, int rows) {
  static EncodeTiled fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiled>(f);
  });
  if (!fn) return set_error(R4Q_ERR_CUDA, "paged_flash_decode: cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[3] = {(cuuint64_t)kHeadDim, (cuuint64_t)c.Hk * c.page, (cuuint64_t)c.n_pages};
  cuuint64_t strides[2] = {(cuuint64_t)kHeadDim, (cuuint64_t)stride};
  cuuint32_t box[3] = {(cuuint32_t)kHeadDim, (cuuint32_t)rows, 1};
  cuuint32_t es[3] = {1, 1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, es,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(R4Q_ERR_CUDA, "paged_flash_decode: tensor map encode failed (%d)", (int)r);
  return R4Q_OK;
}

size_t smem_bytes(int B) {
  return 1024 + (size_t)kWarps * kSlots * 2 * kTileBytes + (size_t)kWarps * 2 * kPartFloats * 4 +
         kWarps * kSlots * 8 + 3 * kWarps * 4 + (size_t)(2 * B + 1) * 4;
}

// A CTA per (sequence, head, group) and no second kernel, when they fit one
// wave and the table holds so few positions that a warp gets two tiles at most.
bool per_segment(int segments, int page, int max_blocks) {
  return segments <= num_sms() && (long)max_blocks * page <= 2L * kWarps * kTile;
}
int groups_of(int H, int Hk) { return Hk * ((H / Hk + kGroup - 1) / kGroup); }

size_t header_bytes(int B) { return ((size_t)(B + 2) * 4 + 15) / 16 * 16; }

}  // namespace

cudaError_t paged_attn_status_word(int** word) { return cudaGetSymbolAddress((void**)word, g_attn_status); }

}  // namespace r4q

using namespace r4q;

extern "C" size_t r4q_paged_flash_decode_workspace_bytes(int B, int H, int Hk, int page, int max_blocks) {
  if (B < 1 || H < 1 || Hk < 1 || page < 1 || max_blocks < 1) return 0;
  if (per_segment(B * groups_of(H, Hk), page, max_blocks)) return 0;
  return header_bytes(B) + (size_t)num_sms() * 2 * kPartFloats * 4;
}

extern "C" int r4q_paged_flash_decode(const void* q, long ldq, const r4q_paged_cache* cache,
                                      const long long* seq_lens, void* o, long ldo, int B, int H, int flags,
                                      void* workspace, size_t ws_bytes, void* stream) {
  AttnArgs a{};
  int st = paged_view("paged_flash_decode", cache, &a.c);
  if (st) return st;
  if (B < 0 || B > kMaxBatch || B > a.c.seqs)
    return set_error(R4Q_ERR_ARG, "paged_flash_decode: batch %d (at most %d and the table's %d rows)", B, kMaxBatch,
                     a.c.seqs);
  if (H < a.c.Hk || H % a.c.Hk || H > 65535)
    return set_error(R4Q_ERR_ARG, "paged_flash_decode: bad heads H=%d Hk=%d", H, a.c.Hk);
  if (flags & ~R4Q_ATTN_FWHT) return set_error(R4Q_ERR_ARG, "paged_flash_decode: unknown flags %d", flags);
  if (B == 0) return R4Q_OK;
  if (!q || !o || !seq_lens) return set_error(R4Q_ERR_ARG, "paged_flash_decode: null pointer");
  if (B > 1 && (ldq < (long)H * kHeadDim || ldo < (long)H * kHeadDim))
    return set_error(R4Q_ERR_ARG, "paged_flash_decode: row strides below H * 128");
  if (!aligned(q, 16) || (B > 1 && ldq % 8) || !aligned(o, 16) || (B > 1 && ldo % 8))
    return set_error(R4Q_ERR_ALIGN, "paged_flash_decode: q and o must be 16-byte aligned, strides multiples of 8");
  a.Hg = H / a.c.Hk;
  a.chunks = (a.Hg + kGroup - 1) / kGroup;
  const int Hc = a.Hc = groups_of(H, a.c.Hk);
  const long cap = (long)a.c.max_blocks * a.c.page;
  if ((cap / kTile + 1) * B * Hc > 1L << 30)
    return set_error(R4Q_ERR_ARG, "paged_flash_decode: %d sequences of %ld positions and %d heads are too many tiles",
                     B, cap, Hc);
  a.per_seg = per_segment(B * Hc, a.c.page, a.c.max_blocks);
  a.by_page = fast_div(a.c.page);
  a.by_Hc = fast_div(Hc);
  a.by_chunks = fast_div(a.chunks);
  a.by_ctas = fast_div(num_sms());
  const size_t need = a.per_seg ? 0 : r4q_paged_flash_decode_workspace_bytes(B, H, a.c.Hk, a.c.page, a.c.max_blocks);
  if (need && (!workspace || ws_bytes < need))
    return set_error(R4Q_ERR_CAPACITY, "paged_flash_decode: workspace %zu < %zu bytes", ws_bytes, need);
  if (need && !aligned(workspace, 16)) return set_error(R4Q_ERR_ALIGN, "paged_flash_decode: workspace misaligned");
  a.q = (const __half*)q; a.ldq = ldq;
  a.seq_lens = seq_lens;
  a.o = (__half*)o; a.ldo = ldo;
  a.B = B; a.H = H; a.fwht = (flags & R4Q_ATTN_FWHT) ? 1 : 0;
  a.two_boxes = a.c.page % kTile != 0;
  a.polls = wait_polls();
  if (need) {
    a.header = (int*)workspace;
    a.parts = (float*)((uint8_t*)workspace + header_bytes(B));
  }
  CUtensorMap tmk, tmv;
  const int rows = a.two_boxes ? kTile / 2 : kTile;
  st = page_map(&tmk, a.c.k, a.c, a.c.k_stride, rows);
  if (!st) st = page_map(&tmv, a.c.v, a.c, a.c.v_stride, rows);
  if (st) return st;
  static std::mutex mu;
  static bool attr_done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lk(mu);
    if (dev >= 64 || !attr_done[dev]) {
      const cudaError_t e = cudaFuncSetAttribute(paged_attn_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 (int)smem_bytes(kMaxBatch));
      if (e != cudaSuccess) {
        cudaGetLastError();
        return set_error(R4Q_ERR_CUDA, "paged_attn_kernel: %s", cudaGetErrorString(e));
      }
      if (dev < 64) attr_done[dev] = true;
    }
  }
  cudaStream_t s = (cudaStream_t)stream;
  const unsigned ctas = a.per_seg ? (unsigned)(B * Hc) : (unsigned)num_sms();
  cudaError_t e = launch_pdl(paged_attn_kernel, dim3(ctas), dim3(kThreads), smem_bytes(B), s, tmk, tmv, a);
  if (e == cudaSuccess && !a.per_seg)
    e = launch_pdl(paged_join_kernel, dim3((unsigned)H, (unsigned)B), dim3(kJoinWarps * 32), 0, s, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(R4Q_ERR_CUDA, "paged_attn_kernel: %s", cudaGetErrorString(e));
  }
  return R4Q_OK;
}
