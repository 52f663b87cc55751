// Latent (MLA) attention of new tokens for sm_100a: each query row over the paged e4m3 cache, all of its first seq_len
// tokens or a list of selected ones, split over the row's tokens and joined.
//
//   s_j = bmm1 q[t, h, :] . kv[slot_j, :]   (576 values);   out[t, h, :] = bmm2 sum_j softmax(s)_j kv[slot_j, 0:512]
//
// Split: a row of n tokens is ceil(n / 128) units of work; the units of all rows, in row order, are cut into equal
// contiguous ranges, one per CTA (two rows or more may share a CTA, one row may span many). A CTA works through its
// range row by row; a row that lies in one range is finished there, the parts of a row cut between ranges go to the
// workspace as (running max m, sum l, unnormalised O) in fp32 and are joined by a second kernel:
//   M = max_i m_i;  O = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i.
// No atomics and a fixed order of the sums: the same inputs give the same bits.
#include <cuda_fp16.h>

#include "common.cuh"
#include "ops.h"

namespace ssb {
namespace {

constexpr int kDq = 576, kDv = 512, kUnit = 128, kTileH = 64;
constexpr int kMaxCtas = 148;                  // ranges a call is cut into at most (the workspace is sized by it)
constexpr float kLog2e = 1.4426950408889634f;

struct Plan {                                   // the row of a CTA's first unit
  int row;
  int64_t first;                                // units before that row
};

// Tokens and units of row t. How many tokens a row's list names is not known before it is read: its share is planned
// by the list's width or, where that is smaller, the tokens it can name.
SSB_DEVICE int row_bound(const MlaDecodeArgs& a, int64_t t) {
  int64_t n = a.indices != nullptr ? a.n_idx : (int64_t)a.width * kUnit;
  if (a.seq_lens != nullptr) n = min(n, (int64_t)a.seq_lens[t]);
  if (a.reqs != nullptr && (a.reqs[t] < 0 || a.reqs[t] >= a.R)) n = 0;
  return n > 0 ? static_cast<int>(n) : 0;
}
SSB_DEVICE int row_units(const MlaDecodeArgs& a, int64_t t) { return (row_bound(a, t) + kUnit - 1) / kUnit; }

// All threads of the CTA (256 or more): this CTA's range [lo, hi) of units and the row that holds unit lo.
constexpr int kScan = 256;
SSB_DEVICE void find_range(const MlaDecodeArgs& a, int cta, int ctas, int64_t* sh, int64_t& lo, int64_t& hi, Plan& p) {
  const int tid = threadIdx.x;
  const bool in = tid < kScan;
  if (in) {
    int64_t sum = 0;
    for (int64_t t = tid; t < a.T; t += kScan) sum += row_units(a, t);
    sh[tid] = sum;
  }
  __syncthreads();
  for (int o = kScan / 2; o > 0; o >>= 1) {
    if (tid < o) sh[tid] += sh[tid + o];
    __syncthreads();
  }
  const int64_t total = sh[0];
  __syncthreads();
  const int64_t used = min((int64_t)ctas, total);      // every range in use holds a unit: a row's CTAs are consecutive
  lo = cta < used ? total * cta / used : total;
  hi = cta < used ? total * (cta + 1) / used : total;
  if (tid == 0) sh[kScan] = a.T, sh[kScan + 1] = 0;
  int64_t base = 0;
  for (int64_t c = 0; c < a.T; c += kScan) {
    const int64_t t = c + tid;
    const int64_t n = in && t < a.T ? row_units(a, t) : 0;
    if (in) sh[tid] = n;
    __syncthreads();
    for (int o = 1; o < kScan; o <<= 1) {
      const int64_t v = in && tid >= o ? sh[tid - o] : 0;
      __syncthreads();
      if (in) sh[tid] += v;
      __syncthreads();
    }
    const int64_t end = base + (in ? sh[tid] : 0), beg = end - n;
    if (n > 0 && beg <= lo && lo < end) sh[kScan] = t, sh[kScan + 1] = beg;
    base += sh[kScan - 1];
    __syncthreads();
    if (base > lo) break;
  }
  p.row = static_cast<int>(sh[kScan]);
  p.first = sh[kScan + 1];
}

SSB_DEVICE float* part_o(const MlaDecodeArgs& a, int tile, int slot) {
  return a.part_o + ((int64_t)tile * 2 * kMaxCtas + slot) * kTileH * kDv;
}
SSB_DEVICE float2* part_ml(const MlaDecodeArgs& a, int tile, int slot) {
  return a.part_ml + ((int64_t)tile * 2 * kMaxCtas + slot) * kTileH;
}

// ---- shared memory ------------------------------------------------------------------------------------------------
constexpr int kSoftWarps = 8;                   // warps 0-7: token quarter warp & 3, heads 32 (warp >> 2) .. + 31
constexpr int kSoftmax = 32 * kSoftWarps;
constexpr int kHalf = 128;                      // threads of one head half
constexpr int kMmaWarp = kSoftWarps;            // warp 8; warps 9-12 gather
constexpr int kGatherWarps = 4;
constexpr int kThreads = kSoftmax + 32 + 32 * kGatherWarps;
constexpr int kChunk = 16384;                   // [128 rows x 128 B], 128-byte swizzle
constexpr int kRope = 8192;                     // [128 rows x 64 B], 64-byte swizzle
constexpr int kRows = 4 * kChunk + kRope;       // 128 rows of 576 bytes: the keys of a unit, or the query tile's parts
constexpr int kOffQ = 0;
constexpr int kOffKv = kRows;                   // two units
constexpr int kOffPlo = 3 * kRows;              // the low parts of P; the high parts take the unit's rope chunk
constexpr int kOffSf = kOffPlo + kRope;         // block scales of P: byte (h % 32) 16 + (h / 32) 4 + token quarter
constexpr int kOffBar = kOffSf + 512;           // mbarriers
constexpr int kOffMisc = kOffBar + 128;         // tmem address, abort flag, last-unit flags
constexpr int kOffMask = kOffMisc + 32;         // uint32 [2][4]: tokens present in a unit
constexpr int kOffScale = kOffMask + 32;        // float2 [64]: base-2 score scale and minus the reference of each head
constexpr int kOffExp = kOffScale + 512;        // float [4][64]: maxima of the token quarters, or their sums
constexpr int kOffSum = kOffExp + 1024;         // float [64]: rescale factors, bmm2 / l
constexpr int kSmem = kOffSum + 256;
static_assert(kOffScale % 16 == 0 && kOffExp % 16 == 0 && kOffSf % 128 == 0 && kSmem <= 232448, "shared memory");
// TMEM columns: O^T as 4 tiles of 128 dims x 64 heads, S^T 128 tokens x (64 high | 64 low), block scales of V (1 against
// the high parts of P, 2^-4 against the low ones) and of P
constexpr uint32_t kColO = 0, kColS = 256, kColOne = 384, kColLow = 388, kColP = 392;
constexpr int kAhead = 4;                       // pages prefetched into L2 beyond the two in shared memory
constexpr float kMaxRise = 64.0f;               // base-2 scores above the reference before the accumulators are rescaled

// Block-scaled instruction descriptor (kind::mxf8f6f4): e4m3 A and B (format 0), ue8m0 scales (bit 23), A and B
// MN-major (bits 15, 16), N >> 3 in [17,23), M >> 4 in [24,29), B's scale byte in [4,6).
__host__ __device__ constexpr uint32_t idesc_mx(int M, int N, int b_byte) {
  return (static_cast<uint32_t>(b_byte) << 4) | (1u << 15) | (1u << 16) | (static_cast<uint32_t>(N >> 3) << 17) |
         (1u << 23) | (static_cast<uint32_t>(M >> 4) << 24);
}
SSB_DEVICE void tc_mma_mx(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t acc, uint32_t sfa,
                          uint32_t sfb) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
      "l"(ad), "l"(bd), "r"(idesc), "r"(acc), "r"(sfa), "r"(sfb)
      : "memory");
}
SSB_DEVICE void tmem_st_x4(uint32_t taddr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(a), "r"(b), "r"(c),
               "r"(d)
               : "memory");
}
SSB_DEVICE void cp_async16(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
SSB_DEVICE void cp_async_arrive_noinc(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
SSB_DEVICE void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// Largest of the 32 lanes' values, NaN ignored (all NaN: NaN).
SSB_DEVICE float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
SSB_DEVICE float ex2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two halves -> two e4m3 bytes (round to nearest even, the first in the low byte) and back.
SSB_DEVICE uint32_t half2_e4m3(__half2 v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(*reinterpret_cast<uint32_t*>(&v)));
  return r;
}
SSB_DEVICE __half2 e4m3_half2(uint32_t b) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(b)));
  return *reinterpret_cast<__half2*>(&r);
}
// v (|v| <= 256) as hi + lo / 16 in e4m3: 8 significant bits, down to a quantum of 2^-13. v enters as two halves (11
// bits, so that the rounding to 8 is the one that counts).
SSB_DEVICE void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 v = __floats2half2_rn(a, b);
  hi = half2_e4m3(v);
  lo = half2_e4m3(__hmul2(__hsub2(v, e4m3_half2(hi)), __float2half2_rn(16.0f)));
}
// Byte offset of 16-byte granule g of row r: a 128-byte-swizzled chunk, a 64-byte-swizzled one.
SSB_DEVICE uint32_t sw128(int r, int g) { return r * 128 + ((g ^ (r & 7)) << 4); }
SSB_DEVICE uint32_t sw64(int r, int g) { return r * 64 + ((g ^ ((r >> 1) & 3)) << 4); }
constexpr uint32_t kSw128 = 2, kSw64 = 4;       // descriptor layout types
// Granule g (0-35) of row r of 576 bytes.
SSB_DEVICE uint32_t row_off(int r, int g) {
  return g < 32 ? (g >> 3) * kChunk + sw128(r, g & 7) : 4 * kChunk + sw64(r, g - 32);
}

// Sums over the 32 lanes of 32 values a lane, transposed: lane l receives the total of value l.
SSB_DEVICE float warp_sum_transposed(float* v, int lane) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float keep = up ? v[i + o] : v[i], send = up ? v[i] : v[i + o];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  return v[0];
}

struct Bars {                                    // kv_full: one a buffer, kv_empty: one a half buffer (64 tokens)
  uint32_t kv_full, kv_empty, q_full, s_full, s_empty, p_full, pv_done, o_full, drain;
};
SSB_DEVICE bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
SSB_DEVICE void tma_prefetch_2d(const CUtensorMap* m, int32_t x, int32_t y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(m)), "r"(x),
               "r"(y)
               : "memory");
}

// One query row's heads h0 .. h0 + 63 into the query tile: rows 0-63 the high parts, 64-127 the low parts of
// q 2^-k (k per head, its largest value in [2^7, 2^8)), zero rows past nh. bf16 has 8 significant bits, so the two e4m3
// parts hold a value exactly unless it is below 2^-14 of the head's largest. Also each head's score scale (its reference
// cleared). Warps 0-7, 8 heads each.
template <bool Q8>
SSB_DEVICE void stage_q(const MlaDecodeArgs& a, uint8_t* smem, int64_t t, int h0, int nh, int warp, int lane) {
  uint8_t* Q = smem + kOffQ;
  float2* scale = reinterpret_cast<float2*>(smem + kOffScale);
  const float unit = a.bmm1 * kLog2e;
  if (Q8) {
    const uint8_t* q = static_cast<const uint8_t*>(a.q) + t * a.ldq;
    uint4 v[9];
#pragma unroll
    for (int j = 0; j < 9; ++j) {
      const int i = warp * 32 + lane + kSoftmax * j, h = i / 36, g = i - h * 36;
      v[j] = h < nh ? *reinterpret_cast<const uint4*>(q + (h0 + h) * a.hsq + g * 16) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < 9; ++j) {
      const int i = warp * 32 + lane + kSoftmax * j, h = i / 36, g = i - h * 36;
      *reinterpret_cast<uint4*>(Q + row_off(h, g)) = v[j];
    }
    if (warp < 2) scale[warp * 32 + lane] = make_float2(unit, 0.0f);
    return;
  }
  const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) + t * a.ldq;
#pragma unroll 1
  for (int i0 = 0; i0 < 8; i0 += 4) {
    uint4 v[4][3];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int h = 8 * warp + i0 + i;
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        const int g = lane + 32 * j;                                  // 72 granules of 8 values
        v[i][j] = h < nh && g < 72 ? *reinterpret_cast<const uint4*>(q + (h0 + h) * a.hsq + 8 * g)
                                   : make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int h = 8 * warp + i0 + i;
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        const uint32_t w[4] = {v[i][j].x, v[i][j].y, v[i][j].z, v[i][j].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, max(w[e] & 0x7FFFu, (w[e] >> 16) & 0x7FFFu));   // bf16 magnitudes
      }
      top = __reduce_max_sync(0xffffffffu, top);
      const int ex = static_cast<int>(top >> 7);                      // the largest value's biased exponent
      const int k = ex == 0 || ex == 255 ? 0 : max(min(ex - 134, 120), -120);
      const float down = __uint_as_float(static_cast<uint32_t>(127 - k) << 23);
      if (lane == 0)
        scale[h] = make_float2(h < nh ? unit * __uint_as_float(static_cast<uint32_t>(127 + k) << 23) : 0.0f, 0.0f);
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        const int g = lane + 32 * j;
        if (g >= 72) continue;
        const uint32_t w[4] = {v[i][j].x, v[i][j].y, v[i][j].z, v[i][j].w};
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // an infinite query value leaves no finite weight: NaN, which e4m3 can carry (it has no infinity)
          const float x = __uint_as_float(w[e] << 16) * down, y = __uint_as_float(w[e] & 0xFFFF0000u) * down;
          split2(isinf(x) ? NAN : x, isinf(y) ? NAN : y, hi[e], lo[e]);
        }
        const uint32_t sub = 8 * (g & 1);                             // 8 values: half a 16-byte granule
        *reinterpret_cast<uint2*>(Q + row_off(h, g >> 1) + sub) = make_uint2(hi[0] | (hi[1] << 16), hi[2] | (hi[3] << 16));
        *reinterpret_cast<uint2*>(Q + row_off(64 + h, g >> 1) + sub) =
            make_uint2(lo[0] | (lo[1] << 16), lo[2] | (lo[3] << 16));
      }
    }
  }
}

// A CTA's share of one row: units [b0, b1) of the row's nb planned ones; every role walks the same segments.
struct Segment {
  int64_t t;
  int b0, b1, nb;
};
struct Walk {
  int64_t t, at, hi, first;
  SSB_DEVICE bool next(const MlaDecodeArgs& a, Segment& s) {
    for (; t < a.T && at < hi; ++t) {
      const int nb = row_units(a, t);
      if (nb == 0) continue;
      const int64_t end = min(hi, first + nb);
      s.t = t, s.b0 = static_cast<int>(at - first), s.b1 = static_cast<int>(end - first), s.nb = nb;
      at = end;
      first += nb;
      ++t;
      return true;
    }
    return false;
  }
};

template <bool Q8>
__global__ void __launch_bounds__(kThreads, 1)
    mla_decode_kernel(const __grid_constant__ CUtensorMap mlat, const __grid_constant__ CUtensorMap mrope,
                      const MlaDecodeArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = blockIdx.x, tile = blockIdx.y;
  const int h0 = tile * kTileH, nh = min(kTileH, a.H - h0);
  const uint32_t sbase = smem_u32(smem), bar = sbase + kOffBar;
  const Bars B = {bar, bar + 16, bar + 48, bar + 56, bar + 64, bar + 72, bar + 80, bar + 88, bar + 96};
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kOffMisc);
  volatile int32_t* abort_flag = reinterpret_cast<volatile int32_t*>(smem + kOffMisc + 4);
  volatile int32_t* last_unit = reinterpret_cast<volatile int32_t*>(smem + kOffMisc + 8);     // [2]
  volatile uint32_t* mask = reinterpret_cast<volatile uint32_t*>(smem + kOffMask);
  if (sbase & 1023) {                                    // the swizzled tiles need it; no static shared memory precedes
    if (tid == 0) raise_status(a.status, kErrCuda);
    return;
  }

  Walk walk;
  {
    int64_t lo, hi;
    Plan p;
    find_range(a, cta, gridDim.x, reinterpret_cast<int64_t*>(smem + kOffPlo), lo, hi, p);
    if (lo >= hi) return;                                // fewer units than CTAs
    walk = {p.row, lo, hi, p.first};
  }
  if (tid == 0) {
    mbar_init(B.kv_full, 33 * kGatherWarps);             // every lane's copies, one arrive a warp for the mask
    mbar_init(B.kv_full + 8, 33 * kGatherWarps);
    for (int i = 0; i < 4; ++i) mbar_init(B.kv_empty + 8 * i, 1);
    mbar_init(B.q_full, kSoftmax);
    mbar_init(B.s_full, 1);
    mbar_init(B.s_empty, kSoftmax);
    mbar_init(B.p_full, kSoftmax);
    mbar_init(B.pv_done, 1);
    mbar_init(B.o_full, 1);
    mbar_init(B.drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();                                       // also: every thread has read the plan's words
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp > kMmaWarp) {
    // ---------------------------------------------------------------- gather: warp w brings tokens 32 w .. 32 w + 31
    const int w = warp - kMmaWarp - 1;
    if (w == 0 && lane == 0) {
      tma_prefetch_desc(&mlat);
      tma_prefetch_desc(&mrope);
    }
    const int cols = a.indices != nullptr ? (a.n_idx + kUnit - 1) / kUnit : 0;
    int u = 0;
    Segment s;
    bool ok = true;
    while (ok && walk.next(a, s)) {
      const int64_t req = a.reqs != nullptr ? a.reqs[s.t] : s.t;
      const int32_t* pages = a.table + req * a.width;
      const int len = a.seq_lens != nullptr ? a.seq_lens[s.t] : 0x7fffffff;
      const int32_t* idx = a.indices != nullptr ? a.indices + s.t * a.ld_idx : nullptr;
      int c0 = s.b0, c1 = s.b1;
      unsigned long long live = ~0ull;                   // bit i: unit c0 + i holds a selected token
      if (idx != nullptr) {                              // the row's planned share as units of list columns
        c0 = static_cast<int>((int64_t)s.b0 * cols / s.nb);
        c1 = static_cast<int>((int64_t)s.b1 * cols / s.nb);
        if (c1 - c0 <= 64) {
          live = 0;
          for (int c = c0; c < c1; ++c) {
            bool any = false;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int col = c * kUnit + 32 * j + lane;
              const int pos = col < a.n_idx ? idx[col] : -1;
              any |= pos >= 0 && pos < len;
            }
            if (__any_sync(0xffffffffu, any)) live |= 1ull << (c - c0);
          }
          if (live == 0) live = 1;                       // nothing selected: one empty unit gives the zeros
        }
      }
      auto slot_at = [&](int c) -> int {                 // cache row of this lane's token of unit c (-1: none)
        int pos = c * kUnit + 32 * w + lane;
        if (idx != nullptr) pos = pos < a.n_idx ? idx[pos] : -1;
        if (pos < 0 || pos >= len || pos / kUnit >= a.width) return -1;
        const int64_t slot = (int64_t)pages[pos / kUnit] * kUnit + pos % kUnit;
        return slot >= 0 && slot < a.cache_rows ? static_cast<int>(slot) : -1;
      };
      auto next_live = [&](int c) {
        while (c < c1 && c - c0 < 64 && !((live >> (c - c0)) & 1)) ++c;
        return c;
      };
      int c = next_live(c0);
      int slot = slot_at(c);
      // the tiles of this warp's lane 0: its half of the unit's tokens (w >> 1), latent chunks 0, 1 and the rope, or 2, 3
      const int ch = 2 * (w & 1);
      auto whole_page = [&](int c, int slot) {           // the same in every lane and warp
        return idx == nullptr && (c + 1) * kUnit <= len && slot >= 0 && slot - (32 * w + lane) + kUnit <= a.cache_rows;
      };
      auto prefetch = [&](int c) {                       // a page some units ahead into L2
        if (lane != 0 || idx != nullptr || c >= c1) return;
        const int sl = slot_at(c);                       // the first token of the warp's quarter
        if (!whole_page(c, sl)) return;
        const int y = sl - 32 * w + 64 * (w >> 1);
        tma_prefetch_2d(&mlat, 128 * ch, y);
        tma_prefetch_2d(&mlat, 128 * ch + 128, y);
        if (ch == 0) tma_prefetch_2d(&mrope, kDv, y);
      };
      for (int i = 0; i < kAhead; ++i) prefetch(c0 + 2 + i);
      while (c < c1) {
        const int buf = u & 1, cn = next_live(c + 1);
        const int slot_n = cn < c1 ? slot_at(cn) : -1;
        prefetch(c + 2 + kAhead);
        if (u >= 2) ok = mbar_wait(B.kv_empty + 16 * buf + 8 * (w >> 1), ((u >> 1) - 1) & 1, abort_flag, a.status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t dst = sbase + kOffKv + buf * kRows, full = B.kv_full + 8 * buf;
        const uint32_t present = __ballot_sync(0xffffffffu, slot >= 0);
        // a whole page comes as tiles; a row's last page, and selected tokens, row by row: rows that are not there have
        // to be zeros (whatever the cache holds there, NaN too, would meet weight 0 in the value product)
        if (whole_page(c, slot)) {
          if (lane == 0) {
            const int hf = w >> 1, y = slot - 32 * w + 64 * hf;
            const uint32_t d0 = dst + ch * kChunk + hf * (kChunk / 2);
            mbar_arrive_expect_tx(full, kChunk + (ch == 0 ? kRope / 2 : 0));
            tma_load_2d(d0, &mlat, 128 * ch, y, full);
            tma_load_2d(d0 + kChunk, &mlat, 128 * ch + 128, y, full);
            if (ch == 0) tma_load_2d(dst + 4 * kChunk + hf * (kRope / 2), &mrope, kDv, y, full);
          } else {
            mbar_arrive(full);
          }
        } else {
          const uint32_t lat = dst + (lane >> 3) * kChunk + 4096 * w;
          const uint8_t* src = a.kv + 16 * lane;
#pragma unroll 16
          for (int r = 0; r < 32; ++r) {                 // a warp instruction a token: its 512 latent bytes
            const int sl = __shfl_sync(0xffffffffu, slot, r);
            cp_async16(lat + sw128(r, lane & 7), src + (int64_t)max(sl, 0) * kDq, sl >= 0);
          }
#pragma unroll
          for (int r = 0; r < 32; r += 8) {              // 8 tokens: their 64 rope bytes
            const int sl = __shfl_sync(0xffffffffu, slot, r + (lane >> 2));
            cp_async16(dst + 4 * kChunk + sw64(32 * w + r + (lane >> 2), lane & 3),
                       a.kv + (int64_t)max(sl, 0) * kDq + kDv + 16 * (lane & 3), sl >= 0);
          }
          cp_async_arrive_noinc(full);                   // fires when this thread's copies have landed
        }
        if (lane == 0) {
          mask[4 * buf + w] = present;
          if (w == 0) last_unit[buf] = cn >= c1;
          mbar_arrive(full);
        }
        ++u;
        c = cn;
        slot = slot_n;
      }
    }
    cp_async_wait_all();
  } else if (warp == kMmaWarp) {
    // ---------------------------------------------------------------- MMA issue (one thread)
    if (lane == 0) {
      constexpr uint32_t idesc_s = idesc_e4m3(128, Q8 ? 64 : 128);
      // descriptors of the operands' first tiles; a tile further on is an addition to the address field
      const uint64_t dq = smem_desc(sbase + kOffQ, 0, 1024, kSw128);
      const uint64_t dqr = smem_desc(sbase + kOffQ + 4 * kChunk, 0, 512, kSw64);
      const uint64_t dk = smem_desc(sbase + kOffKv, 0, 1024, kSw128);
      const uint64_t dkr = smem_desc(sbase + kOffKv + 4 * kChunk, 0, 512, kSw64);
      const uint64_t dv = smem_desc(sbase + kOffKv, kChunk, 1024, kSw128);
      const uint64_t dph = smem_desc(sbase + kOffKv + 4 * kChunk, kRope, 512, kSw64);
      const uint64_t dpl = smem_desc(sbase + kOffPlo, kRope, 512, kSw64);
      const uint64_t dsf = smem_desc(sbase + kOffSf, 0, 128, 0);
      int uq = 0, up = 0, seg = 0;                       // units whose scores, whose values have been issued
      Segment s;
      bool ok = true;
      auto scores = [&](int v) {                         // S^T [tokens, heads] = K Q^T of unit v
        const uint64_t k = dk + (v & 1) * (kRows >> 4), kr = dkr + (v & 1) * (kRows >> 4);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            tc_mma_f8(tmem + kColS, k + ((c * kChunk + ks * 32) >> 4), dq + ((c * kChunk + ks * 32) >> 4), idesc_s,
                      (c | ks) != 0 ? 1u : 0u);
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)                   // the rope chunk: 64 bytes a row
          tc_mma_f8(tmem + kColS, kr + ((ks * 32) >> 4), dqr + ((ks * 32) >> 4), idesc_s, 1u);
        tc_commit(B.s_full);
      };
      auto values = [&](int v, bool fresh) {             // O^T [dims, heads] (+)= V^T P^T of unit v, high then low parts
        const uint64_t kv = dv + (v & 1) * (kRows >> 4), ph = dph + (v & 1) * (kRows >> 4);
        tc_cp_sf(tmem + kColP, dsf);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {                 // 32 tokens a step: one block of scales
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            const uint64_t ad = kv + ((d * kChunk + ks * 4096) >> 4);
            tc_mma_mx(tmem + kColO + 64 * d, ad, ph + ((ks * 2048) >> 4), idesc_mx(128, 64, ks),
                      fresh && ks == 0 ? 0u : 1u, tmem + kColOne, tmem + kColP);
            tc_mma_mx(tmem + kColO + 64 * d, ad, dpl + ((ks * 2048) >> 4), idesc_mx(128, 64, ks), 1u, tmem + kColLow,
                      tmem + kColP);
          }
          if (ks & 1) tc_commit(B.kv_empty + 16 * (v & 1) + 8 * (ks >> 1));     // 64 tokens' rows are free
        }
        tc_commit(B.pv_done);
      };
      while (ok && walk.next(a, s)) {
        ok = mbar_wait(B.q_full, seg & 1, abort_flag, a.status);
        bool fresh = true, last = false;
        unsigned long long t0 = globaltimer();
        while (ok && !(last && up == uq)) {
          // whichever is ready: the next unit's scores first, else the values of the one whose weights are there
          if (!last && mbar_test(B.kv_full + 8 * (uq & 1), (uq >> 1) & 1) &&
              (uq == 0 || mbar_test(B.s_empty, (uq - 1) & 1))) {
            last = last_unit[uq & 1] != 0;
            fence_proxy_async_smem();                    // rows brought by other threads' copies -> the tensor core
            tc_fence_after();
            scores(uq++);
          } else if (up < uq && mbar_test(B.p_full, up & 1)) {
            tc_fence_after();
            values(up++, fresh);
            fresh = false;
          } else {
            if (*abort_flag) ok = false;
            if (globaltimer() - t0 > kWaitNs) {
              *abort_flag = 1;
              raise_status(a.status, kErrTimeout);
              ok = false;
            }
            continue;
          }
          t0 = globaltimer();
        }
        if (ok) tc_commit(B.o_full);
        ++seg;
      }
      tc_commit(B.drain);                                // everything issued has completed when this arrives
      const unsigned long long t0 = globaltimer();
      while (!mbar_try_wait(B.drain, 0) && globaltimer() - t0 <= kWaitNs) {}
    }
  } else {
    // ---------------------------------------------------------------- softmax (warps 0-7): a token and 32 heads a thread
    const int quarter = warp & 3, half = warp >> 2, hb = 32 * half, bid = 1 + half;
    const int row = 32 * quarter + lane;
    const uint32_t tq = tmem + (static_cast<uint32_t>(32 * quarter) << 16);
    float2* scale = reinterpret_cast<float2*>(smem + kOffScale);
    float* part = reinterpret_cast<float*>(smem + kOffExp);
    float* sums = reinterpret_cast<float*>(smem + kOffSum);
    uint8_t* sf = smem + kOffSf;
    if (half == 0) tmem_st_x4(tq + kColOne, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu);   // 1
    else tmem_st_x4(tq + kColLow, 0x7B7B7B7Bu, 0x7B7B7B7Bu, 0x7B7B7B7Bu, 0x7B7B7B7Bu);            // 2^-4
    tmem_st_wait();
    int u = 0, seg = 0;
    Segment s, s_next;
    bool more = walk.next(a, s), ok = true;
    stage_q<Q8>(a, smem, s.t, h0, nh, warp, lane);
    fence_proxy_async_smem();
    tc_fence_before();
    mbar_arrive(B.q_full);
    named_bar(3, kSoftmax);                              // every head's scale is written
    while (more) {
      float l[32];
#pragma unroll
      for (int h = 0; h < 32; ++h) l[h] = 0.0f;
      float ref = -INFINITY;                             // reference of head hb + lane (the same in the 4 quarters)
      bool last = false, fresh = true, unset = true;
      while (!last) {
        const int buf = u & 1;
        ok = mbar_wait(B.s_full, u & 1, abort_flag, a.status);
        if (ok) ok = mbar_wait(B.kv_full + 8 * buf, (u >> 1) & 1, abort_flag, a.status);   // the mask's writes
        tc_fence_after();
        last = last_unit[buf] != 0;
        const uint32_t present = mask[4 * buf + quarter];
        const bool valid = (present >> lane) & 1;
        float p[32];
        auto load_scores = [&]() {                       // base-2 scores less the reference; tokens not there: -inf
          float y[32];
          tmem_ld_32x32b_x32(tq + kColS + hb, p);
          if (!Q8) tmem_ld_32x32b_x32(tq + kColS + 64 + hb, y);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float4 c = *reinterpret_cast<const float4*>(scale + hb + i);
            p[i] = fmaf(Q8 ? p[i] : fmaf(y[i], 0.0625f, p[i]), c.x, c.y);
            p[i + 1] = fmaf(Q8 ? p[i + 1] : fmaf(y[i + 1], 0.0625f, p[i + 1]), c.z, c.w);
          }
          if (present != 0xffffffffu) {
#pragma unroll
            for (int h = 0; h < 32; ++h) p[h] = valid ? p[h] : -INFINITY;
          }
        };
        load_scores();
        float top = p[0];
#pragma unroll
        for (int h = 1; h < 32; ++h) top = fmaxf(top, p[h]);
        // the four quarters agree on the rare path; a failed wait travels the same way
        const bool rise = named_bar_or(bid, kHalf, unset || top > kMaxRise || !ok);
        if (rise) {
          if (named_bar_or(bid, kHalf, !ok)) {
            ok = false;
            break;
          }
          // new references: a head without one, or with scores more than kMaxRise above it, takes the ceiling of this
          // unit's largest score; what it has accumulated is rescaled
          const float old = ref == -INFINITY ? 0.0f : ref;
#pragma unroll
          for (int h = 0; h < 32; ++h) {
            const float m = warp_max(p[h]);
            if (lane == 0) part[64 * quarter + hb + h] = m;
          }
          named_bar(bid, kHalf);
          float m = -INFINITY;
#pragma unroll
          for (int k = 0; k < 4; ++k) m = fmaxf(m, part[64 * k + hb + lane]);
          const bool move = m > -INFINITY && (ref == -INFINITY || m > kMaxRise);
          const float now = move ? ceilf(m + old) : old;
          const float f = move && ref != -INFINITY ? exp2f(old - now) : 1.0f;
          if (move) ref = now;
          unset = __any_sync(0xffffffffu, ref == -INFINITY);
          if (quarter == 0) {
            sums[hb + lane] = f;
            scale[hb + lane].y = -now;
          }
          const bool scaled = __any_sync(0xffffffffu, f != 1.0f);
          named_bar(bid, kHalf);
          if (scaled && !fresh) {
#pragma unroll
            for (int h = 0; h < 32; ++h) l[h] *= sums[hb + h];
            ok = mbar_wait(B.pv_done, (u - 1) & 1, abort_flag, a.status);
            tc_fence_after();
#pragma unroll 1
            for (int d = 0; d < 4; ++d) {
              tmem_ld_32x32b_x32(tq + kColO + 64 * d + hb, p);
              tmem_ld_wait();
#pragma unroll
              for (int h = 0; h < 32; ++h) p[h] *= sums[hb + h];
              tmem_st_32x32b_x32(tq + kColO + 64 * d + hb, p);
            }
            tmem_st_wait();
          }
          load_scores();
        }
        tc_fence_before();
        mbar_arrive(B.s_empty);
        // weights 2^score; then each head's largest over the warp's 32 tokens gives their block scale: its exponent E
        // moves the weights to [2^7, 2^8) at most, the scale 2^(E - 134) moves them back in the product
        uint32_t wh[8], wl[8], mine = 0;
#pragma unroll
        for (int h = 0; h < 32; ++h) {
          p[h] = ex2_fast(p[h]);
          l[h] += p[h];
        }
#pragma unroll
        for (int h = 0; h < 32; h += 4) {
          uint32_t part_hi[2], part_lo[2];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t e = max(__reduce_max_sync(0xffffffffu, __float_as_uint(p[h + k])) & 0x7F800000u, 12u << 23);
            p[h + k] *= __uint_as_float((261u << 23) - e);
            mine = lane == h + k ? e : mine;
          }
          split2(p[h], p[h + 1], part_hi[0], part_lo[0]);
          split2(p[h + 2], p[h + 3], part_hi[1], part_lo[1]);
          wh[h / 4] = part_hi[0] | (part_hi[1] << 16);
          wl[h / 4] = part_lo[0] | (part_lo[1] << 16);
        }
        if (u > 0 && !mbar_wait(B.pv_done, (u - 1) & 1, abort_flag, a.status)) ok = false;   // its P and scales are read
        sf[16 * lane + 4 * half + quarter] = static_cast<uint8_t>((mine >> 23) - 7);
        uint8_t* ph = smem + kOffKv + buf * kRows + 4 * kChunk;
        uint8_t* pl = smem + kOffPlo;
#pragma unroll
        for (int g = 0; g < 2; ++g) {                    // 16 heads a 16-byte granule
          *reinterpret_cast<uint4*>(ph + sw64(row, 2 * half + g)) = make_uint4(wh[4 * g], wh[4 * g + 1], wh[4 * g + 2], wh[4 * g + 3]);
          *reinterpret_cast<uint4*>(pl + sw64(row, 2 * half + g)) = make_uint4(wl[4 * g], wl[4 * g + 1], wl[4 * g + 2], wl[4 * g + 3]);
        }
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(B.p_full);
        fresh = false;
        ++u;
      }
      // ---- the row's sums, the next row's query, then the accumulators ----
      const float ls = warp_sum_transposed(l, lane);
      if (named_bar_or(3, kSoftmax, !ok)) break;
      part[64 * quarter + hb + lane] = ls;
      named_bar(3, kSoftmax);
      float total = 0.0f;
#pragma unroll
      for (int k = 0; k < 4; ++k) total += part[64 * k + hb + lane];
      if (quarter == 0) sums[hb + lane] = total == 0.0f ? 0.0f : a.bmm2 / total;     // a NaN sum stays one
      more = walk.next(a, s_next);
      if (more) {
        stage_q<Q8>(a, smem, s_next.t, h0, nh, warp, lane);
        fence_proxy_async_smem();
        mbar_arrive(B.q_full);
      }
      ok = mbar_wait(B.o_full, seg & 1, abort_flag, a.status);
      if (named_bar_or(3, kSoftmax, !ok)) break;
      tc_fence_after();
      const bool whole = s.b0 == 0 && s.b1 == s.nb;
      const int slot = 2 * cta + (seg == 0 ? 0 : 1);
      if (quarter == 0) {
        const int h = hb + lane;
        if (!whole) part_ml(a, tile, slot)[h] = make_float2(ref, total);
        else if (a.lse != nullptr && h < nh)
          a.lse[s.t * a.H + h0 + h] = total == 0.0f ? -INFINITY : ((ref == -INFINITY ? 0.0f : ref) + log2f(total)) / kLog2e;
        if (half == 0 && lane == 0 && tile == 0) {
          if (s.b0 == 0) a.rows[s.t].first = cta, a.rows[s.t].first_slot = slot;
          if (s.b1 == s.nb) a.rows[s.t].last = cta;
        }
      }
#pragma unroll 1
      for (int d = 0; d < 4; ++d) {                      // 128 dims x 32 heads; a lane holds one dim
        float o[32];
        tmem_ld_32x32b_x32(tq + kColO + 64 * d + hb, o);
        tmem_ld_wait();
        if (whole) {
          __nv_bfloat16* out = a.out + (s.t * a.H + h0 + hb) * kDv + 128 * d + row;
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (hb + i < nh) out[i * kDv] = __float2bfloat16(o[i] * sums[hb + i]);
        } else {
          float* po = part_o(a, tile, slot) + hb * kDv + 128 * d + row;
#pragma unroll
          for (int i = 0; i < 32; ++i) po[i * kDv] = o[i];
        }
      }
      tc_fence_before();
      s = s_next;
      ++seg;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins a row's parts: one CTA per (row, head, 128 output values), warp w taking parts w, w + 4, ...; rows without a
// token get zeros (lse -inf), rows that one CTA finished are left alone.
__global__ void __launch_bounds__(128) mla_join_kernel(const MlaDecodeArgs a) {
  __shared__ float4 so[4][32];
  __shared__ float sl[4];
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y, tile = h / kTileH, hh = h - tile * kTileH;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __nv_bfloat16* out = a.out + (t * a.H + h) * kDv + blockIdx.z * 128;
  const int nb = row_units(a, t);
  if (nb == 0) {
    if (a.reqs != nullptr && threadIdx.x == 0 && (a.reqs[t] < 0 || a.reqs[t] >= a.R)) raise_status(a.status, kErrArgs);
    out[threadIdx.x] = __float2bfloat16(0.0f);
    if (a.lse != nullptr && blockIdx.z == 0 && threadIdx.x == 0) a.lse[t * a.H + h] = -INFINITY;
    return;
  }
  const MlaRowParts rp = a.rows[t];
  if (rp.first == rp.last) return;
  const int parts = rp.last - rp.first + 1;
  auto slot_of = [&](int i) { return i == 0 ? rp.first_slot : 2 * (rp.first + i); };
  float m = -INFINITY;
  for (int i = lane; i < parts; i += 32) m = fmaxf(m, part_ml(a, tile, slot_of(i))[hh].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float l = 0.0f;
  const float mz = m == -INFINITY ? 0.0f : m;            // a part without a token (or all NaN) has m = -inf, f = 0
  for (int i = warp; i < parts; i += 4) {
    const float2 ml = part_ml(a, tile, slot_of(i))[hh];
    const float f = exp2f(ml.x - mz);
    const float4 v = reinterpret_cast<const float4*>(part_o(a, tile, slot_of(i)) + hh * kDv + blockIdx.z * 128)[lane];
    acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y);
    acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
    l = fmaf(f, ml.y, l);
  }
  so[warp][lane] = acc;
  if (lane == 0) sl[warp] = l;
  __syncthreads();
  if (warp != 0) return;
  l = sl[0] + sl[1] + sl[2] + sl[3];
  float4 s = so[0][lane];
#pragma unroll
  for (int w = 1; w < 4; ++w) {
    const float4 v = so[w][lane];
    s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
  }
  const float inv = l == 0.0f ? 0.0f : a.bmm2 / l;
  __nv_bfloat162 lo = __floats2bfloat162_rn(s.x * inv, s.y * inv), hi = __floats2bfloat162_rn(s.z * inv, s.w * inv);
  reinterpret_cast<uint2*>(out)[lane] = make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
  if (a.lse != nullptr && blockIdx.z == 0 && lane == 0)
    a.lse[t * a.H + h] = l == 0.0f ? -INFINITY : (mz + log2f(l)) / kLog2e;
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
int64_t tiles_of(int H) { return (H + kTileH - 1) / kTileH; }
int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

}  // namespace

int64_t mla_decode_workspace_bytes(int64_t T, int H) {
  const int64_t slots = tiles_of(H) * 2 * kMaxCtas;
  return up256(T * (int64_t)sizeof(MlaRowParts)) + up256(slots * kTileH * 8) + slots * kTileH * kDv * 4;
}

int launch_mla_decode(const MlaDecodeArgs& a_in, void* ws, int64_t ws_bytes, cudaStream_t stream) {
  MlaDecodeArgs a = a_in;
  const int eb = a.q_e4m3 ? 1 : 2;
  if (a.T < 0 || a.T > 0x7fffffff || a.H <= 0 || a.H > 128 || a.R <= 0 || a.width <= 0 || a.cache_rows <= 0 || a.cache_rows > 0x7fffffff ||
      (a.indices == nullptr && a.seq_lens == nullptr) ||
      (a.indices != nullptr && (a.n_idx < 0 || a.ld_idx < a.n_idx)) || (a.reqs == nullptr && a.T > a.R))
    return kErrArgs;
  if (a.T == 0) return kOk;
  if (a.q == nullptr || a.kv == nullptr || a.table == nullptr || a.out == nullptr || ws == nullptr ||
      !aligned(a.q, 16) || !aligned(a.kv, 16) || !aligned(a.out, 16) || !aligned(ws, 256) || (a.ldq * eb) % 16 ||
      (a.hsq * eb) % 16 || a.hsq < kDq || (a.T > 1 && a.ldq < kDq))
    return kErrArgs;
  if (ws_bytes < mla_decode_workspace_bytes(a.T, a.H)) return kErrWorkspace;
  const int64_t tiles = tiles_of(a.H), slots = tiles * 2 * kMaxCtas;
  uint8_t* p = static_cast<uint8_t*>(ws);
  a.rows = reinterpret_cast<MlaRowParts*>(p);
  p += up256(a.T * (int64_t)sizeof(MlaRowParts));
  a.part_ml = reinterpret_cast<float2*>(p);
  p += up256(slots * kTileH * 8);
  a.part_o = reinterpret_cast<float*>(p);
  auto* kernel = a.q_e4m3 ? mla_decode_kernel<true> : mla_decode_kernel<false>;
  static bool attr[2] = {false, false};
  if (!attr[a.q_e4m3]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess) return kErrCuda;
    attr[a.q_e4m3] = true;
  }
  CUtensorMap mlat, mrope;
  const int u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  int rc = make_map_2d_ex(&mlat, u8, a.kv, a.cache_rows, kDq, kDq, 128, kUnit / 2, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc == kOk) rc = make_map_2d_ex(&mrope, u8, a.kv, a.cache_rows, kDq, kDq, 64, kUnit / 2, CU_TENSOR_MAP_SWIZZLE_64B);
  if (rc != kOk) return rc;
  kernel<<<dim3((unsigned)(kMaxCtas / tiles), (unsigned)tiles), kThreads, kSmem, stream>>>(mlat, mrope, a);
  if (cudaGetLastError() != cudaSuccess) return kErrCuda;
  mla_join_kernel<<<dim3((unsigned)a.T, (unsigned)a.H, 4), 128, 0, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
}

}  // namespace ssb
