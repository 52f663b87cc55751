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
#include "common.cuh"
#include "ops.h"

namespace ssb {
namespace {

constexpr int kDq = 576, kDv = 512, kUnit = 128, kTileH = 64;
constexpr int kMaxCtas = 148;                  // ranges a call is cut into at most (the workspace is sized by it)
constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

struct Plan {                                   // the row of a CTA's first unit
  int row;
  int64_t first;                                // units before that row
};

// Tokens (selected: list columns) and units of row t.
SSB_DEVICE int row_bound(const MlaDecodeArgs& a, int64_t t) {
  int64_t n = a.indices != nullptr ? a.n_idx : min((int64_t)a.width * kUnit, (int64_t)a.seq_lens[t]);
  if (a.reqs != nullptr && (a.reqs[t] < 0 || a.reqs[t] >= a.R)) n = 0;
  return n > 0 ? static_cast<int>(n) : 0;
}
SSB_DEVICE int row_units(const MlaDecodeArgs& a, int64_t t) { return (row_bound(a, t) + kUnit - 1) / kUnit; }

// All threads of the CTA: this CTA's range [lo, hi) of units and the row that holds unit lo (row = T: nothing to do).
SSB_DEVICE void find_range(const MlaDecodeArgs& a, int cta, int ctas, int64_t* sh, int64_t& lo, int64_t& hi, Plan& p) {
  const int tid = threadIdx.x;
  int64_t sum = 0;
  for (int64_t t = tid; t < a.T; t += blockDim.x) sum += row_units(a, t);
  sh[tid] = sum;
  __syncthreads();
  for (int o = blockDim.x / 2; o > 0; o >>= 1) {
    if (tid < o) sh[tid] += sh[tid + o];
    __syncthreads();
  }
  const int64_t total = sh[0];
  __syncthreads();
  const int64_t used = min((int64_t)ctas, total);      // every range in use holds a unit: a row's CTAs are consecutive
  lo = cta < used ? total * cta / used : total;
  hi = cta < used ? total * (cta + 1) / used : total;
  if (tid == 0) sh[256] = a.T, sh[257] = 0;
  int64_t base = 0;
  for (int64_t c = 0; c < a.T; c += blockDim.x) {
    const int64_t t = c + tid;
    const int64_t n = t < a.T ? row_units(a, t) : 0;
    sh[tid] = n;
    __syncthreads();
    for (int o = 1; o < blockDim.x; o <<= 1) {
      const int64_t v = tid >= o ? sh[tid - o] : 0;
      __syncthreads();
      sh[tid] += v;
      __syncthreads();
    }
    const int64_t end = base + sh[tid], beg = end - n;
    if (n > 0 && beg <= lo && lo < end) sh[256] = t, sh[257] = beg;
    base += sh[blockDim.x - 1];
    __syncthreads();
    if (base > lo) break;
  }
  p.row = static_cast<int>(sh[256]);
  p.first = sh[257];
}

SSB_DEVICE float* part_o(const MlaDecodeArgs& a, int tile, int slot) {
  return a.part_o + ((int64_t)tile * 2 * kMaxCtas + slot) * kTileH * kDv;
}
SSB_DEVICE float2* part_ml(const MlaDecodeArgs& a, int tile, int slot) {
  return a.part_ml + ((int64_t)tile * 2 * kMaxCtas + slot) * kTileH;
}

// Cache row of the j-th token of row t's list (-1: none).
SSB_DEVICE int64_t token_slot(const MlaDecodeArgs& a, int64_t t, int64_t j) {
  const int64_t req = a.reqs != nullptr ? a.reqs[t] : t;
  int64_t pos = j;
  if (a.indices != nullptr) {
    pos = a.indices[t * a.ld_idx + j];
    if (pos < 0 || (a.seq_lens != nullptr && pos >= a.seq_lens[t])) return -1;
  }
  if (pos / kUnit >= a.width) return -1;
  const int64_t page = a.table[req * a.width + pos / kUnit];
  const int64_t slot = page * kUnit + pos % kUnit;
  return page >= 0 && slot < a.cache_rows ? slot : -1;
}

constexpr int kTok = 32;                        // tokens a tile
constexpr int kQLd = 578, kKLd = 578;           // bf16 row pitches in shared memory
constexpr int kOffK = kTileH * kQLd * 2;
constexpr int kOffS = kOffK + kTok * kKLd * 2;
constexpr int kOffStat = kOffS + kTileH * kTok * 4;
constexpr int kOffPlan = kOffStat + 3 * kTileH * 4;
constexpr int kOffSlot = kOffPlan + 260 * 8;
constexpr int kSmem = kOffSlot + kTok * 8;

__global__ void __launch_bounds__(kThreads, 1) mla_decode_kernel(const MlaDecodeArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  __nv_bfloat16* Q = reinterpret_cast<__nv_bfloat16*>(smem);
  __nv_bfloat16* K = reinterpret_cast<__nv_bfloat16*>(smem + kOffK);
  float* Sc = reinterpret_cast<float*>(smem + kOffS);
  float* M = reinterpret_cast<float*>(smem + kOffStat);
  float* L = M + kTileH;
  float* Al = L + kTileH;
  int64_t* sh = reinterpret_cast<int64_t*>(smem + kOffPlan);
  int64_t* slots = reinterpret_cast<int64_t*>(smem + kOffSlot);
  const int tid = threadIdx.x, cta = blockIdx.x, tile = blockIdx.y;
  const int h0 = tile * kTileH, nh = min(kTileH, a.H - h0);
  int64_t lo, hi;
  Plan p;
  find_range(a, cta, gridDim.x, sh, lo, hi, p);
  int64_t at = lo, first = p.first;
  bool head_part = true;                        // the CTA's first segment: partial slot 0, a later one slot 1
  for (int64_t t = p.row; t < a.T && at < hi; ++t) {
    const int nb = row_units(a, t);
    if (nb == 0) continue;
    const int64_t end = min(hi, first + nb);
    const int b0 = static_cast<int>(at - first), b1 = static_cast<int>(end - first), n = row_bound(a, t);
    __syncthreads();
    for (int i = tid; i < kTileH * kDq; i += kThreads) {
      const int h = i / kDq, c = i - h * kDq;
      float v = 0.0f;
      if (h < nh) {
        const int64_t off = t * a.ldq + (h0 + h) * a.hsq + c;
        v = a.q_e4m3 ? e4m3_value(static_cast<const uint8_t*>(a.q)[off])
                     : __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[off]);
      }
      Q[h * kQLd + c] = __float2bfloat16(v);
    }
    if (tid < kTileH) M[tid] = -INFINITY, L[tid] = 0.0f;
    float o[2][kTileH];
#pragma unroll
    for (int h = 0; h < kTileH; ++h) o[0][h] = o[1][h] = 0.0f;
    for (int64_t j0 = (int64_t)b0 * kUnit; j0 < min((int64_t)b1 * kUnit, (int64_t)n); j0 += kTok) {
      __syncthreads();
      if (tid < kTok) slots[tid] = j0 + tid < n ? token_slot(a, t, j0 + tid) : -1;
      __syncthreads();
      for (int i = tid; i < kTok * (kDq / 2); i += kThreads) {
        const int r = i / (kDq / 2), c = i - r * (kDq / 2);
        const int64_t sl = slots[r];
        float2 v = make_float2(0.0f, 0.0f);
        if (sl >= 0) {
          const uint16_t w = reinterpret_cast<const uint16_t*>(a.kv + sl * kDq)[c];
          v = make_float2(e4m3_value(w & 0xFF), e4m3_value(w >> 8));
        }
        *reinterpret_cast<__nv_bfloat162*>(K + r * kKLd + 2 * c) = __floats2bfloat162_rn(v.x, v.y);
      }
      __syncthreads();
      {
        const int h = tid >> 2, g = tid & 3;
        float s[8] = {};
        for (int c = 0; c < kDq; c += 2) {
          const float2 qv = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(Q + h * kQLd + c));
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const float2 kv = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(K + (g + 4 * u) * kKLd + c));
            s[u] = fmaf(qv.y, kv.y, fmaf(qv.x, kv.x, s[u]));
          }
        }
        float mb = -INFINITY;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          s[u] = slots[g + 4 * u] >= 0 ? s[u] * (a.bmm1 * kLog2e) : -INFINITY;
          mb = fmaxf(mb, s[u]);
        }
        mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, 1));
        mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, 2));
        const float m0 = M[h], m1 = fmaxf(m0, mb);
        float ls = 0.0f;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float pv = slots[g + 4 * u] >= 0 ? exp2f(s[u] - (m1 == -INFINITY ? 0.0f : m1)) : 0.0f;
          Sc[h * kTok + g + 4 * u] = pv;
          ls += pv;
        }
        ls += __shfl_xor_sync(0xffffffffu, ls, 1);
        ls += __shfl_xor_sync(0xffffffffu, ls, 2);
        __syncwarp();
        if (g == 0) {
          Al[h] = m0 == -INFINITY ? 0.0f : exp2f(m0 - m1);
          L[h] = L[h] * Al[h] + ls;
          M[h] = m1;
        }
      }
      __syncthreads();
#pragma unroll
      for (int h = 0; h < kTileH; ++h) o[0][h] *= Al[h], o[1][h] *= Al[h];
      for (int j = 0; j < kTok; ++j) {
        const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(K + j * kKLd + 2 * tid));
#pragma unroll
        for (int h = 0; h < kTileH; ++h) {
          const float pv = Sc[h * kTok + j];
          o[0][h] = fmaf(pv, v.x, o[0][h]);
          o[1][h] = fmaf(pv, v.y, o[1][h]);
        }
      }
    }
    __syncthreads();
    const bool whole = b0 == 0 && b1 == nb;
    const int slot = 2 * cta + (head_part ? 0 : 1);
    if (whole) {
#pragma unroll
      for (int h = 0; h < kTileH; ++h) {
        if (h >= nh) break;
        const float inv = L[h] == 0.0f ? 0.0f : a.bmm2 / L[h];         // a NaN sum stays one
        reinterpret_cast<__nv_bfloat162*>(a.out + (t * a.H + h0 + h) * kDv)[tid] =
            __floats2bfloat162_rn(o[0][h] * inv, o[1][h] * inv);
      }
      if (a.lse != nullptr && tid < nh)
        a.lse[t * a.H + h0 + tid] = L[tid] == 0.0f ? -INFINITY : (M[tid] + log2f(L[tid])) / kLog2e;
    } else {
      float* po = part_o(a, tile, slot);
#pragma unroll
      for (int h = 0; h < kTileH; ++h) reinterpret_cast<float2*>(po + h * kDv)[tid] = make_float2(o[0][h], o[1][h]);
      if (tid < kTileH) part_ml(a, tile, slot)[tid] = make_float2(M[tid], L[tid]);
    }
    if (tid == 0 && tile == 0) {
      if (b0 == 0) a.rows[t].first = cta, a.rows[t].first_slot = slot;
      if (b1 == nb) a.rows[t].last = cta;
    }
    head_part = false;
    at = end;
    first += nb;
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
  if (a.T < 0 || a.T > 0x7fffffff || a.H <= 0 || a.H > 128 || a.R <= 0 || a.width <= 0 || a.cache_rows < 0 ||
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
  static bool attr = false;
  if (!attr) {
    if (cudaFuncSetAttribute(mla_decode_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess)
      return kErrCuda;
    attr = true;
  }
  mla_decode_kernel<<<dim3((unsigned)(kMaxCtas / tiles), (unsigned)tiles), kThreads, kSmem, stream>>>(a);
  if (cudaGetLastError() != cudaSuccess) return kErrCuda;
  mla_join_kernel<<<dim3((unsigned)a.T, (unsigned)a.H, 4), 128, 0, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
}

}  // namespace ssb
