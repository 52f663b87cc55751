// KDA decode for sm_100a: the recurrent form of the gated delta rule over short runs of new tokens (one token a request
// in the usual decode step), on the state blocks that the chunked prefill (kda.cu) leaves.
//
// Per head, S [value, key] fp32 from the request's state block, token after token:
//   y = SiLU(sum_w W[c, w] x[t - 3 + w, c])            q | k | v of the head: 384 channels, the conv rows in registers
//   q <- q / sqrt(|q|^2 + 1e-6), k <- k / sqrt(|k|^2 + 1e-6)
//   a_c = exp(lower_bound sigmoid(exp(A_log) (g_c + dt_bias_c))),  b = sigmoid(beta)
//   S <- S diag(a);  u = b (v - S k);  S <- S + u k^T;  o = D^-1/2 S q
// The second product is folded into the first pass over S: with S the decayed state, S' q = S q + u (k . q), so each
// row gives S k and S q together and is touched once. Everything between the bf16 inputs and the bf16 output stays in
// fp32 (the chunked prefill rounds the conv outputs to bf16 for its tensor-core operands; nothing here needs that).
//
// Bound: HBM. A head's 64 KB of state are read and written once a call, 7 D^2 FLOP a token over them; a call moves
// 128 KB a head and request whatever the run's length. One CTA per (request, head), 8 warps, two CTAs an SM; warp w keeps
// value rows 16 w .. 16 w + 15 in registers, a lane 4 key columns of each (one 512-byte row a warp load, 16 loads in
// flight a lane while the conv and the gates are computed). Products and updates as packed fp32 pairs, short
// exponentials and quotients: with the library forms the code outgrew the instruction cache (406 us at 256 requests x 64
// heads, now 351 to 356, the copy rate). Measured against that: 8 lanes a row, which saves 24 of the 31 shuffles of the
// row sums (357 us, then against 347); the states through three 64 KB buffers by bulk copies with two groups of warps on
// every other one (614 us). Runs: each further token costs its arithmetic, little of it beside other CTAs' copies: 24
// requests x 64 heads 39 us with one token each, 45, 60 and 96 with 2, 4 and 8.
#include "common.cuh"
#include "ops.h"

namespace ssb {
namespace {

constexpr int kDim = 128;
constexpr int kDecThreads = 256;
constexpr int kRowsW = 16;             // value rows a warp

// e^x as 2^(x log2 e) with the product's rounding error carried to first order: ex2.approx's own error (2^-22) remains.
// x above 88 counts as 88 (e^x must stay finite, or its correction is inf - inf): as a divisor e^88 makes the quotients
// below 0, as they are there to 2^-126. NaN stays NaN.
SSB_DEVICE float exp_fast(float x) {
  x = x > 88.0f ? 88.0f : x;
  constexpr float kHi = 1.44269502162933349609375f, kLo = 1.925963033500928e-8f;        // log2 e in two parts
  const float t = x * kHi;
  const float r = fmaf(x, kLo, fmaf(x, kHi, -t));
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(t));
  return fmaf(y, fminf(fmaxf(r, -1.0f), 1.0f) * 0.6931471805599453f, y);
}
SSB_DEVICE float sigmoid_fast(float z) { return __fdividef(1.0f, 1.0f + exp_fast(-z)); }
SSB_DEVICE float silu_fast(float y) { return __fdividef(y, 1.0f + exp_fast(-y)); }
SSB_DEVICE float2 bf2(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
// The state is not read again by this call: its stores leave the caches first.
SSB_DEVICE void store_stream(float* p, ulonglong2 v) {
  float4 f;
  f2unpack(v.x, f.x, f.y);
  f2unpack(v.y, f.z, f.w);
  __stcs(reinterpret_cast<float4*>(p), f);
}
SSB_DEVICE float sum2(uint64_t v) {
  float a, b;
  f2unpack(v, a, b);
  return a + b;
}

// Sums over the 32 lanes of 32 values a lane, transposed: lane l receives the total of value l (31 shuffles).
SSB_DEVICE float warp_sum_transposed(float (&v)[32], int lane) {
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

__global__ void __launch_bounds__(kDecThreads, 2) kda_decode_kernel(const __grid_constant__ KdaArgs a) {
  __shared__ __align__(16) float sy[2][4][kDim];       // q | k | v | decay of a token, double-buffered
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r = blockIdx.x / a.H, h = blockIdx.x - r * a.H;
  const int4 sq = __ldg(reinterpret_cast<const int4*>(a.seqs) + r);   // {first row, end row, state block, has state}
  const int s = sq.x, e = sq.y;
  if (s < 0 || e < s || e > a.T || sq.z < 0) {
    if (tid == 0 && h == 0) raise_status(a.status, kErrArgs);
    return;
  }
  if (e == s) return;
  const bool init = sq.w != 0;
  float* S = a.rec_state + (int64_t)sq.z * a.rs_stride + ((int64_t)h * kDim + kRowsW * warp) * kDim + 4 * lane;
  ulonglong2 st[kRowsW];                               // row i of the warp: columns 4 lane .. 4 lane + 3
#pragma unroll
  for (int i = 0; i < kRowsW; ++i)
    st[i] = init ? *reinterpret_cast<const ulonglong2*>(S + i * kDim) : make_ulonglong2(0, 0);

  // threads 0-191: a pair of conv channels each (q 0-63, k 64-127, v 128-191); threads 192-255: a pair of gates
  const bool conv = tid < 192;
  const int pair = tid & 63, part = tid >> 6;
  const int64_t col = (int64_t)part * a.P + h * kDim + 2 * pair;
  __nv_bfloat16* cs = a.conv_state + (int64_t)sq.z * a.cs_stride + col;
  const uint32_t* in = reinterpret_cast<const uint32_t*>(conv ? a.x + col : a.g + h * kDim + 2 * pair);
  const int64_t pitch = (conv ? a.ldx : a.ldg) / 2;
  uint32_t raw0 = 0, raw1 = 0, raw2 = 0;
  if (conv && init) {
    raw0 = *reinterpret_cast<const uint32_t*>(cs);
    raw1 = *reinterpret_cast<const uint32_t*>(cs + 3 * a.P);
    raw2 = *reinterpret_cast<const uint32_t*>(cs + 6 * a.P);
  }
  uint32_t raw = __ldg(in + s * pitch);
  float beta = __bfloat162float(a.beta[(int64_t)s * a.ldb + h]);
#pragma unroll 1
  for (int t = s; t < e; ++t) {
    float* y = &sy[(t - s) & 1][0][0];
    float2 o;
    if (conv) {
      const uint4 wv = __ldg(reinterpret_cast<const uint4*>(a.conv_w + col * 4));   // 2 channels x 4 taps
      const float2 x0 = bf2(raw0), x1 = bf2(raw1), x2 = bf2(raw2), x3 = bf2(raw);
      const float2 p0 = bf2(wv.x), p1 = bf2(wv.y), p2 = bf2(wv.z), p3 = bf2(wv.w);
      o.x = silu_fast(fmaf(p1.y, x3.x, fmaf(p1.x, x2.x, fmaf(p0.y, x1.x, p0.x * x0.x))));
      o.y = silu_fast(fmaf(p3.y, x3.y, fmaf(p3.x, x2.y, fmaf(p2.y, x1.y, p2.x * x0.y))));
      raw0 = raw1, raw1 = raw2, raw2 = raw;
    } else {
      const float2 g = bf2(raw), dt = __ldg(reinterpret_cast<const float2*>(a.dt_bias + h * kDim) + pair);
      const float rate = exp_fast(__ldg(a.a_log + h));
      o.x = exp_fast(a.lower_bound * sigmoid_fast(rate * (g.x + dt.x)));
      o.y = exp_fast(a.lower_bound * sigmoid_fast(rate * (g.y + dt.y)));
    }
    *reinterpret_cast<float2*>(y + part * kDim + 2 * pair) = o;
    const float b = sigmoid_fast(beta);
    if (t + 1 < e) {                                     // the next token's inputs, behind this one's arithmetic
      raw = __ldg(in + (t + 1) * pitch);
      beta = __bfloat162float(a.beta[(int64_t)(t + 1) * a.ldb + h]);
    }
    __syncthreads();
    const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(y + 4 * lane);
    const ulonglong2 k = *reinterpret_cast<const ulonglong2*>(y + kDim + 4 * lane);
    const ulonglong2 dec = *reinterpret_cast<const ulonglong2*>(y + 3 * kDim + 4 * lane);
    float nq = sum2(fma2(q.y, q.y, mul2(q.x, q.x))), nk = sum2(fma2(k.y, k.y, mul2(k.x, k.x)));
    float nd = sum2(fma2(q.y, k.y, mul2(q.x, k.x)));
#pragma unroll
    for (int o2 = 16; o2 > 0; o2 >>= 1) {
      nq += __shfl_xor_sync(0xffffffffu, nq, o2);
      nk += __shfl_xor_sync(0xffffffffu, nk, o2);
      nd += __shfl_xor_sync(0xffffffffu, nd, o2);
    }
    const float rq = a.scale * rsqrtf(nq + 1e-6f), rk = rsqrtf(nk + 1e-6f);
    float d[2 * kRowsW];                                 // of row i: S k at i, S q at 16 + i (k, q not yet normalised)
#pragma unroll
    for (int i = 0; i < kRowsW; ++i) {
      ulonglong2& m = st[i];
      m.x = mul2(m.x, dec.x);
      m.y = mul2(m.y, dec.y);
      d[i] = sum2(fma2(m.y, k.y, mul2(m.x, k.x)));
      d[kRowsW + i] = sum2(fma2(m.y, q.y, mul2(m.x, q.x)));
    }
    const float tot = warp_sum_transposed(d, lane);
    const float sqv = __shfl_xor_sync(0xffffffffu, tot, kRowsW);       // lanes 0-15: S q of their row
    const int row = kRowsW * warp + (lane & 15);
    const float u = b * (y[2 * kDim + row] - tot * rk);                // lanes 0-15: u of their row
    if (lane < kRowsW) a.out[(int64_t)t * a.ldo + h * kDim + row] = __float2bfloat16(sqv * rq + u * (nd * rq * rk));
    const float ur = u * rk;
#pragma unroll
    for (int i = 0; i < kRowsW; ++i) {
      const float ui = __shfl_sync(0xffffffffu, ur, i);
      const uint64_t u2 = f2pack(ui, ui);
      st[i].x = fma2(u2, k.x, st[i].x);
      st[i].y = fma2(u2, k.y, st[i].y);
    }
  }
#pragma unroll
  for (int i = 0; i < kRowsW; ++i) store_stream(S + i * kDim, st[i]);
  if (conv) {                                          // this head's channels of the block: no other CTA touches them
    *reinterpret_cast<uint32_t*>(cs) = raw0;
    *reinterpret_cast<uint32_t*>(cs + 3 * a.P) = raw1;
    *reinterpret_cast<uint32_t*>(cs + 6 * a.P) = raw2;
  }
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace

int launch_kda_decode(const KdaArgs& a, cudaStream_t stream) {
  // empty tensors (no rows, no sequences) have no address
  if ((a.T > 0 && (a.x == nullptr || a.g == nullptr || a.beta == nullptr || a.out == nullptr)) ||
      (a.R > 0 && a.seqs == nullptr) || a.a_log == nullptr || a.dt_bias == nullptr || a.conv_w == nullptr ||
      a.conv_state == nullptr || a.rec_state == nullptr || a.T < 0 || a.T > 0x7fffffff || (a.cs_stride % 2) ||
      (a.rs_stride % 4) || a.cs_stride < 9 * (int64_t)a.P || a.rs_stride < (int64_t)a.H * kDim * kDim ||
      !aligned(a.x, 4) || !aligned(a.g, 4) || !aligned(a.conv_w, 16) || !aligned(a.dt_bias, 8) ||
      !aligned(a.conv_state, 4) || !aligned(a.rec_state, 16) || !aligned(a.seqs, 16) || !aligned(a.beta, 2) ||
      !aligned(a.out, 2))
    return kErrArgs;
  // one row has no pitch: what the caller's tensors state there is not used
  if (a.T > 1 && ((a.ldx % 2) || (a.ldg % 2) || a.ldx < 3 * (int64_t)a.P || a.ldg < a.P || a.ldb < a.H || a.ldo < a.P))
    return kErrArgs;
  if (a.R == 0) return kOk;
  if ((int64_t)a.R * a.H > 0x7fffffff) return kErrArgs;
  kda_decode_kernel<<<(unsigned)(a.R * a.H), kDecThreads, 0, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
}

}  // namespace ssb
