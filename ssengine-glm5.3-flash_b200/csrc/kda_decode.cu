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
// 128 KB a head and request whatever the run's length. One CTA per (request, head), 8 warps; warp w keeps value rows
// 16 w .. 16 w + 15 in registers, a lane 4 key columns of each (one 512-byte row a warp load, 16 loads in flight a lane
// before the conv and the gates are computed, so these hide behind the reads).
#include "common.cuh"
#include "ops.h"

namespace ssb {
namespace {

constexpr int kDim = 128;
constexpr int kDecThreads = 256;
constexpr int kRowsW = 16;             // value rows a warp

SSB_DEVICE float sigmoid_exact(float z) { return 1.0f / (1.0f + expf(-z)); }
SSB_DEVICE float silu_exact(float y) { return y / (1.0f + expf(-y)); }
SSB_DEVICE float2 bf2(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }

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

__global__ void __launch_bounds__(kDecThreads, 2) kda_decode_kernel(const KdaArgs a) {
  __shared__ __align__(16) float sy[2][3][kDim];       // conv outputs q | k | v, double-buffered over tokens
  __shared__ __align__(16) float sa[2][kDim];          // the key channels' decays
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
  float4 st[kRowsW];
#pragma unroll
  for (int i = 0; i < kRowsW; ++i)
    st[i] = init ? *reinterpret_cast<const float4*>(S + i * kDim) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);

  // threads 0-191: a pair of conv channels each (q 0-63, k 64-127, v 128-191); threads 192-255: a pair of gates
  const bool conv = tid < 192;
  const int pair = tid & 63;
  const int64_t col = (int64_t)(tid >> 6) * a.P + h * kDim + 2 * pair;
  float2 w0 = {}, w1 = {}, w2 = {}, w3 = {}, x0 = {}, x1 = {}, x2 = {};
  uint32_t raw0 = 0, raw1 = 0, raw2 = 0;
  __nv_bfloat16* cs = a.conv_state + (int64_t)sq.z * a.cs_stride + col;
  float rate = 0.0f;
  float2 dt = {};
  if (conv) {
    const uint4 wv = __ldg(reinterpret_cast<const uint4*>(a.conv_w + col * 4));   // 2 channels x 4 taps
    const float2 p0 = bf2(wv.x), p1 = bf2(wv.y), p2 = bf2(wv.z), p3 = bf2(wv.w);
    w0 = make_float2(p0.x, p2.x);
    w1 = make_float2(p0.y, p2.y);
    w2 = make_float2(p1.x, p3.x);
    w3 = make_float2(p1.y, p3.y);
    if (init) {
      raw0 = *reinterpret_cast<const uint32_t*>(cs);
      raw1 = *reinterpret_cast<const uint32_t*>(cs + 3 * a.P);
      raw2 = *reinterpret_cast<const uint32_t*>(cs + 6 * a.P);
    }
  } else {
    rate = expf(__ldg(a.a_log + h));
    dt = __ldg(reinterpret_cast<const float2*>(a.dt_bias + h * kDim) + pair);
  }

  for (int t = s; t < e; ++t) {
    const int buf = (t - s) & 1;
    if (conv) {
      const uint32_t raw = __ldg(reinterpret_cast<const uint32_t*>(a.x + (int64_t)t * a.ldx + col));
      x0 = bf2(raw0), x1 = bf2(raw1), x2 = bf2(raw2);
      const float2 x3 = bf2(raw);
      float2 y;
      y.x = fmaf(w3.x, x3.x, fmaf(w2.x, x2.x, fmaf(w1.x, x1.x, w0.x * x0.x)));
      y.y = fmaf(w3.y, x3.y, fmaf(w2.y, x2.y, fmaf(w1.y, x1.y, w0.y * x0.y)));
      *reinterpret_cast<float2*>(&sy[buf][tid >> 6][2 * pair]) = make_float2(silu_exact(y.x), silu_exact(y.y));
      raw0 = raw1, raw1 = raw2, raw2 = raw;
    } else {
      const float2 g = bf2(__ldg(reinterpret_cast<const uint32_t*>(a.g + (int64_t)t * a.ldg + h * kDim) + pair));
      *reinterpret_cast<float2*>(&sa[buf][2 * pair]) =
          make_float2(expf(a.lower_bound * sigmoid_exact(rate * (g.x + dt.x))),
                      expf(a.lower_bound * sigmoid_exact(rate * (g.y + dt.y))));
    }
    const float b = sigmoid_exact(__bfloat162float(a.beta[(int64_t)t * a.ldb + h]));
    __syncthreads();
    float4 q = *reinterpret_cast<const float4*>(&sy[buf][0][4 * lane]);
    float4 k = *reinterpret_cast<const float4*>(&sy[buf][1][4 * lane]);
    const float4 dec = *reinterpret_cast<const float4*>(&sa[buf][4 * lane]);
    const float v = sy[buf][2][kRowsW * warp + (lane & 15)];
    float qq = q.x * q.x + q.y * q.y + q.z * q.z + q.w * q.w;
    float kk = k.x * k.x + k.y * k.y + k.z * k.z + k.w * k.w;
    float qk = q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      qq += __shfl_xor_sync(0xffffffffu, qq, o);
      kk += __shfl_xor_sync(0xffffffffu, kk, o);
      qk += __shfl_xor_sync(0xffffffffu, qk, o);
    }
    const float rq = a.scale / sqrtf(qq + 1e-6f), rk = 1.0f / sqrtf(kk + 1e-6f);
    q = make_float4(q.x * rq, q.y * rq, q.z * rq, q.w * rq);
    k = make_float4(k.x * rk, k.y * rk, k.z * rk, k.w * rk);
    float d[32];                                       // S k of row i at i, scale S q at 16 + i
#pragma unroll
    for (int i = 0; i < kRowsW; ++i) {
      float4& m = st[i];
      m.x *= dec.x, m.y *= dec.y, m.z *= dec.z, m.w *= dec.w;
      d[i] = m.x * k.x + m.y * k.y + m.z * k.z + m.w * k.w;
      d[16 + i] = m.x * q.x + m.y * q.y + m.z * q.z + m.w * q.w;
    }
    const float tot = warp_sum_transposed(d, lane);
    const float sqv = __shfl_xor_sync(0xffffffffu, tot, 16);      // lanes 0-15: S q of their row
    const float u = b * (v - tot);                                // lanes 0-15: u of their row
    if (lane < 16)
      a.out[(int64_t)t * a.ldo + h * kDim + kRowsW * warp + lane] = __float2bfloat16(sqv + u * (qk * rq * rk));
#pragma unroll
    for (int i = 0; i < kRowsW; ++i) {
      const float ui = __shfl_sync(0xffffffffu, u, i);
      float4& m = st[i];
      m.x = fmaf(ui, k.x, m.x), m.y = fmaf(ui, k.y, m.y), m.z = fmaf(ui, k.z, m.z), m.w = fmaf(ui, k.w, m.w);
    }
  }
#pragma unroll
  for (int i = 0; i < kRowsW; ++i) *reinterpret_cast<float4*>(S + i * kDim) = st[i];
  if (conv) {                                          // this head's channels of the block: no other CTA touches them
    *reinterpret_cast<uint32_t*>(cs) = raw0;
    *reinterpret_cast<uint32_t*>(cs + 3 * a.P) = raw1;
    *reinterpret_cast<uint32_t*>(cs + 6 * a.P) = raw2;
  }
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace

int launch_kda_decode(const KdaArgs& a, cudaStream_t stream) {
  if (a.g == nullptr || a.beta == nullptr || a.a_log == nullptr || a.dt_bias == nullptr || a.conv_w == nullptr ||
      a.conv_state == nullptr || a.rec_state == nullptr || a.out == nullptr || a.x == nullptr || a.seqs == nullptr ||
      a.T < 0 || a.T > 0x7fffffff || (a.ldx % 2) || (a.ldg % 2) || a.ldx < 3 * (int64_t)a.P || a.ldg < a.P ||
      a.ldb < a.H || a.ldo < a.P || (a.cs_stride % 2) || (a.rs_stride % 4) || a.cs_stride < 9 * (int64_t)a.P ||
      a.rs_stride < (int64_t)a.H * kDim * kDim || !aligned(a.x, 4) || !aligned(a.g, 4) || !aligned(a.conv_w, 16) ||
      !aligned(a.dt_bias, 8) || !aligned(a.conv_state, 4) || !aligned(a.rec_state, 16) || !aligned(a.seqs, 16) ||
      !aligned(a.beta, 2) || !aligned(a.out, 2))
    return kErrArgs;
  if (a.R == 0) return kOk;
  if ((int64_t)a.R * a.H > 0x7fffffff) return kErrArgs;
  kda_decode_kernel<<<(unsigned)(a.R * a.H), kDecThreads, 0, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
}

}  // namespace ssb
