// KDA over a tree of drafted tokens for sm_100a: every node of a request's tree continues its parent's state (a root's the
// request's state block), all nodes in one launch, the block left as it is.
//
// Per head, with the conv, norms and gates of kda_decode.cu along each node's path (the taps before a root come from the
// block's conv rows): S_i = S_parent diag(a_i) + u_i k_i^T, u_i = b_i (v_i - S_parent diag(a_i) k_i), o_i = D^-1/2 S_i q_i.
// Written out along the path, with A_i the product of the decays on it and A_ij that of the decays below j,
//   u_i = b_i (w_i - sum_{j above i} u_j M_ij),   w_i = v_i - S (A_i k_i),   M_ij = (A_ij k_j) . k_i
//   o_i = S (A_i q_i) + sum_{j on the path} u_j N_ij,                        N_ij = (A_ij k_j) . q_i   (q with D^-1/2)
// and, since the u are linear in the w with scalars of the path alone, o_i = S (A_i q_i) + sum_{j on the path} P_ij w_j with
// P_i (1 + b M) = N_i b: a substitution up each node's path, on scalars. So the state S [value, key] is read once, whatever
// the nodes, no node's own state is formed, and nothing but the scalars goes node after node. The decays multiply up the
// path (each is at most 1; quotients of cumulated ones would overflow).
//
// One CTA a (request, head), 256 threads, two CTAs an SM:
//   conv and gates: a thread a pair of channels of q or k for every second node, of g for every fourth;
//   pairs: a warp a node and those above it, 4 at a time, 4 channels a lane;
//   products: [S (A k) | S (A q)] on the tensor cores, M = 128 value rows, N = 2 nodes, K = 128 keys, tcgen05 kind::f16: S in
//       TMEM and the vectors in shared memory, both as two bf16 parts, three of the four products (what is left out is below
//       2^-16 of a product; the output has 8 bits). S comes straight from global memory, a value row a lane;
//   outputs: w by value rows, as the products lie in TMEM, back there as bf16 parts, and W^T P^T onto S (A q) by the tensor
//       cores, K = nodes.
// The exponentials are the short ones (error about 2^-20 here): nothing computed here is kept but the bf16 outputs.
#include "common.cuh"
#include "kda_math.cuh"
#include "ops.h"

namespace ssb {
namespace {

constexpr int kDim = 128;
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxNodes = 64;
constexpr float kLog2e = 1.4426950408889634f;
// TMEM: S as 64 columns of high and 64 of low parts, later W^T in the same places; the products
constexpr uint32_t kColS = 0, kColLo = 64, kColD = 128, kCols = 256;

template <int N>
struct TreeSmem {
  union {
    struct {
      float k[N][kDim];                    // keys, normalised
      float q[N][kDim];                    // queries, normalised and scaled
    };
    uint8_t op[2][2][2 * N][128];          // A k, A q: high and low parts, 2 chunks of 64 keys [rows x 128 B], swizzled
  };
  union {
    uint32_t in[2][N][kDim / 2];           // inputs of q and k
    float dec[N][kDim];                    // then the decays
    struct {                               // once A k and A q are made
      uint8_t p[2][N][128];                // P: high and low parts [nodes x nodes], swizzled
      uint32_t v[N][kDim / 2];             // inputs of the values
    };
  };
  float pn[N * (N + 1) / 2];               // N_ij: of node i from off[i] on, by distance. Before, bytes: node i's path, in the
                                           // last bytes of its place (overwritten behind their use)
  float pm[N * (N - 1) / 2];               // M_ij: of node i from off[i] - i on, by distance - 1
  float beta[N];
  uint32_t tap[N];                         // bytes: the rows before the node's in the conv, kMaxNodes + j: the j-th newest kept row
  uint16_t off[N + 2];
  int8_t parent[N];
  uint64_t bar[2];
  uint32_t tmem;
  int32_t abort;
};
static_assert(sizeof(uint8_t[2][64][128]) + sizeof(uint32_t[64][64]) == sizeof(float[64][kDim]), "one place");

SSB_DEVICE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
SSB_DEVICE float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
SSB_DEVICE float sigmoid_short(float x) { return rcp(1.0f + ex2(-kLog2e * x)); }
SSB_DEVICE float silu_short(float x) { return x * rcp(1.0f + ex2(-kLog2e * x)); }
SSB_DEVICE float sum2(uint64_t v) {
  float x, y;
  f2unpack(v, x, y);
  return x + y;
}
// Two values as bf16 pairs: the high parts, and what they leave.
SSB_DEVICE void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  const __nv_bfloat162 l = __floats2bfloat162_rn(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xFFFF0000u));
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
SSB_DEVICE void ld8(const float* p, float* v) {              // 32 bytes
  asm volatile("ld.global.nc.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "l"(p));
}
SSB_DEVICE void tmem_ld_x8(uint32_t taddr, float (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "r"(taddr));
}
SSB_DEVICE void tmem_st_x4(uint32_t taddr, const uint32_t (&v)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3])
               : "memory");
}
// D[tmem] (+)= A B with bf16 A in TMEM (a row a lane, 2 values a column) and B in shared memory.
SSB_DEVICE void mma_f16_ta(uint32_t d, uint32_t a, uint64_t bd, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(bd), "r"(idesc), "r"(acc)
      : "memory");
}

SSB_DEVICE void cp_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
SSB_DEVICE void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Four conv taps (0: the oldest) of a node: x[3] its own row's value, the others by `taps`, of which those behind a root are
// the block's kept rows (held[0] the newest).
template <class T, class Row>
SSB_DEVICE void load_taps(T (&x)[4], int i, uint32_t taps, const T (&held)[3], Row row) {
  x[3] = row(i);
#pragma unroll
  for (int e = 0; e < 3; ++e) x[2 - e] = row(static_cast<int>((taps >> (8 * e)) & (kMaxNodes - 1)));
  if (taps & 0x404040u) {
#pragma unroll
    for (int e = 0; e < 3; ++e) {
      const uint32_t t = (taps >> (8 * e)) & 0xFF;
      if (t >= kMaxNodes) x[2 - e] = t == kMaxNodes ? held[0] : t == kMaxNodes + 1 ? held[1] : held[2];
    }
  }
}

template <int N>
__global__ void __launch_bounds__(kThreads, 2) kda_tree_kernel(const __grid_constant__ KdaArgs a) {
  extern __shared__ __align__(1024) uint8_t raw_smem[];
  TreeSmem<N>& sm = *reinterpret_cast<TreeSmem<N>*>(raw_smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r = blockIdx.x / a.H, h = blockIdx.x - r * a.H;
  const int4 sq = __ldg(reinterpret_cast<const int4*>(a.seqs) + r);   // {first row, end row, state block, has state}
  const int s = sq.x, n = sq.y - sq.x;
  if (s < 0 || sq.y < s || sq.y > a.T || n > N || sq.z < 0 || (smem_u32(raw_smem) & 1023)) {
    if (tid == 0 && h == 0) raise_status(a.status, kErrArgs);
    return;
  }
  if (n == 0) return;
  const bool init = sq.w != 0;
  if (warp == 0) {
    tmem_alloc(smem_u32(&sm.tmem), kCols);
    tmem_relinquish();
    if (lane == 0) {
      mbar_init(smem_u32(&sm.bar[0]), 1);
      mbar_init(smem_u32(&sm.bar[1]), 1);
      fence_barrier_init();
    }
  }

  // ---- the state's loads: a value row a lane, half of its keys a thread
  const int quarter = warp & 3, half = warp >> 2, v = 32 * quarter + lane;
  float st[64];
  {
    const float* S = a.rec_state + (int64_t)sq.z * a.rs_stride + ((int64_t)h * kDim + v) * kDim + 64 * half;
    const bool wide = (reinterpret_cast<uintptr_t>(S) & 31) == 0;
#pragma unroll
    for (int c = 0; c < 64; c += 8) {
      if (init && wide) {
        ld8(S + c, st + c);
      } else if (init) {
        const float4 x = __ldg(reinterpret_cast<const float4*>(S + c)), y = __ldg(reinterpret_cast<const float4*>(S + c + 4));
        st[c] = x.x, st[c + 1] = x.y, st[c + 2] = x.z, st[c + 3] = x.w;
        st[c + 4] = y.x, st[c + 5] = y.y, st[c + 6] = y.z, st[c + 7] = y.w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) st[c + j] = 0.0f;
      }
    }
  }
  // ---- the inputs of q and k into shared memory (threads 0-191); the tree (threads 192-255)
  const int pair = tid & 63, part = tid >> 6;
  bool bad = false;
  if (part < 3) {
    const uint32_t* in = reinterpret_cast<const uint32_t*>(a.x + h * kDim + 2 * pair) + s * (a.ldx / 2);
#pragma unroll 4
    for (int i = part; i < 2 * n; i += 3)
      cp_async4(&sm.in[i & 1][i >> 1][pair], in + (i >> 1) * (a.ldx / 2) + (i & 1) * (a.P / 2));
  } else {
    // thread 192 + i: node i, its path walked twice: its length, then its nodes
    const int i = tid - 192;
    const bool node = i < n;
    int p = -1;
    if (node) {
      p = a.parents[s + i];
      bad = p < -1 || p >= i;
      sm.beta[i] = sigmoid_short(__bfloat162float(a.beta[(int64_t)(s + i) * a.ldb + h]));
      sm.parent[i] = static_cast<int8_t>(p);
      // the values' rows are wanted late: on their way to L2
      const __nv_bfloat16* x = a.x + (s + i) * a.ldx + 2 * (int64_t)a.P + h * kDim;
      asm volatile("prefetch.global.L2 [%0];" ::"l"(x));
      asm volatile("prefetch.global.L2 [%0];" ::"l"(x + kDim / 2));
    }
    bad = named_bar_or(1, 64, bad);
    int len = 0;
    uint32_t taps = 0;
    if (node && !bad) {
      int at = p;
      for (int j = 0, kept = kMaxNodes; j < 3; ++j) {
        taps |= static_cast<uint32_t>(at >= 0 ? at : kept++) << (8 * j);
        if (at >= 0) at = sm.parent[at], ++len;
      }
      for (; at >= 0; at = sm.parent[at]) ++len;
      sm.tap[i] = taps;
      ++len;
    }
    int end = len;                                           // the sum of the lengths: a warp each, the second behind the first
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= o) end += x;
    }
    if (i == 31) sm.abort = end;
    named_bar(1, 64);
    if (i >= 32) end += sm.abort;
    if (node && !bad) {
      sm.off[i] = static_cast<uint16_t>(end - len);
      if (i == n - 1) sm.off[n] = static_cast<uint16_t>(end);
      uint8_t* path = reinterpret_cast<uint8_t*>(sm.pn + (end - len)) + 3 * len;
      int at = i;
      for (int d = 0; d < len; ++d) {
        path[d] = static_cast<uint8_t>(at);
        at = sm.parent[at];
      }
    }
  }
  // the gates' inputs: a pair of channels of every fourth node a thread
  uint32_t gin[N / 4];
  {
    const uint32_t* in = reinterpret_cast<const uint32_t*>(a.g + h * kDim + 2 * pair) + s * (a.ldg / 2);
#pragma unroll
    for (int t = 0; t < N / 4; ++t) gin[t] = __ldg(in + min(part + 4 * t, n - 1) * (a.ldg / 2));
  }
  cp_async_wait();
  tc_fence_before();
  if (__syncthreads_or(bad)) {
    if (tid == 0 && h == 0) raise_status(a.status, kErrArgs);
    if (warp == 0) tmem_dealloc(sm.tmem, kCols);
    return;
  }
  if (tid == 0) sm.abort = 0;                                // its place was in use
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  // ---- the state's parts to TMEM
  {
    const uint32_t at = tmem + (static_cast<uint32_t>(32 * quarter) << 16) + kColS + 32 * half;
    float hi[32], lo[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      uint32_t x, y;
      split2(st[2 * j], st[2 * j + 1], x, y);
      hi[j] = __uint_as_float(x), lo[j] = __uint_as_float(y);
    }
    tmem_st_32x32b_x32(at, hi);
    tmem_st_32x32b_x32(at + kColLo, lo);
    tmem_st_wait();
  }

  // ---- the conv of q and k: 4 nodes at a time, every second one
  const __nv_bfloat16* cs = a.conv_state + (int64_t)sq.z * a.cs_stride + h * kDim;              // of q; k, v: + P, + 2 P
  {
    const int which = part & 1;                              // q, k
    uint32_t held[3] = {0, 0, 0};
    if (init)
      for (int j = 0; j < 3; ++j)
        held[j] = *reinterpret_cast<const uint32_t*>(cs + ((int64_t)(2 - j) * 3 + which) * a.P + 2 * pair);
    const uint4 wv = __ldg(reinterpret_cast<const uint4*>(a.conv_w + ((int64_t)which * a.P + h * kDim + 2 * pair) * 4));
    const float2 a0 = bf2(wv.x), a1 = bf2(wv.y), b0 = bf2(wv.z), b1 = bf2(wv.w);               // 2 channels x 4 taps
    const uint64_t p0 = f2pack(a0.x, b0.x), p1 = f2pack(a0.y, b0.y), p2 = f2pack(a1.x, b1.x), p3 = f2pack(a1.y, b1.y);
    const auto row = [&](int j) { return sm.in[which][j][pair]; };
    float* to = (which ? &sm.k[0][0] : &sm.q[0][0]) + 2 * pair;
#pragma unroll 1
    for (int i = half; i < n; i += 8) {
      uint32_t x[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int m = min(i + 2 * j, n - 1);
        load_taps(x[j], m, sm.tap[m], held, row);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint64_t o = fma2(p3, bf2_f2(x[j][3]), fma2(p2, bf2_f2(x[j][2]), fma2(p1, bf2_f2(x[j][1]), mul2(p0, bf2_f2(x[j][0])))));
        float2 y;
        f2unpack(o, y.x, y.y);
        y.x = silu_short(y.x), y.y = silu_short(y.y);
        if (i + 2 * j < n) *reinterpret_cast<float2*>(to + (i + 2 * j) * kDim) = y;
      }
    }
  }
  __syncthreads();
  // ---- the decays, in the place of the inputs
  {
    const float2 dt = __ldg(reinterpret_cast<const float2*>(a.dt_bias + h * kDim) + pair);
    const float rate = -kLog2e * exp_fast(__ldg(a.a_log + h)), lb = a.lower_bound * kLog2e;
#pragma unroll
    for (int t = 0; t < N / 4; ++t) {
      const float2 x = bf2(gin[t]);
      float2 o;
      o.x = ex2(lb * rcp(1.0f + ex2(rate * (x.x + dt.x))));
      o.y = ex2(lb * rcp(1.0f + ex2(rate * (x.y + dt.y))));
      if (part + 4 * t < n) *reinterpret_cast<float2*>(&sm.dec[part + 4 * t][2 * pair]) = o;
    }
  }

  // ---- norms: a warp a node, 4 channels a lane
#pragma unroll 1
  for (int i = warp; i < n; i += kWarps) {
    float4* kp = reinterpret_cast<float4*>(&sm.k[i][4 * lane]);
    float4* qp = reinterpret_cast<float4*>(&sm.q[i][4 * lane]);
    float4 q = *qp, k = *kp;
    const float nk = k.x * k.x + k.y * k.y + k.z * k.z + k.w * k.w, nq = q.x * q.x + q.y * q.y + q.z * q.z + q.w * q.w;
    float t = (lane < 16 ? nk : nq) + __shfl_xor_sync(0xffffffffu, lane < 16 ? nq : nk, 16);   // lanes 0-15: k's, 16-31: q's
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    t = rsqrtf(t + 1e-6f);
    const float rk = __shfl_sync(0xffffffffu, t, 0), rq = a.scale * __shfl_sync(0xffffffffu, t, 16);
    *kp = make_float4(k.x * rk, k.y * rk, k.z * rk, k.w * rk);
    *qp = make_float4(q.x * rq, q.y * rq, q.z * rq, q.w * rq);
  }
  __syncthreads();
  // ---- the pairs of a node and those above it, 4 at a time
#pragma unroll 1
  for (int i = warp; i < n; i += kWarps) {
    const ulonglong2 k = *reinterpret_cast<ulonglong2*>(&sm.k[i][4 * lane]), q = *reinterpret_cast<ulonglong2*>(&sm.q[i][4 * lane]);
    const int at = sm.off[i], len = sm.off[i + 1] - at;
    const uint8_t* path = reinterpret_cast<const uint8_t*>(sm.pn + at) + 3 * len;
    ulonglong2 f = make_ulonglong2(f2pack(1.0f, 1.0f), f2pack(1.0f, 1.0f));                    // the decays below
#pragma unroll 1
    for (int d = 0; d < len; d += 4) {
      int js[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) js[e] = path[min(d + e, len - 1)];
      float t[8];                                              // M of 4 pairs, N of 4 pairs
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const ulonglong2 kj = *reinterpret_cast<ulonglong2*>(&sm.k[js[e]][4 * lane]);
        const ulonglong2 dj = *reinterpret_cast<ulonglong2*>(&sm.dec[js[e]][4 * lane]);
        const uint64_t x = mul2(f.x, kj.x), y = mul2(f.y, kj.y);
        t[e] = sum2(fma2(x, k.x, mul2(y, k.y)));
        t[4 + e] = sum2(fma2(x, q.x, mul2(y, q.y)));
        f.x = mul2(f.x, dj.x), f.y = mul2(f.y, dj.y);
      }
#pragma unroll
      for (int o = 16, m = 4; o >= 4; o >>= 1, m >>= 1) {      // lanes 4 x .. + 3 receive value x
        const bool up = lane & o;
#pragma unroll
        for (int e = 0; e < m; ++e) {
          const float keep = up ? t[e + m] : t[e], send = up ? t[e] : t[e + m];
          t[e] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
      }
      t[0] += __shfl_xor_sync(0xffffffffu, t[0], 2);
      t[0] += __shfl_xor_sync(0xffffffffu, t[0], 1);
      __syncwarp();                                            // the path's bytes are read
      const int e = d + ((lane >> 2) & 3);
      if ((lane & 3) == 0 && e < len) {
        if (lane >= 16) sm.pn[at + e] = t[0];
        else if (e > 0) sm.pm[at - i + e - 1] = t[0];
      }
    }
  }
  // ---- A k and A q as the products' second operand, in the place of k and q; all the warp's paths walked at once
  {
    uint32_t hi[N / kWarps][4], lo[N / kWarps][4];
    {
      ulonglong2 f[N / kWarps];
      int at[N / kWarps];
      bool more = true;
#pragma unroll
      for (int t = 0; t < N / kWarps; ++t) {
        f[t] = make_ulonglong2(f2pack(1.0f, 1.0f), f2pack(1.0f, 1.0f));
        at[t] = warp + kWarps * t < n ? warp + kWarps * t : -1;
      }
#pragma unroll 1
      while (more) {
        more = false;
#pragma unroll
        for (int t = 0; t < N / kWarps; ++t) {
          if (at[t] < 0) continue;
          const ulonglong2 d = *reinterpret_cast<ulonglong2*>(&sm.dec[at[t]][4 * lane]);
          f[t].x = mul2(f[t].x, d.x), f[t].y = mul2(f[t].y, d.y);
          at[t] = sm.parent[at[t]];
          more = true;
        }
      }
#pragma unroll
      for (int t = 0; t < N / kWarps; ++t) {
        const int i = min(warp + kWarps * t, n - 1);
        const ulonglong2 k = *reinterpret_cast<ulonglong2*>(&sm.k[i][4 * lane]), q = *reinterpret_cast<ulonglong2*>(&sm.q[i][4 * lane]);
        const uint64_t y[4] = {mul2(f[t].x, k.x), mul2(f[t].y, k.y), mul2(f[t].x, q.x), mul2(f[t].y, q.y)};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float y0, y1;
          f2unpack(y[e], y0, y1);
          split2(y0, y1, hi[t][e], lo[t][e]);
        }
      }
    }
    __syncthreads();
    const int chunk = lane >> 4, granule = (lane & 15) >> 1, within = (lane & 1) * 8;
#pragma unroll
    for (int t = 0; t < N / kWarps; ++t) {
      const int i = warp + kWarps * t;
      if (i >= n) continue;
      const int at = ((granule ^ (i & 7)) << 4) + within;      // rows i and N + i swizzle alike
      *reinterpret_cast<uint2*>(&sm.op[0][chunk][i][at]) = make_uint2(hi[t][0], hi[t][1]);
      *reinterpret_cast<uint2*>(&sm.op[1][chunk][i][at]) = make_uint2(lo[t][0], lo[t][1]);
      *reinterpret_cast<uint2*>(&sm.op[0][chunk][N + i][at]) = make_uint2(hi[t][2], hi[t][3]);
      *reinterpret_cast<uint2*>(&sm.op[1][chunk][N + i][at]) = make_uint2(lo[t][2], lo[t][3]);
    }
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  const uint32_t bar = smem_u32(&sm.bar[0]);
  if (tid == 0) {
    tc_fence_after();
    constexpr uint32_t idesc = idesc_bf16(128, 2 * N);
    uint32_t acc = 0;
#pragma unroll 1
    for (int t = 0; t < 3; ++t) {                              // high x high, high x low, low x high
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint64_t bd = smem_desc(smem_u32(&sm.op[t == 1][c][0][0]), 0, 1024, 2);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          mma_f16_ta(tmem + kColD, tmem + kColS + (t == 2 ? kColLo : 0) + 32 * c + 8 * ks, bd + 2 * ks, idesc, acc);
          acc = 1;
        }
      }
    }
    tc_commit(bar);
  }
  // ---- meanwhile the values' inputs, and the scalars (threads 192 + i: node i's row of P)
  {
    const uint32_t* in = reinterpret_cast<const uint32_t*>(a.x + 2 * (int64_t)a.P + h * kDim + 2 * pair);
    const int64_t pitch = a.ldx / 2;
#pragma unroll 4
    for (int i = part; i < n; i += 4) cp_async4(&sm.v[i][pair], in + (s + i) * pitch);
  }
  if (part == 3 && tid - 192 < N) {
    const int i = tid - 192;
#pragma unroll
    for (int c = 0; c < 128; c += 16)
      *reinterpret_cast<uint4*>(&sm.p[0][i][c]) = *reinterpret_cast<uint4*>(&sm.p[1][i][c]) = make_uint4(0, 0, 0, 0);
    const int at = i < n ? sm.off[i] : 0, len = i < n ? sm.off[i + 1] - at : 0;
    float* pn = sm.pn + at;
    int m = i;
#pragma unroll 1
    for (int c = 0; c < len; ++c) {
      const float y = pn[c] * sm.beta[m];
      const float* pm = sm.pm + (sm.off[m] - m);
#pragma unroll 4
      for (int e = c + 1; e < len; ++e) pn[e] = fmaf(-y, pm[e - c - 1], pn[e]);
      const __nv_bfloat16 y_hi = __float2bfloat16(y);
      const int to = (((m >> 3) ^ (i & 7)) << 4) + 2 * (m & 7);
      *reinterpret_cast<__nv_bfloat16*>(&sm.p[0][i][to]) = y_hi;
      *reinterpret_cast<__nv_bfloat16*>(&sm.p[1][i][to]) = __float2bfloat16(y - __bfloat162float(y_hi));
      m = sm.parent[m];
    }
  }
  cp_async_wait();
  bool ok = mbar_wait(bar, 0, &sm.abort, a.status);
  fence_proxy_async_smem();
  ok = !__syncthreads_or(!ok);
  tc_fence_after();
  const uint32_t rows = static_cast<uint32_t>(32 * quarter) << 16;
  constexpr int kHalf = N / 2;                                 // a half of the nodes a thread of its value row
  // ---- w = v - S (A k), as bf16 parts in the place of S; zeros past the nodes, whose columns of P are zeros too
  if (ok) {
    float held[3] = {0.0f, 0.0f, 0.0f};
    if (init)
      for (int j = 0; j < 3; ++j) held[j] = __bfloat162float(cs[((int64_t)(2 - j) * 3 + 2) * a.P + v]);
    const uint2 wv = __ldg(reinterpret_cast<const uint2*>(a.conv_w + (2 * (int64_t)a.P + h * kDim + v) * 4));
    const float2 p0 = bf2(wv.x), p1 = bf2(wv.y);
    const auto row = [&](int j) { return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(sm.v[j])[v]); };
#pragma unroll 1
    for (int c = kHalf * half; c < kHalf * (half + 1); c += 8) {
      float y[8], w[8];
      tmem_ld_x8(tmem + rows + kColD + c, y);
      float x[8][4];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = min(c + j, n - 1);
        load_taps(x[j], i, sm.tap[i], held, row);
      }
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float t = silu_short(fmaf(p1.y, x[j][3], fmaf(p1.x, x[j][2], fmaf(p0.y, x[j][1], p0.x * x[j][0]))));
        w[j] = c + j < n ? t - y[j] : 0.0f;
      }
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) split2(w[2 * j], w[2 * j + 1], hi[j], lo[j]);
      tmem_st_x4(tmem + rows + kColS + c / 2, hi);
      tmem_st_x4(tmem + rows + kColS + kColLo + c / 2, lo);
    }
    tmem_st_wait();
  }
  tc_fence_before();
  __syncthreads();
  const uint32_t bar2 = smem_u32(&sm.bar[1]);
  if (ok && tid == 0) {
    tc_fence_after();
    constexpr uint32_t idesc = idesc_bf16(128, N);
#pragma unroll 1
    for (int t = 0; t < 3; ++t) {                              // onto S (A q)
      const uint64_t bd = smem_desc(smem_u32(&sm.p[t == 1][0][0]), 0, 1024, 2);
#pragma unroll
      for (int ks = 0; ks < N / 16; ++ks)
        mma_f16_ta(tmem + kColD + N, tmem + kColS + (t == 2 ? kColLo : 0) + 8 * ks, bd + 2 * ks, idesc, 1u);
    }
    tc_commit(bar2);
  }
  if (ok) ok = mbar_wait(bar2, 0, &sm.abort, a.status);
  if (!__syncthreads_or(!ok)) {
    tc_fence_after();
    __nv_bfloat16* out = a.out + (int64_t)s * a.ldo + h * kDim + v;
#pragma unroll 1
    for (int c = kHalf * half; c < min(kHalf * (half + 1), n); c += 8) {
      float z[8];
      tmem_ld_x8(tmem + rows + kColD + N + c, z);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < n) out[(c + j) * a.ldo] = __float2bfloat16(z[j]);
    }
  } else {
    // products may still be on their way
    const unsigned long long t0 = globaltimer();
    while (!(mbar_try_wait(bar, 0) && mbar_try_wait(bar2, 0)) && globaltimer() - t0 <= 2 * kWaitNs) {}
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, kCols);
  }
}

// TMEM holds two CTAs' columns: shared memory of which three do not fit an SM keeps a third from waiting for them.
template <int N>
constexpr int smem_bytes() {
  static_assert(sizeof(TreeSmem<N>) <= 115712, "two CTAs an SM");
  return sizeof(TreeSmem<N>) > 80 * 1024 ? sizeof(TreeSmem<N>) : 80 * 1024;
}

template <int N>
int launch_nodes(const KdaArgs& a, cudaStream_t stream) {
  static OncePerDevice attr;
  int device = 0;
  const auto set = [] {
    return cudaFuncSetAttribute(kda_tree_kernel<N>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<N>()) ==
           cudaSuccess;
  };
  if (cudaGetDevice(&device) != cudaSuccess || !attr.done(device, set)) return kErrCuda;
  kda_tree_kernel<N><<<(unsigned)(a.R * a.H), kThreads, smem_bytes<N>(), stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
}

}  // namespace

int launch_kda_tree(const KdaArgs& a, cudaStream_t stream) {
  if (!kda_step_args(a) || (a.T > 0 && (a.out == nullptr || a.parents == nullptr)) || !kda_aligned(a.out, 2) ||
      !kda_aligned(a.parents, 4) || (a.T > 1 && a.ldo < a.P) || a.max_nodes < 1 || a.max_nodes > kMaxNodes)
    return kErrArgs;
  if (a.R == 0) return kOk;
  if ((int64_t)a.R * a.H > 0x7fffffff) return kErrArgs;
  if (a.max_nodes <= 16) return launch_nodes<16>(a, stream);
  if (a.max_nodes <= 32) return launch_nodes<32>(a, stream);
  return launch_nodes<64>(a, stream);
}

}  // namespace ssb
