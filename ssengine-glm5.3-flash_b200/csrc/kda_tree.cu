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
// path: each is at most 1, so any depth is safe.
//
// One CTA a (request, head), two or four an SM:
//   conv: a warp a node, 4 channels a lane, of q or k, late of v; gates: a thread a pair of channels of every fourth (eighth)
//       node;
//   norms, pairs, A k and A q: half a warp a node (8 channels a lane), its pairs 2 at a time;
//   products: [S (A k) | S (A q)] on the tensor cores, M = 128 value rows, N = 2 nodes, K = 128 keys, tcgen05 kind::f16: S in
//       TMEM and the vectors in shared memory, both as two bf16 parts, three of the four products (what is left out is below
//       2^-16 of a product; the output has 8 bits). S comes straight from global memory;
//   outputs: w by value rows, as the products lie in TMEM, back there as bf16 parts, and W^T P^T onto S (A q) by the tensor
//       cores, K = nodes.
// The exponentials are the short ones (error about 2^-20 here): nothing computed here is kept but the bf16 outputs.
//
// Bound: not HBM (a head's state is read once, 64 KB, whatever the nodes) but the vectors' arithmetic and the pairs, which
// are on no tensor core. They could be one product in shallow trees: with C the log decays summed along a path, the decays
// between i and j are exp(C_i + c) exp(-(C_j + c)), factors that fp32 and bf16 hold while |lower_bound| times the depth stays
// below about 170 (30 levels and more at -5); deeper ones need this walk. Not built. 48 trees of 32
// to 64 nodes x 64 heads: 262 to 264 us (61 us of bytes), 53,000 warp instructions a CTA (pairs 11,000, conv 14,000, decays
// and norms 9,000, the rest tree, state, scalars and outputs), issue slots 60 % in use, the rest waits for barriers, shared
// memory and the state. 16 trees of 16 to 32 nodes 57 us (15), one tree of 24 nodes, 32 heads 13 us (latency). Each node's
// state formed from its parent's, a CTA a head and node after node, took 1,477 us for the first of these; the products on the
// tensor cores with two CTAs an SM 631; paths as lists 512; outputs as a second product 470; four CTAs an SM up to 32 nodes
// and 512 threads above 352; a node's scalars by half a warp 317; the conv by a warp a node, 4 channels a lane, 300; the
// state by lines 264. Nodes dealt to the warps by the lengths of their paths: 270, the order costs more than it evens out.
#include "common.cuh"
#include "kda_math.cuh"
#include "ops.h"

namespace ssb {
namespace {

constexpr int kDim = 128;
constexpr int kMaxNodes = 64;
constexpr float kLog2e = 1.4426950408889634f;

// How a CTA is made for trees of up to N nodes. Its phases are short and wait on one another (barriers, chains down the
// tree, tensor core and memory latencies), so other CTAs have to fill the SM: up to 32 nodes four of 256 threads, which have
// TMEM for half of the keys at a time; above, where shared memory holds two, 512 threads each.
template <int N>
struct Shape {
  static constexpr int kThreads = N > 32 ? 512 : 256, kWarps = kThreads / 32, kBlocks = N > 32 ? 2 : 4;
  static constexpr int kGroups = kThreads / 64;        // of 64 threads, one a pair of channels; the last looks after the tree
  static constexpr int kParts = kThreads / 128;        // threads of a value row, 32 keys of S each
  static constexpr int kPasses = 4 / kParts;           // over the keys
  // TMEM: S of a pass, high and low parts, later W^T in the same places; [S (A k) | S (A q)]
  static constexpr uint32_t kColS = 0, kColLo = 16 * kParts, kColD = 2 * kColLo, kCols = N > 32 ? 256 : 128;
  static constexpr int kOwn = N > 2 * kWarps ? N / (2 * kWarps) : 1;                   // nodes of half a warp
  static constexpr int kShare = N < 8 * kParts ? 8 : N / kParts;                       // nodes of a thread of a value row
};

template <int N>
struct TreeSmem {
  union {
    struct {
      float k[N][kDim];                    // keys, normalised
      float q[N][kDim];                    // queries, normalised and scaled
    };
    uint8_t op[2][2][2 * N][128];          // A k, A q: high and low parts, 2 chunks of 64 keys [rows x 128 B], swizzled
    float v[N][kDim];                      // then the values
  };
  union {
    uint32_t in[N + 3][2][kDim / 2];       // inputs of q and k, behind them the block's kept rows (N the newest)
    struct {
      union {
        float dec[N][kDim];                // the decays
        struct {                           // once A k and A q are made
          uint8_t p[2][N][128];            // P: high and low parts [nodes x nodes], swizzled
          uint32_t vin[N][kDim / 2];       // inputs of the values
        };
      };
      float pm[N * (N - 1) / 2];           // M_ij: of node i from off[i] - i on, by distance - 1
    };
  };
  float pn[N * (N + 1) / 2];               // N_ij: of node i from off[i] on, by distance. Before, bytes: node i's path, in the
                                           // last bytes of its place (overwritten behind their use)
  float beta[N];
  uint32_t tap[N];                         // bytes: the rows before the node's in the conv, N + j: the j-th newest kept row
  uint16_t off[N + 2];
  int8_t parent[N];
  uint64_t bar[3];
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
// 16 rows x 16 columns: a lane has of rows lane / 4 and + 8 the columns 2 (lane % 4), + 1 (two registers each), then those of
// the next 8 columns.
SSB_DEVICE void tmem_st_16x256(uint32_t taddr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.16x256b.x2.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
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

SSB_DEVICE void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
SSB_DEVICE void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// A pair of channels through the conv (packed weights, the oldest tap's first) and SiLU.
SSB_DEVICE float2 conv_silu(const uint64_t (&p)[4], const uint32_t (&x)[4]) {
  const uint64_t o = fma2(p[3], bf2_f2(x[3]), fma2(p[2], bf2_f2(x[2]), fma2(p[1], bf2_f2(x[1]), mul2(p[0], bf2_f2(x[0])))));
  float2 y;
  f2unpack(o, y.x, y.y);
  return make_float2(silu_short(y.x), silu_short(y.y));
}
SSB_DEVICE void conv_weights(uint64_t (&p)[4], uint4 wv) {                           // 2 channels x 4 taps
  const float2 a0 = bf2(wv.x), a1 = bf2(wv.y), b0 = bf2(wv.z), b1 = bf2(wv.w);
  p[0] = f2pack(a0.x, b0.x), p[1] = f2pack(a0.y, b0.y), p[2] = f2pack(a1.x, b1.x), p[3] = f2pack(a1.y, b1.y);
}

// Two pairs: 4 channels.
SSB_DEVICE float4 conv_silu4(const uint64_t (&p)[2][4], const uint2 (&x)[4]) {
  const uint32_t xa[4] = {x[0].x, x[1].x, x[2].x, x[3].x}, xb[4] = {x[0].y, x[1].y, x[2].y, x[3].y};
  const float2 y = conv_silu(p[0], xa), z = conv_silu(p[1], xb);
  return make_float4(y.x, y.y, z.x, z.y);
}

template <int N>
__global__ void __launch_bounds__(Shape<N>::kThreads, Shape<N>::kBlocks) kda_tree_kernel(const __grid_constant__ KdaArgs a) {
  using C = Shape<N>;
  constexpr int kWarps = C::kWarps, kGroups = C::kGroups, kParts = C::kParts, kOwn = C::kOwn, kShare = C::kShare;
  constexpr int kConvWarps = kWarps - 2;                     // the last two make the lists of the paths meanwhile
  constexpr uint32_t kColS = C::kColS, kColLo = C::kColLo, kColD = C::kColD, kCols = C::kCols;
  extern __shared__ __align__(1024) uint8_t raw_smem[];
  TreeSmem<N>& sm = *reinterpret_cast<TreeSmem<N>*>(raw_smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r = blockIdx.x / a.H, h = blockIdx.x - r * a.H;
  const int4 sq = __ldg(reinterpret_cast<const int4*>(a.seqs) + r);   // {first row, end row, state block, has state}
  const int s = sq.x, n = sq.y - sq.x;
  // the caller's bound, which is at most N, whatever N the call was dispatched to
  if (s < 0 || sq.y < s || sq.y > a.T || n > a.max_nodes || sq.z < 0 || (smem_u32(raw_smem) & 1023)) {
    if (tid == 0 && h == 0) raise_status(a.status, kErrArgs);
    return;
  }
  if (n == 0) return;
  const bool init = sq.w != 0;

  // ---- the state's loads, 32 keys of a pass a thread: 8 keys 8 (lane % 4) .. + 7 of each of the value rows lane / 4 + 8 i,
  // which are 128 bytes of a row for 4 lanes (a row a lane, as TMEM stands, is 4 times the lines a load: 297 us for 48 trees
  // of up to 64 nodes)
  const int quarter = warp & 3, fourth = warp >> 2, v = 32 * quarter + lane;
  const float* S = a.rec_state + (int64_t)sq.z * a.rs_stride + ((int64_t)h * kDim + 32 * quarter) * kDim + 32 * fourth;
  float st[32];
  const auto load_state = [&](int pass) {
    const float* from = S + 32 * kParts * pass + (lane >> 2) * kDim + 8 * (lane & 3);
    const bool wide = (reinterpret_cast<uintptr_t>(from) & 31) == 0;
#pragma unroll
    for (int c = 0; c < 32; c += 8, from += 8 * kDim) {
      if (init && wide) {
        ld8(from, st + c);
      } else if (init) {
        const float4 x = __ldg(reinterpret_cast<const float4*>(from)), y = __ldg(reinterpret_cast<const float4*>(from + 4));
        st[c] = x.x, st[c + 1] = x.y, st[c + 2] = x.z, st[c + 3] = x.w;
        st[c + 4] = y.x, st[c + 5] = y.y, st[c + 6] = y.z, st[c + 7] = y.w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) st[c + j] = 0.0f;
      }
    }
  };
  load_state(0);
  if (C::kPasses > 1 && init) asm volatile("prefetch.global.L2 [%0];" ::"l"(S + 32 * kParts + lane * kDim));
  // ---- the inputs of q and k into shared memory; the tree (the last 64 threads)
  const int pair = tid & 63, part = tid >> 6;
  const __nv_bfloat16* cs = a.conv_state + (int64_t)sq.z * a.cs_stride + h * kDim;            // of q; k, v: + P, + 2 P
  bool bad = false;
  if (part < kGroups - 1) {
    const uint32_t* q = reinterpret_cast<const uint32_t*>(a.x + h * kDim + 2 * pair) + (s + part) * (a.ldx / 2);
    const uint32_t* k = q + a.P / 2;
    const int64_t step = (kGroups - 1) * (a.ldx / 2);
    uint32_t to = smem_u32(&sm.in[part][0][pair]);
#pragma unroll 2
    for (int i = part; i < n; i += kGroups - 1, q += step, k += step, to += (kGroups - 1) * 2 * kDim * 2) {
      cp_async4(to, q);
      cp_async4(to + kDim * 2, k);
    }
    // kept row part (0: the oldest)
    if (part < 3) {
      const uint32_t* kept = reinterpret_cast<const uint32_t*>(cs + (int64_t)part * 3 * a.P + 2 * pair);
      uint32_t(&at)[2][kDim / 2] = sm.in[N + 2 - part];
      if (init) {
        cp_async4(smem_u32(&at[0][pair]), kept);
        cp_async4(smem_u32(&at[1][pair]), kept + a.P / 2);
      } else {
        at[0][pair] = at[1][pair] = 0;
      }
    }
  } else {
    // node i a thread
    const int i = tid - 64 * (kGroups - 1);
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
    if (node && !bad) {
      uint32_t taps = 0;
      for (int j = 0, kept = N, at = p; j < 3; ++j) {
        taps |= static_cast<uint32_t>(at >= 0 ? at : kept++) << (8 * j);
        if (at >= 0) at = sm.parent[at];
      }
      sm.tap[i] = taps;
    }
  }
  // the gates' inputs: a pair of channels of every kGroups-th node a thread
  uint32_t gin[N / kGroups];
  {
    const uint32_t* in = reinterpret_cast<const uint32_t*>(a.g + h * kDim + 2 * pair) + (s + part) * (a.ldg / 2);
    const int64_t step = kGroups * (a.ldg / 2);
#pragma unroll
    for (int t = 0; t < N / kGroups; ++t, in += step)
      if (part + kGroups * t < n) gin[t] = __ldg(in);
  }
  // the conv's weights of q or k and the gates' parameters
  const auto conv_weight = [&](int kind, int j) {              // channels 4 lane + 2 j, + 1
    return __ldg(reinterpret_cast<const uint4*>(a.conv_w + ((int64_t)kind * a.P + h * kDim + 4 * lane + 2 * j) * 4));
  };
  const int kind = warp & 1;                                   // q, k
  uint4 w[2];                                                  // 2 channels x 4 taps each
#pragma unroll
  for (int j = 0; j < 2; ++j) w[j] = conv_weight(kind, j);
  const float2 dt = __ldg(reinterpret_cast<const float2*>(a.dt_bias + h * kDim) + pair);
  const float a_log = __ldg(a.a_log + h);
  if (warp == 0) {                                           // with the loads on their way
    tmem_alloc(smem_u32(&sm.tmem), kCols);
    tmem_relinquish();
    if (lane == 0) {
      sm.abort = 0;
      for (int j = 0; j < 3; ++j) mbar_init(smem_u32(&sm.bar[j]), 1);
      fence_barrier_init();
    }
  }
  cp_async_wait();
  tc_fence_before();
  if (__syncthreads_or(bad)) {
    if (tid == 0 && h == 0) raise_status(a.status, kErrArgs);
    if (warp == 0) tmem_dealloc(sm.tmem, kCols);
    return;
  }
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  // ---- the state's parts to TMEM, by 16 rows: of 32 keys, in 16 columns of pairs, first the pairs 4 c and 4 c + 1 of all c,
  // then 4 c + 2 and 4 c + 3. The products' other operand has them in the same order
  const uint32_t rows = static_cast<uint32_t>(32 * quarter) << 16;
  const auto store_state = [&] {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t hi[8], lo[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {                            // pair (e & 1) + 2 (e >> 2) of row 16 half + 8 (e >> 1 & 1)
        const float* x = st + 16 * half + 8 * (e >> 1 & 1) + 2 * (e & 1) + 4 * (e >> 2);
        split2(x[0], x[1], hi[e], lo[e]);
      }
      const uint32_t to = tmem + rows + (static_cast<uint32_t>(16 * half) << 16) + kColS + 16 * fourth;
      tmem_st_16x256(to, hi);
      tmem_st_16x256(to + kColLo, lo);
    }
    tmem_st_wait();
  };
  store_state();

  // ---- the conv: of q by the even warps, of k by the odd ones, a warp a node, 4 channels a lane
  if (warp >= kConvWarps) {
    // a node's path, a node a thread, walked twice: its length, then its nodes
    const int i = tid - 32 * kConvWarps;
    int len = 0;
    for (int at = i < n ? i : -1; at >= 0; at = sm.parent[at]) ++len;
    int end = len;                                           // the sum of the lengths: a warp each, the second behind the first
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= o) end += x;
    }
    if (i == 31) sm.off[N + 1] = static_cast<uint16_t>(end);
    named_bar(1, 64);
    if (i >= 32) end += sm.off[N + 1];
    if (i < n) {
      sm.off[i] = static_cast<uint16_t>(end - len);
      if (i == n - 1) sm.off[n] = static_cast<uint16_t>(end);
      uint8_t* path = reinterpret_cast<uint8_t*>(sm.pn + (end - len)) + 3 * len;
      int at = i;
      for (int d = 0; d < len; ++d) {
        path[d] = static_cast<uint8_t>(at);
        at = sm.parent[at];
      }
    }
  } else {
    float* to = &(kind ? sm.k : sm.q)[0][4 * lane];
    uint64_t p[2][4];
    conv_weights(p[0], w[0]);
    conv_weights(p[1], w[1]);
#pragma unroll 2
    for (int i = warp >> 1; i < n; i += kConvWarps / 2) {
      const uint32_t taps = sm.tap[i];
      uint2 x[4];
      x[3] = *reinterpret_cast<const uint2*>(&sm.in[i][kind][2 * lane]);
#pragma unroll
      for (int e = 0; e < 3; ++e) x[2 - e] = *reinterpret_cast<const uint2*>(&sm.in[(taps >> (8 * e)) & 0xFF][kind][2 * lane]);
      *reinterpret_cast<float4*>(to + i * kDim) = conv_silu4(p, x);
    }
  }
  __syncthreads();
  // ---- the decays, in the place of the inputs
  {
    const float rate = -kLog2e * exp_fast(a_log), lb = a.lower_bound * kLog2e;
#pragma unroll
    for (int t = 0; t < N / kGroups; ++t) {
      if (part + kGroups * t >= n) continue;
      const float2 x = bf2(gin[t]);
      float2 o;
      o.x = ex2(lb * rcp(1.0f + ex2(rate * (x.x + dt.x))));
      o.y = ex2(lb * rcp(1.0f + ex2(rate * (x.y + dt.y))));
      *reinterpret_cast<float2*>(&sm.dec[part + kGroups * t][2 * pair]) = o;
    }
  }

  // ---- norms: half a warp a node, channels 4 l .. + 3 and 64 + 4 l .. + 3 a lane
  const int l = lane & 15, first = 2 * warp + (lane >> 4);    // node first + 2 kWarps t
  const auto load8 = [&](const float* row, ulonglong2 (&x)[2]) {
    x[0] = *reinterpret_cast<const ulonglong2*>(row + 4 * l);
    x[1] = *reinterpret_cast<const ulonglong2*>(row + 64 + 4 * l);
  };
  const auto dot8 = [](const ulonglong2 (&x)[2], const ulonglong2 (&y)[2]) {
    return sum2(fma2(x[0].x, y[0].x, fma2(x[0].y, y[0].y, fma2(x[1].x, y[1].x, mul2(x[1].y, y[1].y)))));
  };
  const auto scale8 = [](ulonglong2 (&x)[2], uint64_t f) {
    x[0].x = mul2(x[0].x, f), x[0].y = mul2(x[0].y, f), x[1].x = mul2(x[1].x, f), x[1].y = mul2(x[1].y, f);
  };
  const auto mul8 = [](ulonglong2 (&x)[2], const ulonglong2 (&y)[2]) {
    x[0].x = mul2(x[0].x, y[0].x), x[0].y = mul2(x[0].y, y[0].y), x[1].x = mul2(x[1].x, y[1].x), x[1].y = mul2(x[1].y, y[1].y);
  };
  const ulonglong2 ones = make_ulonglong2(f2pack(1.0f, 1.0f), f2pack(1.0f, 1.0f));
#pragma unroll 1
  for (int i0 = 2 * warp; i0 < n; i0 += 2 * kWarps) {
    const int i = min(i0 + (lane >> 4), n - 1);
    ulonglong2 q[2], k[2];
    load8(sm.q[i], q);
    load8(sm.k[i], k);
    const float nk = dot8(k, k), nq = dot8(q, q);
    float t = (l < 8 ? nk : nq) + __shfl_xor_sync(0xffffffffu, l < 8 ? nq : nk, 8);            // l < 8: k's, from 8 on: q's
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    t = rsqrtf(t + 1e-6f);
    const float other = __shfl_xor_sync(0xffffffffu, t, 8);
    const float rk = l < 8 ? t : other, rq = a.scale * (l < 8 ? other : t);
    scale8(q, f2pack(rq, rq));
    scale8(k, f2pack(rk, rk));
    __syncwarp();                                              // the last node may be read by both halves
    if (i == i0 + (lane >> 4)) {
      *reinterpret_cast<ulonglong2*>(&sm.q[i][4 * l]) = q[0], *reinterpret_cast<ulonglong2*>(&sm.q[i][64 + 4 * l]) = q[1];
      *reinterpret_cast<ulonglong2*>(&sm.k[i][4 * l]) = k[0], *reinterpret_cast<ulonglong2*>(&sm.k[i][64 + 4 * l]) = k[1];
    }
  }
  __syncthreads();
  // ---- the pairs of a node and those above it, 2 at a time; A q in the place of q
  ulonglong2 f[kOwn][2];                                       // the decays below, at the end of the path A
  uint32_t nodes[kOwn];                                        // the path: distances l + 16 c in byte c
#pragma unroll
  for (int t = 0; t < kOwn; ++t) {
    nodes[t] = 0;
    if (2 * warp + 2 * kWarps * t >= n) continue;
    const int i = first + 2 * kWarps * t;
    ulonglong2 q[2], k[2];
    f[t][0] = f[t][1] = ones;
    const int im = min(i, n - 1);
    load8(sm.q[im], q);
    load8(sm.k[im], k);
    const int at = sm.off[im], len = sm.off[im + 1] - at;
    const int most = max(len, __shfl_xor_sync(0xffffffffu, len, 16));
    const uint8_t* path = reinterpret_cast<const uint8_t*>(sm.pn + at) + 3 * len;
    for (int c = 0; 16 * c < most; ++c) nodes[t] |= static_cast<uint32_t>(path[min(16 * c + l, len - 1)] & (N - 1)) << (8 * c);
    __syncwarp();                                              // the path's bytes are read
#pragma unroll 1
    for (int d = 0; d < most; d += 2) {
      float x[4];                                              // M of 2 pairs, N of 2 pairs
      const uint32_t word = nodes[t] >> (8 * (d >> 4));
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = __shfl_sync(0xffffffffu, word, (d + e) & 15, 16) & 0xFF;
        ulonglong2 kj[2], dj[2];
        load8(sm.k[j], kj);
        load8(sm.dec[j], dj);
        mul8(kj, f[t]);
        x[e] = dot8(kj, k);
        x[2 + e] = dot8(kj, q);
        if (d + e < len) mul8(f[t], dj);
      }
#pragma unroll
      for (int o = 8, m = 2; m > 0; o >>= 1, m >>= 1) {        // lanes l = 4 c .. + 3 receive value c
        const bool up = l & o;
#pragma unroll
        for (int e = 0; e < m; ++e) {
          const float keep = up ? x[e + m] : x[e], send = up ? x[e] : x[e + m];
          x[e] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
      }
      x[0] += __shfl_xor_sync(0xffffffffu, x[0], 2);
      x[0] += __shfl_xor_sync(0xffffffffu, x[0], 1);
      const int e = d + ((l >> 2) & 1);
      if ((l & 3) == 0 && e < len && i < n) {
        if (l >= 8) sm.pn[at + e] = x[0];
        else if (e > 0) sm.pm[at - i + e - 1] = x[0];
      }
    }
    if (i < n) {
      mul8(q, f[t]);
      *reinterpret_cast<ulonglong2*>(&sm.q[i][4 * l]) = q[0], *reinterpret_cast<ulonglong2*>(&sm.q[i][64 + 4 * l]) = q[1];
    }
  }
  // ---- A k and A q as the products' second operand, in the place of k and q
  {
    uint32_t hi[kOwn][8], lo[kOwn][8];                         // k, then q
#pragma unroll
    for (int t = 0; t < kOwn; ++t) {
      if (2 * warp + 2 * kWarps * t >= n) continue;
      const int i = min(first + 2 * kWarps * t, n - 1);
      ulonglong2 x[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        load8(e ? sm.q[i] : sm.k[i], x);
        if (e == 0) mul8(x, f[t]);
        const uint64_t y[4] = {x[0].x, x[0].y, x[1].x, x[1].y};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float y0, y1;
          f2unpack(y[c], y0, y1);
          split2(y0, y1, hi[t][4 * e + c], lo[t][4 * e + c]);
        }
      }
    }
    __syncthreads();
    // the decays' place is free: P's zeros, the values' inputs
    for (int c = tid; c < 2 * N * 128 / 16; c += C::kThreads) reinterpret_cast<uint4*>(sm.p)[c] = make_uint4(0, 0, 0, 0);
    const uint32_t* in =
        reinterpret_cast<const uint32_t*>(a.x + 2 * (int64_t)a.P + h * kDim + 2 * pair) + (s + part) * (a.ldx / 2);
    const int64_t step = kGroups * (a.ldx / 2);
    uint32_t to = smem_u32(&sm.vin[part][pair]);
#pragma unroll 2
    for (int i = part; i < n; i += kGroups, in += step, to += kGroups * kDim * 2) cp_async4(to, in);
    // channels 4 l .. + 3 of 64, in the state's order of pairs
    const int granule = 4 * (l >> 3) + 2 * (l & 1) + ((l >> 2) & 1), within = (l & 2) * 4;
#pragma unroll
    for (int t = 0; t < kOwn; ++t) {
      const int i = first + 2 * kWarps * t;
      if (i >= n) continue;
      const int at = ((granule ^ (i & 7)) << 4) + within;      // rows i and N + i swizzle alike
#pragma unroll
      for (int e = 0; e < 2; ++e) {                            // A k, A q
#pragma unroll
        for (int c = 0; c < 2; ++c) {                          // channels 4 l, 64 + 4 l
          *reinterpret_cast<uint2*>(&sm.op[0][c][N * e + i][at]) = make_uint2(hi[t][4 * e + 2 * c], hi[t][4 * e + 2 * c + 1]);
          *reinterpret_cast<uint2*>(&sm.op[1][c][N * e + i][at]) = make_uint2(lo[t][4 * e + 2 * c], lo[t][4 * e + 2 * c + 1]);
        }
      }
    }
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  const auto bar = [&](int i) { return smem_u32(&sm.bar[i]); };
  // the products are issued by one lane of the last warp, which has the fewest nodes; the whole warp goes along, so that the
  // addresses stay in uniform registers
  const bool issuer = warp == kWarps - 1;
  const auto products = [&](int pass) {                        // of a pass's keys
    tc_fence_after();
    const bool leader = elect_lane();
    constexpr uint32_t idesc = idesc_bf16(128, 2 * N);
    uint32_t acc = pass;
#pragma unroll 1
    for (int t = 0; t < 3; ++t) {                              // high x high, high x low, low x high
#pragma unroll
      for (int c = 0; c < kParts / 2; ++c) {                   // chunks of 64 keys
        const uint64_t bd = smem_desc(smem_u32(&sm.op[t == 1][kParts / 2 * pass + c][0][0]), 0, 1024, 2);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          if (leader) mma_f16_ta(tmem + kColD, tmem + kColS + (t == 2 ? kColLo : 0) + 32 * c + 8 * ks, bd + 2 * ks, idesc, acc);
          acc = 1;
        }
      }
    }
    if (leader) tc_commit(bar(pass));
    __syncwarp();
  };
  if (issuer) products(0);
  // ---- meanwhile the rest of the inputs, and the scalars
  if (C::kPasses > 1) load_state(1);
  // P_i of half a warp's node: lanes hold the distances l + 16 c; the nodes on the path from i up subtract their share from
  // those above them
#pragma unroll
  for (int t = 0; t < kOwn; ++t) {
    if (2 * warp + 2 * kWarps * t >= n) continue;
    const int i = first + 2 * kWarps * t, im = min(i, n - 1);
    const int at = sm.off[im], len = i < n ? sm.off[im + 1] - at : 0;
    const int most = max(len, __shfl_xor_sync(0xffffffffu, len, 16));
    constexpr int kWords = N / 16;
    float x[kWords], b[kWords];
    int base[kWords];                                          // of the node's M
#pragma unroll
    for (int c = 0; c < kWords; ++c) {
      if (c > 0 && 16 * c >= most) break;
      const int m = (nodes[t] >> (8 * c)) & 0xFF;
      const bool have = 16 * c + l < len;
      x[c] = have ? sm.pn[at + 16 * c + l] : 0.0f;
      b[c] = have ? sm.beta[m] : 0.0f;
      base[c] = sm.off[m] - m;
    }
#pragma unroll
    for (int c = 0; c < kWords; ++c) {
      if (16 * c >= most) break;
#pragma unroll 2
      for (int d = 0; d < min(most - 16 * c, 16); ++d) {
        const float y = __shfl_sync(0xffffffffu, x[c] * b[c], d, 16);
        const float* pm = sm.pm + __shfl_sync(0xffffffffu, base[c], d, 16) + l - d - 1;
#pragma unroll
        for (int e = c; e < kWords; ++e) {
          if (16 * e >= most) break;
          if (16 * e + l > 16 * c + d && 16 * e + l < len) x[e] = fmaf(-y, pm[16 * (e - c)], x[e]);
        }
      }
    }
#pragma unroll
    for (int c = 0; c < kWords; ++c) {
      if (16 * c + l >= len) break;
      const int m = (nodes[t] >> (8 * c)) & 0xFF;
      const float y = x[c] * b[c];
      const __nv_bfloat16 y_hi = __float2bfloat16(y);
      const int to = (((m >> 3) ^ (i & 7)) << 4) + 2 * (m & 7);
      *reinterpret_cast<__nv_bfloat16*>(&sm.p[0][i][to]) = y_hi;
      *reinterpret_cast<__nv_bfloat16*>(&sm.p[1][i][to]) = __float2bfloat16(y - __bfloat162float(y_hi));
    }
  }
  cp_async_wait();
  bool ok = mbar_wait(bar(0), 0, &sm.abort, a.status);
  if (C::kPasses > 1) {                                        // the other half of the keys
    ok = !__syncthreads_or(!ok);
    tc_fence_after();
    if (ok) store_state();
    tc_fence_before();
    __syncthreads();
    if (ok && issuer) products(1);
    if (ok) ok = mbar_wait(bar(1), 0, &sm.abort, a.status);
  }
  uint4 wv[2];                                                 // 2 channels x 4 taps each
#pragma unroll
  for (int j = 0; j < 2; ++j) wv[j] = conv_weight(2, j);
  uint2 held[3] = {};                                          // the values' kept rows, the newest first
  if (init)
    for (int j = 0; j < 3; ++j) {
      const uint32_t* kept = reinterpret_cast<const uint32_t*>(cs + ((int64_t)(2 - j) * 3 + 2) * a.P + 4 * lane);
      held[j] = make_uint2(__ldg(kept), __ldg(kept + 1));
    }
  fence_proxy_async_smem();
  ok = !__syncthreads_or(!ok);
  tc_fence_after();
  // ---- the values, in the place of the products' second operand: a warp a node, 4 channels a lane
  {
    uint64_t p[2][4];
    conv_weights(p[0], wv[0]);
    conv_weights(p[1], wv[1]);
#pragma unroll 1
    for (int i = warp; i < n; i += kWarps) {
      const uint32_t taps = sm.tap[i];
      uint2 x[4];
      x[3] = *reinterpret_cast<const uint2*>(&sm.vin[i][2 * lane]);
#pragma unroll
      for (int e = 0; e < 3; ++e) x[2 - e] = *reinterpret_cast<const uint2*>(&sm.vin[(taps >> (8 * e)) & (N - 1)][2 * lane]);
      if (taps & (N * 0x010101u)) {                            // some are kept rows
#pragma unroll
        for (int e = 0; e < 3; ++e) {
          const uint32_t t = (taps >> (8 * e)) & 0xFF;
          if (t >= N) x[2 - e] = t == N ? held[0] : t == N + 1 ? held[1] : held[2];
        }
      }
      *reinterpret_cast<float4*>(&sm.v[i][4 * lane]) = conv_silu4(p, x);
    }
  }
  __syncthreads();
  // ---- w = v - S (A k), as bf16 parts in the place of S; zeros past the nodes, whose columns of P are zeros too. A w that is
  // not finite concerns the nodes below its own alone, not those whose weight of it is 0: zero in the product, `lost` (bit j:
  // the thread's node j's) makes their outputs NaN
  uint32_t lost = 0;
  if (ok) {
#pragma unroll 1
    for (int c = kShare * fourth; c < min(kShare * (fourth + 1), N); c += 8) {
      float y[8], w[8];
      tmem_ld_x8(tmem + rows + kColD + c, y);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = sm.v[c + j][v];
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = c + j < n ? w[j] - y[j] : 0.0f;
      uint64_t odd = 0;                          // 0 but for values that the parts cannot hold
#pragma unroll
      for (int j = 0; j < 8; j += 2) odd = fma2(mul2(f2pack(w[j], w[j + 1]), f2pack(1.01f, 1.01f)), 0, odd);
      if (sum2(odd) != 0.0f) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!(fabsf(w[j]) < 3.36e38f)) lost |= 1u << (c - kShare * fourth + j), w[j] = 0.0f;
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
  const bool any_lost = __syncthreads_or(lost != 0);
  uint32_t* shared_lost = &sm.vin[0][0];                      // [part][value row]
  if (any_lost) shared_lost[kDim * fourth + v] = lost;
  if (ok && issuer) {
    tc_fence_after();
    const bool leader = elect_lane();
    constexpr uint32_t idesc = idesc_bf16(128, N);
#pragma unroll 1
    for (int t = 0; t < 3; ++t) {                              // onto S (A q)
      const uint64_t bd = smem_desc(smem_u32(&sm.p[t == 1][0][0]), 0, 1024, 2);
#pragma unroll
      for (int ks = 0; ks < N / 16; ++ks)
        if (leader) mma_f16_ta(tmem + kColD + N, tmem + kColS + (t == 2 ? kColLo : 0) + 8 * ks, bd + 2 * ks, idesc, 1u);
    }
    if (leader) tc_commit(bar(2));
    __syncwarp();
  }
  if (ok) ok = mbar_wait(bar(2), 0, &sm.abort, a.status);
  if (!__syncthreads_or(!ok)) {
    tc_fence_after();
    __nv_bfloat16* out = a.out + (int64_t)(s + kShare * fourth) * a.ldo + h * kDim + v;
#pragma unroll 1
    for (int c = kShare * fourth; c < min(kShare * (fourth + 1), n); c += 8) {
      float z[8];
      tmem_ld_x8(tmem + rows + kColD + N + c, z);
      tmem_ld_wait();
      if (any_lost) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          for (int at = c + j < n ? c + j : -1; at >= 0; at = sm.parent[at])
            if (shared_lost[kDim * (at / kShare) + v] >> (at % kShare) & 1) z[j] = NAN;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j, out += a.ldo)
        if (c + j < n) *out = __float2bfloat16(z[j]);
    }
  } else {
    // products may still be on their way
    const unsigned long long t0 = globaltimer();
    while (!(mbar_try_wait(bar(0), 0) && (C::kPasses == 1 || mbar_try_wait(bar(1), 0)) && mbar_try_wait(bar(2), 0)) &&
           globaltimer() - t0 <= 2 * kWaitNs) {}
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, kCols);
  }
}

// TMEM has columns for Shape<N>::kBlocks CTAs: shared memory of which one more does not fit an SM (228 KB, 1 KB of it for
// each) keeps it from waiting for them.
template <int N>
constexpr int smem_bytes() {
  constexpr int most = 228 * 1024 / Shape<N>::kBlocks - 1024, least = 228 * 1024 / (Shape<N>::kBlocks + 1);
  static_assert(sizeof(TreeSmem<N>) <= most, "shared memory");
  return sizeof(TreeSmem<N>) > least ? sizeof(TreeSmem<N>) : least;
}

template <int N>
bool set_smem() {
  return cudaFuncSetAttribute(kda_tree_kernel<N>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<N>()) == cudaSuccess;
}

template <int N>
int launch_nodes(const KdaArgs& a, cudaStream_t stream) {
  kda_tree_kernel<N><<<(unsigned)(a.R * a.H), Shape<N>::kThreads, smem_bytes<N>(), stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
}

}  // namespace

int launch_kda_tree(const KdaArgs& a, cudaStream_t stream) {
  if (!kda_step_args(a) || (a.T > 0 && (a.out == nullptr || a.parents == nullptr)) || !kda_aligned(a.out, 2) ||
      !kda_aligned(a.parents, 4) || (a.T > 1 && a.ldo < a.P) || a.max_nodes < 1 || a.max_nodes > kMaxNodes)
    return kErrArgs;
  if (a.R == 0) return kOk;
  if ((int64_t)a.R * a.H > 0x7fffffff) return kErrArgs;
  static OncePerDevice attr;                     // of all sizes at once: which one a later call takes depends on its trees
  int device = 0;
  const auto set = [] { return set_smem<16>() && set_smem<32>() && set_smem<64>(); };
  if (cudaGetDevice(&device) != cudaSuccess || !attr.done(device, set)) return kErrCuda;
  if (a.max_nodes <= 16) return launch_nodes<16>(a, stream);
  // up to 32 nodes four smaller CTAs an SM, unless the larger ones all run at once: 1 x 24 nodes, 32 heads 13.7 and 11.6 us,
  // 4 x 24, 64 heads 22.3 and 21.2, 4 x 32 24.9 and 23.6, 6 x 24 27.3 and 30.3, 8 x 32 38.7 and 42.8
  const bool at_once = a.R * (int64_t)a.H <= Shape<64>::kBlocks * (int64_t)device_sm_count();
  if (a.max_nodes <= 32 && !at_once) return launch_nodes<32>(a, stream);
  return launch_nodes<64>(a, stream);
}

}  // namespace ssb
