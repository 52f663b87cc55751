// KDA over a tree of drafted tokens for sm_100a: every node of a request's tree continues its parent's state (a root's the
// request's state block), all nodes in one launch, the block left as it is.
//
// Per head, with the conv, norms and gates of kda_decode.cu along each node's path (the taps before a root come from the
// block's conv rows): S_i = S_parent diag(a_i) + u_i k_i^T, u_i = b_i (v_i - S_parent diag(a_i) k_i), o_i = D^-1/2 S_i q_i.
// Written out along the path, with A_i the product of the decays on it and A_ij that of the decays below j,
//   u_i = b_i (v_i - S (A_i k_i) - sum_{j above i} u_j M_ij),   M_ij = (A_ij k_j) . k_i
//   o_i = D^-1/2 (S (A_i q_i) + sum_{j on the path} u_j N_ij),  N_ij = (A_ij k_j) . q_i
// so the state S [value, key] is read once, whatever the nodes, and no node's own state is ever formed: two products of S
// with the nodes' vectors, scalars for the pairs of a node and one above it, and a substitution down the tree for each
// value row. The decays multiply down the path (each is at most 1; quotients of cumulated ones would overflow).
#include "common.cuh"
#include "kda_math.cuh"
#include "ops.h"

namespace ssb {
namespace {

constexpr int kDim = 128;
constexpr int kTreeThreads = 256;
constexpr int kMaxNodes = 64;

template <int N>
struct TreeSmem {
  float k[N][kDim];            // keys, normalised; once the pairs are done, S (A q)
  float dec[N][kDim];          // decays
  float aq[N][kDim];           // queries, then A q
  float ak[N][kDim];           // A k
  float u[N][kDim];            // values, then u
  float m[N][N], n[N][N];      // the pairs
  float beta[N];
  int32_t parent[N];
  int32_t tap[N][3];           // the conv's rows before a node's own, newest first: a node, or -1 - j: the j-th newest kept row
};

template <int N>
__global__ void __launch_bounds__(kTreeThreads) kda_tree_kernel(const __grid_constant__ KdaArgs a) {
  extern __shared__ __align__(16) uint8_t raw_smem[];
  TreeSmem<N>& sm = *reinterpret_cast<TreeSmem<N>*>(raw_smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r = blockIdx.x / a.H, h = blockIdx.x - r * a.H;
  const int4 sq = __ldg(reinterpret_cast<const int4*>(a.seqs) + r);   // {first row, end row, state block, has state}
  const int s = sq.x, n = sq.y - sq.x;
  bool bad = s < 0 || sq.y < s || sq.y > a.T || n > N || sq.z < 0;
  if (!bad && tid < n) {
    const int p = a.parents[s + tid];
    sm.parent[tid] = p;
    bad = p < -1 || p >= tid;
  }
  if (__syncthreads_or(bad)) {
    if (tid == 0 && h == 0) raise_status(a.status, kErrArgs);
    return;
  }
  if (n <= 0) return;
  if (tid < n) {
    int p = tid, kept = 0;
    for (int j = 0; j < 3; ++j) {
      p = p >= 0 ? sm.parent[p] : -1;
      sm.tap[tid][j] = p >= 0 ? p : -1 - kept++;
    }
    sm.beta[tid] = sigmoid_fast(__bfloat162float(a.beta[(int64_t)(s + tid) * a.ldb + h]));
  }
  __syncthreads();
  const bool init = sq.w != 0;

  // ---- conv, gates: a pair of channels a thread, node after node
  const bool conv = tid < 192;
  const int pair = tid & 63, part = tid >> 6;
  const int64_t col = (int64_t)part * a.P + h * kDim + 2 * pair;
  if (conv) {
    const uint32_t* x = reinterpret_cast<const uint32_t*>(a.x + col);
    const int64_t pitch = a.ldx / 2;
    const __nv_bfloat16* cs = a.conv_state + (int64_t)sq.z * a.cs_stride + col;
    uint32_t held[3] = {0, 0, 0};                      // newest first
    if (init)
      for (int j = 0; j < 3; ++j) held[j] = *reinterpret_cast<const uint32_t*>(cs + (int64_t)(2 - j) * 3 * a.P);
    const uint4 wv = __ldg(reinterpret_cast<const uint4*>(a.conv_w + col * 4));     // 2 channels x 4 taps
    const float2 p0 = bf2(wv.x), p1 = bf2(wv.y), p2 = bf2(wv.z), p3 = bf2(wv.w);
    float* to = part == 0 ? &sm.aq[0][0] : part == 1 ? &sm.k[0][0] : &sm.u[0][0];
    for (int i = 0; i < n; ++i) {
      float2 xs[4];
      xs[3] = bf2(__ldg(x + (s + i) * pitch));
      for (int j = 0; j < 3; ++j) {
        const int t = sm.tap[i][j];
        xs[2 - j] = bf2(t >= 0 ? __ldg(x + (s + t) * pitch) : t == -1 ? held[0] : t == -2 ? held[1] : held[2]);
      }
      float2 o;
      o.x = silu_fast(fmaf(p1.y, xs[3].x, fmaf(p1.x, xs[2].x, fmaf(p0.y, xs[1].x, p0.x * xs[0].x))));
      o.y = silu_fast(fmaf(p3.y, xs[3].y, fmaf(p3.x, xs[2].y, fmaf(p2.y, xs[1].y, p2.x * xs[0].y))));
      *reinterpret_cast<float2*>(to + i * kDim + 2 * pair) = o;
    }
  } else {
    const uint32_t* g = reinterpret_cast<const uint32_t*>(a.g + h * kDim + 2 * pair);
    const float2 dt = __ldg(reinterpret_cast<const float2*>(a.dt_bias + h * kDim) + pair);
    const float rate = exp_fast(__ldg(a.a_log + h));
    for (int i = 0; i < n; ++i) {
      const float2 v = bf2(__ldg(g + (s + i) * (a.ldg / 2)));
      float2 o;
      o.x = exp_fast(a.lower_bound * sigmoid_fast(rate * (v.x + dt.x)));
      o.y = exp_fast(a.lower_bound * sigmoid_fast(rate * (v.y + dt.y)));
      *reinterpret_cast<float2*>(&sm.dec[i][2 * pair]) = o;
    }
  }
  __syncthreads();

  // ---- norms: a warp a node, 4 channels a lane
  for (int i = warp; i < n; i += kTreeThreads / 32) {
    float4 q = *reinterpret_cast<float4*>(&sm.aq[i][4 * lane]), k = *reinterpret_cast<float4*>(&sm.k[i][4 * lane]);
    float nq = q.x * q.x + q.y * q.y + q.z * q.z + q.w * q.w, nk = k.x * k.x + k.y * k.y + k.z * k.z + k.w * k.w;
    for (int o = 16; o > 0; o >>= 1) {
      nq += __shfl_xor_sync(0xffffffffu, nq, o);
      nk += __shfl_xor_sync(0xffffffffu, nk, o);
    }
    const float rq = a.scale * rsqrtf(nq + 1e-6f), rk = rsqrtf(nk + 1e-6f);
    *reinterpret_cast<float4*>(&sm.aq[i][4 * lane]) = make_float4(q.x * rq, q.y * rq, q.z * rq, q.w * rq);
    *reinterpret_cast<float4*>(&sm.k[i][4 * lane]) = make_float4(k.x * rk, k.y * rk, k.z * rk, k.w * rk);
  }
  __syncthreads();

  // ---- the pairs of a node and those above it, the decays multiplied up the path
  for (int i = warp; i < n; i += kTreeThreads / 32) {
    const float4 q = *reinterpret_cast<float4*>(&sm.aq[i][4 * lane]), k = *reinterpret_cast<float4*>(&sm.k[i][4 * lane]);
    float4 f = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
    for (int j = i; j >= 0; j = sm.parent[j]) {
      const float4 kj = *reinterpret_cast<float4*>(&sm.k[j][4 * lane]), dj = *reinterpret_cast<float4*>(&sm.dec[j][4 * lane]);
      const float4 t = make_float4(f.x * kj.x, f.y * kj.y, f.z * kj.z, f.w * kj.w);
      float m = t.x * k.x + t.y * k.y + t.z * k.z + t.w * k.w, nn = t.x * q.x + t.y * q.y + t.z * q.z + t.w * q.w;
      for (int o = 16; o > 0; o >>= 1) {
        m += __shfl_xor_sync(0xffffffffu, m, o);
        nn += __shfl_xor_sync(0xffffffffu, nn, o);
      }
      if (lane == 0) sm.m[i][j] = m, sm.n[i][j] = nn;
      f = make_float4(f.x * dj.x, f.y * dj.y, f.z * dj.z, f.w * dj.w);
    }
    *reinterpret_cast<float4*>(&sm.ak[i][4 * lane]) = make_float4(k.x * f.x, k.y * f.y, k.z * f.z, k.w * f.w);
    *reinterpret_cast<float4*>(&sm.aq[i][4 * lane]) = make_float4(q.x * f.x, q.y * f.y, q.z * f.z, q.w * f.w);
  }
  __syncthreads();

  // ---- S (A k) and the substitution (threads 0-127), S (A q) (threads 128-255): a value row a thread
  const int v = tid & 127;
  const bool first = tid < 128;
  float row[kDim];
  {
    const float* S = a.rec_state + (int64_t)sq.z * a.rs_stride + ((int64_t)h * kDim + v) * kDim;
#pragma unroll
    for (int c = 0; c < kDim; c += 4) {
      const float4 w = init ? __ldg(reinterpret_cast<const float4*>(S + c)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      row[c] = w.x, row[c + 1] = w.y, row[c + 2] = w.z, row[c + 3] = w.w;
    }
  }
  for (int i = 0; i < n; ++i) {
    const float4* w = reinterpret_cast<const float4*>(first ? sm.ak[i] : sm.aq[i]);
    float d0 = 0.0f, d1 = 0.0f;
#pragma unroll
    for (int c = 0; c < kDim; c += 8) {
      const float4 w0 = w[c / 4], w1 = w[c / 4 + 1];
      d0 = fmaf(row[c], w0.x, fmaf(row[c + 1], w0.y, fmaf(row[c + 2], w0.z, fmaf(row[c + 3], w0.w, d0))));
      d1 = fmaf(row[c + 4], w1.x, fmaf(row[c + 5], w1.y, fmaf(row[c + 6], w1.z, fmaf(row[c + 7], w1.w, d1))));
    }
    const float d = d0 + d1;
    if (first) {
      float t = sm.u[i][v] - d;
      for (int j = sm.parent[i]; j >= 0; j = sm.parent[j]) t = fmaf(-sm.m[i][j], sm.u[j][v], t);
      sm.u[i][v] = sm.beta[i] * t;
    } else {
      sm.k[i][v] = d;
    }
  }
  __syncthreads();
  for (int i = first ? 0 : 1; i < n; i += 2) {
    float t = sm.k[i][v];
    for (int j = i; j >= 0; j = sm.parent[j]) t = fmaf(sm.n[i][j], sm.u[j][v], t);
    a.out[(int64_t)(s + i) * a.ldo + h * kDim + v] = __float2bfloat16(t);
  }
}

template <int N>
int launch_nodes(const KdaArgs& a, cudaStream_t stream) {
  static OncePerDevice attr;
  int device = 0;
  const auto set = [&] {
    return cudaFuncSetAttribute(kda_tree_kernel<N>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(TreeSmem<N>)) ==
           cudaSuccess;
  };
  if (cudaGetDevice(&device) != cudaSuccess || !attr.done(device, set)) return kErrCuda;
  kda_tree_kernel<N><<<(unsigned)(a.R * a.H), kTreeThreads, sizeof(TreeSmem<N>), stream>>>(a);
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
