// A beam search's selection for sm_100a: of a request's B beams over a vocabulary of V, the k best of
//   score[b] + x[b, v] - log sum_v exp x[b, v]
// in order, equal ones by the lower b V + v. One pass over the logits.
//
// scan: a CTA has one part of one beam's row; each warp keeps the running maximum and sum of exponentials and the k largest
//   (logit, token) it has seen, as 64-bit keys whose order is that of the candidates (equal logits: the lower token is
//   larger). A logit below the warp's k-th key costs one comparison; those above it go to the warp's list in shared memory,
//   which is cut back to its k largest when it is full. The CTA leaves k keys, the maximum and the sum.
// join: a CTA a request: the rows' log sums in 64 bits, then every candidate's score in 64 bits (a beam's own candidates
//   keep the order of their logits, those of different beams are compared at the sums' accuracy). The candidates at or above
//   the best part's k-th go to shared memory and each finds its place by counting those before it.
// Bound: HBM, a read of the logits.
#include "common.cuh"
#include "ops.h"

namespace ssb {
namespace {

constexpr int kScanWarps = 8, kScanThreads = 32 * kScanWarps;
constexpr int kList = 512;                       // keys a warp holds between cuts
constexpr int kJoinThreads = 1024;
constexpr int kMaxK = 64, kMaxBeams = 64;
constexpr int kMaxCandidates = 8192;             // of a request, all parts together
constexpr int kMinPart = 2048;                   // logits a part has at least

// Larger key: larger logit, then lower token. Key 0: none.
SSB_DEVICE uint64_t make_key(float x, uint32_t token) {
  const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);            // -0 counts as 0
  const uint32_t u = b & 0x80000000u ? ~b : b | 0x80000000u;
  return static_cast<uint64_t>(u) << 32 | (0xFFFFFFFFu - token);
}
SSB_DEVICE float key_logit(uint64_t key) {
  const uint32_t u = static_cast<uint32_t>(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}
SSB_DEVICE uint32_t key_token(uint64_t key) { return 0xFFFFFFFFu - static_cast<uint32_t>(key); }

SSB_DEVICE uint64_t warp_max(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor_sync(0xffffffffu, v, o);
    v = w > v ? w : v;
  }
  return v;
}

// e^d, d <= 0: 2^(d log2 e) with the product's rounding error carried to first order (ex2.approx's 2^-22 remains).
SSB_DEVICE float exp_neg(float d) {
  constexpr float kHi = 1.44269502162933349609375f, kLo = 1.925963033500928e-8f;        // log2 e in two parts
  const float t = d * kHi;
  const float r = fmaf(d, kLo, fmaf(d, kHi, -t));
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(t));
  return fmaf(y, fminf(fmaxf(r, -1.0f), 1.0f) * 0.6931471805599453f, y);
}

// The k largest of `count` keys of a list to its front, in order (one warp; keys are distinct). Returns how many.
SSB_DEVICE int cut_list(uint64_t* list, int count, int k, int lane) {
  uint64_t mine[kList / 32];
#pragma unroll
  for (int j = 0; j < kList / 32; ++j) mine[j] = 32 * j + lane < count ? list[32 * j + lane] : 0;
  __syncwarp();
  const int keep = min(k, count);
  for (int i = 0; i < keep; ++i) {
    uint64_t top = 0;
#pragma unroll
    for (int j = 0; j < kList / 32; ++j) top = mine[j] > top ? mine[j] : top;
    top = warp_max(top);
#pragma unroll
    for (int j = 0; j < kList / 32; ++j)
      if (mine[j] == top) mine[j] = 0;
    if (lane == 0) list[i] = top;
  }
  __syncwarp();
  return keep;
}

// Adds the lanes' keys that are above `least` (k-th of the list, 0 while it is short) to the list.
struct WarpList {
  uint64_t* list;
  int count, k;
  uint64_t least;
  float bar;                                     // a logit below it is below `least`
  SSB_DEVICE void add(float x, uint32_t token, int lane) {
    const bool maybe = x >= bar;                 // false for NaN
    if (!__any_sync(0xffffffffu, maybe)) return;
    const uint64_t key = maybe && x > -INFINITY ? make_key(x, token) : 0;
    const bool in = key > least;
    const uint32_t mask = __ballot_sync(0xffffffffu, in);
    if (mask == 0) return;
    if (count + 32 > kList) cut(lane);
    if (in) list[count + __popc(mask & ((1u << lane) - 1))] = key;
    count += __popc(mask);
    __syncwarp();
  }
  SSB_DEVICE void cut(int lane) {
    count = cut_list(list, count, k, lane);
    if (count == k) {
      least = list[k - 1];
      bar = key_logit(least);
    }
    __syncwarp();
  }
};

template <bool kBf16>
__global__ void __launch_bounds__(kScanThreads) beam_scan_kernel(const __grid_constant__ BeamArgs a) {
  __shared__ uint64_t lists[kScanWarps][kList];
  __shared__ float wm[kScanWarps];
  __shared__ double ws[kScanWarps];
  __shared__ int32_t wn[kScanWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t row = blockIdx.x / a.parts;
  const int part = static_cast<int>(blockIdx.x - row * a.parts);
  asm volatile("griddepcontrol.launch_dependents;");
  const float score = a.scores[row];
  if (!(fabsf(score) < INFINITY) || (a.finished != nullptr && a.finished[row])) return;
  const int64_t begin = a.V * part / a.parts, end = a.V * (part + 1) / a.parts;
  const float* xf = static_cast<const float*>(a.x) + (kBf16 ? 0 : row * a.ldx);
  const __nv_bfloat16* xb = static_cast<const __nv_bfloat16*>(a.x) + (kBf16 ? row * a.ldx : 0);
  WarpList L = {lists[warp], 0, a.k, 0, -INFINITY};
  float m = -INFINITY, s = 0.0f;
  for (int64_t i0 = begin + 32 * warp; i0 < end; i0 += kScanThreads) {
    const int64_t i = i0 + lane;
    float x = -INFINITY;
    if (i < end) x = kBf16 ? __bfloat162float(xb[i]) : xf[i];
    if (x > m) {
      s *= m > -INFINITY ? exp_neg(m - x) : 0.0f;
      m = x;
    }
    if (x > -INFINITY || x != x) s += exp_neg(x - m);   // a NaN, or an infinite maximum, makes the sum NaN
    L.add(x, static_cast<uint32_t>(i), lane);
  }
  L.cut(lane);
  // the CTA's maximum and sum, then its k largest
  float top = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  double sum = m > -INFINITY || s != s ? static_cast<double>(s) * exp(static_cast<double>(m) - top) : 0.0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) wm[warp] = top, ws[warp] = sum, wn[warp] = L.count;
  __syncthreads();
  if (warp != 0) return;
  if (lane == 0) {
    float t = -INFINITY;
    for (int w = 0; w < kScanWarps; ++w) t = fmaxf(t, wm[w]);
    double z = 0.0;
    for (int w = 0; w < kScanWarps; ++w)
      if (wm[w] > -INFINITY || ws[w] != ws[w]) z += ws[w] * exp(static_cast<double>(wm[w]) - t);
    BeamPart& p = a.part[row * a.parts + part];
    p.m = t, p.sum = z;
  }
  uint64_t mine[kScanWarps * kMaxK / 32];
#pragma unroll
  for (int j = 0; j < kScanWarps * kMaxK / 32; ++j) {
    const int i = 32 * j + lane, w = i / kMaxK, e = i % kMaxK;
    mine[j] = e < wn[w] ? lists[w][e] : 0;
  }
  uint64_t* out = a.keys + (row * a.parts + part) * a.k;
  for (int i = 0; i < a.k; ++i) {
    uint64_t best = 0;
#pragma unroll
    for (int j = 0; j < kScanWarps * kMaxK / 32; ++j) best = mine[j] > best ? mine[j] : best;
    best = warp_max(best);
#pragma unroll
    for (int j = 0; j < kScanWarps * kMaxK / 32; ++j)
      if (mine[j] == best) mine[j] = 0;
    if (lane == 0) out[i] = best;
  }
}

struct Candidate {
  double score;
  int64_t place;                                 // b V + v
};
// a before b in the result
SSB_DEVICE bool before(const Candidate& a, const Candidate& b) {
  return a.score > b.score || (a.score == b.score && a.place < b.place);
}

__global__ void __launch_bounds__(kJoinThreads) beam_join_kernel(const __grid_constant__ BeamArgs a) {
  extern __shared__ __align__(16) Candidate cand[];
  __shared__ double base[kMaxBeams];             // the rows' log sums, NaN: the beam has no candidate of its logits
  __shared__ Candidate bound[kJoinThreads / 32];
  __shared__ int32_t count;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t g = blockIdx.x;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (tid == 0) count = 0;
  for (int b = warp; b < a.B; b += kJoinThreads / 32) {
    const int64_t row = g * a.B + b;
    const float score = a.scores[row];
    const bool done = a.finished != nullptr && a.finished[row];
    double lse = nan("");
    if (fabsf(score) < INFINITY && !done) {
      float m = -INFINITY;
      for (int p = lane; p < a.parts; p += 32) m = fmaxf(m, a.part[row * a.parts + p].m);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      double z = 0.0;
      for (int p = lane; p < a.parts; p += 32) {
        const BeamPart q = a.part[row * a.parts + p];
        if (q.m > -INFINITY || q.sum != q.sum) z += q.sum * exp(static_cast<double>(q.m) - m);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
      lse = log(z) + m;
    }
    if (lane == 0) base[b] = fabs(lse) < INFINITY ? lse : nan("");
  }
  __syncthreads();
  const int per = a.parts * a.k, total = a.B * per;
  const auto get = [&](int i) {
    const int b = i / per;
    const uint64_t key = base[b] == base[b] ? a.keys[g * total + i] : 0;
    Candidate c = {-INFINITY, int64_t{0x7fffffffffffffff}};
    if (key != 0) {
      c.score = static_cast<double>(a.scores[g * a.B + b]) + (static_cast<double>(key_logit(key)) - base[b]);
      c.place = b * a.V + key_token(key);
    }
    return c;
  };
  // the best k-th candidate of a part: none after it is among the k best
  Candidate bar = {-INFINITY, int64_t{0x7fffffffffffffff}};
  for (int i = tid * a.k + a.k - 1; i < total; i += kJoinThreads * a.k) {
    const Candidate c = get(i);
    if (before(c, bar)) bar = c;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Candidate c = {__shfl_xor_sync(0xffffffffu, bar.score, o), __shfl_xor_sync(0xffffffffu, bar.place, o)};
    if (before(c, bar)) bar = c;
  }
  if (lane == 0) bound[warp] = bar;
  __syncthreads();
  for (int w = 0; w < kJoinThreads / 32; ++w)
    if (before(bound[w], bar)) bar = bound[w];
  for (int i = tid; i < total + a.B; i += kJoinThreads) {
    Candidate c = {-INFINITY, 0};
    if (i < total) {
      c = get(i);
    } else if (a.finished != nullptr && a.finished[g * a.B + i - total]) {
      c.score = a.scores[g * a.B + i - total];
      c.place = (i - total) * a.V + a.pad;
      if (!(fabs(c.score) < INFINITY)) c.score = -INFINITY;
    }
    if (c.score > -INFINITY && !before(bar, c)) cand[atomicAdd(&count, 1)] = c;
  }
  __syncthreads();
  const int n = count;
  for (int i = tid; i < n; i += kJoinThreads) {
    const Candidate c = cand[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += before(cand[j], c);
    if (rank < a.k) {
      a.out_scores[g * a.k + rank] = static_cast<float>(c.score);
      a.out_parents[g * a.k + rank] = static_cast<int32_t>(c.place / a.V);
      a.out_tokens[g * a.k + rank] = c.place % a.V;
    }
  }
  for (int i = n + tid; i < a.k; i += kJoinThreads) {
    a.out_scores[g * a.k + i] = -INFINITY;
    a.out_parents[g * a.k + i] = -1;
    a.out_tokens[g * a.k + i] = -1;
  }
}

// Parts a row is cut into: CTAs for every SM several times over, none short, the candidates of a request within bounds.
int beam_parts(int64_t G, int64_t B, int64_t V, int64_t k) {
  const int64_t rows = G * B;
  int64_t parts = rows > 0 ? (148 * 8 + rows - 1) / rows : 1;
  parts = parts < V / kMinPart ? parts : V / kMinPart;
  parts = parts < kMaxCandidates / (B * k) ? parts : kMaxCandidates / (B * k);
  return static_cast<int>(parts > 1 ? parts : 1);
}
int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

}  // namespace

int64_t beam_workspace_bytes(int64_t G, int64_t B, int64_t V, int64_t k) {
  if (G < 0 || G > (1 << 24) || B < 1 || B > kMaxBeams || V < 1 || V > 0x7fffffff || k < 1 || k > kMaxK) return -1;
  const int64_t n = G * B * beam_parts(G, B, V, k);
  return up256(n * k * 8) + up256(n * static_cast<int64_t>(sizeof(BeamPart)));
}

int launch_beam_select(const BeamArgs& a_in, void* ws, int64_t ws_bytes, cudaStream_t stream) {
  BeamArgs a = a_in;
  const int64_t need = beam_workspace_bytes(a.G, a.B, a.V, a.k);
  if (need < 0 || a.pad < 0 || a.pad >= a.V) return kErrArgs;
  if (a.G == 0) return kOk;
  const auto off = [](const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; };
  if (a.x == nullptr || a.scores == nullptr || a.out_scores == nullptr || a.out_parents == nullptr ||
      a.out_tokens == nullptr || ws == nullptr || off(ws, 256) || off(a.x, a.bf16 ? 2 : 4) || off(a.scores, 4) ||
      off(a.out_scores, 4) || off(a.out_parents, 4) || off(a.out_tokens, 8) || (a.G * a.B > 1 && a.ldx < a.V))
    return kErrArgs;
  if (ws_bytes < need) return kErrWorkspace;
  a.parts = beam_parts(a.G, a.B, a.V, a.k);
  const int64_t rows = a.G * a.B, n = rows * a.parts;
  a.keys = static_cast<uint64_t*>(ws);
  a.part = reinterpret_cast<BeamPart*>(static_cast<uint8_t*>(ws) + up256(n * a.k * 8));
  if (n > 0x7fffffff) return kErrArgs;
  const int smem = (a.B * a.parts * a.k + a.B) * static_cast<int>(sizeof(Candidate));
  static OncePerDevice attr;
  int device = 0;
  const auto set = [] {
    return cudaFuncSetAttribute(beam_join_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (kMaxCandidates + kMaxBeams) * static_cast<int>(sizeof(Candidate))) == cudaSuccess;
  };
  if (cudaGetDevice(&device) != cudaSuccess || !attr.done(device, set)) return kErrCuda;
  (a.bf16 ? beam_scan_kernel<true> : beam_scan_kernel<false>)<<<static_cast<unsigned>(n), kScanThreads, 0, stream>>>(a);
  if (cudaGetLastError() != cudaSuccess) return kErrCuda;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.G));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, beam_join_kernel, a) == cudaSuccess ? kOk : kErrCuda;
}

}  // namespace ssb
