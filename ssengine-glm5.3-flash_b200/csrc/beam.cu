// A beam search's selection for sm_100a: of a request's B beams over a vocabulary of V, the k best of
//   score[b] + x[b, v] - log sum_v exp x[b, v]
// in order, equal ones by the lower b V + v. One pass over the logits.
//
// scan: a CTA has one part of one beam's row, 16 bytes a load. Each warp keeps a sum of exponentials against the
//   largest logit that it has seen, so that this one's term is exactly 1 and no term's exponent is large where the term
//   is: in 32 bits over the terms of one iteration (at most 32 of a lane), in 64 beyond. A new largest logit, a handful
//   a row, rescales the sum by an exponential in 64 bits. Beside it the k largest (logit, token) as 64-bit keys whose
//   order is that of the candidates (equal logits: the lower token is larger). A load's largest logit is compared with
//   a bound of the CTA's k-th largest: the least of its 8 warps' ceil(k / 8)-th largest, at first of the lanes' maxima
//   over their first loads, then of the lists. What is not below goes to the warp's list in shared memory, cut back to
//   its k largest when it is full or the logits seen are four times as many. The CTA leaves k keys, the reference and
//   the sum.
// join: a CTA a request: the rows' log sums, then every candidate's score in 64 bits; a beam's own candidates keep the
//   order of their logits, those of different beams are compared at the sums' accuracy. The candidates at or above the
//   best part's k-th go to shared memory and each finds its place by counting those before it.
// Bound: HBM, a read of the logits. 64 requests x 8 beams over 151,552 fp32 logits, a fifth of the beams finished
// (their logits are not read): 62 us, 0.63 of the copy rate, 59 in a graph; a row is one part there, and its list work
// and the rows' uneven ends are not behind other CTAs' loads. With none finished 89 us, 0.53: 512 rows on 444 places;
// bf16 logits 81; k = 16 108; rows that do not lie on 16 bytes, which come by plain loads, 234 (bf16 140). One request
// of 4 beams: 12 us, two launches and a row's parts over the card.
#include "common.cuh"
#include "ops.h"

namespace ssb {
namespace {

constexpr int kScanWarps = 8, kScanThreads = 32 * kScanWarps, kScanBlocks = 3;
constexpr int kList = 256;                       // keys a warp holds between cuts
constexpr int kGroups = 3;                        // groups of loads on their way to shared memory
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kJoinThreads = 512, kRanked = 64;
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

// The largest of the lanes' keys.
SSB_DEVICE uint64_t warp_max(uint64_t v) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(v >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(v >> 32) == hi ? static_cast<uint32_t>(v) : 0u);
  return static_cast<uint64_t>(hi) << 32 | lo;
}
SSB_DEVICE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
SSB_DEVICE uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// The k largest of the keys that the lanes hold (R each, 0: none; distinct) to out, in order; how many there are.
template <int R>
SSB_DEVICE int take_largest(uint64_t (&mine)[R], uint64_t* out, int k, int lane) {
  int n = 0;
  for (; n < k; ++n) {
    uint64_t top = 0;
#pragma unroll
    for (int j = 0; j < R; ++j) top = mine[j] > top ? mine[j] : top;
    top = warp_max(top);
    if (top == 0) break;
#pragma unroll
    for (int j = 0; j < R; ++j)
      if (mine[j] == top) mine[j] = 0;
    if (lane == 0) out[n] = top;
  }
  __syncwarp();
  return n;
}

// A warp's candidates in shared memory. top: a logit of which the warp has seen ceil(k / 8) as large or larger, so that the
// least `top` of the CTA's 8 warps bounds the CTA's k-th largest from below.
struct WarpList {
  uint64_t key[kList];
  uint64_t least;                                // the warp's k-th largest key, 0 while it is not known
  float top;
  int32_t count;
};
__device__ __noinline__ void cut_list(WarpList& L, int k, int lane) {
  const int count = L.count;
  int n;
  if (count <= 64) {
    uint64_t mine[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) mine[j] = 32 * j + lane < count ? L.key[32 * j + lane] : 0;
    __syncwarp();
    n = take_largest(mine, L.key, k, lane);
  } else {
    uint64_t mine[kList / 32];
#pragma unroll
    for (int j = 0; j < kList / 32; ++j) mine[j] = 32 * j + lane < count ? L.key[32 * j + lane] : 0;
    __syncwarp();
    n = take_largest(mine, L.key, k, lane);
  }
  const int share = (k + kScanWarps - 1) / kScanWarps;
  if (lane == 0) {
    L.count = n;
    if (n == k) L.least = L.key[k - 1];
    if (n >= share) L.top = fmaxf(L.top, key_logit(L.key[share - 1]));
  }
  __syncwarp();
}
// Adds the lanes' logits x that are not below bar and above the list's k-th.
__device__ __noinline__ void offer(WarpList& L, int k, float x, uint32_t token, float bar, int lane) {
  const uint64_t key = make_key(x, token);
  const bool in = x >= bar && x > -INFINITY && key > L.least;          // false for NaN
  const uint32_t mask = __ballot_sync(0xffffffffu, in);
  if (mask == 0) return;
  if (L.count + 32 > kList) cut_list(L, k, lane);
  const int count = L.count;
  if (in) L.key[count + __popc(mask & ((1u << lane) - 1))] = key;
  __syncwarp();
  if (lane == 0) L.count = count + __popc(mask);
  __syncwarp();
}

// What stood against `ref` against the larger `now`. Without a reference there is no sum yet: 0, or NaN.
__device__ __noinline__ double rebase(double total, float ref, float now) {
  return ref > -INFINITY ? total * exp(static_cast<double>(ref) - static_cast<double>(now)) : total;
}

// kSkewed: rows may begin anywhere in a 16-byte piece of memory. A lane's values are the same ones of a row then too, put
// together from two pieces: equal rows get the same sums wherever they lie, and equal candidates stay equal.
template <bool kBf16, bool kSkewed>
__global__ void __launch_bounds__(kScanThreads, kScanBlocks) beam_scan_kernel(const __grid_constant__ BeamArgs a) {
  constexpr int kVec = kBf16 ? 8 : 4, kBytes = 16 / kVec;
  constexpr int kLoads = kSkewed ? 2 : 4;                    // 16-byte loads a lane has on their way
  __shared__ WarpList lists[kScanWarps];
  __shared__ float wm[kScanWarps];
  __shared__ double ws[kScanWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t row = blockIdx.x / a.parts;
  const int part = static_cast<int>(blockIdx.x - row * a.parts);
  asm volatile("griddepcontrol.launch_dependents;");
  const float score = a.scores[row];
  if (!(fabsf(score) < INFINITY) || (a.finished != nullptr && a.finished[row])) return;
  // the row in vectors of 16 bytes
  const char* p = static_cast<const char*>(a.x) + row * a.ldx * kBytes;
  const int32_t V = static_cast<int32_t>(a.V), vectors = (V - 1) / kVec + 1;
  const int32_t begin = static_cast<int32_t>(static_cast<int64_t>(vectors) * part / a.parts);
  const int32_t end = static_cast<int32_t>(static_cast<int64_t>(vectors) * (part + 1) / a.parts);
  const int skew = kSkewed ? static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15) : 0;      // bytes
  const uint4* pieces = reinterpret_cast<const uint4*>(p - skew);
  // vectors all of whose pieces are the row's
  const int32_t lo = max(begin, kSkewed && skew > 0 ? 1 : 0);
  const int32_t hi = min(end, kSkewed ? static_cast<int32_t>((a.V * kBytes + skew) / 16) - 1 : V / kVec);
  const auto load = [&](int32_t i) {                         // -inf where it is not the part's
    if (i >= lo && i < hi) {
      if (!kSkewed) return __ldcs(pieces + i);
      const uint4 q0 = __ldg(pieces + i), q1 = __ldg(pieces + i + 1);
      uint32_t w[8] = {q0.x, q0.y, q0.z, q0.w, q1.x, q1.y, q1.z, q1.w};
#pragma unroll
      for (int j = 0; j < 6; ++j) w[j] = skew & 8 ? w[j + 2] : w[j];
#pragma unroll
      for (int j = 0; j < 5; ++j) w[j] = skew & 4 ? w[j + 1] : w[j];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = __funnelshift_r(w[j], w[j + 1], 8 * (skew & 2));
      return make_uint4(w[0], w[1], w[2], w[3]);
    }
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const int64_t e = static_cast<int64_t>(i) * kVec + j;
      const bool in = i < end && e < a.V;
      if (kBf16) {
        const uint32_t v = in ? reinterpret_cast<const uint16_t*>(p)[e] : 0xFF80u;
        w[j / 2] = j % 2 ? w[j / 2] | v << 16 : v;
      } else {
        w[j] = in ? reinterpret_cast<const uint32_t*>(p)[e] : 0xFF800000u;
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
  // Whole rows come by asynchronous copies, a lane's own places: a group of kLoads vectors is read while the next one is on its
  // way, without registers held for it (64 x 8 beams: 76 us with loads alone, 68 with the next ones in registers).
  extern __shared__ __align__(16) uint4 ring[];
  const auto place = [&](int group, int u) { return ring + ((group % kGroups) * kLoads + u) * kScanThreads + tid; };
  const auto ask = [&](int32_t i0, int group) {
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int32_t i = i0 + u * kScanThreads + lane;
      if (i >= lo && i < hi)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(place(group, u))), "l"(pieces + i) : "memory");
      else
        *place(group, u) = load(i);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const auto values = [](uint4 q, float (&x)[kVec]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (kBf16) x[2 * j] = __uint_as_float(w[j] << 16), x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
      else x[j] = __uint_as_float(w[j]);
    }
  };
  const auto largest = [](uint4 q) {                         // NaN is passed over (unless all are)
    if (!kBf16)
      return fmaxf(fmaxf(__uint_as_float(q.x), __uint_as_float(q.y)), fmaxf(__uint_as_float(q.z), __uint_as_float(q.w)));
    const auto b2 = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
    const __nv_bfloat162 m = __hmax2(__hmax2(b2(q.x), b2(q.y)), __hmax2(b2(q.z), b2(q.w)));
    return fmaxf(__low2float(m), __high2float(m));
  };
  WarpList& L = lists[warp];
  if (lane == 0) L.least = 0, L.top = -INFINITY, L.count = 0;
  __syncthreads();
  float ref = -INFINITY, bar = -INFINITY;                    // the same in all lanes; a logit below bar is no candidate
  uint64_t neg = 0;                                          // -ref, 0 while there is none, as a pair
  double total = 0.0;
  int32_t seen = 0, look = 1;                                // iterations, when to cut the list next
  uint4 q[kLoads];
  const int32_t i1 = begin + 32 * warp, step = kLoads * kScanThreads;
  const auto fetch = [&](int32_t i0, int group) {
    if (kSkewed) {
#pragma unroll
      for (int u = 0; u < kLoads; ++u) q[u] = load(i0 + u * kScanThreads + lane);
    } else {
      asm volatile("cp.async.wait_group %0;" ::"n"(kGroups - 1) : "memory");
#pragma unroll
      for (int u = 0; u < kLoads; ++u) q[u] = *place(group, u);
    }
  };
  if (!kSkewed) {
#pragma unroll
    for (int g = 0; g < kGroups; ++g) ask(i1 + g * step, g);
  }
  fetch(i1, 0);
  {                                                          // at least k logits are as large as the k-th lane's maximum
    float most = largest(q[0]);
#pragma unroll
    for (int u = 1; u < kLoads; ++u) most = fmaxf(most, largest(q[u]));
    uint32_t mine = most > -INFINITY ? static_cast<uint32_t>(make_key(most, 0) >> 32) : 0;
    const int share = (a.k + kScanWarps - 1) / kScanWarps;
    for (int n = 0; n < min(a.k, 32); ++n) {
      const uint32_t best = __reduce_max_sync(0xffffffffu, mine);
      if (best == 0) break;
      if (lane == __ffs(__ballot_sync(0xffffffffu, mine == best)) - 1) mine = 0;
      const float x = key_logit(static_cast<uint64_t>(best) << 32);
      if (n == 0) ref = x, neg = f2pack(-ref, -ref);
      if (n == share - 1 && lane == 0) L.top = x;
      if (n == a.k - 1) bar = x;
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int32_t i0 = i1; i0 < end; i0 += step) {
    if (seen > 0) fetch(i0, seen);
    float tops[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) tops[u] = largest(q[u]);
    if (!kSkewed) ask(i0 + kGroups * step, seen);            // into the places just read
    if (seen == look) {                                      // the list's cut costs as much as an iteration or two
      look *= 4;
      cut_list(L, a.k, lane);
    }
    ++seen;
    {
      // other warps' tops may be read old: they only rise
      float t = lane < kScanWarps ? *static_cast<volatile float*>(&lists[lane].top) : INFINITY;
#pragma unroll
      for (int o = kScanWarps / 2; o > 0; o >>= 1) t = fminf(t, __shfl_xor_sync(0xffffffffu, t, o));
      bar = fmaxf(bar, __shfl_sync(0xffffffffu, t, 0));
      if (L.least != 0) bar = fmaxf(bar, key_logit(L.least));
    }
    uint64_t sum = 0;                                        // of this iteration, as a pair
    const auto flush = [&] {
      float s0, s1;
      f2unpack(sum, s0, s1);
      total += static_cast<double>(s0 + s1);
      sum = 0;
    };
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const float top = tops[u];
      if (__any_sync(0xffffffffu, top >= bar || top > ref)) {
        if (__any_sync(0xffffffffu, top > ref)) {
          float now = top == top ? top : -INFINITY;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, o));
          flush();
          total = rebase(total, ref, now);
          ref = now;
          neg = f2pack(-ref, -ref);
        }
        float x[kVec];
        values(q[u], x);
#pragma unroll
        for (int j = 0; j < kVec; ++j)
          if (__any_sync(0xffffffffu, x[j] >= bar))
            offer(L, a.k, x[j], static_cast<uint32_t>(i0 + u * kScanThreads + lane) * kVec + j, bar, lane);
      }
      float x[kVec];
      values(q[u], x);
      const uint64_t scale = f2pack(kLog2e, kLog2e);
#pragma unroll
      for (int j = 0; j < kVec; j += 2) {
        float t0, t1;
        f2unpack(mul2(add2(f2pack(x[j], x[j + 1]), neg), scale), t0, t1);
        sum = add2(sum, f2pack(ex2(t0), ex2(t1)));           // NaN for a NaN, or an infinite reference
      }
    }
    flush();
  }
  cut_list(L, a.k, lane);
  // the CTA's reference and sum, then its k largest
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) wm[warp] = ref, ws[warp] = total;
  __syncthreads();
  if (warp != 0) return;
  const float m = lane < kScanWarps ? wm[lane] : -INFINITY;
  float t = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
  const double z = lane < kScanWarps ? ws[lane] : 0.0;
  double part_sum = m > -INFINITY ? z * exp_fast(m - t) : z;  // without a reference the sum is 0, or NaN
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) part_sum += __shfl_xor_sync(0xffffffffu, part_sum, o);
  if (lane == 0) a.part[row * a.parts + part] = {part_sum, t};
  uint64_t* out = a.keys + (row * a.parts + part) * a.k;
  int n = 0;
  if (a.k <= 8) {                                            // 64 keys, not 512: 1 x 4 beams 12.2 us instead of 12.8
    uint64_t mine[kScanWarps * 8 / 32];
#pragma unroll
    for (int j = 0; j < kScanWarps * 8 / 32; ++j) {
      const int i = 32 * j + lane, w = i / 8, e = i % 8;
      mine[j] = e < lists[w].count ? lists[w].key[e] : 0;
    }
    n = take_largest(mine, out, a.k, lane);
  } else {
    uint64_t mine[kScanWarps * kMaxK / 32];
#pragma unroll
    for (int j = 0; j < kScanWarps * kMaxK / 32; ++j) {
      const int i = 32 * j + lane, w = i / kMaxK, e = i % kMaxK;
      mine[j] = e < lists[w].count ? lists[w].key[e] : 0;
    }
    n = take_largest(mine, out, a.k, lane);
  }
  for (int i = n + lane; i < a.k; i += 32) out[i] = 0;
}

struct Candidate {
  uint64_t score;                                // a double's bits in an order of its own: larger is better, 0 is none
  uint32_t beam;
  uint32_t at;                                   // its key's place in shared memory, kNoKey: a finished beam's
};
constexpr uint32_t kNoKey = 0xFFFFFFFFu;
// The order of the result: scores, then beams, then a beam's keys. A beam's own candidates go by their logits and tokens also
// where 64 bits of score do not tell them apart (logits near 0 beside the log sum), since its parts chose them so.
struct Bound {
  uint64_t score, key;
  uint32_t beam;
};
// The best of the lanes' bounds.
SSB_DEVICE Bound warp_best(const Bound& x) {
  Bound r;
  r.score = warp_max(x.score);
  r.beam = __reduce_min_sync(0xffffffffu, x.score == r.score ? x.beam : kNoKey);
  r.key = warp_max(x.score == r.score && x.beam == r.beam ? x.key : 0);
  return r;
}
SSB_DEVICE uint64_t order_of(double x) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(x + 0.0));              // -0 counts as 0
  return b >> 63 ? ~b : b | 1ull << 63;
}
SSB_DEVICE double score_of(uint64_t o) {
  return __longlong_as_double(static_cast<int64_t>(o >> 63 ? o & ~(1ull << 63) : ~o));
}
// Shared memory: the parts' keys, then room for every candidate.
__global__ void __launch_bounds__(kJoinThreads) beam_join_kernel(const __grid_constant__ BeamArgs a) {
  extern __shared__ __align__(16) uint64_t keys[];
  __shared__ double lse[kMaxBeams];              // the rows' log sums, NaN: the beam has no candidate of its logits
  __shared__ double given[kMaxBeams];            // the beams' scores
  __shared__ Bound bound[kJoinThreads / 32];
  __shared__ uint64_t group[kJoinThreads / 32];
  __shared__ int32_t rank[kRanked];
  __shared__ int32_t count;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t g = blockIdx.x;
  const int per = a.parts * a.k, total = a.B * per;
  Candidate* cand = reinterpret_cast<Candidate*>(keys + (total + 1) / 2 * 2);
  if (tid == 0) count = 0;
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int i = tid; i < total; i += kJoinThreads) keys[i] = a.keys[g * total + i];     // anything of a beam left out
  for (int b = warp; b < a.B; b += kJoinThreads / 32) {
    const float score = a.scores[g * a.B + b];
    const bool finite = fabsf(score) < INFINITY, done = a.finished != nullptr && a.finished[g * a.B + b];
    double l = nan("");
    if (finite && !done) {
      const BeamPart* part = a.part + (g * a.B + b) * a.parts;
      BeamPart q[4];                             // the first 128 parts, loaded once
      float m = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) q[j] = lane + 32 * j < a.parts ? part[lane + 32 * j] : BeamPart{0.0, -INFINITY};
#pragma unroll
      for (int j = 0; j < 4; ++j) m = fmaxf(m, q[j].m);
      for (int p = lane + 128; p < a.parts; p += 32) m = fmaxf(m, part[p].m);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const auto term = [&](const BeamPart& p) {
        return p.m > -INFINITY || p.sum != p.sum ? p.sum * exp_fast(p.m - m) : 0.0;
      };
      double z = 0.0;
#pragma unroll
      for (int j = 0; j < 4; ++j) z += term(q[j]);
      for (int p = lane + 128; p < a.parts; p += 32) z += term(part[p]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
      l = log(z) + m;
    }
    if (lane == 0) {
      given[b] = score;
      lse[b] = fabs(l) < INFINITY ? l : nan("");
      if (finite && done) cand[atomicAdd(&count, 1)] = {order_of(score), static_cast<uint32_t>(b), kNoKey};
    }
  }
  __syncthreads();
  const auto get = [&](int i) {                  // candidate i, of score 0 where there is none
    const uint32_t b = i / per;
    const uint64_t key = keys[i];
    Bound c = {0, 0, kNoKey};
    if (lse[b] == lse[b] && key != 0) c = {order_of(given[b] + (static_cast<double>(key_logit(key)) - lse[b])), key, b};
    return c;
  };
  // Two bounds of the k-th best: the best k-th candidate of a part, and the least of k groups' best firsts (parts i, i + k,
  // ...). The first is tight where one part has most of the best, the second where they are spread.
  const int lists = a.B * a.parts;
  Bound bar = {0, 0, kNoKey};
  for (int i = tid; i < lists; i += kJoinThreads) {
    const Bound c = get(i * a.k + a.k - 1);
    if (c.score > bar.score || (c.score == bar.score && (c.beam < bar.beam || (c.beam == bar.beam && c.key > bar.key)))) bar = c;
  }
  uint64_t least = ~uint64_t{0};                 // of this warp's groups
  for (int j = warp; j < a.k; j += kJoinThreads / 32) {
    uint64_t best = 0;
    for (int i = j + a.k * lane; i < lists; i += 32 * a.k) best = max(best, get(i * a.k).score);
    least = min(least, warp_max(best));
  }
  bar = warp_best(bar);
  if (lane == 0) bound[warp] = bar, group[warp] = least;
  __syncthreads();
  constexpr int kJoinWarps = kJoinThreads / 32;
  bar = warp_best(bound[lane % kJoinWarps]);
  least = ~warp_max(~group[lane % kJoinWarps]);
  for (int i = tid; i < total; i += kJoinThreads) {
    const Bound c = get(i);
    if (c.score == 0 || c.score < least || c.score < bar.score) continue;
    if (c.score == bar.score && (c.beam > bar.beam || (c.beam == bar.beam && c.key < bar.key))) continue;
    cand[atomicAdd(&count, 1)] = {c.score, c.beam, static_cast<uint32_t>(i)};
  }
  __syncthreads();
  // a candidate's place: those before it, counted by kJoinThreads / kRanked threads
  const int n = count, sharer = tid / kRanked;
  for (int i0 = 0; i0 < n; i0 += kRanked) {
    const int i = i0 + tid % kRanked;
    if (tid < kRanked) rank[tid] = 0;
    __syncthreads();
    if (i < n) {
      const Candidate c = cand[i];
      int r = 0, same = 0;
#pragma unroll 4
      for (int j = sharer; j < n; j += kJoinThreads / kRanked) {
        const uint64_t x = cand[j].score;
        r += x > c.score;
        same += x == c.score;
      }
      if (same > (i % (kJoinThreads / kRanked) == sharer)) {           // others than itself
        for (int j = sharer; j < n; j += kJoinThreads / kRanked) {
          const Candidate x = cand[j];
          if (x.score == c.score && x.beam != c.beam) r += x.beam < c.beam;
          else if (x.score == c.score && x.at != c.at) r += keys[x.at] > keys[c.at];     // a finished beam has one candidate
        }
      }
      if (r > 0) atomicAdd(&rank[tid % kRanked], r);
    }
    __syncthreads();
    if (tid < kRanked && i < n && rank[tid] < a.k) {
      const Candidate c = cand[i];
      const int64_t at = g * a.k + rank[tid];
      a.out_scores[at] = static_cast<float>(score_of(c.score));
      a.out_parents[at] = static_cast<int32_t>(c.beam);
      a.out_tokens[at] = c.at == kNoKey ? a.pad : static_cast<int64_t>(key_token(keys[c.at]));
    }
    __syncthreads();
  }
  for (int i = n + tid; i < a.k; i += kJoinThreads) {
    a.out_scores[g * a.k + i] = -INFINITY;
    a.out_parents[g * a.k + i] = -1;
    a.out_tokens[g * a.k + i] = -1;
  }
}

// Parts a row is cut into, the same for every row (equal rows get equal sums) and on every device: as many as run at
// once, none short, the candidates of a request within bounds. Every part begins and ends with its lists, so a second
// wave costs more than it evens out: cut for 592 CTAs instead of 444, 2 x 4 beams take 18.3 us instead of 13.3, 4 x 8
// 27.8 (21.7), 16 x 4 32.8 (25.4); where rows alone fill the SMs, 64 x 8 beams, one part a row takes 89 us, two 94,
// four 113, and with a fifth finished 59, 75 and 94 (rows that do not lie on 16 bytes: 234, 193 and 197).
constexpr int kAtOnce = 148 * kScanBlocks;
int beam_parts(int64_t G, int64_t B, int64_t V, int64_t k) {
  const int64_t rows = G * B;
  int64_t parts = rows > 0 ? kAtOnce / rows : 1;
  parts = parts < V / kMinPart ? parts : V / kMinPart;
  parts = parts < kMaxCandidates / (B * k) ? parts : kMaxCandidates / (B * k);
  return static_cast<int>(parts > 1 ? parts : 1);
}
constexpr int join_bytes(int candidates, int beams) {
  return (candidates + 1) / 2 * 16 + (candidates + beams) * static_cast<int>(sizeof(Candidate));
}
static_assert(join_bytes(kMaxCandidates, kMaxBeams) + 4096 <= 232448, "shared memory");
constexpr int kRing = kGroups * 4 * kScanThreads * 16;
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
  const int smem = join_bytes(a.B * a.parts * a.k, a.B);
  static OncePerDevice attr;
  int device = 0;
  const auto set = [] {
    const auto most = cudaFuncAttributeMaxDynamicSharedMemorySize;
    return cudaFuncSetAttribute(beam_join_kernel, most, join_bytes(kMaxCandidates, kMaxBeams)) == cudaSuccess &&
           cudaFuncSetAttribute(beam_scan_kernel<false, false>, most, kRing) == cudaSuccess &&
           cudaFuncSetAttribute(beam_scan_kernel<true, false>, most, kRing) == cudaSuccess;
  };
  if (cudaGetDevice(&device) != cudaSuccess || !attr.done(device, set)) return kErrCuda;
  const int64_t bytes = a.bf16 ? 2 : 4;
  const bool skewed = off(a.x, 16) || (rows > 1 && a.ldx * bytes % 16 != 0);
  (a.bf16 ? (skewed ? beam_scan_kernel<true, true> : beam_scan_kernel<true, false>)
          : (skewed ? beam_scan_kernel<false, true> : beam_scan_kernel<false, false>))
      <<<static_cast<unsigned>(n), kScanThreads, skewed ? 0 : kRing, stream>>>(a);
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
