// Latent (MLA) attention of new tokens for sm_100a: each query row over the paged e4m3 cache, all of its first seq_len
// tokens or a list of selected ones, split over the row's tokens and joined.
//
//   s_j = bmm1 q[t, h, :] . kv[slot_j, :]   (576 values);   out[t, h, :] = bmm2 sum_j softmax(s)_j kv[slot_j, 0:512]
//
// Split: a row of n tokens is ceil(n / 64) units of work; the units of all rows, in row order, are cut into equal
// contiguous ranges, one per CTA (two rows or more may share a CTA, one row may span many), or, where rows are few or
// short, each row into parts of its own. A CTA works through its range row by row; a row that lies in one range is
// finished there, the parts of a row cut between ranges go to the workspace as (reference m, sum l, unnormalised O) in
// fp32 and are joined by a second kernel:
//   M = max_i m_i;  O = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i.
// No atomics and a fixed order of the sums: the same inputs give the same bits.
//
// One CTA of 22 warps an SM, over units of 64 tokens and a tile of 64 heads:
//   gather (4 warps): a whole unit of a page as TMA tiles (4 chunks [64 tokens x 128 B] and the rope keys), a row's last
//       units and selected tokens by cp.async row by row, what is not there zero-filled; five units in flight;
//   scores (1 warp issues): S [128 query parts x 64 tokens] = Q K^T, tcgen05 kind::f8f6f4. bf16 queries enter as two
//       e4m3 parts (64 high rows, 64 low ones; `stage_q`): the half of the tensor core that 64 heads alone would leave idle.
//       Q stands in TMEM, which has room for all but 96 bytes a row;
//   softmax (2 sets of 8 warps, every second unit each; 16 tokens of one head a thread): the high and low parts of a head
//       are 16 lanes apart and change places by shuffles. Weights 2^(s - E), E one exponent for a head's 32 tokens, again
//       as two e4m3 parts (8 bits), with 2^E as the ue8m0 block scale of the second product. The accumulators stand
//       against a reference per head, which the sets hand on from unit to unit and which moves only when scores rise 2^64
//       above it;
//   values (1 warp issues): O^T [512 dims x 64 heads] += V^T P^T, kind::mxf8f6f4, 4 tiles of M = 128, N = 64, from the same
//       rows read the other way round.
// TMEM: O^T 256 columns, S of two units 128, Q 120, block scales 8. Shared memory: five units' rows 5 x 36 KB (the high
// parts of P take the place of the rope keys, which only the scores need), the low parts of P 2 x 4 KB, the end of Q 12 KB.
// Bounds: 576 bytes a token from HBM against 128 x 576 + 2 x 64 x 512 products of 8 bits. A unit's bytes take 0.83 us of
// an SM's share of the measured copy rate (1,640 cycles at 1.965 GHz, 1,130 at 1.36), its products 1,340 cycles (18
// instructions of 32, 16 of 48, which read shared memory at its full rate). It takes more than either: 2,000 cycles where
// one row has the card (1 x 131,072), 2,250 under sustained load at 64 rows x 32,768 tokens (386 us a call at 990 W, where
// the power limit holds the clock at 1.36 GHz), 2,700 in single calls at 1.965 GHz (322 us from cold caches, 307 and less
// in short bursts). Which role holds the rest is not shown. 32 rows of 128 to 32,768 tokens 81 us in a burst, 92 sustained;
// 1 x 131,072 tokens 42 us; 1 x 1,000 tokens 18 us, of which the plan is 1.3, the query's staging 5.5, the unit and its
// products 4.5, the parts' stores 2.3 and the join 4.
// Tree form (kTree): a row is a drafted token; it sees its request's context and, of the 64 tokens behind, those of its
// word. What bounds it is the unit's pace again: each row of 64 heads is a tile that reads the pages anew, from L2, at
// 1,940 cycles a unit. 24 rows x 4,001 tokens 35 us (plan and first query a third of it), 8 x 16-32 rows (median 8,192
// tokens) 437 us, 0.56 of the bf16 rate; the e4m3 queries of 64 heads that a stage packs 30.4 us for 32.7 (in a graph)
// and 404 to 434 for 369 to 415 (in turn, with the clock under the power limit falling from run to run). Rows of few
// heads share a tile and its units: 20 x 6-12 rows of 16 heads, e4m3 queries 64 us, 111 with a tile a row. An e4m3 tile
// leaves half of the score product empty: 128 heads a tile would fill it, but their accumulators (512 columns) leave no
// room in TMEM.
// Measured against it (bursts): units of 128 tokens in two slots with a token and 16 heads a thread, whose block maxima
// need warp reductions, 380 us at 64 x 32,768; one warp issuing both products 356 (its waits for scores and for weights
// then follow one another); S of one unit 312. The roles' loops are kept small because they share 28 KB of instruction
// cache: unrolled in full they took 511 us where rolled ones took 485.
#include <cuda_fp16.h>

#include "common.cuh"
#include "ops.h"

namespace ssb {
namespace {

constexpr int kDq = 576, kDv = 512, kPage = 128, kUnit = 64, kTileH = 64;
constexpr int kMaxCtas = kMlaRanges;            // the workspace is sized by it
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kNone = -INFINITY;

constexpr int kSoftWarps = 16;                  // warps 0-15: TMEM lanes 32 (warp & 3) .. (16 heads), tokens 32 (warp >> 2 & 1)
constexpr int kSoftmax = 32 * kSoftWarps;       // .. + 31 of every second unit, those of parity warp >> 3 (a set)
constexpr int kSetWarps = 8;
constexpr int kScoreWarp = kSoftWarps;          // warp 16 issues the score products
constexpr int kValueWarp = kScoreWarp + 1;      // warp 17 the value products
constexpr int kGatherWarp = kValueWarp + 1;     // warps 18-21 bring the cache rows
constexpr int kGatherWarps = 4;
constexpr int kThreads = 32 * (kGatherWarp + kGatherWarps);

// ---- shared memory ------------------------------------------------------------------------------------------------
constexpr int kSlots = 5;                       // units in shared memory
constexpr int kChunk = 8192;                    // [64 rows x 128 B], 128-byte swizzle
constexpr int kRope = 4096;                     // [64 rows x 64 B], 64-byte swizzle
constexpr int kLat = 4 * kChunk;                // a unit's latent rows
constexpr int kOffKv = 0;                       // the latent rows of the units
constexpr int kOffRope = kSlots * kLat;         // their rope keys; once its scores are done, a unit's high parts of P
constexpr int kOffPlo = kOffRope + kSlots * kRope;    // the low parts of P, two units
constexpr int kOffQ = kOffPlo + 2 * kRope;      // the query parts' last 96 bytes: [128 rows x 32 B], 32-byte swizzle, then
constexpr int kOffQRope = kOffQ + 4096;         // [128 rows x 64 B], 64-byte swizzle
constexpr int kOffSf = kOffQRope + 8192;     // block scales of P, two units: byte (h % 32) 16 + unit 8 + (h / 32) 4 + half
constexpr int kOffBar = kOffSf + 512;           // mbarriers
constexpr int kOffMisc = kOffBar + 256;         // tmem address, abort flag, a set's unit with scores far above its references
constexpr int kOffSlot = kOffMisc + 16;         // int4 [5] (8 places): a unit's tokens present (2 words), kLast or not
constexpr int kOffRing = kOffSlot + 128;        // int4 [8]: the same by unit, as the softmax and the values read it
constexpr int kOffRef = kOffRing + 128;         // float [64]: the heads' references
constexpr int kOffRow = kOffRef + 256;          // float [4][64]: maxima and rescale factors, the sums, or maxima of the query
constexpr int kOffSum = kOffRow + 1024;         // float [64]: bmm2 / l
constexpr int kOffPlan = kOffSum + 256;         // int32 [76]: the plan's sums, first row and maxima
constexpr int kSmem = kOffPlan + 304;
static_assert(kOffSlot % 16 == 0 && kOffRow % 16 == 0 && kOffSf % 128 == 0 && kSmem <= 232448, "shared memory");
// TMEM columns: O^T as 4 tiles of 128 dims x 64 heads; S of two units, 64 tokens each; the first 480 bytes of the query
// parts; block scales of V (byte 0, 2^-7, against the high parts of P, byte 1, 2^-11, against the low ones) and of P (2
// columns a unit): all 512. Lanes 32 i + l of S and the
// query parts: the high part of head 16 i + l, l < 16, the low part of head 16 i + l - 16 above
constexpr uint32_t kColO = 0, kColS = 256, kColQ = 384, kColV = 504, kColP = 508;
constexpr float kMaxRise = 64.0f;               // base-2 scores above a head's reference before it moves and O is rescaled
constexpr float kMinE = -100.0f;                // the least exponent of a block
enum : int32_t { kMore = 0, kLast = 1, kEnd = 2 };     // a unit, the last unit of its row, no unit: the row has ended
constexpr uint32_t kSw128 = 2, kSw64 = 4, kSw32 = 6;       // descriptor layout types

// Block-scaled instruction descriptor (kind::mxf8f6f4): e4m3 A and B (format 0), ue8m0 scales (bit 23), A
// MN-major (bit 15), B K-major, N >> 3 in [17,23), M >> 4 in [24,29), B's scale byte in [4,6), A's in [29,31).
__host__ __device__ constexpr uint32_t idesc_mx(int M, int N) {
  return (1u << 15) | (static_cast<uint32_t>(N >> 3) << 17) | (1u << 23) |
         (static_cast<uint32_t>(M >> 4) << 24);
}
// D[tmem] (+)= A B, e4m3 operands with ue8m0 scales for blocks of 32 along the reduction.
SSB_DEVICE void tc_mma_mx(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t acc, uint32_t sfa,
                          uint32_t sfb) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
      "l"(ad), "l"(bd), "r"(idesc), "r"(acc), "r"(sfa), "r"(sfb)
      : "memory");
}
SSB_DEVICE void tmem_ld_x16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
// D[tmem] (+)= A B with e4m3 A in TMEM (a row a lane, 4 values a column) and B in shared memory.
SSB_DEVICE void tc_mma_f8_ta(uint32_t d, uint32_t a, uint64_t bd, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(bd), "r"(idesc), "r"(acc)
      : "memory");
}
SSB_DEVICE void tmem_ld_x4(uint32_t taddr, float (&v)[4]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
               : "r"(taddr));
}
SSB_DEVICE void tmem_st_x16(uint32_t taddr, const float (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
      "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
      : "memory");
}
SSB_DEVICE void tmem_st_x4(uint32_t taddr, uint32_t v) {               // one word in 4 columns
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %1, %1, %1};" ::"r"(taddr), "r"(v) : "memory");
}
SSB_DEVICE void tmem_st_4(uint32_t taddr, const uint32_t (&v)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3])
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
// Transposes 4 x 4 values over 4 neighbouring lanes: v[i] of lane l becomes v[l] of lane i (of the four).
SSB_DEVICE void cross4(float (&v)[4], int lane) {
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i & o) continue;
      const float got = __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + o], o);
      if (up) v[i] = got; else v[i + o] = got;
    }
  }
}
SSB_DEVICE float ex2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
SSB_DEVICE uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
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
// v (|v| <= 256) as hi + lo / 16 in e4m3: 8 significant bits down to 2^-6, a quantum of 2^-13 below. v enters as two
// halves (11 bits, so that the rounding to 8 is the one that counts).
SSB_DEVICE void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 v = __floats2half2_rn(a, b);
  hi = half2_e4m3(v);
  lo = half2_e4m3(__hmul2(__hsub2(v, e4m3_half2(hi)), __float2half2_rn(16.0f)));
}
// The same of two halves with 8 significant bits: hi has the leading 4, lo exactly the others. Below 2^-6, where e4m3 has a
// quantum of 2^-9, (h + 3) - 3 rounds h to it (3 + h lies where halves have that quantum; a larger h has no finer bits and
// comes back unchanged), so that lo has all that hi lost: off by 2^-14 at most, lo's own quantum. Half the conversions of
// `split2`.
SSB_DEVICE void split2_bf16(uint32_t v, uint32_t& hi, uint32_t& lo) {
  const uint32_t h = v & 0xFF80FF80u;
  const __half2 a = *reinterpret_cast<const __half2*>(&v), three = __float2half2_rn(3.0f);
  const __half2 b = __hsub2_rn(__hadd2_rn(*reinterpret_cast<const __half2*>(&h), three), three);
  hi = half2_e4m3(b);
  lo = half2_e4m3(__hmul2(__hsub2(a, b), __float2half2_rn(16.0f)));
}
// Byte offset of 16-byte granule g of row r: a 128-byte-swizzled chunk, a 64-byte-swizzled one.
SSB_DEVICE uint32_t sw128(int r, int g) { return r * 128 + ((g ^ (r & 7)) << 4); }
SSB_DEVICE uint32_t sw32(int r, int g) { return r * 32 + ((g ^ ((r >> 2) & 1)) << 4); }
SSB_DEVICE uint32_t sw64(int r, int g) { return r * 64 + ((g ^ ((r >> 1) & 3)) << 4); }
// ---- barriers -----------------------------------------------------------------------------------------------------
struct Bars {                                    // full, empty: a slot each; s_*, p_full, pv_done, agree, ref_ok, slow: a set
  uint32_t full, empty, q_full, s_full, s_empty, p_full, pv_done, o_full, o_free, drain, agree, ref_ok, slow;
};
// mbar_wait whose second and later tries are out of line: the many waits stay short in the instruction cache.
__device__ __noinline__ bool mbar_wait_more(uint32_t bar, uint32_t parity, volatile int32_t* abort_flag,
                                            int32_t* status) {
  const unsigned long long t0 = globaltimer();
  while (true) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
    if (globaltimer() - t0 > kWaitNs) {
      *abort_flag = 1;
      raise_status(status, kErrTimeout);
      return false;
    }
  }
}
SSB_DEVICE bool mbar_nap(uint32_t bar, uint32_t parity, volatile int32_t* abort_flag, int32_t* status) {
  return mbar_try_wait(bar, parity) || mbar_wait_more(bar, parity, abort_flag, status);
}
// A gather warp that gave up: the tiles it asked for may be on their way into this CTA's shared memory, which is another's
// once the CTA has ended. It waits for the units it has issued; one that another warp left out stays incomplete, but the
// own tiles (microseconds) have landed long before the limit.
__device__ __noinline__ void drain_tiles(uint32_t full, int slot, int round) {
  const unsigned long long t0 = globaltimer();
#pragma unroll 1
  for (int j = 0; j < kSlots; ++j) {
    const int phase = ring_phase(j, slot, round);
    while (phase >= 0 && !mbar_try_wait(full + 8 * j, phase) && globaltimer() - t0 <= kWaitNs / 1000) {}
  }
  __syncwarp();
}
// One arrival for a warp, after all its lanes got here.
SSB_DEVICE void warp_arrive(uint32_t bar, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}
SSB_DEVICE void mbar_arrive_n(uint32_t bar, uint32_t n) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(n) : "memory");
}

// Tree form. Where a row's heads fill half of a tile or less, up to a.group = 64 / H neighbouring rows share one, and with it
// every unit they read: rows of one request with one context length, cut at multiples of the group. The first of them, which
// leads, stands for all in the plan; head h of the tile is head h % H of row h / H behind it.
struct TreeRows {                                // where the rows' requests (null: every row its own), contexts and nodes are
  const int32_t *req, *len;
  const uint64_t* nodes;
  SSB_DEVICE TreeRows(const int32_t* r, const int32_t* l, const uint64_t* n) : req(r), len(l), nodes(n) {}
  SSB_DEVICE explicit TreeRows(const MlaDecodeArgs& a) : req(a.reqs), len(a.seq_lens), nodes(a.ancestors) {}
  SSB_DEVICE bool leads(const MlaDecodeArgs& a, int t) const {
    return t % a.group == 0 || req == nullptr || req[t] != req[t - 1] || len[t] != len[t - 1];
  }
  // Units up to the end of what the rows see that t leads (0: it leads none, a reqs entry outside the table, or a negative
  // length). Positions past 2^31 - 2^7 are past any table.
  SSB_DEVICE int units(const MlaDecodeArgs& a, int t, uint64_t seen) const {
    if (len[t] < 0 || (req != nullptr && static_cast<uint32_t>(req[t]) >= static_cast<uint32_t>(a.R))) return 0;
    const int tokens = min(len[t], 0x7fffff00) + 64 - __clzll(static_cast<long long>(seen));
    return min((tokens + kUnit - 1) / kUnit, kPage / kUnit * a.width);
  }
  // By one thread.
  SSB_DEVICE int units_of(const MlaDecodeArgs& a, int t) const {
    if (!leads(a, t)) return 0;
    uint64_t w = nodes[t];
    for (int i = 1; i < a.group && t + i < a.T && !leads(a, t + i); ++i) w |= nodes[t + i];
    return units(a, t, w);
  }
};
// By a whole warp, whose lanes look at the neighbouring rows at once: the row that leads t, the rows that t leads, the nodes
// that any of those sees, and their units.
SSB_DEVICE int leader_of(const MlaDecodeArgs& a, int t) {
  const TreeRows R(a);
  const int lane = threadIdx.x & 31;
  for (int i = t; true; i -= 32) {
    const uint32_t m = __ballot_sync(0xffffffffu, i - lane < 0 || R.leads(a, max(i - lane, 0)));
    if (m != 0) return i - (__ffs(m) - 1);
  }
}
SSB_DEVICE int rows_led(const MlaDecodeArgs& a, int t) {
  const TreeRows R(a);
  const int lane = threadIdx.x & 31;
  for (int i = 1; true; i += 32) {
    const int j = i + lane;
    const uint32_t m = __ballot_sync(0xffffffffu, j >= a.group || t + j >= a.T || R.leads(a, t + j));
    if (m != 0) return i + __ffs(m) - 1;
  }
}
SSB_DEVICE uint64_t nodes_seen(const MlaDecodeArgs& a, int t) {
  const int lane = threadIdx.x & 31, n = rows_led(a, t);
  const uint64_t w = (lane < n ? a.ancestors[t + lane] : 0) | (lane + 32 < n ? a.ancestors[t + lane + 32] : 0);
  return static_cast<uint64_t>(__reduce_or_sync(0xffffffffu, static_cast<uint32_t>(w >> 32))) << 32 |
         __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(w));
}
SSB_DEVICE int tree_units(const MlaDecodeArgs& a, int t) {
  const TreeRows R(a);
  return R.leads(a, t) ? R.units(a, t, nodes_seen(a, t)) : 0;
}

// ---- the plan -----------------------------------------------------------------------------------------------------
// Tokens and units of row t. How many tokens a row's list names is not known before it is read: its share is planned
// by the list's width or, where that is smaller, the tokens it can name.
template <bool kTree>
SSB_DEVICE int row_units(const MlaDecodeArgs& a, int t) {
  if constexpr (kTree) return tree_units(a, t);            // by a whole warp
  int n = a.indices != nullptr ? a.n_idx : 0x7fffff00;
  if (a.seq_lens != nullptr) n = min(n, a.seq_lens[t]);
  if (a.reqs != nullptr && static_cast<uint32_t>(a.reqs[t]) >= static_cast<uint32_t>(a.R)) n = 0;
  n = n > 0 ? (n + kUnit - 1) / kUnit : 0;
  return a.indices != nullptr ? n : min(n, kPage / kUnit * a.width);
}

// A CTA's share of one row: units [b0, b1) of the row's nb planned ones; every role walks the same segments.
struct Segment {
  int t, b0, b1, nb;
};
// Ranges are cut in units plus `cost` for every row that has any: a row's staging, drain and epilogue take a CTA about as
// long as ten units (32 ragged rows: 85 us at a cost of 4, 80 at 10), none where a range is few units and every cut row
// would lose more (96 selected rows, 21 units a range: 75 us with the cost, 72 without).
struct Walk {
  int t, nb, first, lo, hi, cost;               // next row, its units, the units and costs before it, the range, the cost
};
template <bool kTree>
__device__ __noinline__ bool walk_next(const MlaDecodeArgs& a, Walk& w, Segment& s) {
  bool found = false;
  while (!found && w.first < w.hi) {
    s.t = w.t, s.nb = w.nb;
    s.b0 = max(w.lo - w.first, 0), s.b1 = min(w.hi - w.first, w.nb);
    found = s.b0 < s.b1;
    if (w.nb > 0) w.first += w.nb + w.cost;
    if (++w.t >= a.T) {
      w.first = w.hi;
    } else if (w.first < w.hi) {                           // looked up where the range goes on
      w.nb = row_units<kTree>(a, w.t);
    }
  }
  return found;
}
constexpr int kRowCost = 10, kCostFrom = 24;      // units; ranges of so many units or more bear it

// All threads of the CTA: its range and the row that holds its beginning. sh: 48 words for the warps' sums, 4 for the row.
// False: more CTAs than work, nothing to do here. Where rows are few or short, every row is cut by itself into parts of at
// most `per` units, one a CTA: sum_r ceil(u_r / per) <= units / per + rows CTAs suffice, which fixes `per`. That leaves some
// CTAs out, but each begins one row, where a CTA of equal ranges begins 1 + rows / ctas on average and two or more at
// worst; it is taken where `per` exceeds the equal share by less than those beginnings cost. 34 rows x 1,853 tokens: 38 us
// in equal ranges, 28 in parts; 62 rows of 2,051 selected tokens: 39 and 35; on the other side 41 rows (median 6,427
// tokens, 32 heads): 69 and 77; 48 rows (median 4,096, 16 heads): 50 and 59.
// The tree form's rows are looked at by their neighbours too, one load behind another: up to kPlanRows of them are kept in
// `room` (shared memory that the units take later) with their units (20 x 12 rows of 16 heads: 71 us without, 63 with).
constexpr int kPlanRows = 4096;
template <bool kTree>
SSB_DEVICE bool find_range(const MlaDecodeArgs& a, int cta, int ctas, int32_t* sh, uint8_t* room, Walk& w) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int units = 0, rows = 0, most = 0;
  const bool kept = kTree && a.T <= kPlanRows;
  uint64_t* nodes = reinterpret_cast<uint64_t*>(room);
  int32_t* of = reinterpret_cast<int32_t*>(nodes + kPlanRows);           // units, requests, contexts
  if (kTree && kept) {
#pragma unroll 1
    for (int t = tid; t < a.T; t += kThreads) {
      nodes[t] = a.ancestors[t];
      of[kPlanRows + t] = a.reqs != nullptr ? a.reqs[t] : t;
      of[2 * kPlanRows + t] = a.seq_lens[t];
    }
    __syncthreads();
  }
  const auto units_at = [&](int t) {
    if constexpr (kTree) {
      if (kept) return TreeRows(of + kPlanRows, of + 2 * kPlanRows, nodes).units_of(a, t);
      return TreeRows(a).units_of(a, t);
    } else {
      return row_units<false>(a, t);
    }
  };
#pragma unroll 1
  for (int t = tid; t < a.T; t += kThreads) {
    const int n = units_at(t);
    if (kTree && kept) of[t] = n;
    units += n;
    rows += n > 0;
    if (kTree) most = max(most, n);
  }
  if (kTree) {
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) sh[52 + warp] = most;
  }
  units = __reduce_add_sync(0xffffffffu, units);
  rows = __reduce_add_sync(0xffffffffu, rows);
  if (lane == 0) sh[warp] = units, sh[24 + warp] = rows;
  if (tid == 0) sh[48] = -1;
  __syncthreads();
  units = __reduce_add_sync(0xffffffffu, lane < kThreads / 32 ? sh[lane] : 0);
  rows = __reduce_add_sync(0xffffffffu, lane < kThreads / 32 ? sh[24 + lane] : 0);
  const int spare = max(ctas - rows, 1);
  int per = max((units + spare - 1) / spare, 2);
  if (kTree && 0 < rows && rows <= ctas) {
    // a tree's rows are of one length: floor(ctas / rows) parts of each suffice too (24 rows of 63 units: 11 and not 13)
    const int each = ctas / rows;
    most = __reduce_max_sync(0xffffffffu, lane < kThreads / 32 ? sh[52 + lane] : 0);
    per = max(min(per, (most + each - 1) / each), 2);
  }
  const bool parts = rows < ctas && per <= units / ctas + kRowCost + kRowCost * rows / ctas;
  w.cost = units < kCostFrom * ctas ? 0 : kRowCost;
  if (parts) {
    w.lo = cta;
  } else {
    // every range in use holds a unit: a row's CTAs are consecutive
    const int used = min(ctas, units);
    if (cta >= used) return false;
    const int total = units + rows * w.cost, share = total / used, rem = total - share * used;
    w.lo = cta * share + min(cta, rem);
    w.hi = w.lo + share + (cta < rem);
  }
  if (warp == 0) {
    int base = 0;
#pragma unroll 1
    for (int c = 0; c < a.T; c += 32) {
      const int t = c + lane, nb = t >= a.T ? 0 : kept ? of[t] : units_at(t);
      const int v = nb == 0 ? 0 : parts ? (nb + per - 1) / per : nb + w.cost;
      int end = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, end, o);
        if (lane >= o) end += x;
      }
      end += base;
      const bool hit = end - v <= w.lo && w.lo < end;
      if (hit) sh[48] = t, sh[49] = nb, sh[50] = end - v, sh[51] = v;
      base = __shfl_sync(0xffffffffu, end, 31);
      if (__any_sync(0xffffffffu, hit)) break;
    }
  }
  if (kTree) fence_proxy_async_smem();           // the room's next writes may be tiles
  __syncthreads();
  w.t = sh[48], w.nb = sh[49], w.first = sh[50];
  if (w.t < 0) return false;
  if (parts) {                                  // one segment, written as a range of the row's own units
    const int64_t i = cta - w.first, n = sh[51];
    w.lo = static_cast<int>(w.nb * i / n), w.hi = static_cast<int>(w.nb * (i + 1) / n), w.first = 0;
  }
  return true;
}

// Rows without a token: zeros. One warp.
template <bool kTree>
__device__ __noinline__ void zero_rows(const MlaDecodeArgs& a, int cta, int h0, int nh, int lane) {
#pragma unroll 1
  for (int t = cta; t < a.T; t += gridDim.x) {
    if (row_units<kTree>(a, kTree ? leader_of(a, t) : t) != 0) continue;
    if (lane == 0 && a.reqs != nullptr && static_cast<uint32_t>(a.reqs[t]) >= static_cast<uint32_t>(a.R))
      raise_status(a.status, kErrArgs);
    uint4* o = reinterpret_cast<uint4*>(a.out + ((int64_t)t * a.H + h0) * kDv);
    for (int i = lane; i < nh * kDv / 8; i += 32) o[i] = make_uint4(0, 0, 0, 0);
    for (int i = lane; a.lse != nullptr && i < nh; i += 32) a.lse[(int64_t)t * a.H + h0 + i] = kNone;
  }
}

SSB_DEVICE float* part_o(const MlaDecodeArgs& a, int tile, int slot) {
  return a.part_o + ((int64_t)tile * 2 * kMaxCtas + slot) * kTileH * kDv;
}
SSB_DEVICE float2* part_ml(const MlaDecodeArgs& a, int tile, int slot) {
  return a.part_ml + ((int64_t)tile * 2 * kMaxCtas + slot) * kTileH;
}

// ---- the two products ---------------------------------------------------------------------------------------------
// By a whole warp of which one lane issues: the addresses are the same in every lane, so they stay in uniform registers.
SSB_DEVICE void issue_scores(const Bars& B, uint32_t sbase, int slot, int set, bool leader) {
  constexpr uint32_t idesc = idesc_e4m3(128, kUnit);                 // S [query parts, tokens] = Q K^T
  uint64_t bd = smem_desc(sbase + kOffKv + slot * kLat, 0, 1024, kSw128);
  const uint32_t S = kColS + kUnit * set;
  uint32_t q = kColQ, acc = 0;
#pragma unroll 1
  for (int c = 0; c < 3; ++c) {
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      if (leader) tc_mma_f8_ta(S, q + 8 * ks, bd + 2 * ks, idesc, acc);
      acc = 1;
    }
    q += 32;
    bd += kChunk >> 4;
  }
#pragma unroll
  for (int ks = 0; ks < 3; ++ks)
    if (leader) tc_mma_f8_ta(S, q + 8 * ks, bd + 2 * ks, idesc, 1u);
  if (leader) tc_mma_f8(S, smem_desc(sbase + kOffQ, 0, 256, kSw32), bd + 6, idesc, 1u);
  const uint64_t ar = smem_desc(sbase + kOffQRope, 0, 512, kSw64);
  bd = smem_desc(sbase + kOffRope + slot * kRope, 0, 512, kSw64);
#pragma unroll
  for (int ks = 0; ks < 2; ++ks)                                     // the rope keys: 64 bytes a row
    if (leader) tc_mma_f8(S, ar + 2 * ks, bd + 2 * ks, idesc, 1u);
  if (leader) tc_commit(B.s_full + 8 * set);
}
SSB_DEVICE void issue_values(const Bars& B, uint32_t sbase, int slot, int set, int heads, bool fresh, bool leader) {
  uint64_t ad = smem_desc(sbase + kOffKv + slot * kLat, kChunk, 1024, kSw128);    // O^T [dims, heads] (+)= V^T P^T
  const uint64_t hi0 = smem_desc(sbase + kOffRope + slot * kRope, 0, 512, kSw64);
  const uint64_t lo0 = smem_desc(sbase + kOffPlo + set * kRope, 0, 512, kSw64);
  uint32_t o = kColO;
  const uint32_t sfp = kColP + 2 * set;
  if (leader) tc_cp_sf(kColP, smem_desc(sbase + kOffSf, 0, 128, 0));
#pragma unroll 1
  for (int d = 0; d < 4; ++d) {                                      // 128 dims
    uint32_t acc = fresh ? 0u : 1u;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {                                 // 32 tokens a step: one block of scales
      const uint32_t id = idesc_mx(128, 0) | (static_cast<uint32_t>(heads >> 3) << 17) | (ks << 4);
      if (leader) {
        tc_mma_mx(o, ad + ks * (4096 >> 4), hi0 + 2 * ks, id, acc, kColV, sfp);
        tc_mma_mx(o, ad + ks * (4096 >> 4), lo0 + 2 * ks, id | (1u << 29), 1u, kColV, sfp);
      }
      acc = 1;
    }
    ad += kChunk >> 4;
    o += 64;
  }
  if (leader) {
    tc_commit(B.empty + 8 * slot);
    tc_commit(B.pv_done + 8 * set);
  }
}

// Values 144 part + 16 j .. + 15 of this thread's row of query parts to their place.
SSB_DEVICE void keep_q(uint8_t* smem, uint32_t to, const uint32_t (&w)[4], int part, int j) {
  if (part < 3 || j < 3) {
    tmem_st_4(to, w);
  } else {
    const int row = 32 * ((threadIdx.x >> 5) & 3) + (threadIdx.x & 31);
    uint8_t* at = j < 5 ? smem + kOffQ + sw32(row, j - 3) : smem + kOffQRope + sw64(row, j - 5);
    *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// One query row's heads h0 .. h0 + 63 as the parts of q 2^-k (k per head, its largest value in [2^7, 2^8)) into TMEM (the
// last 96 values: shared memory), zero rows past nh. bf16 has 8 significant bits, so the two e4m3 parts hold a value exactly
// unless it is below 2^-13 of the head's largest (then to 2^-21 of that). First the largest values, 8 threads a head (whole
// lines); then a thread has half of its lane's head's quarter of the row (lanes l and l + 16 share a head), loaded four
// ahead: lane l keeps the high parts, lane l + 16 the low ones, and they exchange the others. e4m3 queries have no low part.
template <bool Q8, bool kTree>
__device__ __noinline__ int stage_q(const MlaDecodeArgs& a, uint8_t* smem, uint32_t tmem, int t, int h0, int nh) {
  int32_t* tops = reinterpret_cast<int32_t*>(smem + kOffRow);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = 16 * (warp & 3) + (lane & 15), part = warp >> 2;      // 144 values
  const bool high = lane < 16, have = h < nh;
  const auto at_head = [&](int x) {                                   // of the tile, as an offset
    if constexpr (kTree)
      if (a.group > 1) return (int64_t)(t + x / a.H) * a.ldq + (int64_t)(x % a.H) * a.hsq;
    return (int64_t)t * a.ldq + (int64_t)(h0 + x) * a.hsq;
  };
  const int64_t off = at_head(min(h, nh - 1)) + 144 * part;
  uint32_t to = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16) + kColQ + 36 * part;
  int k = 0;
  if (Q8) {
    const uint4* q = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.q) + off);
    const bool keep = have && high;
    uint4 v[9];
#pragma unroll
    for (int j = 0; j < 9; ++j) v[j] = __ldg(q + j);                  // 16 values
#pragma unroll
    for (int j = 0; j < 9; ++j, to += 4) {
      const uint32_t w[4] = {keep ? v[j].x : 0, keep ? v[j].y : 0, keep ? v[j].z : 0, keep ? v[j].w : 0};
      keep_q(smem, to, w, part, j);
    }
  } else {
    const __nv_bfloat16* base = static_cast<const __nv_bfloat16*>(a.q);
    {
      const int th = threadIdx.x >> 3, sub = threadIdx.x & 7;
      const uint4* q = reinterpret_cast<const uint4*>(base + at_head(min(th, nh - 1))) + sub;
      uint4 v[9];
#pragma unroll
      for (int j = 0; j < 9; ++j) v[j] = __ldg(q + 8 * j);            // 8 values
      __nv_bfloat162 most = __floats2bfloat162_rn(0.0f, 0.0f);        // magnitudes, NaN kept
#pragma unroll
      for (int j = 0; j < 9; ++j) {
        const __nv_bfloat162* w = reinterpret_cast<const __nv_bfloat162*>(&v[j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) most = __hmax2_nan(most, __habs2(w[e]));
      }
      int top = *reinterpret_cast<int32_t*>(&most) & 0x7FFF7FFF;
      top = max(top & 0xFFFF, top >> 16);
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (sub == 0) tops[th] = top;
    }
    const uint4* q = reinterpret_cast<const uint4*>(base + off) + (high ? 0 : 1);
    uint4 next[4] = {__ldg(q), __ldg(q + 2), __ldg(q + 4), __ldg(q + 6)};
    named_bar(5, kSoftmax);
    const int top = tops[h];
    const int ex = top >> 7;                                          // the largest value's biased exponent
    if (ex != 0) k = max(min(ex - 134, 120), -120);
    // q 2^-k as halves by integer arithmetic on two magnitudes at a time: the exponent's bias changes by 112 + k, what is
    // below 2^-14 becomes 0. An infinite or NaN query value leaves its head no finite score: NaN, which e4m3 can carry (it
    // has no infinity)
    const uint32_t bias = static_cast<uint32_t>(-((112 + k) << 7)) & 0xFFFFu, down = bias | (bias << 16);
    const uint32_t keep = have ? 0xFFFFFFFFu : 0u, bad = have && ex == 255 ? 0x7E007E00u : 0u;
#pragma unroll 1
    for (int j = 0; j < 9; ++j, to += 4) {                            // 16 values, of which this thread has 8
      const uint4 g = next[0];
      next[0] = next[1], next[1] = next[2], next[2] = next[3];
      if (j < 5) next[3] = __ldg(q + 2 * j + 8);
      const uint32_t v[4] = {g.x, g.y, g.z, g.w};
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        split2_bf16((__viaddmax_s16x2_relu(v[i] & 0x7FFF7FFFu, down, 0u) << 3 | (v[i] & 0x80008000u) | bad) & keep,
                    hi[i], lo[i]);
      const uint32_t h01 = hi[0] | (hi[1] << 16), h23 = hi[2] | (hi[3] << 16);
      const uint32_t l01 = lo[0] | (lo[1] << 16), l23 = lo[2] | (lo[3] << 16);
      const uint32_t r01 = __shfl_xor_sync(0xffffffffu, high ? l01 : h01, 16);
      const uint32_t r23 = __shfl_xor_sync(0xffffffffu, high ? l23 : h23, 16);
      const uint32_t w[4] = {high ? h01 : r01, high ? h23 : r23, high ? r01 : l01, high ? r23 : l23};
      keep_q(smem, to, w, part, j);
    }
  }
  fence_proxy_async_smem();
  tmem_st_wait();
  return k;
}

// kTree: a row sees its first seq_len tokens and, of the 64 after them, those that its word names (the nodes on its path).
template <bool Q8, bool kTree>
__global__ void __launch_bounds__(kThreads, 1)
    mla_decode_kernel(const __grid_constant__ CUtensorMap mlat, const __grid_constant__ CUtensorMap mrope,
                      const __grid_constant__ MlaDecodeArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = blockIdx.x, tile = blockIdx.y;
  const int h0 = tile * kTileH, nh = min(kTileH, a.H - h0);
  const auto heads_of = [&](int t) { return kTree && a.group > 1 ? rows_led(a, t) * a.H : nh; };    // heads of its tile
  const uint32_t sbase = smem_u32(smem), bar = sbase + kOffBar;
  const Bars B = {bar,       bar + 40,  bar + 80,  bar + 88,  bar + 104, bar + 120, bar + 136,
                  bar + 152, bar + 160, bar + 168, bar + 176, bar + 192, bar + 208};
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kOffMisc);
  volatile int32_t* abort_flag = reinterpret_cast<volatile int32_t*>(smem + kOffMisc + 4);
  volatile int32_t* far = reinterpret_cast<volatile int32_t*>(smem + kOffMisc + 8);           // [2]
  int4* slots = reinterpret_cast<int4*>(smem + kOffSlot);
  int4* ring = reinterpret_cast<int4*>(smem + kOffRing);
  if (sbase & 1023) {                                    // the swizzled tiles need it; no static shared memory precedes
    if (tid == 0) raise_status(a.status, kErrCuda);
    return;
  }

  asm volatile("griddepcontrol.launch_dependents;");     // the join may be set up meanwhile (it waits for this grid's end)
  if (warp == kScoreWarp) {
    if (lane < 28) {                                     // the barriers, one a lane
      // full: every gather lane's copies and a warp's word
      const uint32_t n = lane < 5 ? 132 : lane < 10 ? 1 : lane == 10 || lane == 20 ? kSoftWarps : lane < 13 ? 2
                         : lane < 17 ? kSetWarps : lane < 20 ? 1 : lane == 21 ? 2 : kSetWarps;
      mbar_init(bar + 8 * lane, n);
    }
    if (lane < 2) far[lane] = 0;
    if (lane == 2) *abort_flag = 0;
    fence_barrier_init();
  } else if (warp == kValueWarp) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  Walk walk;
  if (!find_range<kTree>(a, cta, gridDim.x, reinterpret_cast<int32_t*>(smem + kOffPlan), smem + kOffKv, walk)) {
    if (warp == kValueWarp) {
      zero_rows<kTree>(a, cta, h0, nh, lane);
      tmem_dealloc(0, 512);
    }
    return;
  }
  tc_fence_after();
  constexpr uint32_t tmem = 0;                           // the whole of TMEM: its first lane and column
  if (*tmem_slot != tmem && tid == 0) {
    *abort_flag = 1;
    raise_status(a.status, kErrCuda);
  }

  if (warp >= kGatherWarp) {
    // ---------------------------------------------------------------- gather: warp w brings of a whole unit the latent
    // chunk w (warp 3 also the rope keys); otherwise of tokens 32 (w & 1) .. + 31 the chunks 2 (w >> 1), + 1 and half the rope
    const int w = warp - kGatherWarp, half = w & 1, pair = w >> 1;
    const int cols = a.indices != nullptr ? (a.n_idx + kUnit - 1) / kUnit : 0;
    int slot = 0, round = 0;                             // unit u's slot u % kSlots, and u / kSlots
    Segment s;
    bool ok = true;
    while (ok && walk_next<kTree>(a, walk, s)) {
      const int32_t* pages = a.table + (int64_t)(a.reqs != nullptr ? a.reqs[s.t] : s.t) * a.width;
      const int len = a.seq_lens != nullptr ? a.seq_lens[s.t] : 0x7fffffff;
      // the tokens all seen; those from there on by the rows' words
      const int plain = kTree ? min(len, 0x7fffff00) : len;
      const uint64_t word = kTree ? nodes_seen(a, s.t) : 0;
      const int32_t* idx = a.indices != nullptr ? a.indices + (int64_t)s.t * a.ld_idx : nullptr;
      int c0 = s.b0, c1 = s.b1;
      if (idx != nullptr) {                              // the row's planned share as units of list columns
        c0 = static_cast<int>((int64_t)s.b0 * cols / s.nb);
        c1 = static_cast<int>((int64_t)s.b1 * cols / s.nb);
      }
      // the page of position p (-1: none); the two list entries of a column at this lane (-1: none)
      auto page_of = [&](int p) { return p >= 0 && p / kPage < a.width ? pages[p / kPage] : -1; };
      auto entry = [&](int c, int i) {
        const int col = c * kUnit + 32 * i + lane;
        return idx != nullptr && c < c1 && col < a.n_idx ? idx[col] : -1;
      };
      // the first unit from c on that holds a token (c1: none), e0 and e1 the list entries of unit c; p: the position of
      // this lane's token of it (-1: none)
      auto find = [&](int c, int e0, int e1, int& p) {
        p = -1;
        if (idx == nullptr) {
          if (c < c1) p = c * kUnit + 32 * half + lane;
          if (p >= plain && (!kTree || p - plain >= 64 || !(word >> (p - plain) & 1))) p = -1;
          return min(c, c1);
        }
        while (c < c1) {
          e0 = e0 < len ? e0 : -1, e1 = e1 < len ? e1 : -1;
          if (__any_sync(0xffffffffu, e0 >= 0 || e1 >= 0)) {
            p = half ? e1 : e0;
            break;
          }
          ++c;
          e0 = entry(c, 0), e1 = entry(c, 1);
        }
        return c;
      };
      int p, pn;
      int c = find(c0, entry(c0, 0), entry(c0, 1), p);
      if (c >= c1) c = c0;                               // nothing selected: one empty unit gives the zeros
      int cn = find(c + 1, entry(c + 1, 0), entry(c + 1, 1), pn);
      int page = page_of(p);
      while (c < c1) {
        // the next unit's pages and the list entries of the one after it are on their way while this one is copied (of a
        // dense unit, which is a few instructions, the pages come after it)
        const int page_n = idx != nullptr ? page_of(pn) : -1, e0 = entry(cn + 1, 0), e1 = entry(cn + 1, 1);
        const uint32_t full = B.full + 8 * slot;
        const uint32_t dst = sbase + kOffKv + slot * kLat, rope = sbase + kOffRope + slot * kRope;
        const int64_t row = (int64_t)page * kPage + (p & (kPage - 1));
        const int from = page >= 0 && row < a.cache_rows ? static_cast<int>(row) : -1;
        const uint32_t present = __ballot_sync(0xffffffffu, from >= 0);
        // the slot is free when the values of the unit kSlots before have used it (its words were read before its scores)
        if (round > 0) ok = mbar_nap(B.empty + 8 * slot, (round - 1) & 1, abort_flag, a.status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        // A whole unit of a page (the same in every lane and warp) comes as tiles; a row's last units, and selected tokens,
        // row by row: rows that are not there have to be zeros (whatever the cache holds there, NaN too, would meet weight 0
        // in the value product).
        const int64_t y = (int64_t)page * kPage + ((c * kUnit) & (kPage - 1));
        const bool whole = idx == nullptr && (c + 1) * kUnit <= plain && page >= 0 && y + kUnit <= a.cache_rows;
        if (whole) {
          if (lane == 0) {
            mbar_arrive_expect_tx(full, w == 3 ? kChunk + kRope : kChunk);
            tma_load_2d(dst + w * kChunk, &mlat, 128 * w, static_cast<int>(y), full);
            if (w == 3) tma_load_2d(rope, &mrope, kDv, static_cast<int>(y), full);
          }
        } else {
          // 4 tokens a warp instruction, 128 of their latent bytes; rows 8 apart swizzle alike
          const uint32_t to[2] = {dst + 2 * pair * kChunk + sw128(32 * half + (lane >> 3), lane & 7),
                                  dst + 2 * pair * kChunk + sw128(32 * half + 4 + (lane >> 3), lane & 7)};
          const uint8_t* src = a.kv + 256 * pair + 16 * (lane & 7);
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const int rs = __shfl_sync(0xffffffffu, from, 4 * r + (lane >> 3));
            const uint8_t* at = src + (int64_t)max(rs, 0) * kDq;
            cp_async16(to[r & 1] + (r >> 1) * 1024, at, rs >= 0);
            cp_async16(to[r & 1] + (r >> 1) * 1024 + kChunk, at + 128, rs >= 0);
          }
#pragma unroll
          for (int r = 0; r < 32; r += 16) {             // 16 tokens a warp instruction: half of their 64 rope bytes
            const int rs = __shfl_sync(0xffffffffu, from, r + (lane >> 1)), g = 2 * pair + (lane & 1);
            cp_async16(rope + sw64(32 * half + r + (lane >> 1), g), a.kv + (int64_t)max(rs, 0) * kDq + kDv + 16 * g, rs >= 0);
          }
          cp_async_arrive_noinc(full);                   // fires when this thread's copies have landed
        }
        if (lane == 0) {
          int32_t* told = reinterpret_cast<int32_t*>(slots + slot);
          if (pair == 0) told[half] = static_cast<int32_t>(present);
          if (w == 0) told[2] = cn >= c1 ? kLast : kMore;
          if (kTree && w == 0) told[3] = c;
          mbar_arrive_n(full, whole ? 32 : 1);           // of a whole unit also for the lanes that copied nothing
        }
        if (++slot == kSlots) slot = 0, ++round;
        c = cn;
        p = pn;
        page = idx != nullptr ? page_n : page_of(p);
        cn = find(cn + 1, e0, e1, pn);
      }
    }
    cp_async_wait_all();
    if (!ok) drain_tiles(B.full, slot, round);
  } else if (warp == kValueWarp) {
    // ---------------------------------------------------------------- value products
    zero_rows<kTree>(a, cta, h0, nh, lane);
    __syncwarp();
    const bool leader = elect_lane();
    int u = 0, slot = 0, seg = 0;
    Segment s;
    bool ok = true;
    while (ok && walk_next<kTree>(a, walk, s)) {
      bool last = false, fresh = true;
      const int heads = (heads_of(s.t) + 15) & ~15;
      if (seg > 0) ok = mbar_nap(B.o_free, (seg - 1) & 1, abort_flag, a.status);      // the row before has been read
      while (!last) {
        const int set = u & 1;
        if (ok) ok = mbar_nap(B.p_full + 8 * set, (u >> 1) & 1, abort_flag, a.status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        last = ring[u & 7].z != kMore;
        tc_fence_after();
        issue_values(B, sbase, slot, set, heads, fresh, leader);
        fresh = false;
        ++u;
        if (++slot == kSlots) slot = 0;
      }
      if (ok && leader) tc_commit(B.o_full);
      ++seg;
    }
    if (leader) tc_commit(B.drain);                      // everything issued here has completed when this arrives
  } else if (warp == kScoreWarp) {
    // ---------------------------------------------------------------- score products
    const bool leader = elect_lane();
    int u = 0, slot = 0, round = 0, seg = 0;
    Segment s;
    bool ok = true;
    while (ok && walk_next<kTree>(a, walk, s)) {
      bool last = false;
      const int first = u;
      while (!last) {
        ok = mbar_nap(B.full + 8 * slot, round & 1, abort_flag, a.status);
        if (ok && u > 1) ok = mbar_nap(B.s_empty + 8 * (u & 1), ((u >> 1) - 1) & 1, abort_flag, a.status);
        if (ok && u == first) ok = mbar_nap(B.q_full, seg & 1, abort_flag, a.status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        fence_proxy_async_smem();                        // rows that threads copied -> the tensor core
        tc_fence_after();
        // the unit's words, by unit: entry u & 7 was last read for the values of unit u - 8, which are done (the set that
        // has read S of u - 2 waited for those of u - 6 before it gave the weights of u - 4)
        const int4 word = slots[slot];
        last = word.z != kMore;
        if (leader) {
          ring[u & 7] = word;
          mbar_arrive(B.s_full + 8 * (u & 1));
        }
        issue_scores(B, sbase, slot, u & 1, leader);
        ++u;
        if (++slot == kSlots) slot = 0, ++round;
      }
      // the set that has no further unit of the row is told so, once it has read its last one
      if (ok && u > first + 1) ok = mbar_nap(B.s_empty + 8 * (u & 1), ((u >> 1) - 1) & 1, abort_flag, a.status);
      ok = __all_sync(0xffffffffu, ok);
      if (ok && leader) {
        ring[u & 7] = make_int4(0, 0, kEnd, 0);
        mbar_arrive_n(B.s_full + 8 * (u & 1), 2);
      }
      ++seg;
    }
    if (leader) tc_commit(B.drain);
    const unsigned long long t0 = globaltimer();
    while (!mbar_try_wait(B.drain, 0) && globaltimer() - t0 <= 2 * kWaitNs) {}
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- softmax (warps 0-15): 16 tokens of a head a thread
    const int quarter = warp & 3, half = (warp >> 2) & 1, set = warp >> 3, part = lane >> 4;
    const int mine = 16 * quarter + (lane & 15);
    const uint32_t tq = tmem + (static_cast<uint32_t>(32 * quarter) << 16);
    float* refs = reinterpret_cast<float*>(smem + kOffRef);
    float* rows = reinterpret_cast<float*>(smem + kOffRow);
    float* sums = reinterpret_cast<float*>(smem + kOffSum);
    const uint32_t other = 8 * (set ^ 1), own = 8 * set;
    const bool teller = warp < 4 && lane < 16;           // one thread a head
    if (warp < 4) tmem_st_x4(tq + kColV, 0x7478u);
    int u0 = 0, seg = 0, events = 0;                     // the row's first unit
    Segment s;
    bool more = walk_next<kTree>(a, walk, s), ok = true;
    int heads = heads_of(s.t);
    if (teller) refs[mine] = mine < heads ? kNone : 0.0f;
    int k = stage_q<Q8, kTree>(a, smem, tmem, s.t, h0, heads);     // exponent of head mine's query scale
    tc_fence_before();
    warp_arrive(B.q_full, lane);
    named_bar(5, kSoftmax);                              // every head's reference is written
    while (more) {
      const float c = mine < heads ? a.bmm1 * kLog2e * __uint_as_float(static_cast<uint32_t>(127 + k) << 23) : 0.0f;
      const float c_own = part ? 0.0625f * c : c, c_got = part ? c : 0.0625f * c;
      float l = 0.0f, ref = mine < heads ? kNone : 0.0f; // the sum of the thread's weights, the reference it stands against
      int u = u0 + ((set ^ u0) & 1);
      // in a shared tile, the nodes that this head's row sees, behind `plain` tokens
      const bool shared_tile = kTree && a.group > 1;
      const uint64_t nodes = shared_tile && mine < heads ? a.ancestors[s.t + mine / a.H] : 0;
      const int plain = shared_tile ? min(a.seq_lens[s.t], 0x7fffff00) : 0;
      while (true) {
        ok = mbar_nap(B.s_full + own, events & 1, abort_flag, a.status);
        ++events;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const int4 word = ring[u & 7];
        if (word.z == kEnd) {
          u0 = u;
          break;
        }
        tc_fence_after();
        float v[16];                                     // base-2 scores; tokens not there: -inf
        {
          float x[32];
          tmem_ld_32x32b_x32(tq + kColS + kUnit * set + 32 * half, x);
          tmem_ld_wait();
          tc_fence_before();
          warp_arrive(B.s_empty + own, lane);
          // lanes l and l + 16 have the high and the low part of 32 tokens: each gives the other the half that it does not keep
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float got = __shfl_xor_sync(0xffffffffu, part ? x[i] : x[16 + i], 16);
            v[i] = fmaf(part ? x[16 + i] : x[i], c_own, got * c_got);
          }
        }
        uint32_t present = static_cast<uint32_t>(half ? word.y : word.x);
        if (shared_tile && kUnit * word.w + kUnit > plain) {
          const int from = kUnit * word.w + 32 * half - plain;         // the node of the thread's first token (< 0: context)
          const uint64_t seen = from >= 64 ? 0 : from >= 0 ? nodes >> from : from <= -32 ? ~uint64_t{0}
                                                                          : nodes << -from | ((uint64_t{1} << -from) - 1);
          present &= static_cast<uint32_t>(seen);
          // a token that some rows of the tile see and others do not: whatever its latent values are, the others must not meet
          // NaN times weight 0. Its scores have been formed (NaN for the rows that see it): zeros in the value product do
          uint4* rows16 = reinterpret_cast<uint4*>(smem + kOffKv + (u % kSlots) * kLat);
#pragma unroll 1
          for (int i = 32 * (warp & 7) + lane; i < kLat / 16; i += 32 * kSetWarps) {
            uint4 b = rows16[i];
            const uint32_t n0 = __vcmpeq4(b.x & 0x7F7F7F7Fu, 0x7F7F7F7Fu), n1 = __vcmpeq4(b.y & 0x7F7F7F7Fu, 0x7F7F7F7Fu);
            const uint32_t n2 = __vcmpeq4(b.z & 0x7F7F7F7Fu, 0x7F7F7F7Fu), n3 = __vcmpeq4(b.w & 0x7F7F7F7Fu, 0x7F7F7F7Fu);
            if (n0 | n1 | n2 | n3) rows16[i] = make_uint4(b.x & ~n0, b.y & ~n1, b.z & ~n2, b.w & ~n3);
          }
        }
        if (present != 0xffffffffu) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (!((present >> (16 * part + i)) & 1)) v[i] = kNone;
        }
        float m = kNone;                                 // the largest of the head's 32 tokens, NaN ignored
#pragma unroll
        for (int i = 0; i < 16; ++i) m = fmaxf(m, v[i]);
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
        // the references after the unit before (the other set's)
        if (u != u0) {
          if (!mbar_nap(B.ref_ok + other, ((u - 1) >> 1) & 1, abort_flag, a.status)) ok = false;
          const float now = refs[mine];
          if (now != ref) {
            if (ref != kNone) l *= exp2f(ref - now);
            ref = now;
          }
        }
        // the set agrees on the rare path (a failed wait travels the same way): a head without a reference, or with scores
        // more than kMaxRise above it
        if (__any_sync(0xffffffffu, (ref == kNone ? m > kNone : m - ref > kMaxRise) || !ok) && lane == 0) far[set] = 1;
        warp_arrive(B.agree + own, lane);
        uint32_t wh[4], wl[4];
        float sum, unit;
        int eb;
        bool asked = false;
#pragma unroll 1
        while (true) {
          // weights 2^(score - E + 8) with an exponent E for 32 tokens of a head: the ceiling of the largest of their scores
          // above the head's reference. 2^(E - 8) is their block scale in the product and their weight in the sums; the
          // e4m3 pairs keep 8 bits down to 2^-14 of that largest.
          const float base = ref == kNone ? 0.0f : ref;
          const float e = fminf(fmaxf(ceilf(m - base), kMinE), kMaxRise);
          eb = static_cast<int>(e) + 119;                // biased exponent of 2^(E - 8)
          unit = __uint_as_float(static_cast<uint32_t>(eb) << 23);
          const float off = 8.0f - e;
          uint64_t total = f2pack(0.0f, 0.0f);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t ph[2], pl[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float w0 = ex2_fast(v[4 * i + 2 * j] - base + off), w1 = ex2_fast(v[4 * i + 2 * j + 1] - base + off);
              total = add2(total, f2pack(w0, w1));
              split2(w0, w1, ph[j], pl[j]);
            }
            wh[i] = ph[0] | (ph[1] << 16);
            wl[i] = pl[0] | (pl[1] << 16);
          }
          float t0, t1;
          f2unpack(total, t0, t1);
          sum = t0 + t1;
          if (asked) break;
          asked = true;
          if (!mbar_nap(B.agree + own, (u >> 1) & 1, abort_flag, a.status)) ok = false;
          if (!__any_sync(0xffffffffu, far[set] != 0)) break;
          // new references: the ceiling of this unit's largest score; what has been accumulated is rescaled
          if (lane < 16) rows[64 * half + mine] = m;
          warp_arrive(B.slow + own, lane);
          if (!mbar_nap(B.slow + own, 0, abort_flag, a.status)) ok = false;
          const float most = fmaxf(rows[mine], rows[64 + mine]);
          const bool move = ref == kNone ? most > kNone : most - ref > kMaxRise;
          const float now = move ? ceilf(most) : ref;
          const float f = move && ref != kNone ? exp2f(ref - now) : 1.0f;
          if (half == 0 && lane < 16) {
            refs[mine] = now;
            rows[128 + mine] = f;
          }
          if (half == 0 && quarter == 0 && lane == 0) far[set] = 0;
          warp_arrive(B.slow + own, lane);
          if (!mbar_nap(B.slow + own, 1, abort_flag, a.status)) ok = false;
          ref = now;
          l *= f;
          if (u != u0) {
            if (!mbar_nap(B.pv_done + other, ((u - 1) >> 1) & 1, abort_flag, a.status)) ok = false;
            tc_fence_after();
#pragma unroll 1
            for (int d = 0; d < 8; ++d) {                // 4 tiles of 128 dims, 16 of the warp's 32 heads at a time
              const int h = 32 * half + 16 * (d & 1);
              const uint32_t at = tq + kColO + 64 * (d >> 1) + h;
              float o[16];
              tmem_ld_x16(at, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] *= rows[128 + h + i];
              tmem_st_x16(at, o);
            }
            tmem_st_wait();
          }
        }
        warp_arrive(B.ref_ok + own, lane);
        l = fmaf(sum, unit, l);
        // the values of the set's unit before have read its P
        if (u >= 2 && !mbar_nap(B.pv_done + own, ((u >> 1) - 1) & 1, abort_flag, a.status)) ok = false;
        if (lane < 16)                                   // V's scale is 2^-7
          smem[kOffSf + 16 * (mine & 31) + 8 * set + 4 * (mine >> 5) + half] = static_cast<uint8_t>(eb + 7);
        const int at = sw64(mine, 2 * half + part);
        *reinterpret_cast<uint4*>(smem + kOffRope + (u % kSlots) * kRope + at) = make_uint4(wh[0], wh[1], wh[2], wh[3]);
        *reinterpret_cast<uint4*>(smem + kOffPlo + set * kRope + at) = make_uint4(wl[0], wl[1], wl[2], wl[3]);
        fence_proxy_async_smem();
        tc_fence_before();
        warp_arrive(B.p_full + own, lane);
        if (word.z == kLast) {
          u0 = u + 1;
          break;
        }
        u += 2;
      }
      // ---- the row's sums, the next row's query, then the accumulators ----
      if (named_bar_or(5, kSoftmax, !ok)) break;
      const float last_ref = refs[mine];
      if (ref != last_ref && ref != kNone) l *= exp2f(ref - last_ref);
      ref = last_ref;
      l += __shfl_xor_sync(0xffffffffu, l, 16);
      if (lane < 16) rows[64 * (2 * set + half) + mine] = l;
      named_bar(5, kSoftmax);
      float total = rows[mine] + rows[64 + mine] + rows[128 + mine] + rows[192 + mine];
      if (ref == kNone && total == total) total = 0.0f;                              // no token
      const Segment done = s;
      const int done_heads = heads;
      more = walk_next<kTree>(a, walk, s);
      if (more) heads = heads_of(s.t);
      if (teller) {
        sums[mine] = total == 0.0f ? 0.0f : a.bmm2 / total;                          // a NaN sum stays one
        refs[mine] = mine < heads ? kNone : 0.0f;
      }
      if (more) {
        if (!Q8) named_bar(5, kSoftmax);                 // the sums are read: their place takes the query's maxima
        k = stage_q<Q8, kTree>(a, smem, tmem, s.t, h0, heads);
        tc_fence_before();
        warp_arrive(B.q_full, lane);
      }
      ok = mbar_nap(B.o_full, seg & 1, abort_flag, a.status);
      if (named_bar_or(5, kSoftmax, !ok)) break;
      tc_fence_after();
      const bool whole = done.b0 == 0 && done.b1 == done.nb;
      const int slot = 2 * cta + (seg == 0 ? 0 : 1);
      if (teller) {
        if (!whole) part_ml(a, tile, slot)[mine] = make_float2(ref, total);
        else if (a.lse != nullptr && mine < done_heads)
          a.lse[(int64_t)done.t * a.H + h0 + mine] =
              total == 0.0f ? kNone : ((ref == kNone ? 0.0f : ref) + log2f(total)) * kLn2;
        if (mine == 0 && tile == 0) {
          if (done.b0 == 0) a.rows[done.t].first = cta, a.rows[done.t].first_slot = slot;
          if (done.b1 == done.nb) a.rows[done.t].last = cta;
        }
      }
      const int hb = 16 * (warp >> 2);
      if (!whole) {                                      // a lane has one dim of 16 heads: 128 bytes a warp and head
        float* po = part_o(a, tile, slot) + hb * kDv + 32 * quarter + lane;
#pragma unroll 1
        for (int d = 0; d < 4 && hb < done_heads; ++d, po += 128) {
          float o[16];
          tmem_ld_x16(tq + kColO + 64 * d + hb, o);
          tmem_ld_wait();
#pragma unroll
          for (int h = 0; h < 16; ++h) po[h * kDv] = o[h];
        }
      }
      // a lane has one dim of 4 heads; crossed with its 3 neighbours, 4 dims of head (lane & 3)
      const int e = lane & 3, dim = 32 * quarter + (lane & 28);
      __nv_bfloat16* out = a.out + ((int64_t)done.t * a.H + h0 + hb + e) * kDv + dim;
#pragma unroll 1
      for (int i = 0; i < 16 && hb + i < done_heads && whole; i += 4) {      // 4 heads x 4 tiles of 128 dims
        float o[4][4];
#pragma unroll
        for (int d = 0; d < 4; ++d) tmem_ld_x4(tq + kColO + 64 * d + hb + i, o[d]);
        tmem_ld_wait();
        const float inv = sums[hb + i + e];
        const bool have = hb + i + e < done_heads;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          cross4(o[d], lane);
          const __nv_bfloat162 v0 = __floats2bfloat162_rn(o[d][0] * inv, o[d][1] * inv);
          const __nv_bfloat162 v1 = __floats2bfloat162_rn(o[d][2] * inv, o[d][3] * inv);
          if (have)
            *reinterpret_cast<uint2*>(out + 128 * d) =
                make_uint2(*reinterpret_cast<const uint32_t*>(&v0), *reinterpret_cast<const uint32_t*>(&v1));
        }
        out += 4 * kDv;
      }
      tc_fence_before();
      warp_arrive(B.o_free, lane);
      ++seg;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kValueWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins a row's parts. gridDim.z == 4: one CTA of W = 4 or 16 warps per (row, head, 128 output values), warp w taking parts
// w, w + W, ...; gridDim.z == 1: one of 4 warps per (row, head), a warp 128 values and all the parts (chosen by the
// number of CTAs, below). Rows that one CTA finished, or that have no token, are left alone, and those without a valid
// record: the status tells of them.
constexpr int kJoinWarps = 16;
template <bool kTree>
__global__ void __launch_bounds__(32 * kJoinWarps) mla_join_kernel(const __grid_constant__ MlaDecodeArgs a) {
  __shared__ float4 so[kJoinWarps][32];
  __shared__ float sl[kJoinWarps];
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y, tile = h / kTileH;
  const int64_t t0 = kTree ? leader_of(a, static_cast<int>(t)) : t;                       // the row whose tile this one shares
  const int hh = static_cast<int>((t - t0) * a.H) + h - tile * kTileH;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int units = row_units<kTree>(a, static_cast<int>(t0));     // of the inputs alone
  asm volatile("griddepcontrol.wait;" ::: "memory");       // the parts are written
  if (units == 0) return;
  const MlaRowParts rp = a.rows[t0];
  if (!rp.valid()) {
    if (threadIdx.x == 0) raise_status(a.status, kErrTimeout);
    return;
  }
  if (rp.first == rp.last) return;
  const bool spread = gridDim.z == 4;
  const int parts = rp.last - rp.first + 1, dim = 128 * (spread ? blockIdx.z : warp);
  const int step = spread ? static_cast<int>(blockDim.x) / 32 : 1;
  float m = kNone;
  for (int i = lane; i < parts; i += 32) m = fmaxf(m, part_ml(a, tile, rp.slot(i))[hh].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float l = 0.0f;
  const float mz = m == kNone ? 0.0f : m;                // a part without a token (or all NaN) has m = -inf, f = 0
#pragma unroll 4
  for (int i = spread ? warp : 0; i < parts; i += step) {
    const float2 ml = part_ml(a, tile, rp.slot(i))[hh];
    const float f = exp2f(ml.x - mz);
    const float4 v = reinterpret_cast<const float4*>(part_o(a, tile, rp.slot(i)) + hh * kDv + dim)[lane];
    s.x = fmaf(f, v.x, s.x), s.y = fmaf(f, v.y, s.y);
    s.z = fmaf(f, v.z, s.z), s.w = fmaf(f, v.w, s.w);
    l = fmaf(f, ml.y, l);
  }
  if (spread) {
    so[warp][lane] = s;
    if (lane == 0) sl[warp] = l;
    __syncthreads();
    if (warp != 0) return;
    const int warps = min(parts, step);
#pragma unroll 4
    for (int w = 1; w < warps; ++w) {
      l += sl[w];
      const float4 v = so[w][lane];
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
  }
  const float inv = l == 0.0f ? 0.0f : a.bmm2 / l;       // a NaN sum stays one
  const __nv_bfloat162 lo = __floats2bfloat162_rn(s.x * inv, s.y * inv), hi = __floats2bfloat162_rn(s.z * inv, s.w * inv);
  reinterpret_cast<uint2*>(a.out + (t * a.H + h) * kDv + dim)[lane] =
      make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
  if (a.lse != nullptr && dim == 0 && lane == 0) a.lse[t * a.H + h] = l == 0.0f ? kNone : (mz + log2f(l)) * kLn2;
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
  if (a.T < 0 || a.T > 0x7fffffff || a.H <= 0 || a.H > 128) return kErrArgs;
  if (a.T == 0) return kOk;                              // empty tensors have no address: the others are not looked at
  if (a.R <= 0 || a.width <= 0 || a.cache_rows <= 0 || a.cache_rows > 0x7fffffff ||
      (a.indices == nullptr && a.seq_lens == nullptr) || (a.ancestors != nullptr && a.indices != nullptr) ||
      (a.indices != nullptr && (a.n_idx < 0 || (a.T > 1 && a.ld_idx < a.n_idx))) || (a.reqs == nullptr && a.T > a.R))
    return kErrArgs;
  const int64_t most =                                   // units of a row
      a.indices != nullptr ? (a.n_idx + kUnit - 1) / kUnit : (int64_t)(kPage / kUnit) * a.width;
  if (a.T * (most + kRowCost) > 0x7fffffff) return kErrArgs;
  if (a.q == nullptr || a.kv == nullptr || a.table == nullptr || a.out == nullptr || ws == nullptr ||
      !aligned(a.q, 16) || !aligned(a.kv, 16) || !aligned(a.out, 16) || !aligned(ws, 256) || !aligned(a.ancestors, 8))
    return kErrArgs;
  // one row has no row stride, one head no head stride: what the caller's tensor states there is not used
  if (a.T > 1 && ((a.ldq * eb) % 16 != 0 || a.ldq < kDq)) return kErrArgs;
  if (a.H > 1 && ((a.hsq * eb) % 16 != 0 || a.hsq < kDq)) return kErrArgs;
  if (ws_bytes < mla_decode_workspace_bytes(a.T, a.H)) return kErrWorkspace;
  const int64_t tiles = tiles_of(a.H), slots = tiles * 2 * kMaxCtas;
  uint8_t* p = static_cast<uint8_t*>(ws);
  a.rows = reinterpret_cast<MlaRowParts*>(p);
  p += up256(a.T * (int64_t)sizeof(MlaRowParts));
  a.part_ml = reinterpret_cast<float2*>(p);
  p += up256(slots * kTileH * 8);
  a.part_o = reinterpret_cast<float*>(p);
  const bool tree = a.ancestors != nullptr;
  a.group = tree && a.H <= kTileH / 2 ? kTileH / a.H : 1;
  auto* kernel = tree ? (a.q_e4m3 ? mla_decode_kernel<true, true> : mla_decode_kernel<false, true>)
                      : (a.q_e4m3 ? mla_decode_kernel<true, false> : mla_decode_kernel<false, false>);
  static OncePerDevice attr[4];
  int device = 0;
  const auto set = [&] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) == cudaSuccess;
  };
  if (cudaGetDevice(&device) != cudaSuccess || !attr[2 * tree + a.q_e4m3].done(device, set)) return kErrCuda;
  CUtensorMap mlat = {}, mrope = {};
  if (a.indices == nullptr) {                            // selected tokens are copied row by row
    const int u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
    int rc = make_map_2d_ex(&mlat, u8, a.kv, a.cache_rows, kDq, kDq, 128, kUnit, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc == kOk) rc = make_map_2d_ex(&mrope, u8, a.kv, a.cache_rows, kDq, kDq, 64, kUnit, CU_TENSOR_MAP_SWIZZLE_64B);
    if (rc != kOk) return rc;
  }
  kernel<<<dim3((unsigned)(kMaxCtas / tiles), (unsigned)tiles), kThreads, kSmem, stream>>>(mlat, mrope, a);
  if (cudaGetLastError() != cudaSuccess) return kErrCuda;
  // few rows are cut into many parts each: their CTAs are spread over the parts and the output values. 64 heads, 1 x 131,072
  // tokens: 82 us in all with one CTA a head, 49 with four, 41 with four of 16 warps; 48 rows of 16 heads: 52, 51 and 60;
  // 96 rows of 64: 64 with one, 80 with four
  const unsigned z = a.T * a.H <= 8 * kMaxCtas ? 4 : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.T, (unsigned)a.H, z);
  cfg.blockDim = dim3(a.T * a.H <= kMaxCtas ? 32 * kJoinWarps : 128);
  cfg.stream = stream;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, tree ? mla_join_kernel<true> : mla_join_kernel<false>, a) == cudaSuccess ? kOk : kErrCuda;
}

}  // namespace ssb
