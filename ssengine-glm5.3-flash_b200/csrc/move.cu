// Rows of cache views moved by lists, for sm_100a: beams' states and pages reordered in place, pages forked, accepted
// tokens compacted.
//
// A view is rows of `nbytes` bytes, `stride` apart. For every view, by its list l, and every group g: row dst[l][g][i] takes
// what row src[l][g][i] held before the call, i < n. A group's sources are all read before its rows are written, slice by
// slice: a CTA has one slice of a view's row for one group, 16-byte pieces of every moved row in registers, a barrier, then
// the stores; so the rows of a group may be permuted in place and nothing but the moved bytes is touched.
// Bound: HBM, a read of each source and a write of each moved row. 8 groups of 4 beams, three layers' 4.3 MB states and
// their current pages: 100 us, 0.91 of the copy rate. 64 requests of up to 6 tokens in three layers' latent rows: 7 to 10 us,
// nearly all of it the call's on the host.
#include "common.cuh"
#include "ops.h"

namespace ssb {
namespace {

constexpr int kMoveThreads = 256;
constexpr int kMovePieces = 8;                         // 16-byte pieces a thread
constexpr int kMoveRows = 64;                          // rows of a group

// Kernel parameters are copied at every launch: few views come in a small table.
template <int V>
struct MoveTable {
  MoveView v[V];
};

template <int V>
__global__ void __launch_bounds__(kMoveThreads) move_rows_kernel(const __grid_constant__ MoveTable<V> table,
                                                                 const __grid_constant__ MoveArgs a) {
  __shared__ int32_t ids[2][kMoveRows];
  __shared__ int32_t moved;
  const int tid = threadIdx.x;
  const int64_t item = blockIdx.x;
  int lo = 0, hi = a.views - 1;                        // the last view whose first item is not past this one
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (table.v[mid].first <= item) lo = mid; else hi = mid - 1;
  }
  const MoveView& v = table.v[lo];
  const int64_t slices = (v.nbytes + a.slice - 1) / a.slice;
  const int64_t g = (item - v.first) / slices, slice = item - v.first - g * slices;
  const int64_t at = (v.list * a.groups + g) * a.n;

  // the rows to move: both ids given, within the rows and different, and the first such of its destination
  if (tid < 32) {
    int count = 0;
    for (int i0 = 0; i0 < a.n; i0 += 32) {
      const int i = i0 + tid;
      const int32_t from = i < a.n ? a.src[at + i] : -1, to = i < a.n ? a.dst[at + i] : -1;
      bool go = from >= 0 && to >= 0;
      if (go && (from >= v.rows || to >= v.rows)) {
        go = false;
        raise_status(a.status, kErrArgs);
      }
      for (int j = 0; go && j < i; ++j)                // a source past the rows makes no entry
        if (a.dst[at + j] == to && a.src[at + j] >= 0 && a.src[at + j] < v.rows) go = false;
      go = go && from != to;
      const uint32_t mask = __ballot_sync(0xffffffffu, go);
      if (go) {
        const int k = count + __popc(mask & ((1u << tid) - 1));
        ids[0][k] = from, ids[1][k] = to;
      }
      count += __popc(mask);
    }
    if (tid == 0) moved = count;
  }
  __syncthreads();
  const int m = moved;
  if (m == 0) return;
  const int64_t offset = slice * a.slice;
  const int pieces = static_cast<int>(min(static_cast<int64_t>(a.slice), v.nbytes - offset) / 16), total = m * pieces;
  uint4 held[kMovePieces];
#pragma unroll
  for (int k = 0; k < kMovePieces; ++k) {
    const int i = tid + k * kMoveThreads, row = i / pieces;
    if (i < total)
      held[k] = *reinterpret_cast<const uint4*>(v.base + ids[0][row] * v.stride + offset + 16 * (i - row * pieces));
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kMovePieces; ++k) {
    const int i = tid + k * kMoveThreads, row = i / pieces;
    if (i < total)
      __stcs(reinterpret_cast<uint4*>(v.base + ids[1][row] * v.stride + offset + 16 * (i - row * pieces)), held[k]);
  }
}

}  // namespace

int launch_move_rows(const MoveView* views, const MoveArgs& a_in, cudaStream_t stream) {
  MoveArgs a = a_in;
  if (a.views < 0 || a.views > kMoveViews || a.lists < 0 || a.groups < 0 || a.n < 0 || a.n > kMoveRows) return kErrArgs;
  if (a.views == 0 || a.groups == 0 || a.n == 0) return kOk;
  if (views == nullptr || a.src == nullptr || a.dst == nullptr || (reinterpret_cast<uintptr_t>(a.src) & 3) ||
      (reinterpret_cast<uintptr_t>(a.dst) & 3) || a.lists * a.groups > (int64_t{1} << 40))
    return kErrArgs;
  // a CTA's pieces of all rows of a group fit its registers
  int rows = 1;
  while (rows < a.n) rows *= 2;
  a.slice = kMoveThreads * kMovePieces * 16 / rows;
  MoveTable<kMoveViews> t;
  int64_t items = 0;
  for (int i = 0; i < a.views; ++i) {
    const MoveView& v = views[i];
    if (v.base == nullptr || (reinterpret_cast<uintptr_t>(v.base) & 15) || v.nbytes <= 0 || v.nbytes % 16 != 0 ||
        v.rows < 0 || v.list < 0 || v.list >= a.lists ||
        (v.rows > 1 && (v.stride % 16 != 0 || v.stride < v.nbytes)))
      return kErrArgs;
    t.v[i] = v;
    t.v[i].first = items;
    const int64_t slices = (v.nbytes + a.slice - 1) / a.slice;
    if (slices > 0x7fffffff / a.groups) return kErrArgs;
    items += slices * a.groups;
    if (items > 0x7fffffff) return kErrArgs;
  }
  constexpr int kFew = 8;
  if (a.views <= kFew) {
    MoveTable<kFew> few;
    for (int i = 0; i < a.views; ++i) few.v[i] = t.v[i];
    move_rows_kernel<<<static_cast<unsigned>(items), kMoveThreads, 0, stream>>>(few, a);
  } else {
    move_rows_kernel<<<static_cast<unsigned>(items), kMoveThreads, 0, stream>>>(t, a);
  }
  return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
}

}  // namespace ssb
