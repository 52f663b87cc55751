"""The canonical top-k kernel's own source on CPU threads, with one warp late after every block barrier.

A kernel whose threads agree on its shared counters gives the same result whichever warp is late; one that resets a
counter while a late warp has yet to read it loses the agreement (the warps then meet at different barriers, and columns
are stored past their lists). Each block barrier, warp shuffle and shared atomic of `csrc/topk.cu` becomes its C++
counterpart over 256 threads; the shared lists stand between guard words."""

import re
import subprocess

import numpy as np
import pytest

from oracle import topk as otopk

HOST = r"""
#include <algorithm>
#include <atomic>
#include <barrier>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <memory>
#include <thread>
#include <unistd.h>
#include <vector>
using std::min;
struct Dim { int x; };
thread_local Dim threadIdx;
static Dim blockIdx = {0}, gridDim = {1};
struct float4 { float x, y, z, w; };
static float4 make_float4(float x, float y, float z, float w) { return {x, y, z, w}; }
static int late_warp = -1;
static std::unique_ptr<std::barrier<>> block;
static std::vector<std::unique_ptr<std::barrier<>>> warps;
static uint32_t lanes[8][32];
static void __syncthreads() {
  block->arrive_and_wait();
  if (threadIdx.x >> 5 == late_warp) usleep(1000);
}
template <class F>
static uint32_t warp_op(uint32_t v, F f) {
  const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
  lanes[w][l] = v;
  warps[w]->arrive_and_wait();
  const uint32_t r = f(lanes[w], l);
  warps[w]->arrive_and_wait();
  return r;
}
static uint32_t __shfl_up_sync(uint32_t, uint32_t v, int d) {
  return warp_op(v, [d](uint32_t* a, int l) { return l >= d ? a[l - d] : a[l]; });
}
static uint32_t __shfl_sync(uint32_t, uint32_t v, int s) { return warp_op(v, [s](uint32_t* a, int) { return a[s]; }); }
static uint32_t __ballot_sync(uint32_t, bool v) {
  return warp_op(v, [](uint32_t* a, int) {
    uint32_t r = 0;
    for (int i = 0; i < 32; ++i) r |= a[i] << i;
    return r;
  });
}
static uint32_t atomicAdd(uint32_t* p, uint32_t v) { return __atomic_fetch_add(p, v, __ATOMIC_SEQ_CST); }
static uint32_t __float_as_uint(float f) { uint32_t u; std::memcpy(&u, &f, 4); return u; }
static int __popc(uint32_t v) { return __builtin_popcount(v); }
template <class T>
static T __ldg(const T* p) { return *p; }
static uint32_t* dynamic_shared;
@KERNEL@
int main(int argc, char** argv) {
  // argv: input file {rows, ld, k, cache}, ks, ke, logits; output file; the late warp
  late_warp = std::atoi(argv[3]);
  FILE* f = std::fopen(argv[1], "rb");
  int32_t head[4];
  if (std::fread(head, 4, 4, f) != 4) return 2;
  const int rows = head[0], ld = head[1], k = head[2], cache = head[3];
  std::vector<int32_t> ks(rows), ke(rows), out(rows * k + 2, -7);
  std::vector<float> logits(rows * ld);
  if (std::fread(ks.data(), 4, rows, f) != size_t(rows) || std::fread(ke.data(), 4, rows, f) != size_t(rows) ||
      std::fread(logits.data(), 4, logits.size(), f) != logits.size())
    return 2;
  std::fclose(f);
  const size_t words = cache + kCand + kMaxK, guard = 1 << 16;
  std::vector<uint32_t> shared(words + guard, 0xC0FFEEu);
  dynamic_shared = shared.data();
  block = std::make_unique<std::barrier<>>(kTopkThreads);
  for (int w = 0; w < kTopkWarps; ++w) warps.push_back(std::make_unique<std::barrier<>>(32));
  std::vector<std::thread> threads;
  for (int t = 0; t < kTopkThreads; ++t)
    threads.emplace_back([&, t] {
      threadIdx.x = t;
      topk_canon_kernel(logits.data(), rows, ld, ks.data(), ke.data(), k, out.data() + 1, cache);
      warps[t >> 5]->arrive_and_drop();
      block->arrive_and_drop();
    });
  for (auto& t : threads) t.join();
  for (size_t i = words; i < shared.size(); ++i)
    if (shared[i] != 0xC0FFEEu) return std::printf("a store %zu words past the lists\n", i - words), 1;
  if (out.front() != -7 || out.back() != -7) return std::puts("a store outside the output"), 1;
  f = std::fopen(argv[2], "wb");
  std::fwrite(out.data() + 1, 4, rows * k, f);
  std::fclose(f);
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    from ssengine_b200 import _build

    src = (_build.CSRC / "topk.cu").read_text()
    body = src[src.index("constexpr int kTopkThreads"):src.index("}  // namespace\n")]
    body = body.replace("extern __shared__ uint32_t sm_keys[];", "uint32_t* sm_keys = dynamic_shared;")
    body = re.sub(r"__launch_bounds__\([^)]*\)", "", body)
    for word, to in (("__shared__", "static"), ("__global__", "static"), ("SSB_DEVICE", "static"),
                     ("__restrict__", ""), ("#pragma unroll", "")):
        body = body.replace(word, to)
    d = tmp_path_factory.mktemp("topk")
    (d / "host.cpp").write_text(HOST.replace("@KERNEL@", body))
    subprocess.run(["g++", "-std=c++20", "-O0", "-pthread", "-w", "-o", str(d / "host"), str(d / "host.cpp")], check=True)
    return d / "host"


def rows_with_ties(rng, width, k):
    """Ordinary rows between rows whose threshold value is held by more columns than are needed: a few, more than the
    tie buffer holds, more than the candidate list holds."""
    out = []
    for ties in (0, 40, 0, 3000, 0, width, 0, 7, 0):
        row = rng.standard_normal(width).astype(np.float32)
        if ties:
            at = rng.permutation(width)[:ties + k // 2]
            row[at[:ties]] = 5.0
            row[at[ties:]] = 6.0 + rng.random(at[ties:].size)
        out.append(row)
    return np.stack(out)


# a small row cache: every row takes the long form; a large one: none does
@pytest.mark.parametrize("late,cache", [(-1, 64), (0, 64), (1, 64), (7, 64), (2, 8192)])
def test_a_late_warp_changes_nothing(program, tmp_path, late, cache):
    rng = np.random.default_rng(5)
    width, k = 5000, 24
    logits = rows_with_ties(rng, width, k)
    rows = logits.shape[0]
    ks = rng.integers(0, 5, rows).astype(np.int32)
    ke = np.full(rows, width, np.int32)
    src, dst = tmp_path / "in", tmp_path / "out"
    src.write_bytes(np.array([rows, width, k, cache], np.int32).tobytes() + ks.tobytes() + ke.tobytes() + logits.tobytes())
    # threads that have lost step may wait for one another for good
    run = subprocess.run(["timeout", "60", str(program), str(src), str(dst), str(late)], capture_output=True, text=True)
    assert run.returncode == 0, (run.returncode, run.stdout)
    got = np.frombuffer(dst.read_bytes(), np.int32).reshape(rows, k)
    np.testing.assert_array_equal(got, otopk.canonical_topk(logits, ks, ke, k))
