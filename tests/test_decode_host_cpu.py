"""The decode-step operators' host side and what their kernels share with it, without a GPU."""

import contextlib
import subprocess
import weakref
from types import SimpleNamespace

import pytest


def run_host_program(tmp_path, text):
    """Compiles a program over the library's internal header and runs it on the CPU; it has to print "ok"."""
    from ssengine_b200 import _build

    src, exe = tmp_path / "host.cu", tmp_path / "host"
    src.write_text(text)
    subprocess.run([_build.nvcc(), *_build.ARCH, "-std=c++17", "-O1", f"-I{_build.CSRC}", "-o", str(exe), str(src)],
                   check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout


ROW_PARTS = r"""
#include <cstdio>
#include <cstdint>
#include "ops.h"
using ssb::MlaRowParts;
using ssb::kMlaRanges;
int main() {
  // every record that a plan can write is valid, and its slots are the CTAs' own
  for (int f = 0; f < kMlaRanges; ++f)
    for (int l = f; l < kMlaRanges; ++l)
      for (int s = 0; s < 2; ++s) {
        const MlaRowParts p = {f, l, 2 * f + s, 0};
        if (!p.valid() || p.slot(0) != 2 * f + s) return std::printf("refused %d %d %d\n", f, l, s), 1;
        for (int i = 1; i <= l - f; ++i)
          if (p.slot(i) != 2 * (f + i) || p.slot(i) >= 2 * kMlaRanges)
            return std::printf("slot %d %d %d\n", f, l, i), 1;
      }
  // whatever else memory holds: refused, or within the parts
  const int32_t edge[] = {0, 1, -1, 2, kMlaRanges - 1, kMlaRanges, 2 * kMlaRanges - 1, 2 * kMlaRanges, -2, 294,
                          296, 0x7f800000, 0x7fffffff, static_cast<int32_t>(0x80000000u),
                          static_cast<int32_t>(0xffff8000u), 0x3f800000};
  uint64_t x = 88172645463325252ull;
  auto rnd = [&] { x ^= x << 13, x ^= x >> 7, x ^= x << 17; return static_cast<int32_t>(x >> 20); };
  auto check = [&](const MlaRowParts& p) {
    if (!p.valid()) return true;
    if (p.last < p.first || p.last - p.first >= kMlaRanges) return false;
    for (int i = 0; i <= p.last - p.first; ++i)
      if (p.slot(i) < 0 || p.slot(i) >= 2 * kMlaRanges) return false;
    return true;
  };
  for (int a : edge)
    for (int b : edge)
      for (int c : edge)
        if (!check({a, b, c, 0})) return std::printf("accepted %d %d %d\n", a, b, c), 1;
  for (int n = 0; n < 4000000; ++n) {
    const bool small = n & 1;
    const int32_t a = rnd(), b = rnd(), c = rnd();
    if (!check(small ? MlaRowParts{a % 400, b % 400, c % 400, 0} : MlaRowParts{a, b, c, 0}))
      return std::printf("accepted %d %d %d\n", a, b, c), 1;
  }
  if (MlaRowParts{0, 0x7fffffff, 0, 0}.valid() || MlaRowParts{-1, -1, -2, 0}.valid() || MlaRowParts{3, 2, 6, 0}.valid())
    return std::printf("accepted a range outside\n"), 1;
  std::puts("ok");
}
"""


def test_a_rows_record_stays_within_the_parts_whatever_memory_holds(tmp_path):
    """The join reads parts by a row's record; a CTA that gave up leaves there what the workspace held before."""
    run_host_program(tmp_path, ROW_PARTS)


ONCE = r"""
#include <cstdio>
#include "ops.h"
int main() {
  ssb::OncePerDevice once;
  int calls = 0;
  bool works = false;
  const auto set = [&] { return ++calls, works; };
  if (once.done(0, set) || calls != 1) return std::puts("a failure passed"), 1;
  works = true;
  for (int device : {0, 1, 0, 63, 1, 0, 63})
    if (!once.done(device, set)) return std::puts("refused"), 1;
  if (calls != 4) return std::printf("%d calls for three devices and a failure\n", calls), 1;
  if (!once.done(64, set) || !once.done(64, set) || !once.done(-1, set) || calls != 7) return std::puts("outside"), 1;
  std::puts("ok");
}
"""


def test_kernel_attributes_are_set_on_every_device(tmp_path):
    """Once on each device of the process, again after a failure, and each time for a device beyond the table."""
    run_host_program(tmp_path, ONCE)


class FakeCuda:
    """torch.cuda as `lib.stream_scratch` uses it: streams by handle, buffers on the CPU, a capture that can be on."""

    def __init__(self, monkeypatch):
        import torch

        self.current, self.capturing, self.buffers = 1, set(), []
        empty = torch.empty

        def alloc(n, dtype, device):
            t = empty(n, dtype=dtype)
            self.buffers.append((self.current, weakref.ref(t)))
            return t

        @contextlib.contextmanager
        def stream(s):
            self.current, before = s.cuda_stream, self.current
            yield
            self.current = before

        monkeypatch.setattr(torch, "empty", alloc)
        monkeypatch.setattr(torch.cuda, "stream", stream)
        monkeypatch.setattr(torch.cuda, "current_stream", lambda dev=None: SimpleNamespace(cuda_stream=self.current))
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: self.current in self.capturing)
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: self.current, raising=False)


@pytest.mark.parametrize("explicit", [False, True])
def test_a_captured_call_keeps_no_buffer_that_can_be_outgrown(monkeypatch, explicit):
    """Buffers per stream that grow; in a capture a new one each time, not the stream's kept one nor kept as one: what the
    stream's calls drop later was never the graph's."""
    from ssengine_b200 import lib

    monkeypatch.setattr(lib, "_SCRATCH", {})
    cuda = FakeCuda(monkeypatch)
    get = lambda n: lib.stream_scratch("cuda:0", n, SimpleNamespace(cuda_stream=5) if explicit else None)
    handle = 5 if explicit else 1
    eager = get(1000)
    assert get(600) is eager and cuda.buffers[-1][0] == handle
    cuda.capturing.add(handle)
    captured = get(600)
    again = get(600)
    assert captured is not eager and again is not captured and captured.numel() >= 600
    assert cuda.buffers[-1][0] == handle                    # allocated on the capturing stream, so from the graph's pool
    cuda.capturing.clear()
    assert get(600) is eager
    assert all(t is not captured and t is not again for t in lib._SCRATCH.values())
    larger = get(2000)
    assert larger.numel() >= 2000 and get(600) is larger
    cuda.current = 9
    assert explicit or get(600) is not larger               # another stream, another buffer


class OnDevice:
    """A tensor as the device check sees it."""

    def __init__(self, index, dtype=None, numel=1):
        self.index, self.dtype, self.device, self.shape = index, dtype, f"device {index}", (numel,)
        self.numel = lambda: numel
        self.get_device = lambda: index


def test_calls_refuse_tensors_away_from_the_current_device(monkeypatch):
    import torch

    from ssengine_b200 import lib

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    on = lambda i: [OnDevice(i), OnDevice(i), None, OnDevice(i)]
    word = lambda i, dtype=torch.int32, n=1: OnDevice(i, dtype, n)
    stream = lambda i: SimpleNamespace(cuda_stream=3, device_index=i)
    lib.check_device(on(1))
    lib.check_device(on(1), word(1), stream(1))
    for args in ((on(0),), (on(-1),), (on(1) + [OnDevice(0)],), (on(1) + [OnDevice(-1)],), (on(1), word(-1)),
                 (on(1), word(0)), (on(1), word(1, torch.int64)), (on(1), word(1, n=0)), (on(1), None, stream(0)),
                 (on(0), word(0), stream(0))):
        with pytest.raises(ValueError):
            lib.check_device(*args)


@pytest.mark.parametrize("what", ["a_log", "dt_bias", "status", "conv_weight"])
def test_the_recurrence_checks_every_tensor_it_reads(monkeypatch, what):
    """Each tensor that the kernel reads goes through the device check."""
    import torch

    from ssengine_b200 import lib
    from ssengine_b200.kda import KdaLayer

    seen = []
    monkeypatch.setattr(lib, "check_device", lambda ts, status=None, stream=None: seen.extend([*ts, status]) or 1 / 0)
    H, bf = 2, dict(dtype=torch.bfloat16)
    P = H * 128
    L = KdaLayer(torch.zeros(3 * P, 4, **bf), torch.zeros(H), torch.zeros(P))
    status = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ZeroDivisionError):
        L.decode(torch.zeros(3, 3 * P, **bf), torch.zeros(3, P, **bf), torch.zeros(3, H, **bf),
                 torch.zeros(3, P, **bf), torch.zeros(1, 4, dtype=torch.int32), torch.zeros(2, 3, 3 * P, **bf),
                 torch.zeros(2, H, 128, 128), status=status)
    want = status if what == "status" else getattr(L, what)
    assert any(t is want for t in seen)


@pytest.mark.parametrize("what", ["a_log", "dt_bias"])
def test_gate_parameters_with_strides_are_refused(what):
    """The kernels read heads (and heads x 128) values in a row: a broadcast parameter has one, a strided one others."""
    import torch

    from ssengine_b200.kda import KdaLayer

    H = 2
    P = H * 128
    n = {"a_log": H, "dt_bias": P}
    conv, rec = torch.zeros(2, 3, 3 * P, dtype=torch.bfloat16), torch.zeros(2, H, 128, 128)
    for bad in (lambda k: torch.zeros(1).expand(k), lambda k: torch.zeros(2 * k)[::2]):
        p = {k: bad(v) if k == what else torch.zeros(v) for k, v in n.items()}
        with pytest.raises(AssertionError):
            KdaLayer(torch.zeros(3 * P, 4, dtype=torch.bfloat16), p["a_log"], p["dt_bias"]).c_struct(conv, rec)
    KdaLayer(torch.zeros(3 * P, 4, dtype=torch.bfloat16), torch.zeros(H), torch.zeros(H, 128)).c_struct(conv, rec)


PHASES = r"""
#include <cstdio>
#include "ops.h"
int main() {
  for (int slots = 1; slots <= 8; ++slots) {
    int begun[8] = {}, slot = 0, round = 0;                 // fills of each buffer so far
    for (int unit = 0; unit < 100; ++unit) {
      for (int j = 0; j < slots; ++j)
        if (ssb::ring_phase(j, slot, round) != (begun[j] == 0 ? -1 : (begun[j] - 1) % 2))
          return std::printf("buffer %d of %d after %d units\n", j, slots, unit), 1;
      ++begun[slot];
      if (++slot == slots) slot = 0, ++round;
    }
  }
  std::puts("ok");
}
"""


def test_a_producer_that_gives_up_waits_for_the_copies_it_began(tmp_path):
    """The barrier phase of each buffer's last fill, after any number of units."""
    run_host_program(tmp_path, PHASES)
