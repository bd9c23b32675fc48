"""The read-out operators without a device: where copies begin and end, sizes and scales that
32 bits do not hold, scratch sizes, and the streams of the measured cases."""
import subprocess
from pathlib import Path

import pytest
import torch

from plastix_b200 import _abi, readout
from test_readout import DISTILL, SCORE, SCORE_BWD, FakeContext, refused

CSRC = Path(__file__).resolve().parents[1] / "plastix_b200" / "csrc"

CHUNKS = r"""
#include <cstdio>
#include <vector>
#include "chunk_copy.h"
// Every row of every small array of 16-bit values, copied as the kernels do: chunk by chunk into
// zeros, every byte read inside the array, every value of the row there in the end.
int main() {
  long read = 0;
  for (uint64_t base = 64; base < 80; base += 2)
    for (uint64_t n = 1; n <= 20; ++n)
      for (uint64_t ld = n; ld <= n + 9; ++ld)
        for (uint64_t rows = 1; rows <= 20; ++rows) {
          const uint64_t end = base + 2 * ((rows - 1) * ld + n);
          for (uint64_t r = 0; r < rows; ++r) {
            const uint64_t row = base + 2 * r * ld, row_end = row + 2 * n;
            const bool near = plx::near_edge((uint32_t)r, (uint32_t)rows);
            std::vector<bool> have(row_end + 16);
            for (uint64_t c = row / 16 * 16; c < row_end; c += 16) {
              const plx::ChunkCopy k = near ? plx::chunk_copy(c, row, row_end, base, end)
                                             : plx::ChunkCopy{0, 16, true};
              if (k.to > 16 || k.from > k.to || k.from % 2 || k.to % 2 || (k.whole && k.from)) return 1;
              for (uint64_t b = c + k.from; b < c + k.to; ++b, ++read) {
                if (b < base || b >= end) return 2;
                have[b] = true;
              }
            }
            for (uint64_t b = row; b < row_end; ++b)
              if (!have[b]) return 3;
          }
        }
  std::printf("%ld bytes\n", read);
  return 0;
}
"""


def test_chunks_of_odd_rows_stay_inside_their_array(tmp_path):
    (tmp_path / "chunks.cpp").write_text(CHUNKS)
    subprocess.run(["g++", "-std=c++17", "-O2", f"-I{CSRC}", str(tmp_path / "chunks.cpp"), "-o",
                    str(tmp_path / "chunks")], check=True, capture_output=True, text=True)
    done = subprocess.run([str(tmp_path / "chunks")], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, f"a chunk is wrong ({done.returncode})"


class MetaContext:
    """A context of tensors without memory: every call here is refused before its handle counts."""
    device = torch.device("meta")
    handle = None


@pytest.mark.parametrize("n", [1 << 31, (1 << 32) + 8])
def test_sizes_that_no_32_bit_argument_holds_are_refused(n):
    # 2^32 + 8 would arrive as 8
    c = MetaContext()
    x = torch.empty(1, n, dtype=torch.bfloat16, device="meta")
    small, one = torch.empty(1, 8, device="meta"), torch.empty(1, device="meta")
    ids, values = (torch.empty(1, n, dtype=t, device="meta") for t in (torch.int32, torch.float32))
    for call in (lambda: readout.layer_norm(c, x),
                 lambda: readout.layer_norm_backward(c, x, x, one, one),
                 lambda: readout.log_probs(c, x),
                 lambda: readout.log_probs_backward(c, x, one, one.int(), one),
                 lambda: readout.distill(c, x, ids[:, :4], values[:, :4]),
                 lambda: readout.log_probs(c, small, top=n),
                 lambda: readout.distill(c, small, ids, values)):
        with pytest.raises(ValueError, match="2\\^31"):
            call()
    with pytest.raises(ValueError, match="top"):
        readout.log_probs(c, small, top=-1)


def test_scales_that_leave_the_range_of_32_bits_are_refused():
    """Exponents are taken to base 2: scale * log2 e (or log2 e / temperature) has to be finite,
    or the largest logit's difference of 0 times it would be NaN."""
    for scale in (2.4e38, 3.4e38):
        refused(1, b"scale", "plx_log_probs", *{**SCORE, "scale": scale}.values())
        refused(1, b"scale", "plx_log_probs_backward", *{**SCORE_BWD, "scale": scale}.values())
    for tau in (3e-39, 4e-39):  # 1 / tau is finite
        refused(1, b"too small", "plx_distill", *{**DISTILL, "tau": tau}.values())
    # large, and fine: no rows, so that nothing more is asked of the pointers
    lib = _abi.lib()
    assert lib.plx_log_probs(*{**SCORE, "rows": 0, "scale": 2.3e38}.values()) == 0
    assert lib.plx_distill(*{**DISTILL, "rows": 0, "tau": 3.4e38}.values()) == 0
    assert lib.plx_distill(*{**DISTILL, "rows": 0, "tau": 5e-39}.values()) == 0


def test_a_bias_in_the_backward_call_is_checked():
    c, x, one = FakeContext(), torch.zeros(4, 8), torch.zeros(4)
    for weight, bias in ((None, torch.zeros(7)), (None, torch.zeros(8).bfloat16()), (None, torch.zeros(8, 2)[:, 0])):
        with pytest.raises(ValueError, match="bias"):
            readout.layer_norm_backward(c, x, x, one, one, weight, bias=bias)
    h = x.bfloat16()
    with pytest.raises(ValueError, match="different types"):
        readout.layer_norm_backward(c, h, h, one, one, torch.zeros(8), bias=torch.zeros(8).bfloat16())


@pytest.mark.parametrize("n, most", [(8192, 148), (12288, 148), (16384, 148), (4096, 296), (5120, 296), (2048, 592),
                                     (1024, 1184), (16385, 64)])
def test_layer_norm_scratch_is_what_the_launches_leave(n, most):
    """Column sums of at most as many blocks as run at once with rows this long, two rows of
    32-bit values each; few rows leave a block an SM, of a row or more."""
    size = lambda rows: _abi.lib().plx_layer_norm_scratch_bytes(rows, n) / (8 * n)  # noqa: E731
    assert size(0) == size(1) == 1
    assert size(100) == min(100, most) and size(600) == min(148, most)
    assert size(1 << 20) == most


def test_measured_cases_run_on_the_current_stream(monkeypatch):
    """A pass under another current stream, or on another device, uses that one."""
    from types import SimpleNamespace

    from perf import operators
    from plastix_b200 import runtime

    now = {}

    class FakeRuntimeContext:
        def __init__(self, index=0, stream=None):
            self.device, self.stream = torch.device("cuda", index), stream or now["stream"]

        def use_stream(self, stream):
            self.stream = stream

    seen = []
    monkeypatch.setattr(runtime, "Context", FakeRuntimeContext)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: now["stream"])
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: now["stream"].cuda_stream, raising=False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now["device"])
    monkeypatch.setattr(readout, "layer_norm",
                        lambda ctx, *a, **k: seen.append((ctx.device.index, ctx.stream.cuda_stream)))
    monkeypatch.setattr(operators, "own", True)
    monkeypatch.setattr(operators, "_context", None)
    wanted = [(0, 7), (0, 7), (0, 8), (1, 9), (0, 7)]
    for device, stream in wanted:
        now.update(device=device, stream=SimpleNamespace(cuda_stream=stream))
        x = SimpleNamespace(device=torch.device("cuda", device))
        operators.run({"op": "norm", "train": False, "x": x, "w": None, "b": None})
    assert seen == wanted
