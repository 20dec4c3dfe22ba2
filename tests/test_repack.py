"""Rows of 16-bit elements copied to another stride: what is read lies in the row.

``csrc/repack.cuh`` says which words and elements a thread reads.  It is plain C++
there, so it is compiled for the host and every read is compared with the row's
bounds; the copy itself is tested at every alignment on the GPU."""

import os
import shutil
import subprocess

import pytest
import torch

import practice_cuda_b200
from practice_cuda_b200 import _lib

CSRC = os.path.join(os.path.dirname(practice_cuda_b200.__file__), "csrc")

HOST_CHECK = r"""
#define __host__
#define __device__
#include "repack.cuh"
#include <cstdio>
using namespace pcb::loss;

static int bad = 0;
struct Row {
  const uint16_t* e;
  int cols;
  bool odd;
  uint16_t half(int i) const {
    if (i < 0 || i >= cols) ++bad, std::printf("cols %d odd %d: reads element %d\n", cols, odd, i);
    return i < 0 || i >= cols ? 0xdead : e[i];
  }
  uint32_t pair(int i) const {
    if ((i & 1) != (int)odd) ++bad, std::printf("cols %d odd %d: word at element %d is not aligned\n", cols, odd, i);
    const uint32_t lo = half(i);
    return lo | (uint32_t)half(i + 1) << 16;
  }
};

int main() {
  uint16_t e[40];
  for (int i = 0; i < 40; ++i) e[i] = (uint16_t)(1000 + i);
  for (int cols = 1; cols <= 40; ++cols)
    for (int odd = 0; odd < 2; ++odd)
      for (int j = 0; j < (cols + 1) / 2; ++j) {
        const Row row{e, cols, odd != 0};
        const uint32_t got = join_word_parts(load_word_parts(row, odd != 0, j, cols), odd != 0);
        const uint32_t want = e[2 * j] | (2 * j + 1 < cols ? (uint32_t)e[2 * j + 1] << 16 : 0u);
        if (got != want) ++bad, std::printf("cols %d odd %d word %d: %x for %x\n", cols, odd, j, got, want);
      }
  return bad != 0;
}
"""


def test_reads_stay_in_the_row(tmp_path):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no host compiler")
    source, program = tmp_path / "check.cpp", tmp_path / "check"
    source.write_text(HOST_CHECK)
    subprocess.run([compiler, "-std=c++17", "-I", CSRC, "-o", str(program), str(source)], check=True)
    done = subprocess.run([str(program)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [1, 2, 3, 4, 5, 63, 64, 511, 512, 513, 4096, 4097, 4101])
def test_copy_at_every_alignment(cols):
    for start in range(3):
        for extra in (0, 1, 2, 5):
            base = torch.arange(start + 7 * (cols + extra) + 9, device="cuda").to(torch.int16)
            src = base[start : start + 7 * (cols + extra)].view(7, cols + extra)[:, :cols]
            stride = (cols + 9) // 2 * 2
            dst = torch.full((7, stride), -7, device="cuda", dtype=torch.int16)
            _lib.check(_lib.lib().pcb_repack_u16(src.data_ptr(), 7, cols, src.stride(0), dst.data_ptr(), stride,
                                                 torch.cuda.current_stream().cuda_stream), "pcb_repack_u16")
            assert torch.equal(dst[:, :cols], src)
            assert bool((dst[:, cols:] == -7).all())
