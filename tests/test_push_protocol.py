"""The push transport's flow control, csrc/pa_push_dev.h itself compiled for the host: one block after the other, in any order.  (Lane 0
of a block does all of the protocol; the stand-ins below run that lane.)"""
import os
import subprocess

import pytest

from __graft_entry__ import PKG_DIR

SHIM = r"""
#pragma once
#include <cstdint>
#include <algorithm>
using std::min;
#define __device__
#define __forceinline__ inline
#define __HIP_MEMORY_SCOPE_SYSTEM 0
#define __hip_atomic_load(p, o, s) (*(p))
#define __hip_atomic_store(p, v, o, s) (*(p) = (v))
#define __builtin_amdgcn_s_sleep(k) ((void)0)
static struct { unsigned x; } threadIdx = {0};
static inline void __syncthreads() {}
static inline void __threadfence_system() {}
static long long ticks_now = 0;
static inline long long wall_clock64() { return ++ticks_now; }
static inline unsigned atomicAdd(unsigned *p, unsigned v) { unsigned o = *p; *p += v; return o; }
static inline unsigned atomicOr(unsigned *p, unsigned v) { unsigned o = *p; *p |= v; return o; }
static inline int atomicExch(int *p, int v) { int o = *p; *p = v; return o; }
"""

MAIN = r"""
#include "pa_push_dev.h"
#include <cstdio>
#include <cstdlib>
#include <vector>
// argv: status before | ticks | order of the blocks, as digits | the acknowledgement of every segment ...   (sequence number 5)
int main(int argc, char **argv) {
  int status = atoi(argv[1]);
  const long long ticks = atoll(argv[2]);
  const int nseg = argc - 4, n = 256 * nseg;
  std::vector<unsigned long long> ack, arrive(nseg, 4);
  for (int k = 0; k < nseg; ++k) ack.push_back(strtoull(argv[4 + k], nullptr, 10));
  std::vector<int32_t> idx(n);
  std::vector<double> v(n), dst(n, -1.0);
  std::vector<pa_push_seg> segs(nseg);
  for (int i = 0; i < n; ++i) { idx[i] = i; v[i] = i; }
  for (int k = 0; k < nseg; ++k) segs[k] = {256 * k, 256, dst.data() + 256 * k, nullptr, 0, &arrive[k], &ack[k]};
  unsigned done = 0;
  int ok = 0;
  for (const char *o = argv[3]; *o; ++o)
    pa_push_ipc_block(&ok, idx.data(), n, segs.data(), nseg, v.data(), 5ull, &done, ticks, &status, *o - '0', nseg);
  printf("%d %u", status, done);
  for (int k = 0; k < nseg; ++k) printf(" %llu:%g", arrive[k], dst[256 * k]);
  printf("\n");
}
"""


@pytest.fixture(scope="module")
def block(tmp_path_factory):
    d = tmp_path_factory.mktemp("push")
    (d / "hip").mkdir()
    (d / "hip" / "hip_runtime.h").write_text(SHIM)
    (d / "main.cpp").write_text(MAIN)
    exe = str(d / "push")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-I", str(d), "-I", os.path.join(PKG_DIR, "csrc"), str(d / "main.cpp"), "-o", exe])

    def run(status, ticks, order, *acks):
        r = subprocess.run([exe, str(status), str(ticks), order] + [str(a) for a in acks], capture_output=True, text=True, timeout=20)
        assert r.returncode == 0, r.stderr
        f = r.stdout.split()
        return int(f[0]), int(f[1]), [int(x.split(":")[0]) for x in f[2:]], [float(x.split(":")[1]) for x in f[2:]]
    return run


@pytest.mark.parametrize("order", ["012", "210", "102"])
def test_every_slice_is_announced_when_all_are_delivered(block, order):
    assert block(0, 1000, order, 4, 4, 7) == (0, 0, [5, 5, 5], [0.0, 256.0, 512.0])


@pytest.mark.parametrize("order", ["01", "10"])
@pytest.mark.parametrize("late", [0, 1])
def test_nothing_is_announced_when_one_block_gave_up(block, order, late):
    """The receiver of one slice has not acknowledged: its slice is not written, so no slice may be announced -- also where the block
    that gave up is not the last of the launch.  The counter is ready for the next launch."""
    status, done, arrive, dst = block(0, 1000, order, *[3 if k == late else 4 for k in range(2)])
    assert (status, done, arrive) == (2, 0, [4, 4])
    assert dst[late] == -1.0 and dst[1 - late] == 256.0 * (1 - late)


def test_several_blocks_that_gave_up(block):
    assert block(0, 1000, "3012", 3, 4, 3, 3)[:3] == (2, 0, [4, 4, 4, 4])


@pytest.mark.parametrize("status", [1, 2])
def test_a_wait_ends_at_once_behind_one_that_gave_up(block, status):
    """(a time-out that the run never reaches: 2^60 ticks)"""
    assert block(status, 1 << 60, "01", 3, 3)[1:] == (0, [4, 4], [-1.0, -1.0])


def test_a_flag_that_is_up_is_taken_whatever_the_status(block):
    assert block(1, 1 << 60, "10", 4, 4) == (1, 0, [5, 5], [0.0, 256.0])
