"""Which tiles the workgroups of one launch take, followed on the host: each tile once, also where one launch
runs two products; and which sizes run so."""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "vllm-xpu-kernels_amd", "csrc")

SOURCE = """
#include <vector>
#include "tile_walk.h"
using namespace mi355;
// a kernel's loop over its walk
template <typename W>
static int take(W w, std::vector<int>& got, int total) {
  if (w.t >= w.end) return 0;
  int n = 0;
  for (;;) {
    const bool more = w.more();
    if (w.t < 0 || w.t >= total) return -1;
    ++got[w.t];
    ++n;
    w.next();
    if (!more) return n;
  }
}
static bool once(const std::vector<int>& got) {
  for (int g : got) if (g != 1) return false;
  return true;
}
extern "C" int one(int total, int blocks) {
  std::vector<int> got(total);
  for (int b = 0; b < blocks; ++b) if (take(XcdWalk(total, b, blocks), got, total) < 0) return 0;
  return once(got);
}
// the most tiles of a workgroup, priced 1 of the first and `price` of the second, or -1
extern "C" double two(int first, int second, int extra, int blocks, double price) {
  std::vector<int> a(first), c(second);
  double most = 0;
  for (int b = 0; b < blocks; ++b) {
    const int n = take(XcdWalk(first, b, blocks), a, first), m = take(SecondWalk(first, second, extra, b, blocks), c, second);
    if (n < 0 || m < 0) return -1;
    if (n + price * m > most) most = n + price * m;
  }
  return once(a) && once(c) ? most : -1;
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    d = tmp_path_factory.mktemp("walk")
    src, so = str(d / "walk.cpp"), str(d / "walk.so")
    with open(src, "w") as f:
        f.write(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-D__host__=", "-D__device__=", "-D__forceinline__=inline",
                    "-I" + CSRC, src, "-o", so], check=True)
    lib = ctypes.CDLL(so)
    lib.two.restype = ctypes.c_double
    lib.two.argtypes = [ctypes.c_int] * 4 + [ctypes.c_double]
    return lib


def test_every_tile_is_taken_once(walk):
    for blocks in (8, 16, 256, 512, 768):
        for total in [*range(1, 70), 255, 256, 257, 511, 513, 1000, 2047, 2048, 2049, 9999]:
            assert walk.one(total, blocks), (total, blocks)


def test_every_tile_of_two_products_is_taken_once(walk):
    """Totals that 8 does not divide, so that the last XCD has fewer or none; every number of extra tiles (1 at least) that
    the launch may choose, and more."""
    for first in [*range(1, 40, 3), 255, 256, 257, 300, 391, 392, 504, 511, 600, 900, 1024, 1025]:
        light = 32 - (first + 7) // 8 % 32
        for second in (1, 7, 31, 64, 255, 256, 257, 289, 511, 700, 896, 1500):
            for extra in range(1, (second + 7) // 8 // light + 3):
                assert walk.two(first, second, extra, 256, 1.0) > 0, (first, second, extra)


class Product(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int), ("transposed", ctypes.c_bool), ("I", ctypes.c_int64), ("J", ctypes.c_int64),
                ("R", ctypes.c_int64), ("q", ctypes.c_void_p), ("ldq", ctypes.c_int64), ("p", ctypes.c_void_p),
                ("ldp", ctypes.c_int64), ("out", ctypes.c_void_p), ("ldo", ctypes.c_int64)]


def _together(M, K, rows):
    from vllm_xpu_kernels import capi
    supported = capi.lib["_ZN5mi35522product_pair_supportedERKNS_7ProductES2_"]
    supported.restype = ctypes.c_bool
    ld = (rows + 7) // 8 * 8
    x = Product(1, False, M, K, rows, 16, ld, 16, K, 16, K)
    w = Product(1, True, rows, K, M, 16, ld, 16, K, 16, K)
    return supported(ctypes.byref(x), ctypes.byref(w))


@pytest.mark.parametrize("M,K,N", [(4323, 8456, 684), (3216, 8960, 2039), (4078, 8856, 737)])
def test_the_sizes_of_the_gpu_test_run_in_one_launch(M, K, N):
    """tests/test_gpu_gated_linear.py::test_gradients_together_and_alone compares the bits of one launch with those
    of two: at these sizes there is one."""
    assert _together(M, K, 2 * N)


def test_small_steps_run_in_two_launches():
    assert not _together(61, 2048, 1536) and not _together(1003, 2880, 5760)
