"""The arithmetic that splits paged attention over the device, run on the host:
a small program compiled against the kernels' own headers."""
import os
import shutil
import subprocess

import pytest

from onnx_runtime_dart_b200 import build

pytestmark = pytest.mark.skipif(shutil.which(build.NVCC) is None, reason="needs nvcc")

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>

#include "paged_segments.cuh"

using namespace ortc;

// One sequence of `count` tokens behind `past`, `group` query heads on one KV head.
template <int R, int TK, int EXTRA>
long long places(int count, int past, int group) {
  int32_t cu[2] = {0, count};
  StreamArgs p;
  p.a.c.cu = cu;
  p.a.c.past = &past;
  p.a.c.batch = 1;
  p.a.c.num_tokens = p.a.max_seq = count;
  p.a.c.page_size = 16;
  p.a.c.max_pages = 1 << 26;
  p.a.group = group;
  p.max_rows = INT_MAX;
  StreamPos s;
  return stream_seq<R, TK>(p, s, 0, 0) ? stream_places<EXTRA>(s) : 0;
}

int main(int argc, char** argv) {
  const int count = atoi(argv[1]), past = atoi(argv[2]), group = atoi(argv[3]);
  std::printf("%lld %lld\n", places<16, 64, 2>(count, past, group),
              places<16, 128, 4>(count, past, group));
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cu").write_text(PROGRAM)
    subprocess.run([build.NVCC, *build.ARCH, "-std=c++17", "--expt-relaxed-constexpr", "-I",
                    build.CSRC, "-I", os.path.join(build.HERE, "..", "include"), "-o",
                    str(d / "plan"), str(d / "plan.cu")], check=True, capture_output=True)
    return lambda *args: subprocess.run([str(d / "plan"), *map(str, args)], check=True,
                                        capture_output=True, text=True).stdout.split()


@pytest.mark.parametrize("count,past,group", [
    (1, 0, 1), (131072, 0, 128), (32768, 1000000, 128), (200000, 0, 71), (16777215, 0, 128)])
def test_length_of_the_stream_list(program, count, past, group):
    """Row tiles of 16 times key tiles (64 or 128 keys, and the places a segment's start
    and end count): also where the product passes 32 bits."""
    rows = -(-count * group // 16)
    want = [rows * (-(-(count + past) // tk) + extra) for tk, extra in ((64, 2), (128, 4))]
    assert [int(x) for x in program(count, past, group)] == want
