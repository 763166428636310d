"""What the kernels of the paged KV cache work out or report, run on the host: a small
program compiled against their own headers."""
import os
import shutil
import subprocess

import pytest

from onnx_runtime_dart_b200 import _lib, build

pytestmark = pytest.mark.skipif(shutil.which(build.NVCC) is None, reason="needs nvcc")

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>

#include "kernel_errors.cuh"
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

// The codes written in order, then the status and message, twice.
void report(int n, char** codes) {
  int words[16] = {};
  for (int i = 0; i < n; i++) words[error_word(atoi(codes[i]))] = atoi(codes[i]);
  for (int i = 0; i < 2; i++) {
    std::string msg;
    const int rc = take_kernel_errors(words, &msg);
    std::printf("%d %s\n", rc, msg.c_str());
  }
}

int main(int argc, char** argv) {
  if (argv[1][0] == 'e') {
    report(argc - 2, argv + 2);
    return 0;
  }
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
                                        capture_output=True, text=True).stdout


@pytest.mark.parametrize("count,past,group", [
    (1, 0, 1), (131072, 0, 128), (32768, 1000000, 128), (200000, 0, 71), (16777215, 0, 128)])
def test_length_of_the_stream_list(program, count, past, group):
    """Row tiles of 16 times key tiles (64 or 128 keys, and the places a segment's start
    and end count): also where the product passes 32 bits."""
    rows = -(-count * group // 16)
    want = [rows * (-(-(count + past) // tk) + extra) for tk, extra in ((64, 2), (128, 4))]
    assert [int(x) for x in program(count, past, group).split()] == want


WAIT, LENGTH, PAGE, POSITION = 2, 16, 17, 18


@pytest.mark.parametrize("codes,status,texts", [
    ([], 0, []),
    ([WAIT], _lib.ERR_TIMEOUT, ["exceeded its bound (code 2)"]),
    ([PAGE], _lib.ERR_INVALID_ARG, ["block_table"]),
    ([WAIT, PAGE], _lib.ERR_TIMEOUT, ["exceeded its bound (code 2)", "block_table"]),
    ([LENGTH, WAIT, POSITION, PAGE], _lib.ERR_TIMEOUT,
     ["exceeded its bound (code 2)", "cu_seqlens", "block_table", "cos/sin"]),
    ([POSITION, LENGTH], _lib.ERR_INVALID_ARG, ["cu_seqlens", "cos/sin"])])
def test_reports_do_not_replace_one_another(program, codes, status, texts):
    """A wait that ran out stays reported whatever does not fit besides, and so does all
    else; once."""
    first, second = program("e", *codes).split("\n")[:2]
    rc, msg = first.split(" ", 1)
    assert int(rc) == status
    at = [msg.find(t) for t in texts]
    assert -1 not in at and at == sorted(at)
    assert (msg == "") == (not texts)
    assert second == "0 "
