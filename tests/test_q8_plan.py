"""The 8-bit paged cache's choices of kernels, by sizes (no GPU needed)."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FLAGS = ["-std=c++17", "-O2", "-U_FORTIFY_SOURCE", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover=all",
         "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(ROOT, "baranet-bdml_amd", "csrc")]


def compiled(tmp_path_factory, name, text):
    at = tmp_path_factory.mktemp(name)
    source, exe = str(at / (name + ".cpp")), str(at / name)
    with open(source, "w") as f:
        f.write(text)
    subprocess.run(["g++", *FLAGS, source, "-o", exe], check=True)

    def run(*numbers):
        p = subprocess.run([exe], input=" ".join(map(str, numbers)), capture_output=True, text=True, timeout=60)
        assert p.returncode == 0, p.stderr
        return [[int(x) for x in line.split()] for line in p.stdout.splitlines()]
    return run


def paged_plan():
    """The source that runs a wave of the paged plan's search on the CPU."""
    with open(os.path.join(ROOT, "tests", "paged_plan.cpp")) as f:
        return f.read()


@pytest.fixture(scope="module")
def once(tmp_path_factory):
    return compiled(tmp_path_factory, "once", "#define main paged_plan_main\n" + paged_plan() + """
#undef main
#include "bn_q8_plan.hpp"
int main() {
  long long row_stride;
  int hblocks;
  if (scanf("%lld %d", &row_stride, &hblocks) != 2) return 1;
  printf("%d\\n", decode_reads_once(row_stride, hblocks));
  return 0;
}
""")


@pytest.mark.parametrize("row_stride,group,want", [(64, 1, 1), (64, 8, 1), (64, 16, 1), (64, 17, 0), (64, 20, 0),
                                                   (64, 66, 0), (256, 8, 0), (80, 8, 0), (256, 32, 0)])
def test_rows_that_others_read_stay_in_the_caches(once, row_stride, group, want):
    """A decode's rows go past the caches only if one workgroup alone reads their lines: not with
    several blocks of 16 query heads to a KV head, nor where heads' rows lie beside each other."""
    assert once(row_stride, -(-group // 16)) == [[want]]
