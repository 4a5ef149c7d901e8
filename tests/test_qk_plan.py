"""How the norms of single heads are launched, by sizes (no GPU needed)."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = """
#include <cstdio>
#include "bn_qk_plan.hpp"
using namespace bn;
int main() {
  int n, heads, head_dim;
  while (scanf("%d %d %d", &n, &heads, &head_dim) == 3) {
    const BackPlan d = plan_back(n, heads, head_dim);
    printf("%d %d %d\\n", d.rows, d.groups, (int)d.joins);
  }
  return 0;
}
"""


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    at = tmp_path_factory.mktemp("qk_plan")
    (at / "plan.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-I" + os.path.join(ROOT, "baranet-bdml_amd", "csrc"), str(at / "plan.cpp"), "-o", str(at / "plan")],
                   check=True)

    def run(calls):
        text = "\n".join(" ".join(map(str, c)) for c in calls)
        p = subprocess.run([str(at / "plan")], input=text, capture_output=True, text=True, timeout=60)
        assert p.returncode == 0, p.stderr
        return [[int(x) for x in line.split()] for line in p.stdout.splitlines()]
    return run


CALLS = [(n, heads, d) for d in (16, 32, 64, 128, 256) for heads in (1, 5, 36, 48, 64, 124, 130, 1000, 131070)
         for n in (0, 1, 31, 32, 33, 64, 65, 127, 128, 129, 257, 500, 1023, 1792, 1793, 1820, 2047, 2048, 2049, 8192, 16385, 1 << 23)]


def test_backward_launches_cover_the_rows(plans):
    for (n, heads, d), (rows, groups, joins) in zip(CALLS, plans(CALLS)):
        assert 1 <= rows <= (16 if joins else 8) and groups <= min(n, 1024)
        assert rows * groups >= n or groups == 1024, (n, heads, d)   # (1024 of them take further groups of rows)
        assert not (joins and rows * groups < n)


def test_a_joined_workgroup_has_few_elements(plans):
    """Where the last workgroup adds all sums, there are at most 128, with 64 KB of them, and none has more
    than 32768 elements."""
    some = 0
    for (n, heads, d), (rows, groups, joins) in zip(CALLS, plans(CALLS)):
        if joins:
            some += 1
            assert groups <= 128 and groups * 2 * d * 4 <= 1 << 16
            assert rows * heads * d <= 32768, (n, heads, d)
    assert some > 100
