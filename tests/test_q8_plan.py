"""The 8-bit paged cache's choices of kernels, by sizes (no GPU needed)."""
import os
import random
import subprocess

import pytest

import test_paged_plan as paged

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


CALL = "plan_prefill(dtype ? BN_BF16 : BN_F32, batch, n_rows, n_heads, hkv, cap)"


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """The paged plan's check with this cache's plan in the other caches' place."""
    text = paged_plan()
    assert text.count(CALL) == 1 and text.count('#include "bn_paged_plan.hpp"') == 1
    text = text.replace(CALL, CALL.replace("plan_prefill", "plan_q8")).replace("bn_paged_plan.hpp", "bn_q8_plan.hpp")
    exe = compiled(tmp_path_factory, "q8_plan", text)

    def run(dtype, lens, starts, n_rows, H, Hkv, cap, most=1 << 30):
        first, *rest = exe(int(dtype == "bf16"), len(lens), n_rows, H, Hkv, cap, most, *lens, *starts)
        return first, rest
    return run


def rows_for(units, H, Hkv):
    """The fewest rows of a call with so many units of 128 rows, as the plan counts them."""
    return -(-(-(-units // Hkv) - 1) * 128 * Hkv // H)


@pytest.mark.parametrize("pad", [0, 3])
@pytest.mark.parametrize("case", paged.CASES, ids=lambda c: f"{c[0]}-{len(c[1])}x{max(c[2])}of{max(c[1])}-{c[3]}-{c[4]}")
def test_every_piece_is_dealt_once(plan, case, pad):
    dtype, lens, rows, H, Hkv, cap = case
    paged.deal(plan, dtype, lens, rows, H, Hkv, cap, pad)


@pytest.mark.parametrize("H,Hkv", [(32, 4), (12, 3), (40, 8)])
@pytest.mark.parametrize("cap", [5120, 12288])
@pytest.mark.parametrize("less,R", [(1, 128), (0, 256), (-700, 256)], ids=["below", "at", "above"])
def test_around_the_pipelined_kernels_first_size(plan, H, Hkv, cap, less, R):
    """Ragged batches of one row less than the pipelined kernel takes, of as many, and of more, short of
    the other caches' 2048 units."""
    total = rows_for(1200, H, Hkv) - less
    assert total < rows_for(2048, H, Hkv)
    for batch in (1, total // 512):
        rows, left = [], total
        for b in range(batch - 1):
            rows.append(left * (1 + b % 3) // (2 * batch))
            left -= rows[-1]
        rows.append(left)
        lens = [n + (cap - n) * (b % 4) // 3 if n <= cap else n for b, n in enumerate(rows)]
        assert paged.deal(plan, "bf16", lens, rows, H, Hkv, cap)[0] == R, batch


def test_drawn_calls_between_the_two_rules(plan):
    r = random.Random(11)
    pipelined = 0
    for _ in range(10):
        Hkv = r.choice([1, 2, 3, 4, 8])
        H = Hkv * r.choice([4, 5, 8, 16])
        total = rows_for(r.randint(1000, 2047), H, Hkv)
        batch = r.randint(1, max(1, total // 500))
        cuts = sorted(r.randint(0, total) for _ in range(batch - 1))
        rows = [b - a for a, b in zip([0, *cuts], [*cuts, total])]
        cap = 16 * r.randint(1, 1000)
        lens = [r.choice([n, n + r.randint(0, cap), paged.INT_MAX, 0]) for n in rows]
        pipelined += paged.deal(plan, "bf16", lens, rows, H, Hkv, cap, r.choice([0, 2]))[0] == 256
    assert 2 <= pipelined <= 9
