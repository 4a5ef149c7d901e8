"""How a ragged paged prefill is divided: every unit of 32, 128 or 256 rows of every sequence and KV
head, and every part of a cut one, belongs to exactly one workgroup, and the parts of cut units have
records of their own inside the workspace.  The kernels' own search, run on the CPU (paged_plan.cpp) with
signed overflow, shifts and conversions checked."""
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INT_MAX = 2 ** 31 - 1


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("paged_plan") / "paged_plan")
    subprocess.run(["g++", "-std=c++17", "-O2", "-U_FORTIFY_SOURCE", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(ROOT, "baranet-bdml_amd", "csrc"),
                    os.path.join(ROOT, "tests", "paged_plan.cpp"), "-o", exe], check=True)

    def run(dtype, lens, starts, n_rows, H, Hkv, cap, most=1 << 30):
        text = " ".join(map(str, [int(dtype == "bf16"), len(lens), n_rows, H, Hkv, cap, most, *lens, *starts]))
        p = subprocess.run([exe], input=text, capture_output=True, text=True, timeout=60)
        assert p.returncode == 0, p.stderr
        first, *rest = ([int(x) for x in line.split()] for line in p.stdout.splitlines())
        return first, rest
    return run


def starts_of(rows, first=0):
    out = [first]
    for n in rows:
        out.append(out[-1] + n)
    return out


def deal(plan, dtype, lens, rows, H, Hkv, cap, pad=0):
    starts = starts_of(rows, pad)
    n_rows = starts[-1] + pad
    (R, groups, most, slots, _), found = plan(dtype, lens, starts, n_rows, H, Hkv, cap)
    G = H // Hkv
    want = {(b, g, u) for b, n in enumerate(rows) for g in range(Hkv) for u in range(-(-n * G // R))}
    parts, seen, records = {}, set(), set()
    for block, b, g, unit, part, of, row0, n, slot, tok0, rem0 in found:
        assert (b, g, unit) in want, "a unit that there is not"
        assert (row0, n) == (starts[b], rows[b])
        assert tok0 * G + rem0 == unit * R and 0 <= rem0 < G
        assert 0 <= part < of and parts.setdefault((b, g, unit), of) == of
        assert (b, g, unit, part) not in seen, "a piece that two workgroups take"
        seen.add((b, g, unit, part))
        if of > 1:
            record = slot + part * Hkv
            assert 0 <= record < slots and record not in records
            records.add(record)
    assert len(seen) == sum(parts.values()) and set(parts) == want, "pieces that nobody takes"
    assert len(seen) <= most * Hkv <= groups
    return R, sorted(set(parts.values()))


# dtype, lens (with the new rows), rows, H, Hkv, keys that a table row holds
CASES = [
    ("bf16", [1, 2, 17, 33], [1, 2, 17, 33], 16, 2, 64),
    ("f32", [130, 0, 65, 129], [130, 0, 65, 129], 4, 1, 160),
    ("bf16", [300, 40, 257], [3, 0, 200], 12, 2, 512),
    ("bf16", [9000, 3000, 70, 20000], [5, 64, 1, 3], 16, 2, 20480),
    ("bf16", [3000, 1100, 40], [2100, 767, 33], 32, 4, 4096),
    ("bf16", [17000, 6000], [300, 290], 32, 4, 32768),
    ("f32", [2000, 9000, 3], [700, 5, 3], 8, 2, 9216),
    ("f32", [300] * 80, [9] * 80, 3, 3, 320),
    ("bf16", [700] * 70 + [9000], [10] * 70 + [2], 6, 2, 16384),
    ("bf16", [10, -5, 0], [12, 9, 4], 8, 2, 64),      # more rows than keys
    ("bf16", [4000] * 64, [1] * 63 + [200], 24, 3, 4096),
    ("f32", [8192], [1], 7, 7, 8192),
    ("bf16", [20 + b % 50 for b in range(4300)], [b % 3 // 2 for b in range(4300)], 4, 1, 64),   # runs of a lane past 64
]


@pytest.mark.parametrize("pad", [0, 3])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}-{len(c[1])}x{max(c[2])}of{max(c[1])}-{c[3]}-{c[4]}")
def test_every_piece_is_dealt_once(plan, case, pad):
    dtype, lens, rows, H, Hkv, cap = case
    deal(plan, dtype, lens, rows, H, Hkv, cap, pad)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("H,Hkv", [(4, 1), (16, 1), (32, 1), (64, 1), (64, 2), (512, 1)])
@pytest.mark.parametrize("lens,rows,cap", [
    ([INT_MAX, 40], [70, 40], 144),               # a length past the table beside an ordinary one
    ([40, INT_MAX], [40, 70], 144),
    ([INT_MAX, 40], [7, 4], 144),
    ([1 << 30, 40], [17, 5], 1 << 30),            # the longest that a table can hold
    ([INT_MAX, 0, 5, INT_MAX], [9, 11, 5, 3], 1 << 30),
    ([INT_MAX, -INT_MAX - 1], [30, 30], 4096),
], ids=["past_first", "past_last", "past_few", "longest", "past_and_none", "past_and_negative"])
def test_lengths_past_the_table(plan, dtype, H, Hkv, lens, rows, cap):
    deal(plan, dtype, lens, rows, H, Hkv, cap)


def test_drawn_calls(plan):
    r = random.Random(7)
    for _ in range(25):
        Hkv = r.choice([1, 2, 3, 4, 8])
        H = Hkv * r.choice([1, 3, 4, 5, 8, 16, 32, 40, 64])
        cap = 16 * r.randint(1, 2500)
        batch = r.choice([1, 2, 5, 30, 64, 65, 100])
        most = max(1, min(3000 // batch, 24000 // H // batch))
        rows = [r.choice([0, 1, r.randint(1, most)]) for _ in range(batch)]
        lens = [r.choice([n, n + r.randint(0, cap), r.randint(0, cap), INT_MAX, -3]) for n in rows]
        if sum(rows):
            deal(plan, r.choice(["f32", "bf16"]), lens, rows, H, Hkv, cap, r.choice([0, 2]))


@pytest.mark.parametrize("batch", [1, 70])
def test_tiles_past_32_bits(plan, batch):
    """Many rows of long sequences: the share of a workgroup, in tiles, stays a share."""
    rows = [(1 << 20) // batch] * batch
    (R, *_), found = plan("bf16", [1 << 30] * batch, starts_of(rows), sum(rows), 32, 1, 1 << 30, 5)
    assert len({(b, g, unit, part) for _, b, g, unit, part, *_ in found}) == 5
    assert all(of == 1 for _, _, _, _, _, of, *_ in found)


@pytest.mark.parametrize("dtype,n,H", [("bf16", 1 << 21, 64), ("f32", 1 << 19, 64)])
def test_starts_that_decrease_count_no_further_than_32_bits(plan, dtype, n, H):
    """Row starts out of order count the same rows again and again, here 2^32 units and those of 40 rows
    more: too many, so that no workgroup takes any."""
    R = 128 if dtype == "bf16" else 32
    times = (1 << 32) // (n * H // R)
    starts = [0, n] * times + [n - 40, n]
    (got, *_), found = plan(dtype, [5] * (len(starts) - 1), starts, n, H, 1, 64, 3)
    assert got == R and not found
