"""The 8-bit paged attention at the largest values that its sums take: 2^113 / keys (up to a multiple of
64), with weights of up to 2^15.87 against the first keys'."""
import numpy as np
import pytest
import torch

import bnhip as B
from gpu_util import require_gpu
from paged_util import TD, attention64, attention64_large, check, starts_of
from q8_util import LOW, TABLE, Case8
from test_gpu_paged import host

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def late(lens, dtype):
    """A cache whose values are all but one sign and lie just below the limit, and of whose keys every 64th,
    from the second 64 on, scores 15.87 (log2) above the others with a query of 1, 0, 0, ..: no reference moves."""
    c = Case8(lens, 1, 32, True, seed=9, nan=False, spread=0.0, dtype=dtype)
    top = 2.0 ** (113 - int(np.ceil(np.log2(-(-max(lens) // 64) * 64))))
    byte = int(np.floor(np.log2(top / 448))) + 127
    assert LOW < byte < 247 and 448 * 2.0 ** (byte - 127) <= top < 448 * 2.0 ** (byte - 126)
    code = np.arange(c.codes["v"].size).reshape(c.codes["v"].shape) % 27 + 100   # 36 .. 448
    c.codes["v"], c.bytes["v"][:] = code.astype(np.uint8), byte
    c.v = torch.from_numpy(TABLE[c.codes["v"]] * 2.0 ** (byte - 127))
    c.codes["k"][:], c.bytes["k"][:] = 0, 127
    for b, n in enumerate(lens):
        for j in range(64 + 5 * b, n, 64):
            page, slot = c.place(b, j)
            c.codes["k"][page, 0, slot, 0] = 0x53                                  # 11
    c.k = torch.from_numpy(TABLE[c.codes["k"]])
    return c, top


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H", [1, 4, 20])
@pytest.mark.parametrize("lens", [[128], [1000, 64, 400], [9000]], ids=str)
def test_decode(lens, H, dtype):
    c, top = late(lens, dtype)
    q = torch.zeros((len(lens), H, 64), dtype=TD[dtype])
    q[..., 0] = 1 - torch.arange(H) / 64
    ref, tol = attention64(c, q, [1] * len(lens), scale=1.0)
    check(host(B.paged_q8_decode(q.cuda(), c.cuda(B), scale=1.0)) / top, ref / top, tol / top, "decode")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lens,rows,H", [([128], [1], 4), ([128], [100], 4), ([1000, 64, 400], [40, 3, 200], 8),
                                         ([2048], [2048], 4), ([1100], [1100], 32), ([5200], [5200], 32)], ids=str)
def test_prefill(lens, rows, H, dtype):
    c, top = late(lens, dtype)
    q = torch.zeros((sum(rows), H, 64), dtype=TD[dtype])
    q[..., 0] = 1 - torch.arange(H) / 64
    cache = c.cuda(B)
    ref, tol = attention64_large(c, q.cuda(), rows, scale=1.0)
    o = B.paged_q8_prefill(q.cuda(), cache, torch.from_numpy(starts_of(rows)).cuda(), scale=1.0)
    off = (o.double() - ref).abs() - tol
    assert torch.isfinite(o).all() and (off <= 0).all(), f"{int((off > 0).sum())} past the tolerance, by {off.max():.2e}"
