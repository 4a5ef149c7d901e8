"""The paged KV cache's operators against their plain form in 64 bits (paged_util): lengths around
every tile and page border, empty sequences, ragged rows with padding around them, pages without
memory, places that hold NaN and infinities, odd strides and layouts, any group of heads; then
graphs, streams, shared workspaces and the operators together as a server uses them."""
import numpy as np
import pytest
import torch

import bnhip as B
from gpu_util import require_gpu
from paged_util import D, TD, Case, attention64, attention64_large, check, rotate64, rows_of, starts_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def wide(x, pad, fill=float("nan")):
    """x [n, heads, D] on the device as a column range of a wider tensor (and that tensor)."""
    n, h, d = x.shape
    base = torch.full((n, h * d + pad), fill, dtype=x.dtype, device="cuda")
    v = base[:, pad // 2:pad // 2 + h * d].unflatten(1, (h, d))
    v.copy_(x)
    return v, base


def host(t):
    torch.cuda.synchronize()
    return t.double().cpu().numpy()


def bits(t):
    return t.contiguous().view(torch.int16 if t.dtype == torch.bfloat16 else torch.int32)


# ------------------------------------------------------------------- append
APPENDS = [
    # dtype, lens (after), new rows, Hkv, H, page, layout, theta, q: None / "out" / "in place"
    ("bf16", [1, 17, 300], [1, 1, 1], 4, 32, 16, True, 1e4, "out"),
    ("f32", [1, 17, 300], [1, 1, 1], 4, 32, 16, False, 1e4, "in place"),
    ("bf16", [40, 0, 33, 9], [40, 0, 2, 9], 2, 6, 8, "gaps", 1e4, "out"),
    ("f32", [65, 64, 63], [65, 1, 40], 1, 1, 64, True, 5e5, None),
    ("bf16", [70, 3], [70, 5], 3, 15, 8, False, 0.0, "in place"),      # more rows than the length
    ("f32", [1000, 700], [900, 650], 2, 4, 32, True, 1e4, "out"),      # many rows a workgroup
    ("bf16", [1200, 400, 64], [1200, 1, 64], 4, 8, 128, False, 1e4, "in place"),
    ("bf16", [-3, 5], [2, 5], 2, 2, 16, True, 1e4, "out"),             # a negative length is empty
]


@pytest.mark.parametrize("pad", [0, 3])
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_append(case, pad):
    dtype, lens, rows, Hkv, H, page, layout, theta, q_how = case
    print("append", case, pad, flush=True)
    drop = [(0, 0)] if pad else []
    c = Case(dtype, lens, Hkv, page, layout, seed=len(lens), drop=drop, junk=2**31 - 1, pad_table=pad)
    total = sum(rows) + 2 * pad
    n64 = {w: rows_of(dtype, total, h, 7 + i) for i, (w, h) in enumerate((("k", Hkv), ("v", Hkv), ("q", H)))}
    cache = c.cuda(B)
    k, _ = wide(n64["k"].cuda(), 16)
    v, _ = wide(n64["v"].cuda(), 48)
    q, qbase = wide(n64["q"].cuda(), 16)
    out, obase = wide(torch.full_like(n64["q"], 7.0).cuda(), 32, 7.0)
    st = starts_of(rows, pad)
    starts = None if not pad and all(n == 1 for n in rows) else torch.from_numpy(st).cuda()
    want_k, want_v = c.k.double().numpy(), c.v.double().numpy()
    tol_k = np.zeros_like(want_k)
    eps = torch.finfo(TD[dtype]).eps / 2
    want_q = n64["q"].double().numpy().copy() if q_how == "in place" else np.full((total, H, D), 7.0)
    tol_q = np.zeros_like(want_q)

    def tol(x, y):  # cos and sin off by 2 2^-24 (units: up to 1), two products, a sum; then the type's half step
        pair = np.abs(x).reshape(x.shape[0], -1, 2).sum(2, keepdims=True).repeat(2, 2).reshape(x.shape)
        return 0 * y if theta == 0 else pair * 6 * 2.0 ** -24 + (np.abs(y) + pair * 2.0 ** -21) * eps

    for b, n in enumerate(rows):
        for i in range(n):
            row, pos = pad + sum(rows[:b]) + i, max(lens[b], 0) - n + i
            xq, xk = n64["q"][row].double().numpy(), n64["k"][row].double().numpy()
            want_q[row] = rotate64(xq, pos, theta)
            tol_q[row] = tol(xq, want_q[row])
            at = c.place(b, pos)
            if at:
                want_k[at[0], :, at[1]] = rotate64(xk, pos, theta)
                tol_k[at[0], :, at[1]] = tol(xk, want_k[at[0], :, at[1]])
                want_v[at[0], :, at[1]] = n64["v"][row].double().numpy()
    got = B.paged_append(cache, k, v, q=q if q_how else None, q_out=out if q_how == "out" else None,
                         row_starts=starts, theta=theta)
    gk, gv = host(c.kd), host(c.vd)
    for g, w, t, what in ((gk, want_k, tol_k, "k"), (gv, want_v, 0 * tol_k, "v")):
        same = np.isnan(g) & np.isnan(w) | (g == w)
        off = np.abs(np.where(same, 0, np.where(same, 0, g) - np.where(same, 0, w)))
        assert (off <= t).all(), f"{what}: {int((~(off <= t)).sum())} wrong, worst {np.nanmax(off - t):.2e}"
    if q_how:
        assert got is (out if q_how == "out" else q)
        off = np.abs(host(got) - want_q)
        assert (off <= tol_q).all(), f"q: worst {np.max(off - tol_q):.2e}"
        if q_how == "out":   # around the output nothing was touched
            assert (host(obase)[:, :16] == 7.0).all() and (host(obase)[:, -16:] == 7.0).all()
            assert torch.equal(bits(q), bits(n64["q"].cuda()))
    else:
        assert got is None


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_far_positions(dtype):
    """Angles of far positions: a 32-bit product of position and frequency would be off by 0.06 rad
    at 2^20 and by a whole turn and more at 2^29."""
    page, last = 1 << 15, (1 << 30) - 1
    pos = [2 ** 20 + 1, 123456789, last, 2 ** 24 + 3]
    Bn, Hkv, H = len(pos), 1, 2
    table = np.full((Bn, (1 << 30) // page), -1, np.int32)
    for b, p in enumerate(pos):
        table[b, p // page] = b
    kd = torch.zeros((Bn, Hkv, page, D), dtype=TD[dtype], device="cuda")
    vd = torch.zeros_like(kd)
    cache = B.PagedKV(kd, vd, torch.from_numpy(table).cuda(),
                      torch.tensor([p + 1 for p in pos], dtype=torch.int32, device="cuda"))
    k, v, q = (rows_of(dtype, Bn, h, 3 + h) for h in (1, 1, 2))
    out = B.paged_append(cache, k.cuda(), v.cuda(), q=q.cuda())
    eps = torch.finfo(TD[dtype]).eps / 2
    for b, p in enumerate(pos):
        for got, x in ((out[b], q[b]), (kd[b, :, p % page], k[b])):
            w = rotate64(x.double().numpy(), p, 1e4)
            # the test's own angle, in 64 bits: off by 2^30 2^-52 at most
            t = np.abs(x.double().numpy()).sum() * (6 * 2.0 ** -24 + 2.0 ** -20 * (dtype == "f32") * 2.0 ** -1) + np.abs(w) * eps
            assert (np.abs(host(got) - w) <= t).all(), (b, p)
    assert torch.equal(vd[range(Bn), :, [p % page for p in pos]], v.cuda())


# ------------------------------------------------------------------- decode
EDGES = [0, 1, 2, 7, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 95, 96, 97, 127, 128, 129, 255, 256, 257, 300]
DECODES = [
    # dtype, lens, Hkv, H, page, layout, dropped pages (sequence, index)
    ("bf16", EDGES, 2, 16, 16, True, []),
    ("f32", EDGES, 2, 16, 16, True, []),
    ("bf16", EDGES, 1, 3, 8, False, [(20, 3), (23, 0)]),
    ("f32", EDGES, 3, 15, 32, "gaps", [(20, 3), (23, 0), (2, 0)]),
    ("bf16", EDGES, 1, 16, 64, "gaps", [(16, 0), (20, 1)]),
    ("bf16", EDGES, 1, 20, 128, True, []),             # more heads a KV head than a tile holds
    ("f32", EDGES, 2, 66, 8, False, []),
    ("bf16", EDGES[:14], 5, 5, 8, True, [(13, 1), (13, 7)]),
    ("bf16", [1000], 1, 8, 256, True, [(0, 1)]),
    ("bf16", [513] * 3 + [2000], 4, 32, 16, True, []),
    ("f32", [513] * 3 + [2000], 4, 32, 16, False, []),
    ("bf16", [-7, 0, 0], 2, 2, 16, True, []),           # nothing at all
    ("f32", [50, 2 ** 31 - 1, -2 ** 31], 2, 4, 16, True, []),  # lengths past the table
    ("bf16", [3] * 70 + [1], 8, 8, 16, True, []),
]


@pytest.mark.parametrize("case", DECODES, ids=lambda c: f"{c[0]}-{len(c[1])}x{max(c[1])}-{c[2]}-{c[3]}-p{c[4]}-{c[5]}-d{len(c[6])}")
def test_decode(case):
    dtype, lens, Hkv, H, page, layout, drop = case
    print("decode", case, flush=True)
    big = max(lens) > 10 ** 6
    c = Case(dtype, lens, Hkv, page, layout, drop=drop, seed=H, max_pages=4 if big else None,
             junk=2 ** 31 - 1, pad_table=5)
    q = rows_of(dtype, len(lens), H, 1)
    ref, tol = attention64(c, q, [1] * len(lens))
    cache = c.cuda(B)
    qd, _ = wide(q.cuda(), 32)
    o, obase = wide(torch.full_like(q, 7.0).cuda(), 48, 7.0)
    assert B.paged_decode(qd, cache, o=o, scale=0.125) is o
    check(host(o), ref, tol, "decode")
    assert (host(obase)[:, :24] == 7.0).all() and (host(obase)[:, -24:] == 7.0).all()
    ws = B.paged_workspace(cache, H, len(lens))
    ws.fill_(255)                                       # any contents
    for _ in range(3):                                  # and what an earlier call left
        o2 = B.paged_decode(qd, cache, scale=0.125, workspace=ws)
        assert torch.equal(bits(o2), bits(o)), "a second call differs"


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens", [[20011], [9000, 1, 0, 33], [5000, 40, 7000, 1234, 4000]],
                         ids=lambda x: "-".join(map(str, x)))
def test_decode_long(dtype, lens):
    """Caches cut over many workgroups."""
    print("decode long", dtype, lens, flush=True)
    c = Case(dtype, lens, 2, 64, True, drop=[(0, 17)], seed=3)
    q = rows_of(dtype, len(lens), 8, 5)
    ref, tol = attention64(c, q, [1] * len(lens))
    cache = c.cuda(B)
    ws = B.paged_workspace(cache, 8, len(lens))
    for _ in range(2):
        check(host(B.paged_decode(q.cuda(), cache, scale=0.125, workspace=ws)), ref, tol, "decode")


def test_decode_many_sequences():
    """More sequences than one wave scans at a time, in no order of length."""
    lens = [int(x) for x in np.random.default_rng(0).integers(0, 90, 1300)]
    lens[700] = 3000
    c = Case("bf16", lens, 2, 16, True, seed=1)
    q = rows_of("bf16", len(lens), 4, 2)
    ref, tol = attention64(c, q, [1] * len(lens))
    check(host(B.paged_decode(q.cuda(), c.cuda(B), scale=0.125)), ref, tol, "decode")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_thousands_of_sequences(dtype):
    """More sequences than 64 to a lane of the scans, most of them short, some empty: the three calls."""
    n = 4500
    lens = [int(x) for x in np.random.default_rng(1).integers(0, 40, n)]
    lens[5], lens[4321], lens[n - 1] = 700, 2100, 33
    rows = [min(x, 1 + b % 2) for b, x in enumerate(lens)]
    c = Case(dtype, lens, 1, 16, True, seed=2, nan=False)
    q = rows_of(dtype, sum(rows), 2, 3).cuda()
    cache = c.cuda(B)
    ref, tol = attention64_large(c, q, rows)
    got = B.paged_prefill(q, cache, torch.from_numpy(starts_of(rows)).cuda(), scale=0.125)
    assert ((got.double() - ref).abs() <= tol).all()
    one = rows_of(dtype, n, 2, 4).cuda()
    ref, tol = attention64_large(c, one, [1] * n)
    assert ((B.paged_decode(one, cache, scale=0.125).double() - ref).abs() <= tol).all()
    prefix = c.table[4321, :2].copy()
    for b in range(n):
        c.table[b, :2] = prefix
    ref, tol = attention64_large(c, one, [1] * n)
    got = B.paged_decode_shared(one, cache, torch.from_numpy(prefix).cuda(), 32, scale=0.125)
    assert ((got.double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_decode_extreme_scores(dtype):
    """Scores far apart, equal, and -inf: a key of -inf weighs nothing, keys of -inf alone give zeros
    (where V is finite, 0 is what their weights of 0 give)."""
    c = Case(dtype, [200, 70, 40], 1, 16, True, seed=4, nan=False)
    q = rows_of(dtype, 3, 4, 6)
    q[0] *= 300.0
    q[1] = 0.0
    q[2] = 0.0
    q[2, :, 0] = 1.0
    for j in range(40):
        pg, sl = c.place(2, j)
        c.k[pg, :, sl, 0] = float("-inf") if j != 33 else 1.0
    ref, tol = attention64(c, q, [1] * 3)
    got = host(B.paged_decode(q.cuda(), c.cuda(B), scale=0.125))
    check(got[:2], ref[:2], tol[:2], "decode")
    pg, sl = c.place(2, 33)
    assert (got[2] == c.v[pg, 0, sl].double().numpy()).all()
    c.k[pg, :, sl, 0] = float("-inf")
    got = host(B.paged_decode(q.cuda(), c.cuda(B), scale=0.125))
    assert (got[2] == 0.0).all()


def test_decode_offsets_past_32_bits():
    """A pool whose elements pass 2^32: pages far apart, and keys at both ends."""
    n_pages, page, Hkv = 70000, 512, 1
    free, _ = torch.cuda.mem_get_info()
    kd = torch.empty((n_pages, page, Hkv, D), dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    vd = kd.clone()
    assert kd.numel() > 2 ** 31 and free > 4 * kd.numel()
    table = torch.tensor([[n_pages - 1, 0, n_pages // 2], [69000, 12, 41000]], dtype=torch.int32)
    lens = [3 * page, 2 * page + 5]
    r = torch.Generator().manual_seed(0)
    ks, vs = (torch.randn((2, 3 * page, Hkv, D), generator=r).bfloat16() for _ in range(2))
    for b in range(2):
        for i in range(3):
            for pool, x in ((kd, ks), (vd, vs)):
                pool[int(table[b, i]), 0] = x[b, i * page:(i + 1) * page, 0].cuda()
    cache = B.PagedKV(kd, vd, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"))
    q = torch.randn((2, 8, D), generator=r).bfloat16()
    got = host(B.paged_decode(q.cuda(), cache, scale=0.125))
    st = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    got2 = host(B.paged_prefill(q.cuda(), cache, st, scale=0.125))
    got3 = host(B.paged_decode_shared(q[:1].expand(2, 8, D).contiguous().cuda(),
                                      B.PagedKV(kd, vd, table[:1].expand(2, 3).contiguous().cuda(),
                                                cache.seq_lens), table[0, :2].contiguous().cuda(), 2 * page,
                                      scale=0.125))
    for b in range(2):
        k, v = ks[b, :lens[b], 0].double(), vs[b, :lens[b], 0].double()
        p = torch.softmax(0.125 * q[b].double() @ k.T, 1)
        A = (p @ v.abs()).numpy()
        for g in (got, got2):
            assert (np.abs(g[b] - (p @ v).numpy()) <= A * (4 * 2.0 ** -8)).all()
        k, v = ks[0, :lens[b], 0].double(), vs[0, :lens[b], 0].double()
        p = torch.softmax(0.125 * q[0].double() @ k.T, 1)
        assert (np.abs(got3[b] - (p @ v).numpy()) <= (p @ v.abs()).numpy() * (4 * 2.0 ** -8)).all()


def test_append_offsets_past_32_bits():
    """Rows stored in the last and in a middle page of a pool of more than 2^32 bytes."""
    n_pages, page, Hkv = 70000, 512, 1
    pools = [torch.zeros((n_pages, Hkv, page, D), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    table = torch.tensor([[3, n_pages - 1], [69000, 2]], dtype=torch.int32, device="cuda")
    cache = B.PagedKV(*pools, table, torch.tensor([page + 7, 100], dtype=torch.int32, device="cuda"))
    k, v = (torch.randn((2, Hkv, D), device="cuda").bfloat16() for _ in range(2))
    B.paged_append(cache, k, v, theta=0.0)
    for pool, x in zip(pools, (k, v)):
        assert torch.equal(pool[n_pages - 1, 0, 6], x[0, 0]) and torch.equal(pool[69000, 0, 99], x[1, 0])
        assert int(pool.count_nonzero()) == int(x.count_nonzero())


# ------------------------------------------------------------------- prefill
PREFILLS = [
    # dtype, lens (with the new rows), rows, Hkv, H, page, layout, dropped pages, padding rows
    ("bf16", [1, 2, 17, 33], [1, 2, 17, 33], 2, 16, 16, True, [], 0),
    ("f32", [1, 2, 17, 33], [1, 2, 17, 33], 2, 16, 16, True, [], 0),
    ("bf16", [130, 0, 65, 129], [130, 0, 65, 129], 1, 8, 16, False, [(3, 2)], 3),
    ("f32", [130, 0, 65, 129], [130, 0, 65, 129], 1, 4, 16, False, [(3, 2)], 3),
    ("bf16", [300, 40, 257], [3, 17, 200], 2, 12, 8, "gaps", [(0, 0), (2, 30)], 1),
    ("f32", [300, 40, 257], [3, 17, 200], 2, 10, 64, "gaps", [(0, 0)], 1),
    ("bf16", [200, 64], [199, 64], 1, 1, 128, True, [], 0),
    ("bf16", [100, 31], [64, 31], 1, 20, 8, True, [(0, 5)], 0),
    ("bf16", [10, 5], [12, 9], 2, 8, 16, True, [], 2),      # more rows than keys: the first see nothing
    ("f32", [10, -5], [12, 9], 2, 6, 16, True, [], 2),
    ("bf16", [1000, 700, 3], [5, 1, 1], 4, 32, 32, True, [], 0),   # a few rows behind long caches
    ("f32", [1000, 700, 3], [5, 1, 1], 4, 8, 32, False, [], 0),
    ("bf16", [600, 500], [400, 300], 2, 8, 16, False, [], 0),
    ("f32", [400, 300], [400, 100], 1, 3, 256, True, [], 0),
    ("bf16", [2 ** 31 - 1, 40], [70, 40], 1, 4, 16, True, [], 0),  # a length past the table
]


@pytest.mark.parametrize("case", PREFILLS, ids=lambda c: f"{c[0]}-{'_'.join(map(str, c[2]))}of{max(c[1])}-{c[3]}-{c[4]}-p{c[5]}-{c[6]}-d{len(c[7])}-{c[8]}")
def test_prefill(case):
    dtype, lens, rows, Hkv, H, page, layout, drop, pad = case
    print("prefill", case, flush=True)
    big = max(lens) > 10 ** 6
    c = Case(dtype, lens, Hkv, page, layout, drop=drop, seed=H, max_pages=9 if big else None, junk=-5)
    total = sum(rows) + 2 * pad
    q = rows_of(dtype, total, H, 11)
    ref, tol = attention64(c, q, rows, pad)
    cache = c.cuda(B)
    qd, _ = wide(q.cuda(), 32)
    o, obase = wide(torch.full_like(q, 7.0).cuda(), 16, 7.0)
    st = torch.from_numpy(starts_of(rows, pad)).cuda()
    assert B.paged_prefill(qd, cache, st, o=o, scale=0.125) is o
    got = host(o)
    check(got, ref, tol, "prefill")
    for side in (got[:pad], got[total - pad:], host(obase)[:, :8], host(obase)[:, -8:]):
        assert (side == 7.0).all(), "wrote outside its rows"
    ws = B.paged_workspace(cache, H, total)
    ws.fill_(255)
    for _ in range(3):
        o2 = torch.full_like(q, 7.0).cuda()
        B.paged_prefill(qd, cache, st, o=o2, scale=0.125, workspace=ws)
        assert torch.equal(bits(o2), bits(o)), "a second call differs"


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("H", [16, 32, 64])
@pytest.mark.parametrize("lens,rows", [([2 ** 31 - 1, 40], [70, 40]), ([40, 2 ** 31 - 1, 3], [4, 7, 3])], ids=["many", "few"])
def test_prefill_lengths_past_the_table(dtype, H, lens, rows):
    """A length past the table, in large groups of heads, leaves the sequences beside it their rows."""
    print("prefill past the table", dtype, H, lens, rows, flush=True)
    c = Case(dtype, lens, 1, 16, True, seed=H, max_pages=9)
    q = rows_of(dtype, sum(rows), H, 11)
    ref, tol = attention64(c, q, rows)
    st = torch.from_numpy(starts_of(rows)).cuda()
    o = torch.full_like(q, 7.0).cuda()
    check(host(B.paged_prefill(q.cuda(), c.cuda(B), st, o=o, scale=0.125)), ref, tol, "prefill")


# many rows, and rows behind long caches: each kernel that the host can pick, whole units and cut ones
LARGE = [
    ("bf16", [700, 433, 400], [700, 33, 400], 4, 32, 16),
    ("bf16", [1500, 40, 2100, 900], [1500, 33, 1100, 767], 4, 32, 32),
    ("bf16", [2500, 40, 2800, 3900], [2500, 33, 1100, 1767], 4, 32, 16),
    ("bf16", [1200] * 6, [1200] * 6, 8, 24, 8),
    ("bf16", [40000, 9000], [300, 8500], 4, 20, 32),
    ("bf16", [2900, 3300], [2500, 1001], 4, 20, 16),
    ("bf16", [9000, 3000, 70, 20000], [5, 64, 1, 3], 2, 16, 64),
    ("bf16", [16500, 6000], [300, 290], 4, 32, 64),
    ("bf16", [700] * 70 + [3], [10] * 70 + [2], 2, 6, 16),
    ("bf16", [30000], [4], 1, 1, 16),
    ("f32", [700, 433, 400], [700, 33, 400], 2, 16, 16),
    ("f32", [9000, 3000, 70], [5, 64, 1], 2, 6, 64),
    ("f32", [2000, 1100], [1700, 1100], 4, 16, 16),
    ("f32", [300] * 80, [9] * 80, 3, 3, 8),
]


@pytest.mark.parametrize("case", LARGE, ids=lambda c: f"{c[0]}-{len(c[1])}x{max(c[2])}of{max(c[1])}-{c[3]}-{c[4]}-p{c[5]}")
def test_prefill_large(case):
    dtype, lens, rows, Hkv, H, page = case
    print("prefill large", case, flush=True)
    c = Case(dtype, lens, Hkv, page, True, seed=H, drop=[(0, 3)], nan=False)
    q = rows_of(dtype, sum(rows), H, 11).cuda()
    cache = c.cuda(B)
    st = torch.from_numpy(starts_of(rows)).cuda()
    ws = B.paged_workspace(cache, H, sum(rows))
    ws.fill_(255)
    got = [B.paged_prefill(q, cache, st, scale=0.125, workspace=w) for w in (ws, ws, None)]
    ref, tol = attention64_large(c, q, rows)
    over = (got[0].double() - ref).abs() - tol
    assert (over <= 0).all(), f"{int((over > 0).sum())} past the tolerance, by {float(over.max()):.2e}"
    assert torch.equal(bits(got[0]), bits(got[1])) and torch.equal(bits(got[0]), bits(got[2]))


@pytest.mark.parametrize("lens,rows,Hkv,H", [
    ([1, 0, 17, 300, 1000], [1, 0, 17, 200, 1000], 4, 32),
    ([2000, 65, 64, 63], [700, 65, 1, 63], 4, 20),
    ([5000], [513], 8, 64),
    ([33] * 90, [3] * 90, 8, 64),
], ids=str)
def test_prefill_of_a_roomy_table(lens, rows, Hkv, H):
    """Short sequences in a table with room for long ones, whose kernel runs then; what no row
    sees is NaN and infinite."""
    c = Case("bf16", lens, Hkv, 32, False, seed=H, drop=[(0, 0)], spare=1100)
    q = rows_of("bf16", sum(rows), H, 3).cuda()
    cache = c.cuda(B)
    st = torch.from_numpy(starts_of(rows)).cuda()
    ws = B.paged_workspace(cache, H, sum(rows))
    got = [B.paged_prefill(q, cache, st, scale=0.125, workspace=w) for w in (ws, None)]
    ref, tol = attention64_large(c, q, rows)
    over = (got[0].double() - ref).abs() - tol
    assert (over <= 0).all(), f"{int((over > 0).sum())} past the tolerance, by {float(over.max()):.2e}"
    assert torch.equal(bits(got[0]), bits(got[1]))


def test_prefill_starts_that_decrease_stay_inside():
    """row_starts out of order are the caller's mistake: the rows' values are not defined, but
    nothing outside o is written and the call returns."""
    n = 600
    c = Case("bf16", [4000] * 40, 2, 16, True, seed=1, nan=False, spare=0)
    q = rows_of("bf16", n, 16, 2).cuda()
    cache = c.cuda(B)
    st = torch.tensor([0, n] * 20 + [0], dtype=torch.int32).cuda()
    need = B.paged_workspace(cache, 16, n).numel()
    ws = torch.full((need + 4096,), 77, dtype=torch.uint8, device="cuda")
    out = torch.full((n + 64, 16, D), 7.0, dtype=torch.bfloat16, device="cuda")
    B.paged_prefill(q, cache, st, o=out[32:n + 32], scale=0.125, workspace=ws[:need])
    torch.cuda.synchronize()
    assert (out[:32] == 7.0).all() and (out[n + 32:] == 7.0).all() and (ws[need:] == 77).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("what", ["nan", "inf"])
def test_prefill_hidden_values(dtype, what):
    """The value of a key that a later row sees stays out of the rows before it, whatever it is."""
    n = 140
    c = Case(dtype, [n + 20], 1, 16, True, seed=8, nan=False)
    for j in (45, 90, 131, 159):
        pg, sl = c.place(0, j)
        c.v[pg, 0, sl, ::3] = float(what)
    q = rows_of(dtype, n, 4, 9)
    got = host(B.paged_prefill(q.cuda(), c.cuda(B), torch.tensor([0, n], dtype=torch.int32).cuda(), scale=0.125))
    clean = torch.nan_to_num(c.v.double(), nan=0.0, posinf=0.0)
    whole, c.v = c.v, clean.to(TD[dtype])
    ref, tol = attention64(c, q, [n])
    sees = np.arange(n) + 20 >= 45
    bad = np.zeros(D, bool)
    bad[::3] = True
    check(got[~sees], ref[~sees], tol[~sees], "rows that do not see it")
    check(got[sees][:, :, ~bad], ref[sees][:, :, ~bad], tol[sees][:, :, ~bad], "the other columns")
    assert not np.isfinite(got[sees][:, :, bad]).any()
    c.v = whole


@pytest.mark.parametrize("dtype,Hkv,H,rows", [("f32", 2, 8, 500), ("bf16", 4, 32, 1100), ("bf16", 4, 32, 9000)])
def test_prefill_hidden_values_large(dtype, Hkv, H, rows):
    """The same in calls that the host gives to its other kernels: a value in the middle of the new
    rows, in one column and one KV head."""
    past, j = 70, 70 + rows // 2
    c = Case(dtype, [past + rows], Hkv, 16, True, seed=8, nan=False)
    q = rows_of(dtype, rows, H, 9).cuda()
    st = torch.tensor([0, rows], dtype=torch.int32).cuda()
    cache = c.cuda(B)
    want = B.paged_prefill(q, cache, st, scale=0.125)
    pg, sl = c.place(0, j)
    old = c.vd[pg, 1, sl, 5].clone()
    for bad in (float("nan"), float("inf"), float("-inf")):
        c.vd[pg, 1, sl, 5] = bad
        got = B.paged_prefill(q, cache, st, scale=0.125)
        G = H // Hkv
        hit = torch.zeros(got.shape, dtype=torch.bool, device="cuda")
        hit[j - past:, G:2 * G, 5] = True
        assert not torch.isfinite(got[hit]).any()
        if bad == bad:
            assert (got[hit] == bad).all()
        assert torch.equal(bits(got[~hit]), bits(want[~hit]))
    c.vd[pg, 1, sl, 5] = old


# each prefill kernel: dtype, cached keys, new rows, KV heads, heads, room of the table in pages of 16
KERNELS = [("f32", 20, 140, 1, 4, 0), ("bf16", 20, 140, 1, 4, 0), ("bf16", 20, 140, 4, 32, 0),
           ("bf16", 70, 500, 4, 32, 0), ("bf16", 70, 1100, 4, 32, 0), ("bf16", 0, 4096, 4, 32, 0),
           ("bf16", 70, 1100, 4, 32, 1100), ("f32", 70, 500, 2, 8, 0)]


@pytest.mark.parametrize("kernel", KERNELS, ids=lambda k: "-".join(map(str, k)))
@pytest.mark.parametrize("what", ["key", "query", "inf"])
def test_prefill_scores_of_other_rows(kernel, what):
    """A key that is NaN reaches the rows that see it, one of infinite scores no row that does not, and
    a NaN query none but its own."""
    dtype, past, n, Hkv, H, spare = kernel
    c = Case(dtype, [past + n], Hkv, 16, True, seed=8, nan=False, spare=2 + spare)
    q = rows_of(dtype, n, H, 9).cuda()
    st = torch.tensor([0, n], dtype=torch.int32).cuda()
    cache = c.cuda(B)
    ref, tol = attention64_large(c, q, [n])
    hit = torch.zeros((n, H), dtype=torch.bool, device="cuda")
    G = H // Hkv
    if what == "query":
        for i, h in ((0, 0), (5, H - 1), (n // 2, G // 2), (n - 1, 0)):
            q[i, h, 7] = float("nan")
            hit[i, h] = True
    else:
        i = n // 2 + 3
        pg, sl = c.place(0, past + i)
        c.kd[pg, Hkv - 1, sl, 11] = float("nan") if what == "key" else float("inf")
        hit[i:, H - G:] = True
    got = B.paged_prefill(q, cache, st, scale=0.125)
    over = (got.double() - ref).abs() - tol
    assert (over[~hit] <= 0).all(), f"{int((~(over[~hit] <= 0)).sum())} elements of rows that it must not reach"
    if what == "inf":   # where its score is -inf it weighs nothing, else the row is NaN
        up = hit & (q[:, :, 11] > 0)
        assert torch.isnan(got[up]).all() and torch.isfinite(got[hit & (q[:, :, 11] < 0)]).all()
    else:
        assert torch.isnan(got[hit]).all()


@pytest.mark.parametrize("kernel", KERNELS, ids=lambda k: "-".join(map(str, k)))
def test_prefill_values_of_no_weight(kernel):
    """An infinite element of a key that weighs nothing makes that element of the rows that see it infinite
    or NaN, in tiles that all rows of a workgroup see and in others."""
    dtype, past, n, Hkv, H, spare = kernel
    c = Case(dtype, [past + n], Hkv, 16, True, seed=8, nan=False, spare=2 + spare)
    q = rows_of(dtype, n, H, 9).cuda().abs()
    st = torch.tensor([0, n], dtype=torch.int32).cuda()
    cache = c.cuda(B)
    hit = torch.zeros((n, D), dtype=torch.bool, device="cuda")
    for j, d in ((3, 5), (past + n // 2, 8), (past + n - 2, 63)):
        pg, sl = c.place(0, j)
        c.kd[pg, :, sl] = -1000.0
        hit[max(j - past, 0):, d] = True
    ref, tol = attention64_large(c, q, [n])
    for j, d in ((3, 5), (past + n // 2, 8), (past + n - 2, 63)):
        pg, sl = c.place(0, j)
        c.vd[pg, :, sl, d] = float("inf")
    hit = hit[:, None].expand(n, H, D)
    got = B.paged_prefill(q, cache, st, scale=0.125)
    over = (got.double() - ref).abs() - tol
    assert not torch.isfinite(got[hit]).any() and (over[~hit] <= 0).all()
    last = B.paged_decode(q[-1:].contiguous(), cache, scale=0.125)
    assert torch.equal(torch.isfinite(last)[0], ~hit[-1])


@pytest.mark.parametrize("dtype,Bn,P", [("f32", 40, 304), ("bf16", 40, 304), ("bf16", 100, 16384)])
def test_shared_scores_of_other_rows(dtype, Bn, P):
    """The same behind a shared prefix: sequences that end before the key, and a NaN query among the batch."""
    H, Hkv, page, dirty = 32, 4, 16, P - 40
    lens = [P + b % 5 if b % 3 else P - 64 - b for b in range(Bn)]
    c = Case(dtype, lens, Hkv, page, True, seed=P, nan=False)
    q = rows_of(dtype, Bn, H, 1).cuda()
    cache = c.cuda(B)
    prefix = c.table[1, :P // page].copy()
    own = c.table.copy()
    c.table[:, :P // page] = prefix     # attention64_large takes the prefix from each table
    ref, tol = attention64_large(c, q, [1] * Bn)
    c.table[:] = own
    cache.k_pages[int(prefix[dirty // page]), 1, dirty % page, 3] = float("nan")
    q[4, 9] = float("nan")
    got = B.paged_decode_shared(q, cache, torch.from_numpy(prefix).cuda(), P, scale=0.125)
    hit = torch.zeros((Bn, H), dtype=torch.bool, device="cuda")
    hit[torch.tensor([x > dirty for x in lens]), H // Hkv:2 * H // Hkv] = True
    hit[4, 9] = True
    assert torch.isnan(got[hit]).all()
    over = (got.double() - ref).abs() - tol
    assert (over[~hit] <= 0).all(), f"{int((~(over[~hit] <= 0)).sum())} elements of rows that it must not reach"


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_prefill_extreme_scores(dtype):
    """Growing scores (the running maximum moves at every tile), then huge ones."""
    n = 150
    c = Case(dtype, [n + 70], 1, 16, True, seed=8, nan=False)
    for j in range(n + 70):
        pg, sl = c.place(0, j)
        c.k[pg, 0, sl] = c.k[pg, 0, sl] * (1 + j)
    q = rows_of(dtype, n, 8, 9)
    ref, tol = attention64(c, q, [n])
    got = host(B.paged_prefill(q.cuda(), c.cuda(B), torch.tensor([0, n], dtype=torch.int32).cuda(), scale=0.125))
    check(got, ref, tol, "prefill")


def test_prefill_without_starts_is_decode():
    c = Case("bf16", [5, 100, 64], 2, 16, True, seed=2)
    q = rows_of("bf16", 3, 16, 3)
    ref, tol = attention64(c, q, [1] * 3)
    check(host(B.paged_prefill(q.cuda(), c.cuda(B), scale=0.125)), ref, tol, "prefill")


# ------------------------------------------------------------------- shared prefix
SHARED = [
    # dtype, prefix, own keys per sequence, Hkv, H, page, layout
    ("bf16", 0, [1, 40, 5], 2, 16, 16, True),
    ("bf16", 1, [1, 40, 5], 2, 16, 16, True),
    ("f32", 33, [1, 40, 5], 2, 6, 16, False),
    ("bf16", 64, [1, 70, 0, 5, 129], 1, 8, 64, True),
    ("f32", 64, [1, 70, 0, 5, 129], 1, 8, 64, True),
    ("bf16", 300, [3, 1, 1, 90] * 9, 2, 16, 16, False),
    ("f32", 300, [3, 1, 1, 90] * 9, 2, 4, 8, "gaps"),
    ("bf16", 1000, [10], 1, 20, 32, True),
    ("bf16", 129, [-100, -129, -1, 20, -300], 2, 12, 16, "gaps"),   # shorter than the prefix, empty
    ("f32", 129, [-100, -129, -1, 20, -300], 2, 12, 16, True),
    ("bf16", 2500, [1] * 40 + [700], 1, 3, 128, True),
    ("bf16", 70, [0] * 300, 1, 8, 8, True),
]


@pytest.mark.parametrize("case", SHARED, ids=lambda c: f"{c[0]}-P{c[1]}-{len(c[2])}-{c[3]}-{c[4]}-p{c[5]}-{c[6]}")
def test_shared(case):
    dtype, P, own, Hkv, H, page, layout = case
    print("shared", case, flush=True)
    lens = [P + n for n in own]
    c = Case(dtype, lens, Hkv, page, layout, seed=P, nan=False)
    # the common keys in pages of their own; what the tables say of pages wholly below P is not looked at
    n_prefix = -(-P // page)
    r = np.random.default_rng(P + 1)
    extra = [torch.from_numpy(r.standard_normal((n_prefix, Hkv, page, D)).astype(np.float32)).to(TD[dtype])
             for _ in range(2)]
    prefix = np.arange(c.n_pages, c.n_pages + n_prefix, dtype=np.int32)
    c.k, c.v = torch.cat([c.k, extra[0]]), torch.cat([c.v, extra[1]])
    c.n_pages += n_prefix
    c.table[:, :P // page] = 2 ** 31 - 1
    if P % page:
        c.v[-1, :, P % page:] = float("nan")
        for b in range(len(lens)):      # and a shared page's part of the sequence's copy neither
            if 0 <= c.table[b, P // page] < c.n_pages:
                c.v[int(c.table[b, P // page]), :, :P % page] = float("nan")
    q = rows_of(dtype, len(lens), H, 1)
    ref, tol = attention64(c, q, [1] * len(lens), prefix=prefix, prefix_len=P)
    cache = c.cuda(B)
    qd, _ = wide(q.cuda(), 32)
    o, obase = wide(torch.full_like(q, 7.0).cuda(), 48, 7.0)
    pd = torch.from_numpy(prefix).cuda()
    assert B.paged_decode_shared(qd, cache, pd, P, o=o, scale=0.125) is o
    check(host(o), ref, tol, "shared")
    assert (host(obase)[:, :24] == 7.0).all() and (host(obase)[:, -24:] == 7.0).all()
    ws = B.paged_workspace(cache, H, len(lens), P)
    ws.fill_(255)
    for _ in range(3):
        o2 = B.paged_decode_shared(qd, cache, pd, P, scale=0.125, workspace=ws)
        assert torch.equal(bits(o2), bits(o)), "a second call differs"


@pytest.mark.parametrize("case", [("bf16", 2048, 200, 700, 4, 32, 16), ("bf16", 4096, 150, 3000, 8, 8, 32),
                                  ("bf16", 640, 700, 90, 4, 20, 64), ("f32", 1024, 70, 900, 4, 16, 16),
                                  ("bf16", 4096, 210, 700, 4, 32, 16), ("bf16", 16384, 100, 300, 1, 16, 32),
                                  ("bf16", 16384, 100, 100, 4, 20, 64)],
                         ids=lambda c: "-".join(map(str, c)))
def test_shared_large(case):
    """Large batches (the pipelined kernel) and own keys cut over workgroups; some sequences shorter
    than the prefix, some empty, a page of the prefix and one of a sequence without memory."""
    dtype, P, Bn, own, Hkv, H, page = case
    r = np.random.default_rng(P)
    lens = [P + int(x) for x in r.integers(0, own + 1, Bn)]
    lens[3], lens[5], lens[7], lens[11] = 0, P - 100, P, 17
    c = Case(dtype, lens, Hkv, page, True, seed=P, nan=False, drop=[(9, P // page)])
    prefix = c.table[Bn - 1, :P // page].copy()
    prefix[2] = -1
    q = rows_of(dtype, Bn, H, 1).cuda()
    cache = c.cuda(B)
    pd = torch.from_numpy(prefix).cuda()
    ws = B.paged_workspace(cache, H, Bn, P)
    ws.fill_(255)
    got = [B.paged_decode_shared(q, cache, pd, P, scale=0.125, workspace=w) for w in (ws, ws, None)]
    pages_of = c.table.copy()
    for b in range(Bn):     # attention64_large takes the prefix from each table
        c.table[b, :P // page] = prefix
    ref, tol = attention64_large(c, q, [1] * Bn)
    c.table[:] = pages_of
    over = (got[0].double() - ref).abs() - tol
    assert (over <= 0).all(), f"{int((over > 0).sum())} past the tolerance, by {float(over.max()):.2e}"
    assert torch.equal(bits(got[0]), bits(got[1])) and torch.equal(bits(got[0]), bits(got[2]))


@pytest.mark.parametrize("Bn,P", [(100, 1024), (100, 16384)], ids=["few", "many"])
def test_shared_prefix_values_that_short_sequences_do_not_see(Bn, P):
    """Infinite and NaN values of the prefix behind the end of some sequences: these come out as
    without them, bit for bit, and the others carry them."""
    H, Hkv, page, dirty = 32, 4, 32, P - 40
    lens = [P + b % 5 if b % 3 else P - 64 - b for b in range(Bn)]
    c = Case("bf16", lens, Hkv, page, True, seed=P, nan=False)
    q = rows_of("bf16", Bn, H, 1).cuda()
    cache = c.cuda(B)
    prefix = torch.from_numpy(c.table[1, :P // page].copy()).cuda()
    ws = B.paged_workspace(cache, H, Bn, P)
    clean = B.paged_decode_shared(q, cache, prefix, P, scale=0.125, workspace=ws)
    at = (int(c.table[1, dirty // page]), slice(None), dirty % page)
    cache.v_pages[at][:, 3] = float("inf")
    cache.v_pages[at][:, 40] = float("nan")
    cache.v_pages[at][:, 41] = float("-inf")
    got = B.paged_decode_shared(q, cache, prefix, P, scale=0.125, workspace=ws)
    sees = torch.tensor([n > dirty for n in lens]).cuda()
    assert torch.equal(bits(got[~sees]), bits(clean[~sees])) and torch.isfinite(clean.float()).all()
    assert (got[sees][..., 3] == float("inf")).all() and (got[sees][..., 41] == float("-inf")).all()
    assert torch.isnan(got[sees][..., 40]).all()
    rest = [d for d in range(64) if d not in (3, 40, 41)]
    assert torch.equal(bits(got[sees][..., rest].contiguous()), bits(clean[sees][..., rest].contiguous()))


def test_shared_prefix_page_without_memory():
    c = Case("bf16", [90, 120, 70], 2, 16, True, seed=2)
    prefix = c.table[0, :4].copy()
    prefix[1] = -1
    q = rows_of("bf16", 3, 8, 3)
    ref, tol = attention64(c, q, [1] * 3, prefix=prefix, prefix_len=64)
    got = B.paged_decode_shared(q.cuda(), c.cuda(B), torch.from_numpy(prefix).cuda(), 64, scale=0.125)
    check(host(got), ref, tol, "shared")


@pytest.mark.parametrize("dtype,lens,rows,H", [("bf16", [9000, 300, 17], [1, 1, 1], 32), ("f32", [900, 0, 17], [1, 1, 1], 8),
                                               ("bf16", [3000, 300, 17], [700, 290, 17], 32), ("f32", [900, 300, 17], [70, 290, 17], 8),
                                               ("bf16", [20000, 6000], [300, 290], 32), ("bf16", [6000] * 2, [4400, 4500], 32)], ids=str)
def test_outputs_in_the_queries_place(dtype, lens, rows, H):
    """o may be q itself: decode, prefill and a shared prefix give the same bits."""
    c = Case(dtype, lens, 4, 16, True, seed=H, nan=False, spare=2)
    cache = c.cuda(B)
    q = rows_of(dtype, sum(rows), H, 5).cuda()
    st = torch.from_numpy(starts_of(rows)).cuda()
    prefix = cache.page_table[0, :16].contiguous()
    one = q[:len(lens)]
    for x, call in ((q, lambda q, o: B.paged_prefill(q, cache, st, o=o, scale=0.125)),
                    (one, lambda q, o: B.paged_decode(q, cache, o=o, scale=0.125)),
                    (one, lambda q, o: B.paged_decode_shared(q, cache, prefix, 250, o=o, scale=0.125))):
        want = call(x, None)
        for _ in range(3):
            y = x.clone()
            assert call(y, y) is y
            assert torch.equal(bits(y), bits(want))


# ------------------------------------------------------------------- graphs, streams
def big_case():
    c = Case("bf16", [3000, 17, 900, 2100], 2, 16, True, seed=5, nan=False)
    return c, c.cuda(B)


@pytest.mark.parametrize("op", ["decode", "prefill", "shared"])
def test_graphs_share_a_workspace(op):
    """Two graphs with one workspace, replayed in turn with eager calls on it and changed lengths
    in between: each replay equals the eager call."""
    c, cache = big_case()
    q = rows_of("bf16", 8, 16, 6).cuda()
    st = torch.tensor([0, 4, 5, 5, 8], dtype=torch.int32).cuda()
    pages = cache.page_table[0, :40].contiguous()
    ws = B.paged_workspace(cache, 16, 8, 600)
    ws.fill_(77)

    def call(x, o):
        if op == "decode":
            B.paged_decode(x[:4], cache, o=o[:4], scale=0.125, workspace=ws)
        elif op == "prefill":
            B.paged_prefill(x, cache, st, o=o, scale=0.125, workspace=ws)
        else:
            B.paged_decode_shared(x[:4], cache, pages, 600, o=o[:4], scale=0.125, workspace=ws)

    xs, outs, graphs = [q, (q * 0.5)], [], []
    s = torch.cuda.Stream()
    for x in xs:
        o = torch.zeros_like(q)
        with torch.cuda.stream(s):
            call(x, o)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(x, o)
        outs.append(o)
        graphs.append(g)
    for step, lens in enumerate(([3000, 17, 900, 2100], [1, 0, 640, 3000], [2999, 300, 601, 5], [3000, 17, 900, 2100])):
        cache.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        for x, o, g in zip(xs, outs, graphs):
            o.zero_()
            g.replay()
            torch.cuda.synchronize()
            got = o.clone()
            want = torch.zeros_like(q)
            call(x, want)
            torch.cuda.synchronize()
            assert torch.equal(bits(got), bits(want)), f"step {step}"
            junk = torch.empty_like(ws)
            if step == 1:
                ws.copy_(junk.random_(0, 256))


def test_a_graph_of_cut_units():
    """Long sequences, whose units of 256 rows are cut and added up in the launch, replayed from a
    graph under other lengths, with eager calls of another shape on the same workspace between."""
    lens, rows = [17000, 6000, 20000], [300, 1, 45]
    c = Case("bf16", lens, 2, 64, True, seed=3, nan=False)
    cache = c.cuda(B)
    q = rows_of("bf16", sum(rows), 32, 6).cuda()
    st = torch.from_numpy(starts_of(rows)).cuda()
    ws = B.paged_workspace(cache, 32, sum(rows))
    o = torch.zeros_like(q)
    B.paged_prefill(q, cache, st, o=o, scale=0.125, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        B.paged_prefill(q, cache, st, o=o, scale=0.125, workspace=ws)
    for now in (lens, [300, 1, 45], [16999, 0, 9000], lens):
        cache.seq_lens.copy_(torch.tensor(now, dtype=torch.int32))
        o.zero_()
        g.replay()
        torch.cuda.synchronize()
        got = o.clone()
        assert torch.equal(bits(got), bits(B.paged_prefill(q, cache, st, scale=0.125)))
        B.paged_decode(q[:3], cache, scale=0.125, workspace=ws)
        B.paged_prefill(q[:7], cache, torch.tensor([0, 4, 4, 7], dtype=torch.int32).cuda(), scale=0.125, workspace=ws)
    c.lens = lens
    ref, tol = attention64_large(c, q, rows)
    over = (got.double() - ref).abs() - tol
    assert (over <= 0).all(), f"{int((over > 0).sum())} past the tolerance, by {float(over.max()):.2e}"


def test_calls_on_two_streams():
    """Calls in flight at once, each with its own workspace or the pool's."""
    c, cache = big_case()
    q = rows_of("bf16", 4, 16, 6).cuda()
    want = B.paged_decode(q, cache, scale=0.125)
    pages = cache.page_table[0, :40].contiguous()
    want_s = B.paged_decode_shared(q, cache, pages, 600, scale=0.125)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    wss = [B.paged_workspace(cache, 16, 4, 600), B.paged_workspace(cache, 16, 4, 600), None]
    got = []
    for _ in range(5):
        for s, ws in zip(streams, wss):
            with torch.cuda.stream(s):
                got.append((B.paged_decode(q, cache, scale=0.125, workspace=ws), want))
                got.append((B.paged_decode_shared(q, cache, pages, 600, scale=0.125, workspace=ws), want_s))
    torch.cuda.synchronize()
    for g, w in got:
        assert torch.equal(bits(g), bits(w))


@pytest.mark.parametrize("op", ["decode", "prefill", "shared"])
def test_calls_on_a_given_stream(op):
    """stream=: the output is not memory that the present stream still writes, and once dropped it is not
    the present stream's while the call's is at work."""
    c, cache = big_case()
    q = rows_of("bf16", 4, 16, 6).cuda()
    st = torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32).cuda()
    pages = cache.page_table[0, :40].contiguous()
    ws = B.paged_workspace(cache, 16, 4, 600)
    work = torch.zeros((8192, 8192), dtype=torch.bfloat16, device="cuda")
    s = torch.cuda.Stream()

    def call(stream=None):
        if op == "decode":
            return B.paged_decode(q, cache, scale=0.125, workspace=ws, stream=stream)
        if op == "prefill":
            return B.paged_prefill(q, cache, st, scale=0.125, workspace=ws, stream=stream)
        return B.paged_decode_shared(q, cache, pages, 600, scale=0.125, workspace=ws, stream=stream)

    def busy():     # some milliseconds
        for _ in range(4):
            torch.mm(work, work)

    want = call()
    torch.cuda.synchronize()
    for _ in range(3):
        t = torch.empty_like(q)
        busy()
        t.fill_(7.0)
        at = t.data_ptr()
        del t       # free for the present stream's next tensor, written when busy() is through
        o = call(s)
        assert o.data_ptr() != at
        torch.cuda.synchronize()
        assert torch.equal(bits(o), bits(want))
        with torch.cuda.stream(s):
            busy()
        o = call(s)
        at = o.data_ptr()
        del o
        t = torch.empty_like(q)
        assert t.data_ptr() != at
        torch.cuda.synchronize()


def test_host_memory_is_refused():
    c = Case("bf16", [5, 9], 2, 16, True)
    kv = B.PagedKV(c.k, c.v, torch.from_numpy(c.table.copy()), torch.tensor([5, 9], dtype=torch.int32))
    q = rows_of("bf16", 2, 4, 1)
    s, m = B.status_of("bn_paged_decode", kv.ref, q.data_ptr(), q.data_ptr(), 4, 256, 256, 0.125, None, 0, None)
    assert s == B.BN_ERR_NOT_DEVICE and "only GPU implementation available" in m


def test_a_workspace_after_starts_that_decrease():
    """A call with row_starts out of order leaves nothing in its workspace that a later one trips over."""
    for n, H, Hkv in ((600, 16, 2), (40, 8, 1)):
        c = Case("bf16", [5000] * 40, Hkv, 16, True, seed=n, nan=False, spare=0)
        q = rows_of("bf16", n, H, 2).cuda()
        cache = c.cuda(B)
        good = torch.tensor([0] + [n // 2] * 39 + [n], dtype=torch.int32).cuda()
        ws = B.paged_workspace(cache, H, n)
        want = B.paged_prefill(q, cache, good, scale=0.125)
        for bad in ([0, n] * 20 + [0], [n, 0] * 20 + [n], [0] + [n, n // 2] * 20, list(range(40, -1, -1))):
            B.paged_prefill(q, cache, torch.tensor(bad, dtype=torch.int32).cuda(), scale=0.125, workspace=ws)
            for _ in range(2):
                got = B.paged_prefill(q, cache, good, scale=0.125, workspace=ws)
                assert torch.equal(bits(got), bits(want))


# ------------------------------------------------------------------- together
@pytest.mark.parametrize("dtype,page,layout", [("f32", 16, True), ("bf16", 8, False), ("bf16", 32, True)])
def test_a_server_run(dtype, page, layout):
    """Prompts of three users arrive and are answered token by token: append and prefill, one more
    chunk for one of them, then append and decode steps, and a shared-prefix decode over the same
    tables; every output against 64 bits over the cache's own (checked) contents."""
    Hkv, H, prompt = 2, 8, [37, 5, 64]
    room = [120] * 3
    c = Case(dtype, room, Hkv, page, layout, seed=21, nan=True)
    c.k[:], c.v[:] = float("nan"), float("nan")       # nothing is there before it is appended
    cache = c.cuda(B)
    eps = torch.finfo(TD[dtype]).eps / 2
    r = np.random.default_rng(5)
    truth_k = {}

    def step(rows, op):
        c.lens = [a + n for a, n in zip(c.lens, rows)]
        cache.seq_lens.copy_(torch.tensor(c.lens, dtype=torch.int32))
        n = sum(rows)
        qkv = torch.from_numpy(r.standard_normal((n, (H + 2 * Hkv) * D)).astype(np.float32)).to(TD[dtype])
        x = qkv.cuda()
        q, k, v = (t.unflatten(1, (-1, D)) for t in x.split([H * D, Hkv * D, Hkv * D], 1))
        st = torch.from_numpy(starts_of(rows)).cuda()
        B.paged_append(cache, k, v, q=q, row_starts=st)
        o = op(q, st)
        torch.cuda.synchronize()
        c.k, c.v = c.kd.cpu().contiguous(), c.vd.cpu().contiguous()
        at = 0
        for b, m in enumerate(rows):
            for i in range(m):
                j = c.lens[b] - m + i
                raw = qkv[at + i].double().numpy().reshape(-1, D)
                turned = rotate64(raw[:H + Hkv], j, 1e4)
                pg, sl = c.place(b, j)
                pair = 2 * np.abs(raw).max() * 6 * 2.0 ** -24
                assert (np.abs(c.k[pg, :, sl].double().numpy() - turned[H:]) <= pair + np.abs(turned[H:]) * eps * 1.01).all()
                assert (c.v[pg, :, sl].double().numpy() == raw[H + Hkv:]).all()
                assert (np.abs(host(q[at + i]) - turned[:H]) <= pair + np.abs(turned[:H]) * eps * 1.01).all()
            at += m
        ref, tol = attention64(c, q.cpu(), rows)
        check(host(o), ref, tol, f"lengths {c.lens}")

    c.lens = [0, 0, 0]
    step(prompt, lambda q, st: B.paged_prefill(q, cache, st, scale=0.125))
    step([0, 30, 2], lambda q, st: B.paged_prefill(q, cache, st, scale=0.125))
    for _ in range(6):
        step([1, 1, 1], lambda q, st: B.paged_decode(q.contiguous(), cache, scale=0.125))
    # the last two users' tables start like the first one's: their copies of its pages
    common = 32
    for b in (1, 2):
        for i in range(common // page):
            cache.page_table[b, i] = cache.page_table[0, i]
            c.table[b, i] = c.table[0, i]
    pages = cache.page_table[0, :common // page].contiguous()
    for _ in range(2):
        step([1, 1, 1], lambda q, st: B.paged_decode_shared(q.contiguous(), cache, pages, common, scale=0.125))
