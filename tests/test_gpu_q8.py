"""The paged KV cache in 8 bits against its plain form in 64 bits (q8_util): codes and scales of
appended rows, older rows of a block under a larger scale, values read back, and the attention over
the pages: lengths around every block, tile and page border, empty sequences, ragged rows with padding
around them, pages without memory, places that hold NaN, odd strides and layouts, any group of heads."""
import numpy as np
import pytest
import torch

import bnhip as B
from gpu_util import require_gpu
from paged_util import D, TD, attention64, attention64_large, check, rotate64, rows_of, starts_of
from q8_util import BLOCK, HIGH, LOW, TABLE, Case8, byte_of, codes_of, half_step, scale_of, store
from test_gpu_paged import bits, host, wide

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def same_bytes(got, want, what):
    got, want = got.cpu().numpy(), np.asarray(want)
    if "codes" in what:      # two codes are NaN
        got, want = (np.where(x == 255, 127, x) for x in (got, want))
    bad = np.argwhere(got != want)
    assert not len(bad), f"{what}: {len(bad)} bytes differ, first at {bad[0]}: {got[tuple(bad[0])]} for {want[tuple(bad[0])]}"


# --------------------------------------------------------------------- read
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_every_code_under_every_scale(dtype):
    codes = np.tile(np.arange(1024) % 256, 256).astype(np.uint8).reshape(256, 1, 16, D)
    byte = np.arange(256, dtype=np.uint8).reshape(256, 1, 1)
    table = torch.arange(256, dtype=torch.int32, device="cuda").view(1, 256)
    cache = B.PagedQ8(*(torch.from_numpy(x).cuda() for x in (codes, codes, byte, byte)), table,
                      torch.tensor([4096], dtype=torch.int32, device="cuda"))
    st = torch.tensor([0, 4096], dtype=torch.int32, device="cuda")
    k, v = B.paged_q8_read(cache, st, n_rows=4096, dtype=TD[dtype])
    with np.errstate(over="ignore"):
        want = (TABLE[codes] * scale_of(byte)[..., None]).astype(np.float32)   # exact, or past the range
    big = torch.from_numpy(want).to(TD[dtype]).cuda().view(4096, 1, D)
    for got in (k, v):
        assert torch.equal(torch.isnan(got), torch.isnan(big))
        assert torch.equal(torch.nan_to_num(got, 0.0), torch.nan_to_num(big, 0.0))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("page,layout,pad", [(16, True, 0), (32, False, 3), (128, "gaps", 2)])
def test_read(dtype, page, layout, pad):
    lens = [300, 0, 17, 16, 15, 1, 40, -5, 33]
    rows = [300, 0, 5, 16, 20, 1, 33, 2, 32]      # 20: more rows than the length
    c = Case8(lens, 3, page, layout, seed=page, drop=[(0, 0)], junk=2 ** 31 - 1, pad_table=pad)
    cache = c.cuda(B)
    total = sum(rows) + 2 * pad
    st = torch.from_numpy(starts_of(rows, pad)).cuda()
    outs = [wide(torch.full((total, 3, D), 7.0, dtype=TD[dtype]).cuda(), 16, 7.0) for _ in range(2)]
    for which in ("both", "k", "v"):
        for o, base in outs:
            base.fill_(7.0)
        k, v = (o if which in ("both", n) else None for (o, _), n in zip(outs, "kv"))
        got = B.paged_q8_read(cache, st, k=k, v=v)
        assert got[0] is k and got[1] is v
        for (o, base), name in zip(outs, "kv"):
            want = np.full((total, 3, D), 7.0)
            if which in ("both", name):
                at = pad
                for b, n in enumerate(rows):
                    for i in range(n):
                        place = c.place(b, max(lens[b], 0) - n + i)
                        want[at + i] = getattr(c, name)[place[0], :, place[1]].numpy() if place else 0.0
                    at += n
            assert (host(o) == want).all(), (which, name)
            assert (host(base)[:, :8] == 7.0).all() and (host(base)[:, -8:] == 7.0).all()
    one = B.paged_q8_read(cache)                  # without row_starts: the last row of each
    for b, n in enumerate(lens):
        place = c.place(b, max(n, 0) - 1)
        for got, name in zip(one, "kv"):
            assert (host(got)[b] == (getattr(c, name)[place[0], :, place[1]].numpy() if place else 0.0)).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_read_many_rows(dtype):
    """More bytes than the caches keep (another kernel), ragged, with padding around."""
    Hkv, page, n = 4, 64, 130000 if dtype == "bf16" else 70000
    lens = [n - 3000, 2500, 777]
    r = torch.Generator(device="cuda").manual_seed(3)
    need = [-(-x // page) for x in lens]
    order = torch.randperm(sum(need) + 3, generator=r, device="cuda").int()
    table = torch.full((3, max(need)), -1, dtype=torch.int32, device="cuda")
    for b, m in enumerate(need):
        table[b, :m] = order[sum(need[:b]):sum(need[:b + 1])]
    codes = [torch.randint(0, 127, (sum(need) + 3, Hkv, page, D), generator=r, device="cuda", dtype=torch.uint8) for _ in "kv"]
    sc = [torch.randint(110, 140, (sum(need) + 3, Hkv, page // BLOCK), generator=r, device="cuda", dtype=torch.uint8) for _ in "kv"]
    cache = B.PagedQ8(*codes, *sc, table, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    st = torch.from_numpy(starts_of(lens, 5)).cuda()
    outs = [torch.full((sum(lens) + 12, Hkv, D), 7.0, dtype=TD[dtype], device="cuda") for _ in "kv"]
    B.paged_q8_read(cache, st, k=outs[0], v=outs[1])
    values = torch.from_numpy(TABLE).float().cuda()
    for o, c, s in zip(outs, codes, sc):
        at = 5
        assert (o[:5] == 7.0).all() and (o[-7:] == 7.0).all()
        for b, m in enumerate(lens):
            j = torch.arange(m, device="cuda")
            pg, sl = table[b, j // page].long(), j % page
            want = torch.ldexp(values[c[pg, :, sl].long()], s[pg, :, sl // BLOCK].int()[..., None] - 127)
            assert torch.equal(o[at:at + m].float(), want)
            at += m


# ------------------------------------------------------------------- append
APPENDS = [
    # dtype, lens (after), new rows, Hkv, H, page, layout, theta, q: None / "out" / "in place", norms
    ("bf16", [1, 17, 300], [1, 1, 1], 4, 32, 16, True, 1e4, "out", "qk"),
    ("f32", [1, 17, 300], [1, 1, 1], 4, 32, 16, False, 1e4, "in place", ""),
    ("bf16", [40, 0, 33, 9], [40, 0, 2, 9], 2, 6, 32, "gaps", 1e4, "out", "k"),
    ("f32", [65, 64, 63], [65, 1, 40], 1, 1, 64, True, 5e5, None, "k"),
    ("bf16", [70, 3], [70, 5], 3, 15, 16, False, 0.0, "in place", "q"),     # more rows than the length
    ("f32", [1000, 700], [900, 650], 2, 4, 32, True, 1e4, "out", "qk"),
    ("bf16", [1200, 400, 64], [1200, 1, 64], 4, 8, 128, False, 1e4, "in place", ""),
    ("bf16", [-3, 5], [2, 5], 2, 2, 16, True, 1e4, "out", "qk"),            # a negative length is empty
    ("f32", [31, 47, 100], [30, 16, 3], 5, 10, 16, "gaps", 1e4, "out", "qk"),
]


def normed64(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


@pytest.mark.parametrize("pad", [0, 3])
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_append(case, pad):
    dtype, lens, rows, Hkv, H, page, layout, theta, q_how, norms = case
    print("append", case, pad, flush=True)
    eps = 1e-3
    c = Case8(lens, Hkv, page, layout, seed=len(lens), drop=[(0, 0)] if pad else [], junk=2 ** 31 - 1, pad_table=pad)
    total = sum(rows) + 2 * pad
    new = {w: rows_of(dtype, total, h, 7 + i) for i, (w, h) in enumerate((("k", Hkv), ("v", Hkv), ("q", H)))}
    w = {n: (1 + 0.3 * rows_of("f32", 1, 1, 90 + i)[0, 0]).to(TD[dtype]) for i, n in enumerate("qk")}
    cache = c.cuda(B)
    k, _ = wide(new["k"].cuda(), 16)
    v, _ = wide(new["v"].cuda(), 48)
    q, _ = wide(new["q"].cuda(), 16)
    out, obase = wide(torch.full_like(new["q"], 7.0).cuda(), 32, 7.0)
    starts = None if not pad and all(n == 1 for n in rows) else torch.from_numpy(starts_of(rows, pad)).cuda()
    got = B.paged_q8_append(cache, k, v, q=q if q_how else None, q_out=out if q_how == "out" else None,
                            row_starts=starts, theta=theta, eps=eps,
                            q_weight=w["q"].cuda() if "q" in norms and q_how else None,
                            k_weight=w["k"].cuda() if "k" in norms else None)
    half = torch.finfo(TD[dtype]).eps / 2
    want_q = new["q"].double().numpy().copy() if q_how == "in place" else np.full((total, H, D), 7.0)
    tol_q = np.zeros_like(want_q)

    def formed(x, pos, name, normed):
        """(value, what 32-bit arithmetic is off at most) of rows before the last rounding."""
        y, rel = x, 0.0
        if normed:      # a sum of 64 squares, a root, three products
            y, rel = normed64(x, w[name].double().numpy(), eps), (64 / 2 + 8) * 2.0 ** -24
        size = np.abs(y).reshape(y.shape[0], -1, 2).sum(2, keepdims=True).repeat(2, 2).reshape(y.shape)
        if theta:
            y = rotate64(y, pos, theta)
        return y, size * ((6 if theta else 0) * 2.0 ** -24 + rel)

    err = {n: np.zeros((c.n_pages, Hkv, page, D)) for n in "kv"}
    exact = {n: np.full((c.n_pages, Hkv, page, D), np.nan) for n in "kv"}
    for b, n in enumerate(rows):
        at = pad + sum(rows[:b])
        first = max(lens[b], 0) - n
        made = {"k": [], "v": []}
        for i in range(n):
            x = {m: new[m][at + i].double().numpy() for m in "kvq"}
            want_q[at + i], e = formed(x["q"], first + i, "q", "q" in norms)
            tol_q[at + i] = e + (np.abs(want_q[at + i]) + e) * half
            yk, ek = formed(x["k"], first + i, "k", "k" in norms)
            made["k"].append(yk)
            made["v"].append(x["v"])
            place = c.place(b, first + i)
            if place:
                err["k"][place[0], :, place[1]] = ek
                exact["k"][place[0], :, place[1]], exact["v"][place[0], :, place[1]] = yk, x["v"]
        if n:
            for m in "kv":
                store(c, b, first, np.array(made[m]), m)
    for name, pool, sc in (("k", c.kc, c.kb), ("v", c.vc, c.vb)):
        same_bytes(sc, c.bytes[name], f"{name} scales")
        g, want = pool.cpu().numpy(), c.codes[name]
        old = np.isnan(exact[name])
        assert (g[old] == want[old]).all(), f"{name}: other places changed"
        byte = np.repeat(c.bytes[name], BLOCK, 2)[..., None] * np.ones(D, int)
        val = TABLE[g[~old]] * scale_of(byte[~old])
        x = exact[name][~old]
        unit = 2.0 ** (byte[~old].astype(float) - 127)
        # nearest: off by half a step, of the value's own binade or (rounded up into it) the next one's border
        lim = half_step(x / unit, 127) * unit + err[name][~old]
        assert (np.abs(val - x) <= lim).all(), f"{name}: {(np.abs(val - x) > lim).sum()} not the nearest"
        flips = (g[~old] != want[~old]).mean() if x.size else 0
        assert flips <= 1e-3, f"{name}: {flips:.1e} of codes differ"
        if name == "v" or (theta == 0 and "k" not in norms):   # nothing before the rounding: exactly
            assert flips == 0
    if q_how:
        assert got is (out if q_how == "out" else q)
        off = np.abs(host(got) - want_q)
        assert (off <= tol_q).all(), f"q: worst {np.max(off - tol_q):.2e}"
        if q_how == "out":
            assert (host(obase)[:, :16] == 7.0).all() and (host(obase)[:, -16:] == 7.0).all()
            assert torch.equal(bits(q), bits(new["q"].cuda()))
    else:
        assert got is None


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_row_by_row(dtype):
    """Rows of growing and falling size, one a call: older rows of the block under the larger scales."""
    r = np.random.default_rng(3)
    c = Case8([0, 0], 2, 32, True, nan=True, max_pages=2, seed=1)
    c.table[:] = [[1, 0], [2, -1]]
    for n in c.codes.values():
        n[:] = 0x5a                                 # what earlier owners left, scales too
    for n in c.bytes.values():
        n[:] = 200
    cache = c.cuda(B)
    c.td.copy_(torch.from_numpy(c.table))
    for step in range(45):
        c.lens = [step + 1, step + 1]
        c.ld.fill_(step + 1)
        size = 2.0 ** r.integers(-20, 20, (2, 2, 1)) if step % 5 else 1.0
        new = {n: torch.from_numpy(r.standard_normal((2, 2, D)) * size).to(TD[dtype]) for n in "kv"}
        B.paged_q8_append(cache, new["k"].cuda(), new["v"].cuda(), theta=0.0)
        for n, pool, sc in (("k", c.kc, c.kb), ("v", c.vc, c.vb)):
            for b in range(2):
                store(c, b, step, new[n][b:b + 1].double().numpy(), n)
            same_bytes(sc, c.bytes[n], f"{n} scales, step {step}")
            same_bytes(pool, c.codes[n], f"{n} codes, step {step}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_borders_of_the_scales(dtype):
    """A block's largest element at, above and below 448 times a power of two; zeros; the least and the
    largest numbers; infinite and NaN elements."""
    f = torch.finfo(TD[dtype])
    up = 1 + f.eps
    tops = [448.0, 448.0 * up, 448.0 * (1 - f.eps / 2), 256.0, 0.0, 2.0 ** -126, 2.0 ** -133, 2.0 ** -109, f.max,
            -f.max, 1.75 * 2.0 ** 127, 1.75 * 2.0 ** 127 * up, 240 * 2.0 ** 119, -448.0, 3e-39, 1.0]
    n = len(tops)
    x = torch.zeros((n * 16, 1, D), dtype=torch.float64)
    r = np.random.default_rng(1)
    for i, t in enumerate(tops):
        x[16 * i:16 * i + 16] = torch.from_numpy(r.uniform(-1, 1, (16, 1, D)) * abs(t) * 2.0 ** r.integers(-12, 0, (16, 1, 1)))
        x[16 * i + i, 0, 3 * i] = t
    x = x.to(TD[dtype])
    x[5, 0, 5], x[6, 0, 6], x[7, 0, 7] = float("inf"), float("-inf"), float("nan")
    x[16 * 4:16 * 5, 0, :] = 0
    x[16 * 4, 0, 0] = float("nan")                  # nothing finite but zeros
    c = Case8([n * 16], 1, 16, True, nan=False, seed=2)
    cache = c.cuda(B)
    st = torch.tensor([0, n * 16], dtype=torch.int32, device="cuda")
    B.paged_q8_append(cache, x.cuda(), x.cuda(), row_starts=st, theta=0.0)
    for name, pool, sc in (("k", c.kc, c.kb), ("v", c.vc, c.vb)):
        store(c, 0, 0, x.double().numpy(), name)
        same_bytes(sc, c.bytes[name], "scales")
        same_bytes(pool, c.codes[name], "codes")
    # and no value read back is infinite that was not
    k, _ = B.paged_q8_read(cache, st, n_rows=n * 16, dtype=torch.float32)
    bad = ~torch.isfinite(x).cuda()
    assert torch.equal(~torch.isfinite(k), bad)


def test_append_far_positions():
    page, last = 1 << 15, (1 << 30) - 1
    pos = [2 ** 20 + 1, 123456789, last, 2 ** 24 + 3]
    table = np.full((4, (1 << 30) // page), -1, np.int32)
    for b, p in enumerate(pos):
        table[b, p // page] = b
    codes = torch.zeros((4, 1, page, D), dtype=torch.uint8, device="cuda")
    sc = torch.full((4, 1, page // 16), 90, dtype=torch.uint8, device="cuda")
    cache = B.PagedQ8(codes, codes.clone(), sc, sc.clone(), torch.from_numpy(table).cuda(),
                      torch.tensor([p + 1 for p in pos], dtype=torch.int32, device="cuda"))
    k, v, q = (rows_of("f32", 4, h, 3 + h) for h in (1, 1, 2))
    out = B.paged_q8_append(cache, k.cuda(), v.cuda(), q=q.cuda())
    got, _ = B.paged_q8_read(cache, dtype=torch.float32)
    for b, p in enumerate(pos):
        w = rotate64(q[b].double().numpy(), p, 1e4)
        size = np.abs(q[b].double().numpy()).sum()
        assert (np.abs(host(out[b]) - w) <= size * (6 * 2.0 ** -24 + 2.0 ** -21)).all(), (b, p)
        w = rotate64(k[b].double().numpy(), p, 1e4)
        lim = half_step(w, byte_of(np.abs(w).max())) + np.abs(k[b].double().numpy()).sum() * (6 * 2.0 ** -24 + 2.0 ** -21)
        assert (np.abs(host(got[b]) - w) <= lim).all(), (b, p)


def test_offsets_past_32_bits():
    """Pages whose codes lie past 4 GiB: appended, read back and attended to."""
    page, Hkv, n_pages = 4096, 4, 4200              # 1 MiB a page
    codes = [torch.zeros((n_pages, Hkv, page, D), dtype=torch.uint8, device="cuda") for _ in range(2)]
    sc = [torch.full((n_pages, Hkv, page // 16), 120, dtype=torch.uint8, device="cuda") for _ in range(2)]
    table = torch.tensor([[n_pages - 1, 5], [4099, n_pages - 2]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([100, 4096 + 30], dtype=torch.int32, device="cuda")
    cache = B.PagedQ8(*codes, *sc, table, lens)
    rows = [100, 60]
    k, v, q = (rows_of("bf16", 160, h, h).cuda() for h in (4, 4, 8))
    st = torch.tensor([0, 100, 160], dtype=torch.int32, device="cuda")
    B.paged_q8_append(cache, k, v, row_starts=st, theta=0.0)
    got = B.paged_q8_read(cache, st, n_rows=160)
    for g, x in zip(got, (k, v)):
        byte = 127 - 8 + 3                           # sizes up to 2^3.. : a code's half step is 2^-4 of its value at most
        assert ((g.double() - x.double()).abs() <= x.double().abs() * 2.0 ** -4 + 2.0 ** (byte - 127 - 10)).all()
    o = B.paged_q8_prefill(q, cache, st, scale=0.125)
    kk, vv = (torch.cat([torch.zeros(4096 + 30 - 60, 4, D, device="cuda"), g[100:].float()]).double() for g in got)
    for seq, kk, vv, qq, oo, n in ((0, got[0][:100].double(), got[1][:100].double(), q[:100], o[:100], 100),
                                   (1, kk, vv, q[100:], o[100:], 60)):
        L = kk.shape[0]
        for h in range(8):
            s = 0.125 * qq[:, h].double() @ kk[:, h // 2].T
            hid = torch.arange(L, device="cuda")[None] > (L - n + torch.arange(n, device="cuda"))[:, None]
            p = torch.softmax(s.masked_fill(hid, -np.inf), 1)
            ref, size = p @ vv[:, h // 2], p @ vv[:, h // 2].abs()
            # bf16 probabilities and output; scores and sums in 32 bits, as q8_util
            assert ((oo[:, h].double() - ref).abs() <= ref.abs() * 2.0 ** -9 + size * (2.0 ** -8 + 2.0 ** -10)).all()
    lone = B.paged_q8_decode(q[[99, 159]].contiguous(), cache, scale=0.125)
    assert ((lone.double() - o[[99, 159]].double()).abs() <= 2.0 ** -7 * o[[99, 159]].double().abs() + 2.0 ** -7).all()


def test_append_starts_that_decrease_stay_inside():
    """Rows are clamped to the tensors: nothing outside them or the table is touched."""
    c = Case8([40, 30, 20], 2, 16, True, seed=5)
    cache = c.cuda(B)
    new = rows_of("bf16", 30, 2, 1).cuda()
    qbase = torch.full((32, 4, D), 7.0, dtype=torch.bfloat16, device="cuda")
    for starts in ([25, 10, 40, 5], [-100, 50, 7, 2 ** 31 - 1], [2 ** 31 - 1, -2 ** 31, 3, 0], [30, 20, 10, 0]):
        st = torch.tensor(starts, dtype=torch.int32, device="cuda")
        B.paged_q8_append(cache, new, new, q=qbase[1:31].clone(), q_out=qbase[1:31], row_starts=st)
        B.paged_q8_read(cache, st, n_rows=30)
        torch.cuda.synchronize()
        assert (qbase[0] == 7.0).all() and (qbase[31] == 7.0).all()


def test_thousands_of_sequences():
    """More sequences than one step of the search for a unit's tells apart, ragged, most of few rows."""
    r = np.random.default_rng(0)
    rows = r.integers(0, 3, 5000)
    rows[[3, 700, 4999]] = [90, 33, 17]
    lens = np.where(rows > 0, rows + r.integers(0, 20, 5000), 0)
    c = Case8([int(x) for x in lens], 1, 16, True, nan=True, seed=4)
    cache = c.cuda(B)
    total = int(rows.sum())
    x = rows_of("bf16", total, 1, 9)
    st = torch.from_numpy(starts_of(rows)).cuda()
    B.paged_q8_append(cache, x.cuda(), (-x).cuda(), row_starts=st, theta=0.0)
    at = 0
    for b, n in enumerate(rows):
        if n:
            store(c, b, int(lens[b] - n), x[at:at + n].double().numpy(), "k")
            store(c, b, int(lens[b] - n), -x[at:at + n].double().numpy(), "v")
        at += n
    for name, pool, sc in (("k", c.kc, c.kb), ("v", c.vc, c.vb)):
        same_bytes(sc, c.bytes[name], f"{name} scales")
        same_bytes(pool, c.codes[name], f"{name} codes")


# ---------------------------------------------------------------- attention
EDGES = [0, 1, 2, 7, 8, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65, 95, 96, 97, 127, 128, 129, 255, 256, 257, 300]
DECODES = [
    # lens, Hkv, H, page, layout, dropped pages (sequence, index)
    (EDGES, 2, 16, 16, True, []),
    (EDGES, 1, 3, 16, False, [(20, 3), (23, 0)]),
    (EDGES, 3, 15, 32, "gaps", [(20, 2), (23, 0), (2, 0)]),
    (EDGES, 1, 16, 64, "gaps", [(16, 0), (20, 1)]),
    (EDGES, 1, 20, 128, True, []),             # more heads a KV head than a tile holds
    (EDGES, 2, 66, 16, False, []),
    (EDGES[:14], 5, 5, 16, True, [(13, 1), (13, 2)]),
    ([1000], 1, 8, 256, True, [(0, 1)]),
    ([513] * 3 + [2000], 4, 32, 16, True, []),
    ([513] * 3 + [2000], 4, 32, 16, False, []),
    ([-7, 0, 0], 2, 2, 16, True, []),           # nothing at all
    ([50, 2 ** 31 - 1, -2 ** 31], 2, 4, 16, True, []),  # lengths past the table
    ([3] * 70 + [1], 8, 8, 16, True, []),
]


DTYPES = pytest.mark.parametrize("dtype", ["bf16", "f32"])


@DTYPES
@pytest.mark.parametrize("case", DECODES, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{c[1]}-{c[2]}-p{c[3]}-{c[4]}-d{len(c[5])}")
def test_decode(case, dtype):
    lens, Hkv, H, page, layout, drop = case
    print("decode", case, dtype, flush=True)
    big = max(lens) > 10 ** 6
    c = Case8(lens, Hkv, page, layout, drop=drop, seed=H, max_pages=4 if big else None, junk=2 ** 31 - 1, pad_table=5,
              dtype=dtype)
    q = rows_of(dtype, len(lens), H, 1)
    ref, tol = attention64(c, q, [1] * len(lens))
    cache = c.cuda(B)
    qd, _ = wide(q.cuda(), 32)
    o, obase = wide(torch.full_like(q, 7.0).cuda(), 48, 7.0)
    assert B.paged_q8_decode(qd, cache, o=o, scale=0.125) is o
    check(host(o), ref, tol, "decode")
    assert (host(obase)[:, :24] == 7.0).all() and (host(obase)[:, -24:] == 7.0).all()
    ws = B.paged_q8_workspace(cache, H, len(lens))
    ws.fill_(255)                                       # any contents
    for _ in range(3):                                  # and what an earlier call left
        o2 = B.paged_q8_decode(qd, cache, scale=0.125, workspace=ws)
        assert torch.equal(bits(o2), bits(o)), "a second call differs"


@DTYPES
@pytest.mark.parametrize("lens,Hkv,H", [([20011], 2, 8), ([9000, 1, 0, 33], 2, 8), ([5000, 40, 7000, 1234, 4000], 2, 8),
                                        ([12000, 700], 1, 1), ([12000, 700, 3000], 1, 5), ([7000, 9000], 1, 12),
                                        ([5000] * 3, 3, 45)], ids=str)
def test_decode_long(lens, Hkv, H, dtype):
    """Caches cut over many workgroups."""
    print("decode long", lens, Hkv, H, dtype, flush=True)
    c = Case8(lens, Hkv, 64, True, drop=[(0, 17)], seed=3, dtype=dtype)
    q = rows_of(dtype, len(lens), H, 5)
    ref, tol = attention64(c, q, [1] * len(lens))
    cache = c.cuda(B)
    ws = B.paged_q8_workspace(cache, H, len(lens))
    for _ in range(2):
        check(host(B.paged_q8_decode(q.cuda(), cache, scale=0.125, workspace=ws)), ref, tol, "decode")


@pytest.mark.parametrize("n,H,dtype", [(1300, 4, "bf16"), (1300, 4, "f32"), (4000, 1, "bf16"), (2500, 32, "bf16")])
def test_decode_many_sequences(n, H, dtype):
    """More sequences than threads, and more in a share than its list and its places hold."""
    lens = [int(x) for x in np.random.default_rng(0).integers(0, 90, n)]
    lens[700], lens[900:1000] = 3000, [0] * 100
    c = Case8(lens, 2 if H > 1 else 1, 16, True, seed=1, dtype=dtype)
    q = rows_of(dtype, len(lens), H, 2)
    ref, tol = attention64(c, q, [1] * len(lens))
    check(host(B.paged_q8_decode(q.cuda(), c.cuda(B), scale=0.125)), ref, tol, "decode")


@DTYPES
@pytest.mark.parametrize("call", ["decode", "prefill"])
def test_extreme_scores(call, dtype):
    """Scores far apart, so that the largest arrives late, and scales at both ends of their range."""
    lens = [200, 131, 97]
    c = Case8(lens, 1, 32, True, seed=8, spread=6.0, dtype=dtype)
    q = (40 * rows_of(dtype, 3, 4, 1).float()).to(TD[dtype])
    ref, tol = attention64(c, q, [1] * 3)
    cache = c.cuda(B)
    st = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")
    o = B.paged_q8_decode(q.cuda(), cache, scale=0.125) if call == "decode" else \
        B.paged_q8_prefill(q.cuda(), cache, st, scale=0.125)
    check(host(o), ref, tol, call)
    for byte, x in ((LOW, 2.0 ** -117), (HIGH - 20, 2.0 ** 100)):
        c = Case8([70], 1, 32, True, seed=9, nan=False, spread=0.0, dtype=dtype)
        c.bytes["v"][:] = byte
        c.v = torch.from_numpy(TABLE[c.codes["v"]] * x)
        ref, tol = attention64(c, q[:1], [1])
        cache = c.cuda(B)
        o = B.paged_q8_decode(q[:1].cuda(), cache, scale=2.0 ** -6) if call == "decode" else \
            B.paged_q8_prefill(q[:1].cuda(), cache, st[:2].contiguous(), scale=2.0 ** -6)
        ref, tol = attention64(c, q[:1], [1], scale=2.0 ** -6)
        check(host(o) / x, ref / x, tol / x + 2.0 ** -9 * (byte == LOW), call)   # (subnormal bf16 outputs may be zeros)


PREFILLS = [
    # lens, rows, Hkv, H, page, layout, dropped, padding
    ([40, 0, 33, 9], [40, 0, 2, 9], 2, 6, 16, "gaps", [], 3),
    (EDGES, [min(n, 1 + i % 7) for i, n in enumerate(EDGES)], 2, 16, 16, True, [], 0),
    (EDGES, EDGES, 1, 4, 32, False, [(20, 1), (23, 0)], 2),
    ([300, 150, 64], [300, 3, 64], 4, 32, 64, True, [(0, 1)], 5),
    ([300, 5], [17, 9], 3, 15, 16, "gaps", [], 0),      # more rows than the length
    ([257], [130], 1, 20, 16, True, [], 0),
    ([500, 700], [33, 65], 1, 66, 128, False, [], 1),
    ([-3, 5, 2 ** 31 - 1], [2, 5, 3], 2, 2, 16, True, [], 0),
]


@DTYPES
@pytest.mark.parametrize("case", PREFILLS, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{max(c[1])}-{c[2]}-{c[3]}-p{c[4]}-{c[5]}-d{len(c[6])}")
def test_prefill(case, dtype):
    lens, rows, Hkv, H, page, layout, drop, pad = case
    print("prefill", case, dtype, flush=True)
    big = max(lens) > 10 ** 6
    c = Case8(lens, Hkv, page, layout, drop=drop, seed=H, max_pages=4 if big else None, junk=-5, pad_table=2, dtype=dtype)
    n = sum(rows) + 2 * pad
    q = rows_of(dtype, n, H, 1)
    ref, tol = attention64(c, q, rows, pad)
    cache = c.cuda(B)
    qd, _ = wide(q.cuda(), 32)
    o, obase = wide(torch.full_like(q, 7.0).cuda(), 16, 7.0)
    st = torch.from_numpy(starts_of(rows, pad)).cuda()
    assert B.paged_q8_prefill(qd, cache, st, o=o, scale=0.125) is o
    got = host(o)
    check(got, ref, tol, "prefill")
    assert (got[np.isnan(ref)] == 7.0).all(), "rows of no sequence were written"
    assert (host(obase)[:, :8] == 7.0).all() and (host(obase)[:, -8:] == 7.0).all()
    ws = B.paged_q8_workspace(cache, H, n)
    ws.fill_(255)
    some = torch.from_numpy(~np.isnan(ref)).cuda()
    for _ in range(2):
        o2 = B.paged_q8_prefill(qd, cache, st, scale=0.125, workspace=ws)
        assert torch.equal(bits(o2[some]), bits(o[some])), "a second call differs"


LARGE = [
    # lens, rows, Hkv, H, page, layout
    ([2000], [2000], 4, 32, 16, True),
    ([1500, 700, 1111, 33], [1500, 690, 800, 33], 4, 32, 16, True),
    ([9000], [256], 1, 8, 64, True),
    ([3000, 5000], [768, 700], 2, 16, 32, False),
    ([6000], [4500], 4, 32, 64, True),
    ([20000], [300], 4, 32, 128, True),
    ([17000, 600], [1500, 600], 2, 16, 64, False),
    ([900, 3300, 1100], [620, 3200, 1001], 4, 32, 16, False),  # just enough rows for units of 256
]


@DTYPES
@pytest.mark.parametrize("case", LARGE, ids=lambda c: f"{'-'.join(map(str, c[0]))}-{'-'.join(map(str, c[1]))}-{c[2]}-{c[3]}-p{c[4]}-{c[5]}")
def test_prefill_large(case, dtype):
    lens, rows, Hkv, H, page, layout = case
    print("prefill large", case, dtype, flush=True)
    c = Case8(lens, Hkv, page, layout, seed=1, drop=[(0, 20)], dtype=dtype)
    q = rows_of(dtype, sum(rows), H, 4).cuda()
    cache = c.cuda(B)
    ref, tol = attention64_large(c, q, rows)
    st = torch.from_numpy(starts_of(rows)).cuda()
    ws = B.paged_q8_workspace(cache, H, sum(rows))
    ws.fill_(255)
    for _ in range(2):
        o = B.paged_q8_prefill(q, cache, st, scale=0.125, workspace=ws)
        off = (o.double() - ref).abs() - tol
        assert torch.isfinite(o).all() and (off <= 0).all(), f"{int((off > 0).sum())} past the tolerance, by {off.max():.2e}"


@DTYPES
@pytest.mark.parametrize("rows,lens", [([50], [70]), ([3, 3, 3], [40, 100, 20]), ([700], [900]), ([2100], [2200]),
                                       ([4200], [17000])], ids=str)
def test_a_hidden_nan_stays_hidden(rows, lens, dtype):
    """NaN values and keys of later positions reach the rows that see them and no other."""
    Hkv, H = 1, 8
    c = Case8(lens, Hkv, 64, True, seed=6, dtype=dtype)
    cache = c.cuda(B)
    q = rows_of(dtype, sum(rows), H, 4).cuda()
    st = torch.from_numpy(starts_of(rows)).cuda()
    ref, tol = attention64_large(c, q, rows)
    j = lens[0] - rows[0] // 2                       # a key that half of the first sequence's rows see
    pg, sl = c.place(0, j)
    from_row = j - (lens[0] - rows[0])               # the first row that sees it
    sees = torch.zeros(sum(rows), dtype=torch.bool, device="cuda")
    sees[from_row:rows[0]] = True
    for pool, what in ((c.vc, "v"), (c.kc, "k")):
        kept = pool[pg, 0, sl].clone()
        pool[pg, 0, sl, 5] = 0x7f
        o = B.paged_q8_prefill(q, cache, st, scale=0.125)
        near = (o.double() - ref).abs() <= tol       # (a NaN is not)
        hit = torch.zeros_like(near)
        hit[sees] = True
        if what == "v":
            hit &= torch.arange(D, device="cuda") == 5
        assert torch.isnan(o[hit]).all() and near[~hit].all(), what
        pool[pg, 0, sl] = kept


def test_outputs_in_the_queries_place():
    c = Case8([300, 40, 77], 2, 16, True, seed=2)
    cache = c.cuda(B)
    q = rows_of("bf16", 30, 8, 4).cuda()
    st = torch.tensor([0, 20, 21, 30], dtype=torch.int32, device="cuda")
    o = B.paged_q8_prefill(q, cache, st)
    x = q.clone()
    assert B.paged_q8_prefill(x, cache, st, o=x) is x and torch.equal(bits(x), bits(o))
    q = rows_of("bf16", 3, 8, 5).cuda()
    o = B.paged_q8_decode(q, cache)
    assert torch.equal(bits(B.paged_q8_decode(q, cache, o=q)), bits(o))


def test_prefill_without_starts_is_decode():
    c = Case8([300, 0, 77], 2, 16, True, seed=2)
    cache = c.cuda(B)
    q = rows_of("bf16", 3, 8, 4).cuda()
    assert torch.equal(bits(B.paged_q8_prefill(q, cache)), bits(B.paged_q8_decode(q, cache)))


# ------------------------------------------------------- graphs and streams
def step(cache, k, v, q, q_rot, o, st, ws, weights, decode):
    B.paged_q8_append(cache, k, v, q=q, q_out=q_rot, row_starts=st, q_weight=weights[0], k_weight=weights[1])
    if decode:
        return B.paged_q8_decode(q_rot, cache, o=o, workspace=ws)
    return B.paged_q8_prefill(q_rot, cache, st, o=o, workspace=ws)


@pytest.mark.parametrize("decode", [True, False], ids=["decode", "prefill"])
def test_a_graph_follows_the_table_and_the_lengths(decode):
    """Append and attention captured once; replayed as the sequences grow, with eager work between."""
    lens = [700, 40, 2500]
    rows = [1, 1, 1] if decode else [90, 3, 600]
    H, Hkv, n = 8, 2, sum(rows)
    cases = [Case8([x + 100 for x in lens], Hkv, 32, True, seed=5, nan=False) for _ in range(2)]
    caches = [c.cuda(B) for c in cases]
    k, v, q = (torch.zeros((n, h, D), dtype=torch.bfloat16, device="cuda") for h in (Hkv, Hkv, H))
    w = [(1 + 0.1 * rows_of("f32", 1, 1, i)[0, 0]).bfloat16().cuda() for i in range(2)]
    q_rot, o = torch.empty_like(q), torch.empty_like(q)
    st = None if decode else torch.from_numpy(starts_of(rows)).cuda()
    ws = B.paged_q8_workspace(caches[0], H, n)
    args = (caches[0], k, v, q, q_rot, o, st, ws, w, decode)
    cases[0].ld.copy_(torch.tensor(lens, dtype=torch.int32))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(*args)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step(*args)
    for c in cases:      # both caches as they were
        for have, want in ((c.kc, c.codes["k"]), (c.vc, c.codes["v"]), (c.kb, c.bytes["k"]), (c.vb, c.bytes["v"])):
            have.copy_(torch.from_numpy(want))
    for i in range(5):
        new = [rows_of("bf16", n, t.shape[1], 50 + 3 * i + j) for j, t in enumerate((k, v, q))]
        for t, x in zip((k, v, q), new):
            t.copy_(x)
        for c in cases:
            c.ld.copy_(torch.tensor([x + 17 * i for x in lens], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = o.clone()
        eager = step(caches[1], k, v, q, torch.empty_like(q), torch.empty_like(q), st, None, w, decode)
        assert torch.equal(bits(got), bits(eager)), f"replay {i}"
        for a, b in zip((cases[0].kc, cases[0].vc, cases[0].kb, cases[0].vb),
                        (cases[1].kc, cases[1].vc, cases[1].kb, cases[1].vb)):
            assert torch.equal(a, b), f"replay {i}: caches differ"


def test_two_graphs_share_a_workspace():
    H, Hkv = 8, 2
    c = Case8([6000, 300, 9], Hkv, 64, True, seed=5)
    cache = c.cuda(B)
    qd, qp = rows_of("bf16", 3, H, 1).cuda(), rows_of("bf16", 700, H, 2).cuda()
    st = torch.tensor([0, 600, 691, 700], dtype=torch.int32, device="cuda")
    ws = B.paged_q8_workspace(cache, H, 700)
    od, op = torch.empty_like(qd), torch.empty_like(qp)
    graphs = []
    for run in (lambda: B.paged_q8_decode(qd, cache, o=od, workspace=ws),
                lambda: B.paged_q8_prefill(qp, cache, st, o=op, workspace=ws)):
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            run()
            side.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                run()
        graphs.append(g)
    want = B.paged_q8_decode(qd, cache), B.paged_q8_prefill(qp, cache, st)
    for i in range(4):
        od.zero_(), op.zero_()
        for g in graphs if i % 2 else graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(bits(od), bits(want[0])) and torch.equal(bits(op), bits(want[1])), i


def test_calls_on_a_given_stream():
    c = Case8([3000, 40], 2, 16, True, seed=2)
    cache = c.cuda(B)
    q = rows_of("bf16", 2, 8, 4).cuda()
    st = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    want = (B.paged_q8_decode(q, cache), B.paged_q8_prefill(q, cache, st), *B.paged_q8_read(cache))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        got = (B.paged_q8_decode(q, cache, stream=side), B.paged_q8_prefill(q, cache, st, stream=side),
               *B.paged_q8_read(cache, stream=side))
        torch.cuda.current_stream().wait_stream(side)
        for a, b in zip(got, want):
            assert torch.equal(bits(a), bits(b))


def test_host_memory_is_refused():
    c = Case8([30], 2, 16, True, seed=2)
    cache = c.cuda(B)
    c.ld = c.ld.cpu()
    view = B.BnPagedQ8(*[getattr(cache.view, n) for n, _ in B.BnPagedQ8._fields_])
    view.seq_lens = c.ld.data_ptr()
    import ctypes as C
    q = rows_of("bf16", 1, 8, 4).cuda()
    s, m = B.status_of("bn_paged_q8_decode", C.byref(view), B.BN_BF16, q.data_ptr(), q.data_ptr(), 8, 512, 512, 0.125,
                       None, 0, None)
    assert s == B.BN_ERR_NOT_DEVICE, m


# ----------------------------------------------------------- used together
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("page,layout", [(16, True), (64, False)])
def test_a_server_run(dtype, page, layout):
    """Prompts, then decode steps, then one conversation taken out and put into another cache: every
    attention call against 64 bits over what the cache held, and the cache's values against the rows."""
    Hkv, H, prompts, steps = 2, 8, [37, 5, 130], 21
    r = np.random.default_rng(1)
    c = Case8([n + steps for n in prompts], Hkv, page, layout, seed=7, dtype=dtype)
    for x in c.codes.values():
        x[:] = 127                                   # nothing is there yet
    for x in c.bytes.values():
        x[:] = 255
    cache = c.cuda(B)
    w = [(1 + 0.2 * rows_of("f32", 1, 1, i)[0, 0]).to(TD[dtype]) for i in range(2)]
    ws = B.paged_q8_workspace(cache, H, sum(prompts))
    kept = {b: [] for b in range(3)}                 # the keys and values that went in, 64 bits
    lens = list(prompts)
    for turn in range(steps + 1):
        rows = prompts if turn == 0 else [1, 1, 1]
        if turn:
            lens = [n + 1 for n in lens]
        n = sum(rows)
        k, v, q = (torch.from_numpy(r.standard_normal((n, h, D))).to(TD[dtype]) for h in (Hkv, Hkv, H))
        c.ld.copy_(torch.tensor(lens, dtype=torch.int32))
        st = torch.from_numpy(starts_of(rows)).cuda() if turn == 0 else None
        q_rot = B.paged_q8_append(cache, k.cuda(), v.cuda(), q=q.cuda(), row_starts=st, q_weight=w[0].cuda(),
                                  k_weight=w[1].cuda(), eps=1e-5)
        at = 0
        for b, m in enumerate(rows):
            for i in range(m):
                kk = rotate64(normed64(k[at + i].double().numpy(), w[1].double().numpy(), 1e-5), lens[b] - m + i, 1e4)
                kept[b].append((kk, v[at + i].double().numpy()))
            at += m
        qb = q_rot
        o = B.paged_q8_prefill(qb, cache, st, scale=0.125, workspace=ws) if turn == 0 else \
            B.paged_q8_decode(qb, cache, scale=0.125, workspace=ws)
        # what the cache holds now, read back, is what the attention is measured by
        for pool, sc, name in ((c.kc, c.kb, "k"), (c.vc, c.vb, "v")):
            setattr(c, name, torch.from_numpy(TABLE[pool.cpu().numpy()] *
                                              np.repeat(scale_of(sc.cpu().numpy()), BLOCK, 2)[..., None]))
        c.lens = list(lens)
        ref, tol = attention64(c, qb.cpu(), rows)
        check(host(o), ref, tol, f"turn {turn}")
    all_rows = torch.from_numpy(starts_of(lens)).cuda()
    back = B.paged_q8_read(cache, all_rows, n_rows=sum(lens), dtype=torch.float32)
    at = 0
    for b, n in enumerate(lens):
        for got, i in zip(back, (0, 1)):
            x = np.array([e[i] for e in kept[b]])
            g = host(got[at:at + n])
            # a row is rounded under its block's last scale, perhaps once more on the way there
            top = np.array([np.abs(x[j // 16 * 16:j // 16 * 16 + 16]).max(axis=(0, 2)) for j in range(n)])
            lim = np.abs(x) * 2.0 ** -4 + (top / 224)[..., None] * 2 * 2.0 ** -10 + 1e-5
            assert (np.abs(g - x) <= lim).all(), (b, i, (np.abs(g - x) - lim).max())
        at += n
    # into a cache of another geometry: the same values again
    n = lens[2]
    d = Case8([n], Hkv, 32, True, seed=8)
    other = d.cuda(B)
    one = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    B.paged_q8_append(other, *(x[-n:].contiguous() for x in back), row_starts=one, theta=0.0)
    again = B.paged_q8_read(other, one, n_rows=n, dtype=torch.float32)
    for a, x in zip(again, back):
        assert torch.equal(a, x[-n:])
