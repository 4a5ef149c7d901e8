"""Inputs and the plain 64-bit form of the 8-bit paged cache's operators, for their tests.

Attention: the cache's values are bf16 numbers, so paged_util's tolerances hold, those of the queries' type.
Rounding to the cache: a value is off by at most half a step of e4m3 (2^-4 of itself, 2^-10 of the
scale below 2^-6 of it) and by what the 32-bit arithmetic before it was off.
"""
import numpy as np
import torch

from paged_util import D, Case

BLOCK, LOW, HIGH = 16, 10, 247


def e4m3_table():
    """The 256 codes' values, float64."""
    b = np.arange(256)
    e, m = b >> 3 & 15, (b & 7).astype(np.float64)
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0)) * np.where(b & 128, -1.0, 1.0)
    v[[127, 255]] = np.nan
    return v


TABLE = e4m3_table()


def scale_of(byte):
    return 2.0 ** (np.clip(np.asarray(byte).astype(int), LOW, HIGH) - 127.0)


def byte_of(amax):
    """The smallest byte whose power of two times 448 reaches amax."""
    if not amax > 0:
        return LOW
    n = int(np.ceil(np.log2(amax / 448)))
    while amax <= 448 * 2.0 ** (n - 1):
        n -= 1
    while amax > 448 * 2.0 ** n:
        n += 1
    return int(np.clip(n + 127, LOW, HIGH))


def codes_of(x, byte):
    """float64 values -> codes under a byte, nearest, ties to even; infinite and NaN: 0x7f."""
    x = np.asarray(x, np.float64)
    y = np.clip(np.where(np.isfinite(x), x, 0) / 2.0 ** (int(byte) - 127), *((-240, 240) if byte == HIGH else (-448, 448)))
    a = np.abs(y)
    step = 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(a, 2.0 ** -30))), -6) - 3)
    a = np.round(a / step) * step                     # numpy rounds ties to even
    c = np.searchsorted(TABLE[:127], a).astype(np.uint8)
    assert (TABLE[c] == a).all()
    c = c | np.where(np.signbit(y), 128, 0).astype(np.uint8)
    return np.where(np.isfinite(x), c, 127).astype(np.uint8)


def half_step(x, byte):
    """Half of e4m3's step at x under a byte."""
    s = 2.0 ** (int(byte) - 127)
    a = np.maximum(np.abs(x) / s, 2.0 ** -30)
    return 2.0 ** (np.maximum(np.floor(np.log2(a)), -6) - 4) * s


class Case8(Case):
    """A case whose cache is in 8 bits: k, v are its values (bf16 exactly); places that no visible key
    has hold NaN codes, and blocks without one scales of any byte."""

    def __init__(self, lens, Hkv=2, page=16, layout=True, seed=0, nan=True, spread=1.0, dtype="bf16", **kw):
        super().__init__("bf16", lens, Hkv, page, layout, seed=seed, nan=False, **kw)
        self.dtype = dtype                                # that of queries and outputs
        r = np.random.default_rng(seed + 1000)
        blocks = page // BLOCK
        seen = np.zeros((self.n_pages, page), bool)
        for b, n in enumerate(self.lens):
            for j in range(min(max(n, 0), self.max_pages * page)):
                pg = self.table[b, j // page]
                if 0 <= pg < self.n_pages:
                    seen[pg, j % page] = True
        self.seen = seen
        some = seen.reshape(self.n_pages, blocks, BLOCK).any(2)
        self.codes, self.bytes = {}, {}
        for name in "kv":
            x = getattr(self, name).double().numpy().reshape(self.n_pages, Hkv, blocks, BLOCK * D)
            x = x * 2.0 ** (spread * r.standard_normal((self.n_pages, Hkv, blocks, 1)).clip(-2, 2))
            byte = np.array([byte_of(a) for a in np.abs(x).max(3).ravel()], np.uint8).reshape(x.shape[:3])
            unit = 2.0 ** (byte.astype(float) - 127)[..., None]
            code = codes_of(x / unit, 127).reshape(self.n_pages, Hkv, page, D)
            value = TABLE[code] * np.repeat(unit[..., 0], BLOCK, 2)[..., None]
            setattr(self, name, torch.from_numpy(value))
            if nan:
                code = np.where(seen[:, None, :, None], code, [127, 255][name == "v"]).astype(np.uint8)
                junk = r.choice([0, 255, 254, 1, 130], size=byte.shape).astype(np.uint8)
                byte = np.where(some[:, None], byte, junk).astype(np.uint8)
            self.codes[name], self.bytes[name] = code, byte

    def pool8(self, x):
        x = torch.from_numpy(x)
        if self.head_major is True:
            return x.cuda()
        if self.head_major is False:
            return x.transpose(1, 2).contiguous().cuda().transpose(1, 2)
        s = torch.full((x.shape[0] * 2, x.shape[1], x.shape[2] + 1, D + 16), 127, dtype=torch.uint8)
        s[::2, :, :-1, :D] = x        # "gaps": every stride with room in it
        return s.cuda()[::2, :, :-1, :D]

    def scales8(self, x):
        x = torch.from_numpy(x)
        if self.head_major == "gaps":
            s = torch.full((x.shape[0], x.shape[1] + 1, x.shape[2] + 3), 255, dtype=torch.uint8)
            s[:, :-1, :x.shape[2]] = x
            return s.cuda()[:, :-1, :x.shape[2]]
        return x.cuda()

    def cuda(self, B):
        self.kc, self.vc = self.pool8(self.codes["k"]), self.pool8(self.codes["v"])
        self.kb, self.vb = self.scales8(self.bytes["k"]), self.scales8(self.bytes["v"])
        self.kd, self.vd = self.k.cuda(), self.v.cuda()          # values, for attention64_large
        self.td = torch.from_numpy(self.full_table).cuda()[:, :self.max_pages]
        self.ld = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        return B.PagedQ8(self.kc, self.vc, self.kb, self.vb, self.td, self.ld)


def store(case, b, first, x64, name, err=None):
    """The cache after rows x64 [n, Hkv, D] (float64) were appended to sequence b at positions first ..:
    case.codes and case.bytes are updated; returns nothing.  (x64 holds the values before rounding.)"""
    codes, bts = case.codes[name], case.bytes[name]
    n = x64.shape[0]
    for g in range(case.Hkv):
        for blk in range(first // BLOCK, (first + n - 1) // BLOCK + 1):
            lo, hi = max(first, blk * BLOCK), min(first + n, (blk + 1) * BLOCK)
            at = case.place(b, lo) if lo >= 0 else None
            if at is None:
                continue
            page, slot = at
            x = x64[lo - first:hi - first, g]
            a = np.abs(x[np.isfinite(x)])
            byte = byte_of(a.max() if a.size else 0.0)
            before = int(np.clip(bts[page, g, slot // BLOCK], LOW, HIGH))
            if lo % BLOCK:
                if byte > before:
                    old = slice(slot - lo % BLOCK, slot)
                    codes[page, g, old] = codes_of(TABLE[codes[page, g, old]] * scale_of(before), byte)
                byte = max(byte, before)
            codes[page, g, slot:slot + hi - lo] = codes_of(x, byte)
            bts[page, g, slot // BLOCK] = byte
