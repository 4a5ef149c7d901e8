"""Inputs and the plain 64-bit form of the paged KV cache's operators, for their tests.

A tolerance here is the sum of what each rounding on the way can do:
  * an output of type T is off by half a step, eps(T)/2 of its value;
  * with bf16 the probabilities enter the product with V as bf16 values, each off by half a step
    (eps/2 = 2^-8 of itself), which moves an output by at most 2^-8 of A = sum p|v| / sum p, and the
    sum of probabilities, rounded or not, by as much again;
  * a score is a sum of 64 products in 32 bits, scaled into the exponent: off by at most
    (64 + 8) 2^-24 S with S = scale sum|q||k|, and an exponential of it is off by twice that (of
    itself, both in numerator and denominator), at most 2^-22 more for the exponential;
  * sums over n keys in 32 bits are off by at most n 2^-24 of the sum of the terms' sizes, in
    numerator and denominator.
"""
import numpy as np
import torch

D = 64
TD = {"f32": torch.float32, "bf16": torch.bfloat16}


class Case:
    """A pool, a table and lengths on the CPU; cuda() puts them on the device.

    lens: keys per sequence; rows: new rows per sequence.  Every place of the pool that no visible
    key has, and every page in no table, holds NaN (nan=True)."""

    def __init__(self, dtype, lens, Hkv=2, page=16, head_major=True, spare=2, seed=0, drop=(), nan=True,
                 max_pages=None, pad_table=0, junk=-1):
        r = np.random.default_rng(seed)
        self.dtype, self.lens, self.Hkv, self.page = dtype, list(lens), Hkv, page
        B = len(self.lens)
        need = [-(-max(n, 0) // page) for n in self.lens]
        self.max_pages = max(need + [1]) + spare if max_pages is None else max_pages
        need = [min(n, self.max_pages) for n in need]
        self.n_pages = sum(need) + 3
        order = r.permutation(self.n_pages).astype(np.int32)
        self.full_table = np.full((B, self.max_pages + pad_table), junk, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.full_table[b, :n] = order[at:at + n]
            at += n
        for b, j in drop:
            self.full_table[b, j] = [-1, self.n_pages, -2147483648, 2147483647][(b + j) % 4]
        self.table = self.full_table[:, :self.max_pages]
        shape = (self.n_pages, Hkv, page, D)
        self.k, self.v = (torch.from_numpy(r.standard_normal(shape).astype(np.float32)).to(TD[dtype])
                          for _ in range(2))
        if nan:
            seen = np.zeros((self.n_pages, page), bool)
            for b, n in enumerate(self.lens):
                for j in range(min(max(n, 0), self.max_pages * page)):
                    pg = self.table[b, j // page]
                    if 0 <= pg < self.n_pages:
                        seen[pg, j % page] = True
            hide = torch.from_numpy(~seen)[:, None, :, None].expand(shape)
            self.k = self.k.masked_fill(hide, float("nan"))
            self.v = self.v.masked_fill(hide, float("nan"))
            self.v[hide & (torch.arange(D) % 2 == 0)] = float("inf")
        self.head_major = head_major

    def pool(self, x):
        """x [n_pages, Hkv, page, D] on the device in the case's layout, as that view."""
        if self.head_major is True:
            return x.cuda()
        if self.head_major is False:
            return x.transpose(1, 2).contiguous().cuda().transpose(1, 2)
        s = torch.full((x.shape[0] * 2, x.shape[1], x.shape[2] + 1, D + 8), float("nan"), dtype=x.dtype)
        s[::2, :, :-1, :D] = x        # "gaps": every stride with room in it
        return s.cuda()[::2, :, :-1, :D]

    def cuda(self, B):
        self.kd, self.vd = self.pool(self.k), self.pool(self.v)
        self.td = torch.from_numpy(self.full_table).cuda()[:, :self.max_pages]
        self.ld = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        return B.PagedKV(self.kd, self.vd, self.td, self.ld)

    def place(self, b, j, prefix=None, prefix_len=0):
        """(page, slot) of key j of sequence b, or None."""
        if j < 0 or j >= self.max_pages * self.page:
            return None
        pg = int(prefix[j // self.page]) if j < prefix_len else int(self.table[b, j // self.page])
        return (pg, j % self.page) if 0 <= pg < self.n_pages else None


def starts_of(rows, first=0):
    return np.concatenate([[first], first + np.cumsum(rows)]).astype(np.int32)


def rows_of(dtype, n, heads, seed, stride=None):
    r = np.random.default_rng(seed)
    x = torch.from_numpy(r.standard_normal((n, heads, D)).astype(np.float32)).to(TD[dtype])
    return x


def attention64(case, q, rows, first=0, scale=0.125, prefix=None, prefix_len=0):
    """(o, tol) [n_rows, H, D] float64; rows that belong to no sequence: NaN in both."""
    n_rows, H, _ = q.shape
    G = H // case.Hkv
    o = np.full((n_rows, H, D), np.nan)
    tol = np.full((n_rows, H, D), np.nan)
    eps = torch.finfo(TD[case.dtype]).eps / 2
    at = first
    for b, n in enumerate(rows):
        length = max(case.lens[b], 0)
        places = [case.place(b, j, prefix, prefix_len) for j in range(min(length, case.max_pages * case.page))]
        js = np.array([j for j, p in enumerate(places) if p], int)
        pg = np.array([p[0] for p in places if p], int)
        sl = np.array([p[1] for p in places if p], int)
        k = case.k[pg, :, sl].double().numpy() if len(js) else np.zeros((0, case.Hkv, D))
        v = case.v[pg, :, sl].double().numpy() if len(js) else np.zeros((0, case.Hkv, D))
        for i in range(n):
            if at + i >= n_rows:
                break
            vis = js <= length - n + i
            o[at + i] = 0.0
            tol[at + i] = 0.0
            if not vis.any():
                continue
            for h in range(H):
                kk, vv, qq = k[vis, h // G], v[vis, h // G], q[at + i, h].double().numpy()
                s = scale * (kk @ qq)
                p = np.exp(s - s.max())
                L = p.sum()
                o[at + i, h] = p @ vv / L
                A = p @ np.abs(vv) / L
                S = scale * float((np.abs(kk) @ np.abs(qq)).max())
                rel = 2 * (2 * (72 * 2.0 ** -24 * S) + 2.0 ** -22 + len(kk) * 2.0 ** -24)
                if case.dtype == "bf16":
                    rel += 2 * eps
                tol[at + i, h] = eps * np.abs(o[at + i, h]) + rel * A
        at += n
    return o, tol


def check(got, ref, tol, what=""):
    got = np.asarray(got, np.float64)
    some = ~np.isnan(ref)
    assert np.isfinite(got[some]).all(), f"{what}: not finite"
    over = np.abs(got - ref)[some] - tol[some]
    assert (over <= 0).all(), f"{what}: {int((over > 0).sum())} of {over.size} past the tolerance, by {over.max():.2e}"


def rotate64(x, pos, theta):
    """x [heads, D] float64 numpy at a position."""
    if theta == 0:
        return x
    a = pos * float(np.float32(theta)) ** (-np.arange(0, D, 2) / D)
    c, s = np.cos(a), np.sin(a)
    y = np.empty_like(x)
    y[:, 0::2] = x[:, 0::2] * c - x[:, 1::2] * s
    y[:, 1::2] = x[:, 0::2] * s + x[:, 1::2] * c
    return y


def attention64_large(case, q, rows, scale=0.125, prefix=None, prefix_len=0):
    """attention64 for large cases: (o, tol) as float64 tensors, computed on q's device by products
    in 64 bits per sequence and head (no padding rows)."""
    n_rows, H, _ = q.shape
    G = H // case.Hkv
    o = torch.zeros((n_rows, H, D), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    eps = torch.finfo(TD[case.dtype]).eps / 2
    kd, vd = case.kd, case.vd
    at = 0
    for b, n in enumerate(rows):
        length = min(max(case.lens[b], 0), case.max_pages * case.page)
        pages = torch.from_numpy(case.table[b, :-(-length // case.page)].astype(np.int64)).to(q.device)
        if prefix is not None:
            pages[:-(-prefix_len // case.page)] = torch.from_numpy(prefix.astype(np.int64)).to(q.device)
            if prefix_len % case.page and length > prefix_len:
                raise ValueError("prefix must end with a page")
        j = torch.arange(length, device=q.device)
        hidden = j[None, :] > (length - n + torch.arange(n, device=q.device))[:, None]
        gone = (pages < 0) | (pages >= case.n_pages)
        hidden |= gone[j // case.page][None, :]
        pages = pages.masked_fill(gone, 0)
        if length == 0:
            at += n
            continue
        for g in range(case.Hkv):
            k, v = (x[pages, g].reshape(-1, D)[:length].double() for x in (kd, vd))
            k, v = k.masked_fill(gone[j // case.page][:, None], 0), v.masked_fill(gone[j // case.page][:, None], 0)
            for h in range(g * G, (g + 1) * G):
                x = q[at:at + n, h].double()
                s = (x @ k.T).mul_(scale).masked_fill_(hidden, -np.inf)
                p = torch.softmax(s, 1).nan_to_num_(0.0)
                o[at:at + n, h] = p @ v
                A = p @ v.abs()
                S = scale * (x.abs() @ k.abs().T).max(1, keepdim=True).values
                rel = 2 * (2 * (72 * 2.0 ** -24 * S) + 2.0 ** -22 + length * 2.0 ** -24) + \
                    (2 * eps if case.dtype == "bf16" else 0.0)
                tol[at:at + n, h] = eps * o[at:at + n, h].abs() + rel * A
        at += n
    return o, tol
