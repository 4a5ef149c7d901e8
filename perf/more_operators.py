"""Timed calls of a paged KV cache held in 8 bits, and of the norms of single heads that feed it.

The cache holds keys and values as e4m3 numbers under a power of two for every 16 keys of a page and
KV head, half the memory of the bf16 cache and half the bytes that a decode step reads.  Queries and
keys may be normed, head by head, before they are turned.  Each case is one pass through one of six
operators, at the shapes of TinyLLaMA-1.1B (32 query heads, 4 KV heads of 64), the model that the
repository's configurations, tests and benchmark use, and at its neighbours.  A case names its
operator:

``norm``      RMSNorm of every query and key head, and the rotation by the position, in one pass
``gradient``  the same backward: gradients of the rows and of the two weights
``append``    the new rows of a batch: normed and turned, K and V rounded and stored in the pages;
              then the blocks of 16 keys that they lie in, read back (older rows of the first block
              among them, which a larger scale rounds again)
``read``      the last keys of every sequence as bf16 rows
``decode``    one query row per sequence against its pages
``prefill``   the new rows of a ragged batch (prompts, or chunks behind cached keys), causal

``run`` in its plain form is the same in elementary torch operations in 32 bits, ``exact`` in 64.
"""
import math
import os
import sys

import numpy as np
import torch

own = False  # true: run() calls the library's operators

D = 64          # head_dim, fixed by the attention kernels
BLOCK = 16      # keys of a page that have a scale in common
THETA = 10000.0
EPS = 1e-5
_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_E4M3 = torch.float8_e4m3fn


def _case(op, batch, shortest, longest, rows_from=1, rows_to=1, heads=32, kv_heads=4, dtype="bf16",
          page=16, head_major=True, norm=True):
    """shortest..longest: keys per sequence behind the call's rows (decode: the new row's key among
    them); rows_from..rows_to: the call's rows per sequence."""
    return dict(op=op, batch=batch, shortest=shortest, longest=longest, rows_from=rows_from,
                rows_to=rows_to, heads=heads, kv_heads=kv_heads, dtype=dtype, page=page,
                head_major=head_major, norm=norm)


def listed():
    return [
        # a decode step of a small server without a cache of this library: launches count
        dict(name="norm_step", **_case("norm", 16, 1, 4000)),
        # a training batch: the headline prefill configuration, 4 x 2048 rows
        dict(name="norm_batch", **_case("norm", 4, 0, 0, 2048, 2048)),
        # the fp32 model's sequences of odd lengths, packed
        dict(name="gradient_fp32", **_case("gradient", 3, 0, 0, 57, 777, dtype="fp32")),
        # the long-context configuration: one sequence of 16384 rows
        dict(name="gradient_long", **_case("gradient", 1, 0, 0, 16384, 16384)),
        # a decode step of a full batch: one row each, somewhere in a block of older rows
        dict(name="append_step", **_case("append", 64, 511, 4095)),
        # a batch of prompts
        dict(name="append_prompts", **_case("append", 4, 0, 0, 2048, 2048)),
        # a finished conversation taken out of the cache
        dict(name="read_one", **_case("read", 1, 0, 0, 1237, 1237)),
        # a long document's keys for another cache
        dict(name="read_long", **_case("read", 2, 0, 0, 40000, 65536, page=64)),
        # a full batch, ragged U[512, 4096]: the serving configuration
        dict(name="decode_batch", **_case("decode", 64, 512, 4096)),
        # three users, one of them with a very long history
        dict(name="decode_long", **_case("decode", 3, 5003, 131072, page=64)),
        # prompts of different lengths that arrived together, behind earlier turns of their own
        dict(name="prefill_prompts", **_case("prefill", 7, 0, 700, 33, 1500)),
        # one long document behind an equally long one
        dict(name="prefill_long", **_case("prefill", 1, 8192, 8192, 8192, 8192, page=64)),
    ]


def _log(rng, lo, hi):
    """An integer in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the same ranges, no dearer than its operator's largest listed one."""
    while True:
        case = _draw(rng)
        if all(work(case)[k] <= max(work(c)[k] for c in listed() if c["op"] == case["op"])
               for k in ("bytes", "flops")):
            return case


def _draw(rng):
    heads, kv_heads = rng.choice([(32, 4), (32, 4), (32, 4), (32, 8), (16, 4), (12, 4), (8, 8), (20, 4)])
    kind = dict(heads=heads, kv_heads=kv_heads, page=rng.choice([16, 16, 32, 64, 128]),
                head_major=rng.random() < 0.7)
    op = rng.choice(["norm", "gradient", "append", "append", "read", "decode", "decode", "prefill", "prefill"])
    if op in ("norm", "gradient", "append"):
        fp32 = rng.random() < 0.3
        batch = _log(rng, 1, 64)
        most = (16384 if op == "gradient" else 8192) // batch // (4 if fp32 else 1)
        to = min(_log(rng, 1, 16384), most)
        past = rng.choice([0, _log(rng, 1, 8192)])
        norm = op != "append" or rng.random() < 0.6
        return _case(op, batch, past // 3, past, max(1, to // 4), max(1, to), dtype="fp32" if fp32 else "bf16",
                     norm=norm, **kind)
    if op == "read":
        batch = _log(rng, 1, 64)
        to = min(_log(rng, 1, 65536), (1 << 16) // batch)
        past = rng.choice([0, 0, _log(rng, 1, 2048)])
        return _case(op, batch, past // 3, past, max(1, to // rng.choice([1, 5])), max(1, to), **kind)
    if op == "decode":
        longest = _log(rng, 16, 65536)
        batch = max(1, min(_log(rng, 1, 128), (1 << 17) // longest))
        shortest = max(1, int(longest * rng.choice([1.0, rng.uniform(0.02, 1.0)])))
        return _case(op, batch, shortest, longest, **kind)
    while True:
        batch, to, past = _log(rng, 1, 12), _log(rng, 2, 8192), rng.choice([0, _log(rng, 16, 16384)])
        if batch * to * (to // 2 + past) <= (1 << 27) * 2 // 3:   # (row, key) pairs
            return _case(op, batch, past // 2, past, max(1, int(to * rng.uniform(0.1, 1.0))), to, **kind)


# ------------------------------------------------------------------- inputs
def _spread(lo, hi, n):
    """n integers over [lo, hi], the first of them hi, in no order."""
    return [hi] + [lo + int((hi - lo) * ((i * 0.6180339887498949) % 1.0)) for i in range(1, n)]


def _sizes(case):
    """(the call's rows, keys with them) of every sequence."""
    rows = _spread(case["rows_from"], case["rows_to"], case["batch"])
    past = _spread(case["shortest"], case["longest"], case["batch"])[::-1]
    return rows, past if case["op"] == "decode" else [p + n for p, n in zip(past, rows)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    op, B, H, Hkv, ps = case["op"], case["batch"], case["heads"], case["kv_heads"], case["page"]
    rows, lens = _sizes(case)
    total = sum(rows)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def index(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    starts = index([0] + rows).cumsum(0).to(torch.int32)
    t = dict(case=case, starts=starts, lens=index(lens))
    if op in ("norm", "gradient", "append"):
        # the projection's output, a row per token: Q | K | V
        t["qkv"] = normal(total, (H + 2 * Hkv) * D).to(dt)
        t["wq"], t["wk"] = ((1 + 0.2 * normal(D)).to(dt) for _ in range(2))
    if op in ("norm", "gradient"):
        row = torch.arange(total, device="cuda")
        b = torch.searchsorted(starts[1:].contiguous(), row.to(torch.int32), right=True)
        t["positions"] = (t["lens"][b] - starts[b + 1] + row).to(torch.int32)
        t["q_out"], t["k_out"] = (torch.zeros((total, h, D), dtype=dt, device="cuda") for h in (H, Hkv))
        if op == "gradient":
            t["gq"], t["gk"] = normal(total, H, D).to(dt), normal(total, Hkv, D).to(dt)
            if own:
                t["workspace"] = _library().qk_norm_rope_workspace(total, H, Hkv)
        if own:
            _library()
        return t

    # the pages of every sequence, anywhere in the pool
    need = [-(-n // ps) for n in lens]
    n_pages = sum(need) + 5
    order = np.random.default_rng(seed).permutation(n_pages).astype(np.int32)
    table = np.full((B, max(need) + 2), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    t["table"] = torch.from_numpy(table).cuda()
    for name in ("k", "v"):
        # what earlier calls stored: the largest code of a block lies in (224, 448]
        x = normal(n_pages, Hkv, ps // BLOCK, BLOCK * D)
        x *= torch.exp2(0.5 * normal(n_pages, Hkv, ps // BLOCK, 1).clamp(-2, 2))
        k = _power(x.abs().amax(-1, keepdim=True))
        codes = _round(x, k).view(torch.uint8).view(n_pages, Hkv, ps, D)
        if not case["head_major"]:
            codes = codes.transpose(1, 2).contiguous().transpose(1, 2)
        t[name], t[name + "_scale"] = codes, (k[..., 0] + 127).to(torch.uint8)
    if op == "append":
        t["q_out"] = torch.zeros((total, H, D), dtype=dt, device="cuda")
        # the rows of the first new row's block that were there before it
        t["back"] = index([0] + [n + (length - n) % BLOCK for n, length in zip(rows, lens)]).cumsum(0).to(torch.int32)
    if op in ("append", "read"):
        n = int(t["back" if op == "append" else "starts"][-1])
        t["k_rows"], t["v_rows"] = (torch.zeros((n, Hkv, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    if op in ("decode", "prefill"):
        t["q"] = normal(total, H, D).to(dt)
        t["o"] = torch.zeros((total, H, D), dtype=dt, device="cuda")
    # what the program knows on the host
    t["rows"], t["host_lens"] = rows, lens
    if own:
        bnhip = _library()
        t["cache"] = bnhip.PagedQ8(t["k"], t["v"], t["k_scale"], t["v_scale"], t["table"], t["lens"])
        if op in ("decode", "prefill"):
            t["workspace"] = bnhip.paged_q8_workspace(t["cache"], H, total)
    return t


def _library():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "baranet-bdml_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import bnhip
    return bnhip


# ------------------------------------------------------------------- a pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _split(t):
    """Q, K and V of the projection's rows, as views."""
    case = t["case"]
    H, Hkv, n = case["heads"], case["kv_heads"], t["qkv"].shape[0]
    x = t["qkv"]
    return (x[:, :H * D].view(n, H, D), x[:, H * D:(H + Hkv) * D].view(n, Hkv, D),
            x[:, (H + Hkv) * D:].view(n, Hkv, D))


def _run_own(t):
    bnhip, case = sys.modules["bnhip"], t["case"]
    op = case["op"]
    if op == "norm":
        q, k, _ = _split(t)
        bnhip.qk_norm_rope(q, k, t["wq"], t["wk"], EPS, positions=t["positions"], theta=THETA,
                           q_out=t["q_out"], k_out=t["k_out"])
        return dict(q=t["q_out"], k=t["k_out"])
    if op == "gradient":
        q, k, _ = _split(t)
        dq, dk, dwq, dwk = bnhip.qk_norm_rope_backward(
            q, k, t["wq"], t["wk"], t["gq"], t["gk"], EPS, positions=t["positions"], theta=THETA,
            dq=t["q_out"], dk=t["k_out"], workspace=t["workspace"])
        return dict(q=dq, k=dk, wq=dwq, wk=dwk)
    if op == "append":
        q, k, v = _split(t)
        starts = None if case["rows_to"] == 1 else t["starts"]
        norms = dict(q_weight=t["wq"], k_weight=t["wk"], eps=EPS) if case["norm"] else {}
        bnhip.paged_q8_append(t["cache"], k, v, q=q, q_out=t["q_out"], row_starts=starts, theta=THETA, **norms)
        bnhip.paged_q8_read(t["cache"], t["back"], k=t["k_rows"], v=t["v_rows"])
        return dict(k=t["k_rows"], v=t["v_rows"], q=t["q_out"])
    if op == "read":
        bnhip.paged_q8_read(t["cache"], t["starts"], k=t["k_rows"], v=t["v_rows"])
        return dict(k=t["k_rows"], v=t["v_rows"])
    if op == "decode":
        return bnhip.paged_q8_decode(t["q"], t["cache"], o=t["o"], workspace=t["workspace"])
    return bnhip.paged_q8_prefill(t["q"], t["cache"], t["starts"], o=t["o"], workspace=t["workspace"])


def _turn(pos):
    """Cosines and sines [rows, 1, D/2] of pos * theta^(-2p/D); the angles in 64 bits."""
    freq = THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device=pos.device) / D)
    angle = pos.double()[:, None] * freq
    return angle.cos().float()[:, None], angle.sin().float()[:, None]


def _rotate(x, cos, sin):
    """Adjacent pairs of each head turned, in 32 bits."""
    out = torch.empty_like(x)
    out[..., 0::2] = x[..., 0::2] * cos - x[..., 1::2] * sin
    out[..., 1::2] = x[..., 0::2] * sin + x[..., 1::2] * cos
    return out


def _normed(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()


def _power(amax):
    """The smallest k with amax <= 448 2^k, within what the scales can say."""
    m, e = torch.frexp(amax)
    return torch.where(amax > 0, e - 9 + (m > 0.875).int(), -117).clamp(-117, 120)


def _round(x, k):
    """x as e4m3 numbers under 2^k."""
    return torch.ldexp(x, -k).clamp(-448, 448).to(_E4M3)


def _run_plain(t):
    case = t["case"]
    op, H, Hkv = case["op"], case["heads"], case["kv_heads"]
    G, scale = H // Hkv, 1.0 / math.sqrt(D)
    if op == "norm":
        q, k, _ = _split(t)
        turn = _turn(t["positions"])
        t["q_out"].copy_(_rotate(_normed(q.float(), t["wq"]), *turn))
        t["k_out"].copy_(_rotate(_normed(k.float(), t["wk"]), *turn))
        return dict(q=t["q_out"], k=t["k_out"])
    if op == "gradient":
        q, k, _ = _split(t)
        cos, sin = _turn(t["positions"])

        def back(x, w, dy, dx):
            x, w = x.float(), w.float()
            g = _rotate(dy.float(), cos, -sin)
            r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
            u, wg = x * r, g * w
            dx.copy_(r * (wg - u * (wg * u).mean(-1, keepdim=True)))
            return dx, (g * u).sum((0, 1))

        dq, dwq = back(q, t["wq"], t["gq"], t["q_out"])
        dk, dwk = back(k, t["wk"], t["gk"], t["k_out"])
        return dict(q=dq, k=dk, wq=dwq, wk=dwk)
    if op == "append":
        _store(t)
        return dict(**_back(t, t["back"]), q=t["q_out"])
    if op == "read":
        return _back(t, t["starts"])
    if op == "decode":
        q = t["q"].float().view(-1, Hkv, G, D)
        longest = max(t["host_lens"])
        j = torch.arange(longest, device=q.device)
        page = t["table"][:, j // case["page"]].long().clamp(min=0)
        slot = (j % case["page"])[None].expand_as(page)
        k, v = (_values(t, n, page, slot).transpose(1, 2).contiguous() for n in "kv")   # [B, Hkv, L, D]
        s = (q @ k.transpose(2, 3)) * scale
        s = s.masked_fill((j[None, :] >= t["lens"][:, None])[:, None, None], -math.inf)
        t["o"].copy_((_softmax(s) @ v).reshape(-1, H, D))
        return t["o"]
    at = 0
    for b, (n, length) in enumerate(zip(t["rows"], t["host_lens"])):
        j = torch.arange(length, device=t["q"].device)
        page, slot = t["table"][b, j // case["page"]].long(), j % case["page"]
        k = _values(t, "k", page, slot).permute(1, 2, 0).contiguous()   # [Hkv, D, L]
        v = _values(t, "v", page, slot).transpose(0, 1).contiguous()    # [Hkv, L, D]
        for r0 in range(0, n, 1024):
            m = min(1024, n - r0)
            q = t["q"][at + r0:at + r0 + m].float().view(m, Hkv, G, D)
            s = (q.permute(1, 2, 0, 3).reshape(Hkv, G * m, D) @ k).view(Hkv, G, m, length) * scale
            last = length - n + r0 + torch.arange(m, device=k.device)
            s = s.masked_fill(j[None, :] > last[:, None], -math.inf)
            o = (_softmax(s).view(Hkv, G * m, length) @ v).view(Hkv, G, m, D)
            t["o"][at + r0:at + r0 + m] = o.permute(2, 0, 1, 3).reshape(m, H, D).to(t["o"].dtype)
        at += n
    return t["o"]


def _places(t, starts, n):
    """(sequence, position, page, slot) of n rows, those of sequence b its last ones."""
    row = torch.arange(n, device=starts.device)
    b = torch.searchsorted(starts[1:].contiguous(), row.to(torch.int32), right=True)
    pos = t["lens"][b] - starts[b + 1] + row
    ps = t["case"]["page"]
    return b, pos, t["table"][b, pos // ps].long(), (pos % ps).long()


def _values(t, name, page, slot):
    """What the cache holds in the places, in 32 bits: [..., Hkv, D]."""
    k = t[name + "_scale"][page, :, slot // BLOCK].int() - 127
    return torch.ldexp(t[name][page, :, slot].view(_E4M3).float(), k[..., None])


def _back(t, starts):
    _, _, page, slot = _places(t, starts, t["k_rows"].shape[0])
    for name in "kv":
        t[name + "_rows"].copy_(_values(t, name, page, slot))
    return dict(k=t["k_rows"], v=t["v_rows"])


def _store(t):
    """Norm, rotation, rounding and storing of the new rows."""
    q, k, v = (x.float() for x in _split(t))
    _, pos, page, slot = _places(t, t["starts"], q.shape[0])
    if t["case"]["norm"]:
        q, k = _normed(q, t["wq"]), _normed(k, t["wk"])
    cos, sin = _turn(pos)
    t["q_out"].copy_(_rotate(q, cos, sin))
    # sequences whose first new row comes behind older ones in its block: those rows, in 32 bits
    first = t["starts"][:-1].long()
    head, at = page[first], slot[first] // BLOCK
    old = torch.arange(BLOCK, device=q.device) < slot[first, None] % BLOCK      # [B, 16]
    inside = at[:, None] * BLOCK + torch.arange(BLOCK, device=q.device)
    heads = torch.arange(k.shape[1], device=q.device)
    for name, x in (("k", _rotate(k, cos, sin)), ("v", v)):
        codes, scales = t[name], t[name + "_scale"]
        n_pages, Hkv, blocks = scales.shape
        amax = torch.zeros((n_pages * blocks, Hkv), device=x.device)
        block = page * blocks + slot // BLOCK
        amax.scatter_reduce_(0, block[:, None].expand(-1, Hkv), x.abs().amax(-1), "amax")
        power = _power(amax).view(n_pages, blocks, Hkv)
        before = scales[head, :, at].int() - 127                                # [B, Hkv]
        merged = torch.where(old.any(1)[:, None], torch.maximum(before, power[head, at]), power[head, at])
        power[head, at] = merged
        rows = _values(t, name, head[:, None].expand_as(inside), inside)        # [B, 16, Hkv, D]
        again = _round(rows, merged[:, None, :, None]).view(torch.uint8)
        kept = codes[head[:, None], :, inside]
        codes[head[:, None, None], heads, inside[:, :, None]] = torch.where(old[:, :, None, None], again, kept)
        k_of_row = power[page, slot // BLOCK]                                   # [rows, Hkv]
        scales[page, :, slot // BLOCK] = (k_of_row + 127).to(torch.uint8)
        codes[page, :, slot] = _round(x, k_of_row[..., None]).view(torch.uint8)


def _softmax(s):
    """Rows of scores to probabilities; a row of -inf alone gives zeros."""
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    return p / p.sum(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)


# ------------------------------------------------------------------- its cost
def work(case):
    e, H, Hkv, op = 2 if case["dtype"] == "bf16" else 4, case["heads"], case["kv_heads"], case["op"]
    rows, lens = _sizes(case)
    total = sum(rows)
    held = D + 1 / BLOCK  # bytes of a row in the cache, with its part of the scale
    if op == "norm":       # read and written once; squares, two scalings and a rotation
        return {"bytes": 2 * total * (H + Hkv) * D * e, "flops": 7 * total * (H + Hkv) * D}
    if op == "gradient":   # rows and gradients read, gradients written
        return {"bytes": 3 * total * (H + Hkv) * D * e, "flops": 16 * total * (H + Hkv) * D}
    if op == "append":     # rows read, q written; K and V written in 8 bits, read back and written as bf16
        back = sum(n + (length - n) % BLOCK for n, length in zip(rows, lens))
        return {"bytes": int(total * (2 * H + 2 * Hkv) * D * e + 2 * Hkv * (total * held + back * (held + 2 * D))),
                "flops": 7 * total * (H + Hkv) * D + 4 * total * Hkv * D}
    if op == "read":
        return {"bytes": int(2 * total * Hkv * (held + 2 * D)), "flops": 2 * total * Hkv * D}
    pairs = sum(n * (length - n) + n * (n + 1) // 2 for n, length in zip(rows, lens))
    return {"bytes": int(2 * sum(lens) * Hkv * held) + 2 * total * H * D * e, "flops": 4 * pairs * H * D}


# ------------------------------------------------------------------- the same in 64 bits
def _turned64(x, pos, sign=1.0):
    """x [n, heads, D] float64, each pair a complex number times exp(i angle)."""
    turn = torch.exp(torch.arange(D // 2, dtype=torch.float64, device=x.device) * (-2.0 / D * math.log(THETA)))
    a = sign * pos.double()[:, None, None] * turn
    z = torch.view_as_complex(x.contiguous().view(*x.shape[:-1], D // 2, 2))
    return torch.view_as_real(z * torch.complex(a.cos(), a.sin())).reshape(x.shape)


def _normed64(x, w):
    return x / (torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / D + EPS).sqrt() * w.double()


def _held64(x, power):
    """x [..., D] float64 rounded to the nearest e4m3 number times 2^power, ties to even."""
    y = x / torch.exp2(power.double())
    exponent = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -30))).clamp(min=-6)
    step = torch.exp2(exponent - 3)
    return (torch.round(y / step) * step).clamp(-448, 448) * torch.exp2(power.double())


def _pool64(t, name):
    """The whole pool's values, [n_pages, Hkv, page, D] float64."""
    byte = torch.arange(256, device="cuda")
    sign, e, m = 1 - 2.0 * (byte >> 7), byte >> 3 & 15, (byte & 7).double()
    values = sign * torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.exp2(e.double() - 10))
    power = t[name + "_scale"].double() - 127
    return values[t[name].long()] * torch.exp2(power).repeat_interleave(BLOCK, 2)[..., None]


def exact(case, seed):
    t = prepare(case, seed)
    rows, lens = _sizes(case)
    op, H, Hkv, ps = case["op"], case["heads"], case["kv_heads"], case["page"]
    G, at = H // Hkv, 0
    if op in ("norm", "gradient"):
        pos, out = t["positions"], {}
        n = pos.shape[0]
        for name, x, w in (("q", t["qkv"][:, :H * D].reshape(n, H, D).double(), t["wq"]),
                           ("k", t["qkv"][:, H * D:(H + Hkv) * D].reshape(n, Hkv, D).double(), t["wk"])):
            if op == "norm":
                out[name] = _turned64(_normed64(x, w), pos)
                continue
            g = _turned64(t["g" + name].double(), pos, -1.0)
            ms = x.square().sum(-1, keepdim=True) / D + EPS
            wg = g * w.double()
            out[name] = wg / ms.sqrt() - x * (wg * x).sum(-1, keepdim=True) / (D * ms ** 1.5)
            out["w" + name] = (g * x / ms.sqrt()).flatten(0, 1).sum(0)
        return out
    if op in ("append", "read"):
        n_back = [n + ((length - n) % BLOCK if op == "append" else 0) for n, length in zip(rows, lens)]
        new = {}
        if op == "append":
            pos = torch.cat([torch.arange(length - n, length, device="cuda") for n, length in zip(rows, lens)])
            x = t["qkv"].double().view(-1, H + 2 * Hkv, D)
            q, k, v = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
            if case["norm"]:
                q, k = _normed64(q, t["wq"]), _normed64(k, t["wk"])
            new = dict(q=_turned64(q, pos), k=_turned64(k, pos), v=v)
        out = {}
        for name in "kv":
            pool, power, got, at = _pool64(t, name), t[name + "_scale"].double() - 127, [], 0
            for b, (n, length, back) in enumerate(zip(rows, lens, n_back)):
                j = torch.arange(length - back, length, device="cuda")
                page = t["table"][b, j // ps].long()
                held = pool[page, :, j % ps]                     # [back, Hkv, D]
                if op == "append":
                    past = back - n                              # older rows of the first block
                    full = torch.zeros((-(-back // BLOCK) * BLOCK, Hkv, D), dtype=torch.float64, device="cuda")
                    full[:past], full[past:back] = held[:past], new[name][at:at + n]
                    blocks = full.view(-1, BLOCK, Hkv, D)
                    biggest = blocks.clone()
                    biggest[0, :past] = 0                        # they are under the scale that they had
                    a = biggest.abs().amax((1, 3))
                    k = torch.ceil(torch.log2(a / 448))
                    k = torch.where(a > 448 * torch.exp2(k), k + 1, torch.where(a <= 448 * torch.exp2(k - 1), k - 1, k))
                    k = k.clamp(-117, 120)
                    if past:
                        k[0] = torch.maximum(k[0], power[page[0], :, int(j[0]) % ps // BLOCK])
                    held = _held64(blocks, k[:, None, :, None].expand(-1, BLOCK, -1, 1)).view(-1, Hkv, D)[:back]
                got.append(held)
                at += n
            out[name] = torch.cat(got)
        if op == "append":
            out["q"] = new["q"]
        return out
    o = torch.empty(t["o"].shape, dtype=torch.float64, device="cuda")
    k64, v64 = _pool64(t, "k"), _pool64(t, "v")
    for b, (n, length) in enumerate(zip(rows, lens)):
        pages = t["table"][b, :-(-length // ps)].long()
        hidden = None
        if n > 1:
            hidden = torch.ones(n, length, dtype=torch.bool, device="cuda").triu(length - n + 1)
        for g in range(Hkv):
            k, v = (p[pages, g].reshape(-1, D)[:length] for p in (k64, v64))
            for h in range(g * G, (g + 1) * G):
                s = t["q"][at:at + n, h].double() @ k.T / math.sqrt(D)
                if hidden is not None:
                    s.masked_fill_(hidden, -math.inf)
                s.sub_(torch.logsumexp(s, dim=1, keepdim=True)).exp_()
                o[at:at + n, h] = s @ v
        at += n
    return o
