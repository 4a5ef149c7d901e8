"""Timed calls of the paged KV cache: appending to it, and the attention that reads it.

A server keeps the keys and values of all its sequences in one pool of pages; a table per sequence
says which pages hold its keys.  Each case is one pass through one of the four operators, at the
shapes of TinyLLaMA-1.1B (32 query heads, 4 KV heads of 64), the model that the repository's
configurations, tests and benchmark use, and at its neighbours.  A case names its operator:

``append``   the new rows of a batch: K and Q rotated by their positions, K and V stored in the pages
``decode``   one query row per sequence against its pages
``prefill``  the new rows of a ragged batch (prompts, or chunks behind cached keys), causal
``shared``   decode of a batch whose first keys are common to all and read once

``run`` in its plain form is the same in elementary torch operations in 32 bits, ``exact`` in 64.
"""
import math
import os
import sys

import numpy as np
import torch

own = False  # true: run() calls the library's operators

D = 64          # head_dim, fixed by the kernels
THETA = 10000.0
_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _case(op, batch, shortest, longest, rows_from=1, rows_to=1, prefix=0, heads=32, kv_heads=4,
          dtype="bf16", page=16, head_major=True):
    """shortest..longest: keys per sequence behind the call's new rows (shared: behind the prefix
    too, the new row's key among them); rows_from..rows_to: new rows per sequence."""
    return dict(op=op, batch=batch, shortest=shortest, longest=longest, rows_from=rows_from,
                rows_to=rows_to, prefix=prefix, heads=heads, kv_heads=kv_heads, dtype=dtype, page=page,
                head_major=head_major)


def listed():
    return [
        # a decode step of a small server: 16 new tokens; the smallest call, launches count
        dict(name="append_step", **_case("append", 16, 1, 4000)),
        # the fp32 model's prompts of odd lengths
        dict(name="append_fp32", **_case("append", 3, 0, 0, 57, 777, dtype="fp32")),
        # a batch of prompts: the headline prefill configuration, 4 x 2048 rows
        dict(name="append_prompts", **_case("append", 4, 0, 0, 2048, 2048)),
        # the fp32 model's decode step behind its 512-token prompt
        dict(name="decode_fp32", **_case("decode", 1, 640, 640, dtype="fp32")),
        # a full batch, ragged U[512, 4096]: the serving configuration
        dict(name="decode_batch", **_case("decode", 64, 512, 4096)),
        # three users, one of them with a very long history
        dict(name="decode_long", **_case("decode", 3, 5003, 131072, page=64)),
        # the fp32 model's 512-token prompt, one layer
        dict(name="prefill_fp32", **_case("prefill", 1, 0, 0, 512, 512, dtype="fp32")),
        # prompts of different lengths that arrived together
        dict(name="prefill_prompts", **_case("prefill", 7, 0, 0, 33, 1500)),
        # chunked prefill: the next 256 rows of three long prompts
        dict(name="prefill_chunks", **_case("prefill", 3, 1000, 8192, 256, 256, page=32)),
        # one long document behind an equally long one
        dict(name="prefill_long", **_case("prefill", 1, 8192, 8192, 8192, 8192, page=64)),
        # a full batch behind one system prompt, short conversations of their own
        dict(name="shared_prompt", **_case("shared", 64, 1, 500, prefix=2048)),
        # many samples of one long document
        dict(name="shared_document", **_case("shared", 200, 1, 1000, prefix=16387, page=32)),
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
    fp32 = rng.random() < 0.25
    kind = dict(heads=heads, kv_heads=kv_heads, dtype="fp32" if fp32 else "bf16",
                page=rng.choice([8, 16, 16, 32, 64, 128]), head_major=rng.random() < 0.7)
    op = rng.choice(["append", "decode", "decode", "prefill", "prefill", "shared"])
    if op == "append":
        batch = _log(rng, 1, 64)
        to = min(_log(rng, 1, 4096), 8192 // batch // (4 if fp32 else 1))
        past = rng.choice([0, _log(rng, 1, 8192)])
        return _case(op, batch, past // 3, past, max(1, to // 4), max(1, to), **kind)
    if op == "decode":
        longest = _log(rng, 16, 65536)
        batch = max(1, min(_log(rng, 1, 128), (1 << 17) // longest // (2 if fp32 else 1)))
        shortest = max(1, int(longest * rng.choice([1.0, rng.uniform(0.02, 1.0)])))
        return _case(op, batch, shortest, longest, **kind)
    if op == "prefill":
        most = (1 << 27) // 20 if fp32 else (1 << 27) * 2 // 3   # (row, key) pairs
        while True:
            batch, to, past = _log(rng, 1, 12), _log(rng, 2, 8192), rng.choice([0, _log(rng, 16, 16384)])
            if batch * to * (to // 2 + past) <= most:
                return _case(op, batch, past // 2, past, max(1, int(to * rng.uniform(0.1, 1.0))), to, **kind)
    prefix = _log(rng, 64, 16384)
    longest = _log(rng, 1, 2000)
    batch = min(_log(rng, 2, 200), max(2, (1 << 16) // longest))
    return _case(op, batch, max(1, longest // 5), longest, prefix=prefix, **kind)


# ------------------------------------------------------------------- inputs
def _spread(lo, hi, n):
    """n integers over [lo, hi], the first of them hi, in no order."""
    return [hi] + [lo + int((hi - lo) * ((i * 0.6180339887498949) % 1.0)) for i in range(1, n)]


def _sizes(case):
    """(new rows, keys with the new ones) of every sequence."""
    rows = _spread(case["rows_from"], case["rows_to"], case["batch"])
    past = _spread(case["shortest"], case["longest"], case["batch"])[::-1]
    if case["op"] in ("append", "prefill"):
        return rows, [p + n for p, n in zip(past, rows)]
    return rows, [case["prefix"] + p for p in past]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    B, H, Hkv, ps = case["batch"], case["heads"], case["kv_heads"], case["page"]
    rows, lens = _sizes(case)
    total = sum(rows)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dt)

    # the pages of every sequence, anywhere in the pool; the full pages of a common prefix are
    # everyone's, and a page that it shares with a sequence's own keys is that sequence's copy
    common = case["prefix"] // ps
    need = [-(-n // ps) for n in lens]
    n_prefix = -(-case["prefix"] // ps)
    n_pages = n_prefix + sum(n - common for n in need) + 5
    order = np.random.default_rng(seed).permutation(n_pages).astype(np.int32)
    max_pages = max(need) + 2
    table = np.full((B, max_pages), -1, np.int32)
    prefix_pages, at = order[:n_prefix], n_prefix
    for b, n in enumerate(need):
        table[b, :common] = prefix_pages[:common]
        table[b, common:n] = order[at:at + n - common]
        at += n - common

    def pool():
        if case["head_major"]:
            return normal(n_pages, Hkv, ps, D)
        return normal(n_pages, ps, Hkv, D).transpose(1, 2)

    k, v = pool(), pool()
    if case["prefix"] % ps:
        own_copy = torch.from_numpy(table[:, common].astype(np.int64)).cuda()
        for p in (k, v):
            p[own_copy, :, :case["prefix"] % ps] = p[int(prefix_pages[-1]), :, :case["prefix"] % ps]
    t = dict(case=case, k=k, v=v, table=torch.from_numpy(table).cuda(),
             lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
             starts=torch.tensor([0] + rows, device="cuda").cumsum(0).to(torch.int32))
    if case["op"] == "append":
        # the projection's output, a row per token: Q | K | V
        t["qkv"] = normal(total, (H + 2 * Hkv) * D)
        t["q_out"] = torch.zeros((total, H, D), dtype=dt, device="cuda")
    else:
        t["q"] = normal(total, H, D)
        t["o"] = torch.zeros((total, H, D), dtype=dt, device="cuda")
    if case["op"] == "shared":
        t["prefix_pages"] = torch.from_numpy(prefix_pages).cuda()
    # what the program knows on the host
    t["rows"], t["host_lens"] = rows, lens
    if own:
        bnhip = _library()
        t["cache"] = bnhip.PagedKV(t["k"], t["v"], t["table"], t["lens"])
        if case["op"] != "append":
            t["workspace"] = bnhip.paged_workspace(t["cache"], H, total, case["prefix"])
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
    if case["op"] == "append":
        q, k, v = _split(t)
        starts = None if case["rows_to"] == 1 else t["starts"]
        bnhip.paged_append(t["cache"], k, v, q=q, q_out=t["q_out"], row_starts=starts, theta=THETA)
        return dict(k=t["k"], v=t["v"], q=t["q_out"])
    if case["op"] == "decode":
        return bnhip.paged_decode(t["q"], t["cache"], o=t["o"], workspace=t["workspace"])
    if case["op"] == "prefill":
        return bnhip.paged_prefill(t["q"], t["cache"], t["starts"], o=t["o"], workspace=t["workspace"])
    return bnhip.paged_decode_shared(t["q"], t["cache"], t["prefix_pages"], case["prefix"], o=t["o"],
                                     workspace=t["workspace"])


def _rotate(x, pos):
    """Adjacent pairs of each head turned by pos * theta^(-2p/D); the angles in 64 bits."""
    freq = THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device=x.device) / D)
    angle = pos.double()[:, None] * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    y = x.float()
    out = torch.empty_like(y)
    out[..., 0::2] = y[..., 0::2] * cos - y[..., 1::2] * sin
    out[..., 1::2] = y[..., 0::2] * sin + y[..., 1::2] * cos
    return out.to(x.dtype)


def _keys(pool, table, first, n):
    """Keys first .. first + n - 1 of every sequence of the table: [B, n, Hkv, D] in 32 bits
    (entries without a page read page 0: the caller masks them)."""
    ps = pool.shape[2]
    j = first + torch.arange(n, device=pool.device)
    page = table[:, j // ps].long().clamp(min=0)
    return pool[page, :, (j % ps)[None].expand_as(page)].float()


def _softmax(s):
    """Rows of scores to probabilities; a row of -inf alone gives zeros."""
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    return p / p.sum(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)


def _run_plain(t):
    case = t["case"]
    B, H, Hkv, ps = case["batch"], case["heads"], case["kv_heads"], case["page"]
    G, scale = H // Hkv, 1.0 / math.sqrt(D)
    if case["op"] == "append":
        q, k, v = _split(t)
        row = torch.arange(q.shape[0], device=q.device)
        b = torch.searchsorted(t["starts"][1:].contiguous(), row.to(torch.int32), right=True)
        pos = t["lens"][b] - t["starts"][b + 1] + row
        page, slot = t["table"][b, pos // ps].long(), (pos % ps).long()
        t["k"][page, :, slot] = _rotate(k, pos)
        t["v"][page, :, slot] = v
        t["q_out"].copy_(_rotate(q, pos))
        return dict(k=t["k"], v=t["v"], q=t["q_out"])
    if case["op"] == "prefill":
        at = 0
        for b, (n, length) in enumerate(zip(t["rows"], t["host_lens"])):
            table = t["table"][b:b + 1]
            k = _keys(t["k"], table, 0, length)[0].permute(1, 2, 0).contiguous()   # [Hkv, D, L]
            v = _keys(t["v"], table, 0, length)[0].transpose(0, 1).contiguous()    # [Hkv, L, D]
            j = torch.arange(length, device=k.device)
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
    # one row per sequence: the scores of a common prefix for all of them at once, then each
    # sequence's own keys, padded to the longest
    P, longest = case["prefix"], max(t["host_lens"]) - case["prefix"]
    q = t["q"].float().view(B, Hkv, G, D)
    k, v = (_keys(p, t["table"], P, longest).transpose(1, 2).contiguous() for p in (t["k"], t["v"]))
    s = (q @ k.transpose(2, 3)) * scale                                   # [B, Hkv, G, longest]
    j = P + torch.arange(longest, device=q.device)
    s = s.masked_fill((j[None, :] >= t["lens"][:, None])[:, None, None], -math.inf)
    if P == 0:
        o = _softmax(s) @ v
    else:
        table = t["prefix_pages"][None]
        kp = _keys(t["k"], table, 0, P)[0].permute(1, 2, 0).contiguous()  # [Hkv, D, P]
        vp = _keys(t["v"], table, 0, P)[0].transpose(0, 1).contiguous()   # [Hkv, P, D]
        sp = (q.transpose(0, 1).reshape(Hkv, B * G, D) @ kp) * scale
        p = _softmax(torch.cat([sp.view(Hkv, B, G, P).transpose(0, 1), s], -1))
        o = (p[..., :P].transpose(0, 1).reshape(Hkv, B * G, P) @ vp).view(Hkv, B, G, D).transpose(0, 1)
        o = o + p[..., P:].contiguous() @ v
    t["o"].copy_(o.reshape(B, H, D))
    return t["o"]


# ------------------------------------------------------------------- its cost
def work(case):
    e, H, Hkv = 2 if case["dtype"] == "bf16" else 4, case["heads"], case["kv_heads"]
    rows, lens = _sizes(case)
    total = sum(rows)
    if case["op"] == "append":   # read and written once; a rotation is three operations an element
        return {"bytes": 2 * total * (H + 2 * Hkv) * D * e, "flops": 3 * total * (H + Hkv) * D}
    pairs = sum(n * (length - n) + n * (n + 1) // 2 for n, length in zip(rows, lens))
    keys = sum(lens) - (case["batch"] - 1) * case["prefix"]
    return {"bytes": e * D * (2 * keys * Hkv + 2 * total * H), "flops": 4 * pairs * H * D}


# ------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    t = prepare(case, seed)
    rows, lens = _sizes(case)
    H, Hkv, ps = case["heads"], case["kv_heads"], case["page"]
    G, at = H // Hkv, 0
    if case["op"] == "append":
        out = dict(k=t["k"].double(), v=t["v"].double(),
                   q=torch.empty(t["q_out"].shape, dtype=torch.float64, device="cuda"))
        new = t["qkv"].double()
        for b, (n, length) in enumerate(zip(rows, lens)):
            x = new[at:at + n].view(n, H + 2 * Hkv, D // 2, 2)
            pos = torch.arange(length - n, length, dtype=torch.float64, device="cuda")
            turn = torch.exp(torch.arange(D // 2, dtype=torch.float64, device="cuda")
                             * (-2.0 / D * math.log(THETA)))
            z = torch.view_as_complex(x[:, :H + Hkv].contiguous())
            a = pos[:, None, None] * turn
            z = torch.view_as_real(z * torch.complex(a.cos(), a.sin())).reshape(n, H + Hkv, D)
            out["q"][at:at + n] = z[:, :H]
            j = np.arange(length - n, length)
            page = t["table"][b].cpu().numpy()[j // ps]
            where = (torch.from_numpy(page).long().cuda(), slice(None), torch.from_numpy(j % ps).cuda())
            out["k"][where] = z[:, H:]
            out["v"][where] = x[:, H + Hkv:].reshape(n, Hkv, D)
            at += n
        return out
    o = torch.empty(t["o"].shape, dtype=torch.float64, device="cuda")
    for b, (n, length) in enumerate(zip(rows, lens)):
        pages = t["table"][b, :-(-length // ps)].long()
        hidden = None
        if n > 1:
            hidden = torch.ones(n, length, dtype=torch.bool, device="cuda").triu(length - n + 1)
        for g in range(Hkv):
            k, v = (p[pages, g].reshape(-1, D)[:length].double() for p in (t["k"], t["v"]))
            for h in range(g * G, (g + 1) * G):
                s = t["q"][at:at + n, h].double() @ k.T / math.sqrt(D)
                if hidden is not None:
                    s.masked_fill_(hidden, -math.inf)
                s.sub_(torch.logsumexp(s, dim=1, keepdim=True)).exp_()
                o[at:at + n, h] = s @ v
        at += n
    return o
