"""Norms of single heads with the rotation in the same pass, and the backward pass, against the formulas in
64 bits and against differences.

Tolerances: a head's mean of squares is a sum of D products in 32 bits, its root and reciprocal two units
more, then two products, the rotation's sine and cosine (2 units each), two products and a sum: a value is off
by at most (D / 2 + 20) 2^-24 of the sizes of the pair that it came from, and half a step of its type."""
import numpy as np
import pytest
import torch

import bnhip as B
from gpu_util import require_gpu
from paged_util import TD
from test_gpu_paged import bits, host, wide

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def turn(x, pos, theta, back=False):
    """x [rows, heads, D] float64 turned by the rows' positions."""
    if theta == 0:
        return x
    d = x.shape[-1]
    a = np.asarray(pos, np.float64)[:, None] * float(np.float32(theta)) ** (-np.arange(0, d, 2) / d)
    c, s = np.cos(a)[:, None], np.sin(a)[:, None] * (-1 if back else 1)
    y = np.empty_like(x)
    y[..., 0::2] = x[..., 0::2] * c - x[..., 1::2] * s
    y[..., 1::2] = x[..., 0::2] * s + x[..., 1::2] * c
    return y


def pair(x):
    a = np.abs(x)
    return (a[..., 0::2] + a[..., 1::2]).repeat(2, -1)


def forward64(x, w, pos, eps, theta):
    u = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    return turn(u, pos, theta), pair(u)


def backward64(x, w, dy, pos, eps, theta):
    """(dx, dw, sizes of dx's terms, sizes of dw's terms)"""
    d = x.shape[-1]
    g = turn(dy, pos, theta, True)
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    u, wg, size = x * r, w * g, pair(dy)
    dot = (wg * u).sum(-1, keepdims=True) / d
    some = (np.abs(w) * size * np.abs(u)).sum(-1, keepdims=True) / d
    return r * (wg - u * dot), (g * u).sum((0, 1)), r * (np.abs(w) * size + np.abs(u) * some), \
        (size * np.abs(u)).sum((0, 1))


def made(dtype, n, H, Hkv, D, seed=0):
    r = np.random.default_rng(seed)

    def t(*shape, size=1.0):
        return torch.from_numpy(size * r.standard_normal(shape)).to(TD[dtype])
    x = dict(q=t(n, H, D), k=t(n, max(Hkv, 1), D), gq=t(n, H, D), gk=t(n, max(Hkv, 1), D))
    x["wq"], x["wk"] = ((1 + 0.3 * torch.from_numpy(r.standard_normal(D))).to(TD[dtype]) for _ in range(2))
    if n > 2:
        x["q"][1] *= 1e-3                     # rows of other sizes, and one of zeros
        x["k"][2] = 0
    return x


CASES = [
    # dtype, rows, H, Hkv, D, theta, positions: None / offset / "given"
    ("bf16", 1, 32, 4, 64, 1e4, None),
    ("f32", 1, 32, 4, 64, 1e4, 77),
    ("bf16", 37, 6, 3, 64, 1e4, "given"),
    ("f32", 37, 5, 1, 64, 5e5, "given"),
    ("bf16", 333, 32, 4, 64, 0.0, None),
    ("bf16", 9, 4, 2, 128, 1e4, -5),
    ("f32", 9, 3, 3, 128, 1e4, "given"),
    ("bf16", 7, 2, 2, 256, 1e6, "given"),
    ("f32", 7, 1, 1, 256, 1e4, None),
    ("bf16", 50, 3, 1, 16, 1e4, "given"),
    ("f32", 50, 7, 2, 32, 1e4, "given"),
    ("bf16", 20, 8, 0, 64, 1e4, "given"),      # queries alone
    ("f32", 3000, 4, 2, 64, 1e4, None),        # several rows a workgroup
    ("bf16", 9001, 3, 1, 64, 1e4, "given"),
    ("bf16", 5, 300, 1, 32, 1e4, None),
]


def positions_of(how, n):
    if how == "given":
        p = np.random.default_rng(5).integers(-3, 1 << 20, n)
        p[0] = 2 ** 31 - 1
        return torch.from_numpy(p.astype(np.int32)).cuda(), 0, p
    off = how or 0
    return None, off, np.arange(n) + off


@pytest.mark.parametrize("place", ["new", "wide", "in place"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_forward(case, place):
    dtype, n, H, Hkv, D, theta, how = case
    print("norm", case, place, flush=True)
    x = made(dtype, n, H, Hkv, D)
    pos, off, p = positions_of(how, n)
    q, k = (wide(x[t].cuda(), 16)[0] for t in "qk")
    qo, qb = wide(torch.full_like(x["q"], 7.0).cuda(), 32, 7.0) if place == "wide" else (q if place == "in place" else None, None)
    ko = k if place == "in place" else None
    if not Hkv:
        k = ko = None
    got = B.qk_norm_rope(q, k, x["wq"].cuda(), x["wk"].cuda() if Hkv else None, 1e-5, positions=pos, position_offset=off,
                         theta=theta, q_out=qo, k_out=ko)
    half = torch.finfo(TD[dtype]).eps / 2
    for t, o in zip("qk", got):
        if o is None:
            assert t == "k" and not Hkv
            continue
        want, size = forward64(x[t].double().numpy(), x["w" + t].double().numpy(), p, 1e-5, theta)
        err = size * ((D / 2 + 20) * 2.0 ** -24)
        # a position's angle in the test is off by 2^31 2^-52 at most
        tol = err + size * 2.0 ** -20 * (dtype == "f32") + (np.abs(want) + err) * half
        offs = np.abs(host(o) - want)
        assert (offs <= tol).all(), (t, (offs - tol).max())
    if place == "wide":
        assert (host(qb)[:, :16] == 7.0).all() and (host(qb)[:, -16:] == 7.0).all()


@pytest.mark.parametrize("place", ["new", "of the gradients", "of the rows"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_backward(case, place):
    dtype, n, H, Hkv, D, theta, how = case
    print("norm backward", case, place, flush=True)
    x = made(dtype, n, H, Hkv, D, 1)
    pos, off, p = positions_of(how, n)
    q, k, gq, gk = (wide(x[t].cuda(), 16)[0] for t in ("q", "k", "gq", "gk"))
    dq, dk = {"new": (None, None), "of the gradients": (gq, gk), "of the rows": (q, k)}[place]
    if not Hkv:
        k = gk = dk = None
    ws = B.qk_norm_rope_workspace(n, H, Hkv, D)
    ws.fill_(255)
    got = B.qk_norm_rope_backward(q, k, x["wq"].cuda(), x["wk"].cuda() if Hkv else None, gq, gk, 1e-5, positions=pos,
                                  position_offset=off, theta=theta, dq=dq, dk=dk, workspace=ws if place == "new" else None)
    half = torch.finfo(TD[dtype]).eps / 2
    unit = (2 * D + 60) * 2.0 ** -24 + 2.0 ** -20 * (how == "given")
    for t, dx, dw, heads in (("q", got[0], got[2], H), ("k", got[1], got[3], Hkv)):
        if not heads:
            assert dx is None and dw is None
            continue
        want, want_w, size, size_w = backward64(x[t].double().numpy(), x["w" + t].double().numpy(),
                                                x["g" + t].double().numpy(), p, 1e-5, theta)
        tol = size * unit + (np.abs(want) + size * unit) * half
        offs = np.abs(host(dx) - want)
        assert (offs <= tol).all(), (t, (offs - tol).max())
        # a thread adds up every 256 / (D / 8)-th head's element in turn at most, then few sums of those
        depth = n * heads / (256 / (D / 8)) + 1024 / 32 + 30
        assert dw.dtype == torch.float32
        offs = np.abs(host(dw) - want_w)
        assert (offs <= size_w * (unit + depth * 2.0 ** -24)).all(), (t, offs.max())


def test_gradients_against_differences():
    """The formula's gradients in 64 bits against central differences, and the kernel's against those."""
    r = np.random.default_rng(2)
    n, H, D, eps, theta = 3, 2, 16, 1e-3, 1e4
    x, dy, w, pos = r.standard_normal((n, H, D)), r.standard_normal((n, H, D)), 1 + 0.3 * r.standard_normal(D), np.arange(n)
    x, dy, w = (a.astype(np.float32).astype(np.float64) for a in (x, dy, w))
    loss = lambda x, w: (forward64(x, w, pos, eps, theta)[0] * dy).sum()  # noqa: E731
    dx, dw, *_ = backward64(x, w, dy, pos, eps, theta)
    h = 1e-6
    num = np.zeros_like(x)
    for i in np.ndindex(x.shape):
        e = np.zeros_like(x)
        e[i] = h
        num[i] = (loss(x + e, w) - loss(x - e, w)) / (2 * h)
    # central differences: h^2 times third derivatives of order 10^2, and 2^-52 of the loss over h
    assert np.abs(num - dx).max() <= 1e-8 + 1e-7
    numw = np.array([(loss(x, w + h * (np.arange(D) == i)) - loss(x, w - h * (np.arange(D) == i))) / (2 * h) for i in range(D)])
    assert np.abs(numw - dw).max() <= 1e-8 + 1e-7
    t = lambda a: torch.from_numpy(a.astype(np.float32)).cuda()  # noqa: E731
    got = B.qk_norm_rope_backward(t(x), t(x), t(w), t(w), t(dy), t(dy), eps, theta=theta)
    for g in got[:2]:
        assert np.abs(host(g) - num).max() <= 1e-4
    for g in got[2:]:
        assert np.abs(host(g) - numw).max() <= 1e-4


@pytest.mark.parametrize("n", [0, 700, 9001])
def test_weights_gradients_are_the_same_every_time(n):
    x = made("bf16", n, 8, 2, 64, 3)
    a = [x[t].cuda() for t in ("q", "k", "wq", "wk", "gq", "gk")]
    first = B.qk_norm_rope_backward(*a)
    for _ in range(3):
        for g, f in zip(B.qk_norm_rope_backward(*a), first):
            assert torch.equal(g, f)
    if n == 0:
        assert (first[2] == 0).all() and (first[3] == 0).all()


@pytest.mark.parametrize("D,H,Hkv,sizes", [
    (64, 32, 4, [1, 1820, 129, 5000, 128, 1821, 700, 300]),  # sums added by the last workgroup and by another launch
    (256, 3, 1, [700, 3, 512, 9000, 513, 32, 33]),
    (16, 40, 1, [2048, 100, 2049, 8193, 5, 2000]),
])
def test_a_workspace_goes_from_call_to_call(D, H, Hkv, sizes):
    """One workspace, never cleared, for calls of other sizes behind each other: every call's gradients are
    those of a fresh workspace, and the weights' those of 64 bits."""
    ws = B.qk_norm_rope_workspace(max(sizes), H, Hkv, D)
    ws.fill_(0x5b)
    x = made("bf16", max(sizes), H, Hkv, D, 4)
    a = {t: x[t].cuda() for t in x}
    for n in sizes:
        print("workspace", D, n, flush=True)
        args = a["q"][:n], a["k"][:n], a["wq"], a["wk"], a["gq"][:n], a["gk"][:n]
        got = [B.qk_norm_rope_backward(*args, workspace=ws) for _ in range(3)]
        fresh = B.qk_norm_rope_backward(*args)
        for g in got:
            for u, v in zip(g, fresh):
                assert torch.equal(u, v), n
        for t, dw, heads in (("q", fresh[2], H), ("k", fresh[3], Hkv)):
            _, want, _, size = backward64(x[t][:n].double().numpy(), x["w" + t].double().numpy(), x["g" + t][:n].double().numpy(), np.arange(n),
                                          1e-5, 1e4)
            depth = n * heads / (256 / (D / 8)) + 1024 / 32 + 30
            assert (np.abs(host(dw) - want) <= size * ((2 * D + 60 + depth) * 2.0 ** -24)).all(), (n, t)


def test_infinite_and_nan_elements_stay_in_their_head():
    x = made("f32", 4, 3, 1, 64, 3)
    x["q"][1, 1, 7], x["q"][2, 0, 3] = float("nan"), float("inf")
    clean = made("f32", 4, 3, 1, 64, 3)
    q = B.qk_norm_rope(x["q"].cuda(), None, x["wq"].cuda(), None)[0]
    w = B.qk_norm_rope(clean["q"].cuda(), None, x["wq"].cuda(), None)[0]
    hit = torch.zeros(4, 3, dtype=torch.bool)
    hit[1, 1] = hit[2, 0] = True
    assert torch.equal(q.cpu()[~hit], w.cpu()[~hit])
    assert torch.isnan(q.cpu()[1, 1]).all() and torch.isnan(q.cpu()[2, 0, 2])


def test_a_graph_of_both_directions():
    n, H, Hkv, D = 300, 8, 2, 64
    x = made("bf16", n, H, Hkv, D)
    t = {m: v.cuda() for m, v in x.items()}
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    out = {m: torch.empty_like(t[m]) for m in ("q", "k", "gq", "gk")}
    ws = B.qk_norm_rope_workspace(n, H, Hkv)

    def both():
        B.qk_norm_rope(t["q"], t["k"], t["wq"], t["wk"], positions=pos, q_out=out["q"], k_out=out["k"])
        return B.qk_norm_rope_backward(t["q"], t["k"], t["wq"], t["wk"], t["gq"], t["gk"], positions=pos, dq=out["gq"],
                                       dk=out["gk"], workspace=ws)[2:]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        both()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            dw = both()
    for i in range(4):
        new = made("bf16", n, H, Hkv, D, 10 + i)
        for m in t:
            t[m].copy_(new[m])
        pos.add_(1000 * i)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out.values()] + [d.clone() for d in dw]
        want = list(B.qk_norm_rope(t["q"], t["k"], t["wq"], t["wk"], positions=pos)) + \
            list(B.qk_norm_rope_backward(t["q"], t["k"], t["wq"], t["wk"], t["gq"], t["gk"], positions=pos))
        for a, b in zip(got, want):
            assert torch.equal(a, b), i


def test_no_key_heads_give_a_key_weight_no_gradient():
    x = made("f32", 40, 8, 2, 64)
    a = {t: x[t].cuda() for t in x}
    none = a["k"][:, :0]
    q, k = B.qk_norm_rope(a["q"], none, a["wq"], a["wk"])
    torch.full((2, 64), 7.0, device="cuda")  # what the gradients' memory held before
    dq, dk, dwq, dwk = B.qk_norm_rope_backward(a["q"], none, a["wq"], a["wk"], a["gq"], none)
    alone = B.qk_norm_rope_backward(a["q"], None, a["wq"], None, a["gq"], None)
    assert k.shape == dk.shape == (40, 0, 64) and (dwk == 0).all()
    assert torch.equal(dq, alone[0]) and torch.equal(dwq, alone[2]) and alone[3] is None
    assert torch.equal(q, B.qk_norm_rope(a["q"], None, a["wq"], None)[0])


def test_on_a_given_stream():
    x = made("f32", 500, 8, 2, 64)
    a = [x[t].cuda() for t in ("q", "k", "wq", "wk", "gq", "gk")]
    want = [*B.qk_norm_rope(*a[:4]), *B.qk_norm_rope_backward(*a)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = [*B.qk_norm_rope(*a[:4], stream=side), *B.qk_norm_rope_backward(*a, stream=side)]
    torch.cuda.current_stream().wait_stream(side)
    for g, w in zip(got, want):
        assert torch.equal(g, w)


def test_a_training_step_through_the_attention():
    """Norm and rotation, attention, and both backward: the gradients of the projection's rows and of the
    weights against 64 bits."""
    Bn, S, H, Hkv, D = 1, 96, 8, 2, 64
    x = made("bf16", S, H, Hkv, D)
    r = np.random.default_rng(8)
    v, do = (torch.from_numpy(r.standard_normal((S, h, D))).bfloat16() for h in (Hkv, H))
    c = {m: t.cuda() for m, t in x.items()}
    qr, kr = B.qk_norm_rope(c["q"], c["k"], c["wq"], c["wk"])
    o, lse = B.gqa_prefill_lse(qr[None], kr[None], v.cuda()[None])
    dqr, dkr, dv = B.gqa_prefill_backward(qr[None], kr[None], v.cuda()[None], o, do.cuda()[None], lse)
    got = B.qk_norm_rope_backward(c["q"], c["k"], c["wq"], c["wk"], dqr[0], dkr[0])
    leaves = [x[t].double().requires_grad_() for t in ("q", "k", "wq", "wk")]

    def norm(t, w):
        u = t / (t.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w
        a = torch.arange(S, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
        z = torch.view_as_complex(u.reshape(*u.shape[:-1], D // 2, 2)) * torch.polar(torch.ones_like(a), a)[:, None]
        return torch.view_as_real(z).flatten(-2)
    q64, k64 = norm(leaves[0], leaves[2]), norm(leaves[1], leaves[3])
    s = torch.einsum("ihd,jhd->hij", q64, k64.repeat_interleave(H // Hkv, 1)) / 8
    s = s.masked_fill(torch.ones(S, S, dtype=torch.bool).triu(1), -np.inf)
    o64 = torch.einsum("hij,jhd->ihd", s.softmax(-1), v.double().repeat_interleave(H // Hkv, 1))
    (o64 * do.double()).sum().backward()
    for g, leaf in zip(got, leaves):
        # bf16 tensors and products on the way: each rounding 2^-8 of the sizes, of which some ten in a row
        off = (g.double().cpu() - leaf.grad).norm() / leaf.grad.norm()
        assert off <= 10 * 2.0 ** -8, off
