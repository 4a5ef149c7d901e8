"""The 8-bit paged cache's calls and the norms of single heads refuse on the host what they cannot take,
before any device work (made-up addresses, never dereferenced: no GPU needed)."""
import ctypes as C

import pytest
import torch

import bnhip as B

CACHE = dict(k=0x10000, v=0x20000, k_scale=0x50001, v_scale=0x60003, page_table=0x30000, seq_lens=0x40000,
             page_stride=4 * 16 * 64, head_stride=16 * 64, row_stride=64, scale_page_stride=4, scale_head_stride=1,
             table_stride=8, batch=3, n_pages=24, max_pages=8, page_size=16, n_kv_heads=4, head_dim=64)


def cache(**kw):
    return B.BnPagedQ8(*[{**CACHE, **kw}[n] for n, _ in B.BnPagedQ8._fields_])


def ref(c):
    c = cache() if c is None else c
    return C.byref(c) if c else None


def append(c=None, dtype=B.BN_BF16, k=0x1000, v=0x2000, q=0x3000, qo=0x4000, starts=0x5000, n=7, H=32, ks=2560, vs=2560,
           qs=2560, qos=2048, theta=1e4, wq=0x6000, wk=0x7000, eps=1e-5):
    return B.status_of("bn_paged_q8_append", ref(c), dtype, k, v, q, qo, starts, n, H, ks, vs, qs, qos, theta, wq, wk,
                       eps, None)


def read(c=None, dtype=B.BN_BF16, k=0x1000, v=0x2000, starts=0x5000, n=7, ks=256, vs=512):
    return B.status_of("bn_paged_q8_read", ref(c), dtype, k, v, starts, n, ks, vs, None)


def decode(c=None, dtype=B.BN_BF16, q=0x1000, o=0x2000, H=32, qs=2048, os=2048, scale=0.125, ws=None, wsb=0):
    return B.status_of("bn_paged_q8_decode", ref(c), dtype, q, o, H, qs, os, scale, ws, wsb, None)


def prefill(c=None, dtype=B.BN_BF16, q=0x1000, o=0x2000, starts=0x3000, n=7, H=32, qs=2048, os=2048, scale=0.125,
            ws=None, wsb=0):
    return B.status_of("bn_paged_q8_prefill", ref(c), dtype, q, o, starts, n, H, qs, os, scale, ws, wsb, None)


CALLS = {"Paged Q8 append": append, "Paged Q8 read": read, "Paged Q8 decode": decode, "Paged Q8 prefill": prefill}
INVALID, SHAPE, UNSUPPORTED = B.BN_ERR_INVALID_ARG, B.BN_ERR_SHAPE, B.BN_ERR_UNSUPPORTED


@pytest.mark.parametrize("kw,status,msg", [
    (dict(n_pages=-1), SHAPE, "negative"),
    (dict(max_pages=-1), SHAPE, "negative"),
    (dict(n_kv_heads=0), SHAPE, "num_kv_heads"),
    (dict(n_kv_heads=65536), UNSUPPORTED, "65535"),
    (dict(head_dim=128), UNSUPPORTED, "head_dim must be 64"),
    (dict(page_size=8), UNSUPPORTED, "at least 16"),
    (dict(page_size=24), UNSUPPORTED, "power of two"),
    (dict(page_size=1 << 21, max_pages=1), UNSUPPORTED, "2^20"),
    (dict(max_pages=1 << 27), UNSUPPORTED, "2^30"),
    (dict(row_stride=(1 << 24) + 16), UNSUPPORTED, "2^24"),
    (dict(row_stride=48), INVALID, "strides"),
    (dict(row_stride=72), INVALID, "strides"),
    (dict(page_stride=1 << 30), UNSUPPORTED, "2^30"),
    (dict(table_stride=7), SHAPE, "overlap"),
    (dict(k=0), INVALID, "NULL"),
    (dict(v_scale=0), INVALID, "NULL"),
    (dict(seq_lens=0), INVALID, "NULL"),
    (dict(k=0x10008), UNSUPPORTED, "16-byte"),
    (dict(page_table=0x30002), UNSUPPORTED, "4-byte"),
    (dict(scale_page_stride=0), INVALID, "scale strides"),
    (dict(scale_head_stride=0), INVALID, "scale strides"),
    (dict(scale_head_stride=-1), INVALID, "scale strides"),
    (dict(page_size=64, scale_head_stride=3), INVALID, "scale strides"),
])
@pytest.mark.parametrize("name", sorted(CALLS))
def test_cache_refusals(name, kw, status, msg):
    s, m = CALLS[name](cache(**kw))
    assert s == status and m.startswith(name + ":") and msg in m, m


@pytest.mark.parametrize("name", sorted(CALLS))
def test_null_cache_and_empty_batch(name):
    s, m = CALLS[name](False)
    assert s == INVALID and "cache is NULL" in m
    c = cache(batch=0, k=0, v=0, k_scale=0, v_scale=0, page_table=0, seq_lens=0)
    assert CALLS[name](c) == (B.BN_OK, "")


@pytest.mark.parametrize("call,kw,status,msg", [
    (append, dict(dtype=B.BN_U32), UNSUPPORTED, "dtype"),
    (append, dict(n=-1), SHAPE, "negative number of rows"),
    (append, dict(n=(1 << 23) + 1), UNSUPPORTED, "2^23 rows"),
    (append, dict(starts=None), SHAPE, "one row per sequence"),
    (append, dict(starts=0x5002), UNSUPPORTED, "row_starts"),
    (append, dict(q=None, wq=None), INVALID, "together"),
    (append, dict(qo=None), INVALID, "together"),
    (append, dict(q=None, qo=None), INVALID, "q_weight without q"),
    (append, dict(H=30), SHAPE, "num_heads"),
    (append, dict(theta=-1.0), INVALID, "theta"),
    (append, dict(theta=float("nan")), INVALID, "theta"),
    (append, dict(eps=-1.0), INVALID, "eps"),
    (append, dict(eps=float("inf")), INVALID, "eps"),
    (append, dict(wk=0x7008), UNSUPPORTED, "weights"),
    (append, dict(k=None), INVALID, "k is NULL"),
    (append, dict(v=None), INVALID, "v is NULL"),
    (append, dict(ks=255), SHAPE, "k row stride"),
    (append, dict(vs=260), UNSUPPORTED, "v must be"),
    (append, dict(q=0x3004), UNSUPPORTED, "q must be"),
    (append, dict(qos=2040), SHAPE, "q_out row stride"),
    (append, dict(qo=0x3000), INVALID, "in q's place"),
    (read, dict(dtype=7), UNSUPPORTED, "dtype"),
    (read, dict(n=-1), SHAPE, "negative number of rows"),
    (read, dict(n=(1 << 23) + 1), UNSUPPORTED, "2^23 rows"),
    (read, dict(starts=None), SHAPE, "one row per sequence"),
    (read, dict(k=None, v=None), INVALID, "k and v are NULL"),
    (read, dict(ks=255), SHAPE, "k row stride"),
    (read, dict(k=None, vs=252), SHAPE, "v row stride"),
    (read, dict(v=0x2008), UNSUPPORTED, "v must be"),
    (decode, dict(dtype=B.BN_U32), UNSUPPORTED, "dtype"),
    (decode, dict(H=30), SHAPE, "num_heads"),
    (decode, dict(H=4 * 16384), UNSUPPORTED, "65535"),
    (decode, dict(scale=0.0), INVALID, "scale"),
    (decode, dict(scale=float("inf")), INVALID, "scale"),
    (decode, dict(q=None), INVALID, "q is NULL"),
    (decode, dict(o=0x2008), UNSUPPORTED, "o must be"),
    (decode, dict(os=2047), SHAPE, "o row stride"),
    (prefill, dict(dtype=B.BN_U32), UNSUPPORTED, "dtype"),
    (prefill, dict(starts=None), SHAPE, "one row per sequence"),
    (prefill, dict(n=-2), SHAPE, "negative number of rows"),
    (prefill, dict(n=(1 << 26)), UNSUPPORTED, "2^30"),
    (prefill, dict(qs=2052), UNSUPPORTED, "q must be"),
])
def test_argument_refusals(call, kw, status, msg):
    s, m = call(**kw)
    assert s == status and msg in m, m


def test_no_rows_is_nothing_to_do():
    assert append(n=0, k=None, v=None) == (B.BN_OK, "")
    assert read(n=0, k=None, v=None) == (B.BN_OK, "")
    assert prefill(n=0, q=None, o=None) == (B.BN_OK, "")


def test_a_workspace_too_small_is_refused():
    c = cache(max_pages=4096, table_stride=4096, n_pages=20000)
    for call, n in ((decode, 3), (prefill, 700)):
        need = B.lib().bn_paged_q8_workspace_size(C.byref(c), 32, n)
        if need:
            s, m = call(c, ws=0x10000, wsb=need - 1, **({} if call is decode else dict(n=n)))
            assert s == INVALID and "workspace" in m
            s, m = call(c, ws=0x10008, wsb=need, **({} if call is decode else dict(n=n)))
            assert s == UNSUPPORTED and "16-byte" in m
    assert B.lib().bn_paged_q8_workspace_size(None, 32, 3) == 0
    assert B.lib().bn_paged_q8_workspace_size(C.byref(cache(page_size=8)), 32, 3) == 0


@pytest.mark.parametrize("batch,hkv,heads,keys", [(1, 4, 32, 4096), (7, 4, 32, 4096), (7, 4, 32, 40000), (64, 8, 64, 1 << 20),
                                                  (2, 1, 4, 16384), (300, 3, 15, 500)])
def test_a_workspace_does_for_fewer_rows(batch, hkv, heads, keys):
    c = cache(batch=batch, n_kv_heads=hkv, max_pages=-(-keys // 16), table_stride=-(-keys // 16), n_pages=1 << 21)
    rows = sorted({*range(1, 400), *range(400, 40000, 97), *range(1100 * 128 // heads, 1300 * 128 // heads)})
    need = [B.lib().bn_paged_q8_workspace_size(C.byref(c), heads, n) for n in rows]
    assert need[0] > 0 and all(a <= b for a, b in zip(need, need[1:]))


# ------------------------------------------------- norms of single heads
def norm(dtype=B.BN_BF16, q=0x1000, k=0x2000, wq=0x3000, wk=0x4000, qo=0x5000, ko=0x6000, pos=0x7000, n=5, H=8, Hkv=2, D=64,
         qs=512, ks=512, qos=512, kos=128, offset=0, eps=1e-5, theta=1e4):
    return B.status_of("bn_qk_norm_rope", dtype, q, k, wq, wk, qo, ko, pos, n, H, Hkv, D, qs, ks, qos, kos, offset, eps,
                       theta, None)


def back(dtype=B.BN_BF16, q=0x1000, k=0x2000, wq=0x3000, wk=0x4000, gq=0x5000, gk=0x6000, dq=0x8000, dk=0x9000, dwq=0xa004,
         dwk=0xb000, pos=0x7000, n=5, H=8, Hkv=2, D=64, qs=512, ks=512, gqs=512, gks=128, dqs=512, dks=128, offset=0,
         eps=1e-5, theta=1e4, ws=None, wsb=0):
    return B.status_of("bn_qk_norm_rope_backward", dtype, q, k, wq, wk, gq, gk, dq, dk, dwq, dwk, pos, n, H, Hkv, D, qs,
                       ks, gqs, gks, dqs, dks, offset, eps, theta, ws, wsb, None)


@pytest.mark.parametrize("kw,status,msg", [
    (dict(dtype=B.BN_U32), UNSUPPORTED, "dtype"),
    (dict(n=-1), SHAPE, "negative number of rows"),
    (dict(n=(1 << 23) + 1), UNSUPPORTED, "2^23"),
    (dict(H=0), SHAPE, "num_heads"),
    (dict(Hkv=-1), SHAPE, "num_kv_heads"),
    (dict(H=65536, qs=1 << 23), UNSUPPORTED, "65535"),
    (dict(D=48), UNSUPPORTED, "head_dim"),
    (dict(D=8), UNSUPPORTED, "head_dim"),
    (dict(D=512), UNSUPPORTED, "head_dim"),
    (dict(eps=-1e-5), INVALID, "eps"),
    (dict(eps=float("nan")), INVALID, "eps"),
    (dict(theta=float("inf")), INVALID, "theta"),
    (dict(k=None), INVALID, "together"),
    (dict(Hkv=0), INVALID, "together"),
    (dict(wq=None), INVALID, "weight is NULL"),
    (dict(wk=None), INVALID, "weight is NULL"),
    (dict(wq=0x3008), UNSUPPORTED, "weights"),
    (dict(q=None), INVALID, "q is NULL"),
    (dict(qs=511), SHAPE, "q row stride"),
    (dict(ks=516), UNSUPPORTED, "k must be"),
    (dict(pos=0x7002), UNSUPPORTED, "positions"),
])
@pytest.mark.parametrize("call", [norm, back])
def test_norm_refusals(call, kw, status, msg):
    s, m = call(**kw)
    assert s == status and m.startswith("QK norm") and msg in m, m


@pytest.mark.parametrize("call,kw,status,msg", [
    (norm, dict(qo=None), INVALID, "q_out is NULL"),
    (norm, dict(ko=0x6008), UNSUPPORTED, "k_out must be"),
    (norm, dict(qo=0x1000, qos=1024), INVALID, "in its input's place"),
    (back, dict(gq=None), INVALID, "dq_out is NULL"),
    (back, dict(dk=None), INVALID, "dk is NULL"),
    (back, dict(dwq=None), INVALID, "gradient of a weight"),
    (back, dict(dwk=None), INVALID, "gradient of a weight"),
    (back, dict(dwq=0xa002), UNSUPPORTED, "4-byte"),
    (back, dict(dq=0x5000, dqs=1024), INVALID, "in an input's place"),
    (back, dict(ws=0x10000, wsb=16), INVALID, "workspace of"),
    (back, dict(ws=0x10008, wsb=1 << 20), UNSUPPORTED, "workspace must be"),
])
def test_norm_argument_refusals(call, kw, status, msg):
    s, m = call(**kw)
    assert s == status and msg in m, m


def test_norm_of_no_rows():
    assert norm(n=0, q=None, k=None, qo=None, ko=None) == (B.BN_OK, "")


# ------------------------------------------------- the binding
def q8(**kw):
    t = dict(k=torch.zeros((5, 2, 32, 64), dtype=torch.uint8), s=torch.zeros((5, 2, 2), dtype=torch.uint8),
             table=torch.zeros((3, 4), dtype=torch.int32), lens=torch.zeros(3, dtype=torch.int32))
    t.update(kw)
    return B.PagedQ8(t["k"], t.get("v", t["k"]), t["s"], t.get("vs", t["s"]), t["table"], t["lens"])


def test_python_wrappers_refuse():
    kv = q8()
    assert kv.view.page_size == 32 and kv.view.n_kv_heads == 2 and kv.view.batch == 3
    k = torch.zeros((5, 2, 32, 64), dtype=torch.uint8)
    s = torch.zeros((5, 2, 2), dtype=torch.uint8)
    kv8 = q8(k=k.view(torch.float8_e4m3fn), s=s.view(torch.float8_e8m0fnu))
    assert kv8.view.scale_page_stride == 4 and kv8.view.scale_head_stride == 2
    for bad in (dict(v=k[:4]), dict(k=k.bfloat16()), dict(v=k.view(torch.float8_e4m3fn)), dict(k=k[:, :, :24]),
                dict(s=s[:, :1]), dict(s=s.int()), dict(vs=s.view(torch.float8_e8m0fnu)),
                dict(s=torch.zeros((5, 2, 4), dtype=torch.uint8)[..., ::2]), dict(table=torch.zeros((3, 4))),
                dict(lens=torch.zeros(2, dtype=torch.int32)), dict(k=k[..., ::2])):
        with pytest.raises(ValueError, match="PagedQ8"):
            q8(**bad)
    q = torch.zeros((3, 8, 64), dtype=torch.bfloat16)
    kn = q[:, :2].contiguous()
    for call, match in (
            (lambda: B.paged_q8_decode(q[:2], kv), "paged_q8_decode: q"),
            (lambda: B.paged_q8_decode(q.half(), kv), "float32 or bfloat16"),
            (lambda: B.paged_q8_decode(q, kv, o=q[:, :4]), "paged_q8_decode: o"),
            (lambda: B.paged_q8_decode(q, kv, o=q.float()), "paged_q8_decode: o"),
            (lambda: B.paged_q8_prefill(torch.zeros((7, 8, 64), dtype=torch.bfloat16), kv), "one row per sequence"),
            (lambda: B.paged_q8_prefill(q, kv, torch.zeros(3, dtype=torch.int32)), "row_starts"),
            (lambda: B.paged_q8_append(kv, q, kn), "paged_q8_append: k"),
            (lambda: B.paged_q8_append(kv, kn, kn.float()), "paged_q8_append: v"),
            (lambda: B.paged_q8_append(kv, kn.half(), kn), "float32 or bfloat16"),
            (lambda: B.paged_q8_append(kv, kn, kn, q_out=q), "q_out without q"),
            (lambda: B.paged_q8_append(kv, kn, kn, k_weight=torch.zeros(64)), "k_weight"),
            (lambda: B.paged_q8_append(kv, kn, kn, q=q, q_weight=torch.zeros(32, dtype=torch.bfloat16)), "q_weight"),
            (lambda: B.paged_q8_append(kv, kn, kn), "not on a GPU"),
            (lambda: B.paged_q8_read(kv, torch.zeros(4, dtype=torch.int32)), "n_rows"),
            (lambda: B.paged_q8_read(kv, k=kn[:2]), "one row per sequence"),
            (lambda: B.paged_q8_read(kv, k=kn, v=kn.float()), "paged_q8_read: v"),
            (lambda: B.paged_q8_decode(q, kv, workspace=torch.empty(1 << 20, dtype=torch.uint8, device="meta")),
             "workspace"),
            (lambda: B.qk_norm_rope(q, kn, q[0, 0], None), "together"),
            (lambda: B.qk_norm_rope(q, kn, q[0, 0], q[0, 0, :32]), "k_weight"),
            (lambda: B.qk_norm_rope(q.half(), None, q[0, 0].half(), None), "float32 or bfloat16"),
            (lambda: B.qk_norm_rope(q, None, q[0, 0], None, positions=torch.zeros(3)), "positions"),
            (lambda: B.qk_norm_rope(q, None, q[0, 0], None), "not on a GPU")):
        with pytest.raises(ValueError, match=match):
            call()


def test_outputs_are_memory_of_the_stream_that_writes_them(monkeypatch):
    """The binding makes a call's outputs under the stream that it is given."""
    made = []
    monkeypatch.setattr(B, "made_on", lambda stream, make: made.append(stream) or make())
    monkeypatch.setattr(B, "call", lambda *a: None)
    monkeypatch.setattr(B, "_cache_stream", lambda cache, stream: 0)
    monkeypatch.setattr(B, "_qk_args", lambda op, q, *a: (B.BN_BF16, 0, None, 0, 0, *q.shape[:2], (q.shape[2], q.dtype, q.device)))
    kv, st, q = q8(), object(), torch.zeros((3, 8, 64), dtype=torch.bfloat16)
    starts = torch.zeros(4, dtype=torch.int32)
    for call, n in ((lambda: B.paged_q8_decode(q, kv, stream=st), 1),
                    (lambda: B.paged_q8_prefill(q, kv, starts, stream=st), 1),
                    (lambda: B.paged_q8_read(kv, starts, n_rows=3, stream=st), 2),
                    (lambda: B.qk_norm_rope(q, q, q[0, 0], q[0, 0], stream=st), 2),
                    (lambda: B.qk_norm_rope_backward(q, q, q[0, 0], q[0, 0], q, q, stream=st), 3)):
        made.clear()
        call()
        assert made == [st] * n


@pytest.mark.parametrize("H,Hkv,D", [(32, 4, 64), (3, 1, 256), (40, 0, 16), (64, 8, 128)])
def test_a_workspace_of_the_norms_does_for_fewer_rows(H, Hkv, D):
    need = [B.lib().bn_qk_norm_rope_backward_workspace_size(n, H, Hkv, D) for n in [*range(0, 3000), 8191, 8192, 1 << 23]]
    assert need[1] > 0 and all(a <= b for a, b in zip(need, need[1:]))
