"""The paged KV cache's calls refuse on the host what they cannot take, before any device work
(made-up addresses, never dereferenced: no GPU needed)."""
import ctypes as C

import pytest
import torch

import bnhip as B

CACHE = dict(k=0x10000, v=0x20000, page_table=0x30000, seq_lens=0x40000, page_stride=4 * 16 * 64,
             head_stride=16 * 64, row_stride=64, table_stride=8, dtype=B.BN_BF16, batch=3, n_pages=24,
             max_pages=8, page_size=16, n_kv_heads=4, head_dim=64)


def cache(**kw):
    return B.BnPagedKV(*[{**CACHE, **kw}[n] for n, _ in B.BnPagedKV._fields_])


def append(c=None, k=0x1000, v=0x2000, q=0x3000, qo=0x4000, starts=0x5000, n=7, H=32, ks=2560, vs=2560,
           qs=2560, qos=2048, theta=1e4):
    c = cache() if c is None else c
    return B.status_of("bn_paged_append", C.byref(c) if c else None, k, v, q, qo, starts, n, H, ks, vs,
                       qs, qos, theta, None)


def decode(c=None, q=0x1000, o=0x2000, H=32, qs=2048, os=2048, scale=0.125, ws=None, wsb=0):
    c = cache() if c is None else c
    return B.status_of("bn_paged_decode", C.byref(c) if c else None, q, o, H, qs, os, scale, ws, wsb, None)


def prefill(c=None, q=0x1000, o=0x2000, starts=0x3000, n=7, H=32, qs=2048, os=2048, scale=0.125, ws=None,
            wsb=0):
    c = cache() if c is None else c
    return B.status_of("bn_paged_prefill", C.byref(c) if c else None, q, o, starts, n, H, qs, os, scale,
                       ws, wsb, None)


def shared(c=None, q=0x1000, o=0x2000, H=32, qs=2048, os=2048, scale=0.125, pages=0x3000, P=40, ws=None,
           wsb=0):
    c = cache() if c is None else c
    return B.status_of("bn_paged_decode_shared", C.byref(c) if c else None, q, o, H, qs, os, scale,
                       pages, P, ws, wsb, None)


CALLS = {"Paged append": append, "Paged decode": decode, "Paged prefill": prefill,
         "Paged decode (shared prefix)": shared}


@pytest.mark.parametrize("kw,status,msg", [
    (dict(dtype=B.BN_U32), B.BN_ERR_UNSUPPORTED, "dtype"),
    (dict(batch=-1), B.BN_ERR_SHAPE, "negative"),
    (dict(n_pages=-1), B.BN_ERR_SHAPE, "negative"),
    (dict(max_pages=-1), B.BN_ERR_SHAPE, "negative"),
    (dict(n_kv_heads=0), B.BN_ERR_SHAPE, "num_kv_heads"),
    (dict(head_dim=128), B.BN_ERR_UNSUPPORTED, "head_dim must be 64"),
    (dict(page_size=0), B.BN_ERR_UNSUPPORTED, "power of two"),
    (dict(page_size=24), B.BN_ERR_UNSUPPORTED, "power of two"),
    (dict(page_size=4), B.BN_ERR_UNSUPPORTED, "at least 8"),
    (dict(row_stride=(1 << 24) + 8), B.BN_ERR_UNSUPPORTED, "2^24"),
    (dict(page_size=-16), B.BN_ERR_UNSUPPORTED, "power of two"),
    (dict(page_size=1 << 21, max_pages=1), B.BN_ERR_UNSUPPORTED, "2^20"),
    (dict(page_size=1 << 25, max_pages=1, n_pages=1), B.BN_ERR_UNSUPPORTED, "2^20"),
    (dict(max_pages=1 << 27), B.BN_ERR_UNSUPPORTED, "2^30"),
    (dict(batch=(1 << 20) + 1), B.BN_ERR_SHAPE | B.BN_ERR_UNSUPPORTED, ""),
    (dict(row_stride=32), B.BN_ERR_INVALID_ARG, "strides"),
    (dict(row_stride=68), B.BN_ERR_INVALID_ARG, "strides"),
    (dict(head_stride=0), B.BN_ERR_INVALID_ARG, "strides"),
    (dict(page_stride=-4096), B.BN_ERR_INVALID_ARG, "strides"),
    (dict(page_stride=1 << 30), B.BN_ERR_UNSUPPORTED, "2^30"),
    (dict(table_stride=7), B.BN_ERR_SHAPE, "overlap"),
    (dict(k=0), B.BN_ERR_INVALID_ARG, "NULL"),
    (dict(v=0), B.BN_ERR_INVALID_ARG, "NULL"),
    (dict(page_table=0), B.BN_ERR_INVALID_ARG, "NULL"),
    (dict(seq_lens=0), B.BN_ERR_INVALID_ARG, "NULL"),
    (dict(k=0x10008), B.BN_ERR_UNSUPPORTED, "16-byte"),
    (dict(page_table=0x30002), B.BN_ERR_UNSUPPORTED, "4-byte"),
    (dict(seq_lens=0x40001), B.BN_ERR_UNSUPPORTED, "4-byte"),
])
@pytest.mark.parametrize("name", sorted(CALLS))
def test_cache_refusals(name, kw, status, msg):
    s, m = CALLS[name](cache(**kw))
    if "batch" in kw and kw["batch"] > 0:  # one row each: the row counts disagree first where they are given
        assert s in (B.BN_ERR_SHAPE, B.BN_ERR_UNSUPPORTED) and m.startswith(name + ":")
        return
    assert s == status, m
    assert m.startswith(name + ":") and msg in m, m


@pytest.mark.parametrize("name", sorted(CALLS))
def test_null_cache_and_empty_batch(name):
    s, m = CALLS[name](False)
    assert s == B.BN_ERR_INVALID_ARG and "cache is NULL" in m
    c = cache(batch=0, k=0, v=0, page_table=0, seq_lens=0)
    assert CALLS[name](c) == (B.BN_OK, "")


@pytest.mark.parametrize("call,kw,status,msg", [
    (append, dict(n=-1), B.BN_ERR_SHAPE, "negative number of rows"),
    (append, dict(n=(1 << 23) + 1), B.BN_ERR_UNSUPPORTED, "2^23 rows"),
    (append, dict(starts=None), B.BN_ERR_SHAPE, "one row per sequence"),
    (append, dict(starts=0x5002), B.BN_ERR_UNSUPPORTED, "row_starts"),
    (append, dict(q=None), B.BN_ERR_INVALID_ARG, "together"),
    (append, dict(qo=None), B.BN_ERR_INVALID_ARG, "together"),
    (append, dict(H=30), B.BN_ERR_SHAPE, "num_heads"),
    (append, dict(theta=-1.0), B.BN_ERR_INVALID_ARG, "theta"),
    (append, dict(theta=float("nan")), B.BN_ERR_INVALID_ARG, "theta"),
    (append, dict(theta=float("inf")), B.BN_ERR_INVALID_ARG, "theta"),
    (append, dict(k=None), B.BN_ERR_INVALID_ARG, "k is NULL"),
    (append, dict(v=None), B.BN_ERR_INVALID_ARG, "v is NULL"),
    (append, dict(ks=255), B.BN_ERR_SHAPE, "k row stride"),
    (append, dict(vs=260), B.BN_ERR_UNSUPPORTED, "v must be"),
    (append, dict(q=0x3004), B.BN_ERR_UNSUPPORTED, "q must be"),
    (append, dict(qos=2040), B.BN_ERR_SHAPE, "q_out row stride"),
    (append, dict(qo=0x3000), B.BN_ERR_INVALID_ARG, "in q's place"),
    (decode, dict(H=30), B.BN_ERR_SHAPE, "num_heads"),
    (decode, dict(H=0), B.BN_ERR_SHAPE, "num_heads"),
    (decode, dict(H=4 * 16384), B.BN_ERR_UNSUPPORTED, "65535"),
    (decode, dict(scale=0.0), B.BN_ERR_INVALID_ARG, "scale"),
    (decode, dict(scale=float("inf")), B.BN_ERR_INVALID_ARG, "scale"),
    (decode, dict(q=None), B.BN_ERR_INVALID_ARG, "q is NULL"),
    (decode, dict(o=None), B.BN_ERR_INVALID_ARG, "o is NULL"),
    (decode, dict(o=0x2008), B.BN_ERR_UNSUPPORTED, "o must be"),
    (decode, dict(qs=2044), B.BN_ERR_SHAPE, "q row stride"),
    (decode, dict(os=2052), B.BN_ERR_UNSUPPORTED, "o must be"),
    (decode, dict(ws=0x9008, wsb=1 << 40), B.BN_ERR_UNSUPPORTED, "workspace must be"),
    (prefill, dict(n=-3), B.BN_ERR_SHAPE, "negative number of rows"),
    (prefill, dict(starts=None), B.BN_ERR_SHAPE, "one row per sequence"),
    (prefill, dict(scale=-1.0), B.BN_ERR_INVALID_ARG, "scale"),
    (prefill, dict(q=0x1002), B.BN_ERR_UNSUPPORTED, "q must be"),
    (shared, dict(P=-1), B.BN_ERR_SHAPE, "prefix length"),
    (shared, dict(pages=None), B.BN_ERR_INVALID_ARG, "prefix_pages"),
    (shared, dict(pages=0x3001), B.BN_ERR_UNSUPPORTED, "prefix_pages"),
])
def test_argument_refusals(call, kw, status, msg):
    s, m = call(**kw)
    assert s == status, m
    assert msg in m, m


def test_no_rows_is_nothing_to_do():
    assert append(n=0) == (B.BN_OK, "")
    assert prefill(n=0) == (B.BN_OK, "")


def test_workspace_sizes():
    L = B.lib()
    c = cache()
    for n in (0, 1, 7, 1000):
        for P in (0, 1, 5000):
            need = L.bn_paged_workspace_size(C.byref(c), 32, n, P)
            assert need < 1 << 32
    for bad in (cache(dtype=B.BN_U32), cache(head_dim=32), cache(n_kv_heads=0), cache(page_size=3)):
        assert L.bn_paged_workspace_size(C.byref(bad), 32, 3, 0) == 0
    assert L.bn_paged_workspace_size(None, 32, 3, 0) == 0
    assert L.bn_paged_workspace_size(C.byref(c), 30, 3, 0) == 0
    assert L.bn_paged_workspace_size(C.byref(c), 32, -1, 0) == 0


@pytest.mark.parametrize("dtype", [B.BN_F32, B.BN_BF16])
def test_a_workspace_does_for_fewer_rows(dtype):
    L = B.lib()
    for pages, batch, hkv in ((8, 3, 2), (600, 3, 4), (1024, 70, 4), (4096, 1, 3), (9000, 5, 8)):
        c = cache(dtype=dtype, batch=batch, max_pages=pages, table_stride=pages, n_kv_heads=hkv)
        rows = sorted({n + d for n in (*range(0, 40), *(2 ** i * j for i in range(6, 15) for j in (4, 5, 6, 7)))
                       for d in (0, 1)})
        need = [L.bn_paged_workspace_size(C.byref(c), 8 * hkv, n, 0) for n in rows]
        assert need == sorted(need)
        need = [L.bn_paged_workspace_size(C.byref(c), 8 * hkv, batch, P)
                for P in (0, 1, 100, 1000, 4000, 5000, 16000, 17000, 30000, 60000, 140000) if P <= pages * 16]
        assert need == sorted(need)


def test_a_workspace_too_small_is_refused():
    L = B.lib()
    c = cache(batch=64, max_pages=1024, table_stride=1024, n_pages=4096)
    for call, P in ((decode, 0), (shared, 5000)):
        need = L.bn_paged_workspace_size(C.byref(c), 32, 64, P)
        if need:
            s, m = call(c, ws=0x9000, wsb=need - 1, **(dict(P=P) if P else {}))
            assert s == B.BN_ERR_INVALID_ARG and "workspace" in m


def test_python_wrappers_refuse():
    k = torch.zeros((5, 2, 16, 64), dtype=torch.bfloat16)
    table = torch.zeros((3, 4), dtype=torch.int32)
    lens = torch.zeros(3, dtype=torch.int32)
    kv = B.PagedKV(k, k.clone(), table, lens)
    assert kv.view.page_size == 16 and kv.view.n_kv_heads == 2 and kv.view.batch == 3
    for bad in (dict(v=k[:4]), dict(v=k.float()), dict(k=k.half(), v=k.half()), dict(table=table.long()),
                dict(lens=lens.long()), dict(lens=lens[:2]), dict(table=table[0]), dict(k=k[..., ::2], v=k[..., ::2]),
                dict(table=torch.zeros((3, 8), dtype=torch.int32)[:, ::2])):
        a = dict(k=k, v=k, table=table, lens=lens, **{})
        a.update(bad)
        with pytest.raises(ValueError, match="PagedKV"):
            B.PagedKV(a["k"], a["v"], a["table"], a["lens"])
    q = torch.zeros((3, 8, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="paged_decode: q"):
        B.paged_decode(q[:2], kv)
    with pytest.raises(ValueError, match="dtype"):
        B.paged_decode(q.float(), kv)
    with pytest.raises(ValueError, match="contiguous"):
        B.paged_decode(torch.zeros((3, 64, 8), dtype=torch.bfloat16).transpose(1, 2), kv)
    with pytest.raises(ValueError, match="paged_decode: o"):
        B.paged_decode(q, kv, o=q[:, :4])
    with pytest.raises(ValueError, match="one row per sequence"):
        B.paged_prefill(torch.zeros((7, 8, 64), dtype=torch.bfloat16), kv)
    with pytest.raises(ValueError, match="row_starts"):
        B.paged_prefill(q, kv, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="row_starts"):
        B.paged_prefill(q, kv, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError, match="prefix_pages"):
        B.paged_decode_shared(q, kv, torch.zeros(2, dtype=torch.int32), 33)
    with pytest.raises(ValueError, match="prefix_pages"):
        B.paged_decode_shared(q, kv, torch.zeros(2), 3)
    kn = torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="paged_append: k"):
        B.paged_append(kv, q, kn)
    with pytest.raises(ValueError, match="paged_append: v"):
        B.paged_append(kv, kn, kn[:2])
    with pytest.raises(ValueError, match="q_out without q"):
        B.paged_append(kv, kn, kn, q_out=q)


def test_python_wrappers_refuse_other_devices():
    from types import SimpleNamespace
    k = torch.zeros((5, 2, 16, 64), dtype=torch.bfloat16)
    kv = B.PagedKV(k, k.clone(), torch.zeros((3, 4), dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
    q = torch.zeros((3, 8, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="not on a GPU"):
        B.paged_decode(q, kv)
    with pytest.raises(ValueError, match="workspace"):
        B.paged_decode(q, kv, workspace=torch.empty(1 << 20, dtype=torch.uint8, device="meta"))
    with pytest.raises(ValueError, match="workspace"):
        B.paged_prefill(q, kv, workspace=torch.empty((1 << 10, 2), dtype=torch.uint8)[:, 0])
    kv.device = torch.device("cuda:0")  # what follows looks at the stream alone
    with pytest.raises(ValueError, match="stream"):
        B._cache_stream(kv, SimpleNamespace(device=torch.device("cuda:1"), cuda_stream=0))
    assert B._cache_stream(kv, SimpleNamespace(device=torch.device("cuda:0"), cuda_stream=7)) == 7


@pytest.mark.parametrize("call,c,kw", [
    (shared, dict(batch=1 << 20, max_pages=16, table_stride=16), dict(H=128, qs=8192, os=8192, P=200)),
    (shared, dict(batch=1 << 20, max_pages=16, table_stride=16, dtype=B.BN_F32), dict(H=512, qs=32768, os=32768, P=1)),
    (prefill, dict(batch=1 << 20, n_kv_heads=64), dict(n=1 << 20, H=64, qs=4096, os=4096)),
    (prefill, dict(batch=1, dtype=B.BN_F32), dict(n=1 << 25, H=32)),
    (prefill, dict(batch=1 << 20, dtype=B.BN_F32), dict(n=1 << 22, H=240, qs=16384, os=16384)),
], ids=["shared", "shared_fp32", "many_sequences", "many_rows_fp32", "both_fp32"])
def test_launches_past_32_bits_are_refused(call, c, kw):
    s, m = call(cache(**c), **kw)
    assert s == B.BN_ERR_UNSUPPORTED and "2^32 threads" in m, m


@pytest.mark.parametrize("call,c,kw", [
    (shared, dict(batch=1 << 20, max_pages=16, table_stride=16), dict(H=124, qs=8192, os=8192, P=200)),
    (prefill, dict(batch=1 << 20, n_kv_heads=4), dict(n=(1 << 22), H=32)),
    (prefill, dict(batch=1 << 20, n_kv_heads=4, dtype=B.BN_F32), dict(n=(1 << 22), H=32)),
    (prefill, dict(batch=1), dict(n=1 << 25, H=32)),
    (prefill, dict(batch=1, dtype=B.BN_F32), dict(n=(1 << 25) - (1 << 16), H=32)),
    (decode, dict(batch=1 << 20), dict(H=1020, qs=65536, os=65536)),
], ids=["shared", "many", "many_fp32", "rows", "rows_fp32", "decode"])
def test_large_calls_below_that_are_not(call, c, kw):
    s, m = call(cache(**c), **kw)      # past every check of the arguments: no device, or none of its memory
    assert s in (B.BN_ERR_HIP, B.BN_ERR_NOT_DEVICE), m


def test_too_many_kv_heads_are_refused():
    """Also in an append without queries, whose pieces of a row are counted in 32 bits."""
    for heads in (65536, 1 << 26, 1 << 30):
        s, m = append(cache(batch=1, n_kv_heads=heads), q=None, qo=None, n=1, ks=heads * 64, vs=heads * 64)
        assert s == B.BN_ERR_UNSUPPORTED and "65535" in m, m


def outputs_of(stream):
    """Every call of the binding that makes its outputs, with the given stream: {name: outputs}."""
    k = torch.zeros((5, 2, 16, 64), dtype=torch.bfloat16)
    kv = B.PagedKV(k, k.clone(), torch.zeros((3, 4), dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
    q3, st = torch.zeros((3, 8, 64), dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32)
    q, kc = torch.zeros((2, 6, 8, 64), dtype=torch.bfloat16), torch.zeros((2, 6, 2, 64), dtype=torch.bfloat16)
    x, w, lens = torch.zeros((3, 512)), torch.zeros((1, 512)), torch.zeros(2, dtype=torch.int32)
    lse = torch.zeros((2, 8, 6))
    return {
        "paged_decode": B.paged_decode(q3, kv, stream=stream),
        "paged_prefill": B.paged_prefill(q3, kv, st, stream=stream),
        "paged_decode_shared": B.paged_decode_shared(q3, kv, lens, 20, stream=stream),
        "gqa_prefill": B.gqa_prefill(q, kc, kc, stream=stream),
        "gqa_prefill_lse": B.gqa_prefill_lse(q, kc, kc, stream=stream),
        "gqa_prefill_backward": B.gqa_prefill_backward(q, kc, kc, q, q, lse, stream=stream),
        "gqa_decode": B.gqa_decode(q[:, 0].contiguous(), kc, kc, lens, stream=stream),
        "gqa_decode_planned": B.gqa_decode_planned(q[:, 0].contiguous(), kc, kc, lens, [0, 0], stream=stream),
        "fused_head_attention": B.fused_head_attention(x, x[:, :128], x[:, :128], 8, 2, stream=stream),
        "add_rmsnorm": B.add_rmsnorm(x, x, w, 1e-5, stream=stream),
        "silu_mul": B.silu_mul(x, x, stream=stream),
        "linear_rope": B.linear_rope(x, torch.zeros((512, 64)), stream=stream),
    }


def test_outputs_are_memory_of_the_stream_that_writes_them(monkeypatch):
    """A block that work of the present stream still uses is not the output of a call on another, and is not
    handed out again while either works on it."""
    import contextlib
    under, made, kept = [None], {}, {}

    @contextlib.contextmanager
    def on(stream):
        under.append(stream)
        yield
        under.pop()

    def tracked(make):
        def run(*a, **kw):
            t = make(*a, **kw)
            made[t.data_ptr()] = under[-1]
            return t
        return run

    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: "present")
    monkeypatch.setattr(torch, "empty_like", tracked(torch.empty_like))
    monkeypatch.setattr(torch, "empty", tracked(torch.empty))
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: kept.__setitem__(t.data_ptr(), s))
    monkeypatch.setattr(B, "call", lambda *a: None)
    monkeypatch.setattr(B, "stream_of", lambda s: s)
    monkeypatch.setattr(B, "_cache_stream", lambda cache, s: s)
    for stream, keeps in (("other", "present"), ("present", None), (None, None)):
        kept.clear()
        for name, out in outputs_of(stream).items():
            for t in out if isinstance(out, tuple) else (out,):
                assert made[t.data_ptr()] == stream, name
                assert kept.get(t.data_ptr()) == keeps, name
