"""CPU tests of the attention step over a cache in 8 bits: the C entry points and the ops refuse before any launch, schemas and
shapes.  No kernel runs here."""
import ctypes as C
import struct

import pytest
import torch

from exl3rocm import _lib, paged, paged8

P = C.c_void_p(0x1000)
ODD = C.c_void_p(0x1008)
FIELDS = ["k", "v", "k_scale", "v_scale", "k_ldp", "k_ldt", "k_ldh", "v_ldp", "v_ldt", "v_ldh", "ks_ldp", "ks_ldb", "ks_ldh", "vs_ldp", "vs_ldb",
          "vs_ldh", "pages", "page_size", "kv_heads", "head_dim"]


def cache(**k):
    c = dict(k=0x1000, v=0x1000, k_scale=0x1004, v_scale=0x1008, k_ldp=8192, k_ldt=128, k_ldh=4096, v_ldp=8192, v_ldt=128, v_ldh=4096, ks_ldp=4,
             ks_ldb=1, ks_ldh=2, vs_ldp=4, vs_ldb=1, vs_ldh=2, pages=8, page_size=32, kv_heads=2, head_dim=128)
    assert list(c) == FIELDS and set(k) <= set(c)
    c.update(k)
    return struct.pack("=16q4i", *c.values())


BAD_CACHES = [dict(k=0), dict(v=0), dict(k_scale=0), dict(v_scale=0), dict(k=0x1008), dict(v=0x1001), dict(k_scale=0x1002), dict(v_scale=0x1001),
              dict(k_ldp=8200), dict(k_ldt=120), dict(v_ldh=4104), dict(k_ldt=-128), dict(v_ldt=1 << 27), dict(ks_ldp=-1), dict(vs_ldb=-1), dict(ks_ldh=-2),
              dict(pages=-1), dict(pages=1 << 27), dict(page_size=0), dict(page_size=8), dict(page_size=40), dict(page_size=65552), dict(kv_heads=0),
              dict(kv_heads=1025), dict(head_dim=96), dict(head_dim=512)]


def attention(L, c=cache(), **k):
    a = dict(q=P, q_ldt=128, q_ldh=128, cache=c, table=P, ld=4, cols=4, cu=P, seq=P, out=P, o_ldt=128, o_ldh=128, tokens=2, requests=1, hq=4,
             scale=1.0, window=0, dtype=0, ws=P, nbytes=1 << 30, stream=None)
    a.update(k)
    return L.exl3_paged_attention8(*a.values())


def write(L, c=cache(), **k):
    a = dict(q=P, q_ldt=128, q_ldh=128, k=P, k_ldt=128, k_ldh=128, v=P, v_ldt=128, v_ldh=128, pos=P, slots=P, out=P, cache=c, inv=P, m=1.0, tokens=2,
             hq=4, rot=128, inter=0, dtype=1, stream=None)
    a.update(k)
    return L.exl3_rope_kv_write8(*a.values())


def read(L, c=cache(), **k):
    a = dict(cache=c, slots=P, k=P, v=P, tokens=2, dtype=1, stream=None)
    a.update(k)
    return L.exl3_kv_read8(*a.values())


def test_caches_are_refused():
    L = _lib.lib()
    for call in (attention, write, read):
        assert call(L, None) == _lib.EINVAL
        for bad in BAD_CACHES:
            assert call(L, cache(**bad)) == _lib.EINVAL, (call, bad)
        # an empty batch launches nothing; strides that address nothing may be anything
        assert call(L, cache(pages=1, k_ldp=3, vs_ldp=-9), tokens=0) == _lib.OK
        assert call(L, cache(kv_heads=1, k_ldh=3, ks_ldh=-1), tokens=0) == _lib.OK
        assert call(L, cache(page_size=16, ks_ldb=-1), tokens=0) == _lib.OK
        assert call(L, cache(pages=0, k=0, v_scale=0), tokens=0) == _lib.OK


def test_attention_refusals():
    L = _lib.lib()
    for bad in (dict(q=None), dict(table=None), dict(cu=None), dict(seq=None), dict(out=None), dict(q=ODD), dict(out=ODD), dict(q_ldt=4), dict(q_ldh=-8),
                dict(o_ldh=12), dict(hq=3), dict(hq=0), dict(hq=2048), dict(ld=3), dict(cols=-1, ld=0), dict(window=-1), dict(window=(1 << 30) + 1),
                dict(dtype=2), dict(tokens=-1), dict(requests=20000), dict(requests=-1), dict(tokens=1 << 23), dict(cols=1 << 27, ld=1 << 27)):
        assert attention(L, **bad) == _lib.EINVAL, bad
    assert attention(L, ws=None) == _lib.EWORKSPACE
    assert attention(L, ws=ODD) == _lib.EWORKSPACE
    assert attention(L, nbytes=L.exl3_paged_attention_workspace_size() - 1) == _lib.EWORKSPACE


def test_write_and_read_refusals():
    L = _lib.lib()
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(pos=None), dict(slots=None), dict(out=None), dict(inv=None), dict(q=ODD), dict(v=ODD),
                dict(out=ODD), dict(q_ldh=100), dict(k_ldt=-128), dict(v_ldh=12), dict(rot=3), dict(rot=130), dict(rot=-2), dict(hq=1), dict(hq=1025),
                dict(dtype=5), dict(tokens=-1), dict(tokens=1 << 23)):
        assert write(L, **bad) == _lib.EINVAL, bad
    for bad in (dict(slots=None), dict(k=None), dict(v=None), dict(k=ODD), dict(v=ODD), dict(dtype=2), dict(tokens=-1), dict(tokens=1 << 23)):
        assert read(L, **bad) == _lib.EINVAL, bad


# ---------------------------------------------------------------------------------------------
# the ops, on host tensors whose entry points are replaced
# ---------------------------------------------------------------------------------------------
@pytest.fixture
def called(monkeypatch):
    got = []
    for m in (paged, paged8):
        monkeypatch.setattr(m, "_gpu", lambda t, what: t.get_device())
    monkeypatch.setattr(paged, "_raw_stream", lambda gpu: 0)
    monkeypatch.setattr(paged, "_workspaces", {(-1, 0): torch.zeros(16, dtype=torch.uint8)})
    monkeypatch.setattr(paged8, "_entry", lambda name: lambda *a: got.append((name, a)) or 0)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: -1, raising=False)
    return got


def args():
    q, k = torch.zeros(5, 4, 64, dtype=torch.bfloat16), torch.zeros(5, 2, 64, dtype=torch.bfloat16)
    i = torch.zeros(5, dtype=torch.int64)
    return q, k, k.clone(), i, i, *paged8.new_cache8(3, 32, 2, 64, device="cpu"), torch.zeros(32, dtype=torch.float64)


def test_new_cache():
    kc, vc, ks, vs = paged8.new_cache8(3, 48, 2, 64, device="cpu")
    assert kc.shape == vc.shape == (3, 48, 2, 64) and ks.shape == vs.shape == (3, 3, 2)
    assert kc.stride() == (6144, 64, 3072, 1) and ks.stride() == (6, 1, 3)         # a page holds a head's tokens together
    assert kc.dtype is torch.int8 and ks.dtype is torch.float32
    for page in (8, 0, 24):
        with pytest.raises(RuntimeError, match="multiple of 16"):
            paged8.new_cache8(3, page, 2, 64, device="cpu")


def test_calls_reach_the_entry_points(called):
    q, k, v, pos, slots, kc, vc, ks, vs, f = args()
    c = struct.pack("=16q4i", kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), 4096, 64, 2048, 4096, 64, 2048, 4, 1, 2, 4, 1, 2, 3, 32, 2, 64)
    op = torch.ops.exl3rocm
    out = op.rope_kv_write8(q, k, v, pos, slots, kc, vc, ks, vs, f, 1.5, True)
    assert called.pop() == ("exl3_rope_kv_write8", (q.data_ptr(), 256, 64, k.data_ptr(), 128, 64, v.data_ptr(), 128, 64, pos.data_ptr(), slots.data_ptr(),
                                                    out.data_ptr(), c, f.data_ptr(), 1.5, 5, 4, 64, True, 1, 0))
    rk, rv = op.kv_read8(kc, vc, ks, vs, slots, torch.bfloat16)
    assert rk.shape == rv.shape == (5, 2, 64) and rk.dtype is torch.bfloat16
    assert called.pop() == ("exl3_kv_read8", (c, slots.data_ptr(), rk.data_ptr(), rv.data_ptr(), 5, 1, 0))
    assert op.kv_read8(kc, vc, ks, vs, slots)[0].dtype is torch.float16
    table, cu, seq = torch.zeros(2, 7, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    out = op.paged_attention8(q, kc, vc, ks, vs, table[:, :5], cu, seq, 0.25, 9)
    name, a = called.pop()
    assert name == "exl3_paged_attention8" and a[3] == c and out.shape == q.shape
    assert a[:3] + a[4:-3] == (q.data_ptr(), 256, 64, table.data_ptr(), 7, 5, cu.data_ptr(), seq.data_ptr(), out.data_ptr(), 256, 64, 5, 2, 4, 0.25, 9, 1)


def test_ops_refuse(called):
    q, k, v, pos, slots, kc, vc, ks, vs, f = args()
    cache4 = (kc, vc, ks, vs)
    table, cu, seq = torch.zeros(2, 7, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    op = torch.ops.exl3rocm
    wide = paged8.new_cache8(3, 32, 2, 128, device="cpu")
    bad_caches = [(kc.byte(), vc, ks, vs), (kc, vc.half(), ks, vs), (kc, vc[:2], ks, vs), (kc, vc, ks.double(), vs), (kc, vc, ks, vs.half()),
                  (kc, vc, ks[:, :1], vs), (kc, vc, ks, vs[..., :1]), (kc[..., :32], vc[..., :32], ks, vs), (kc[:, :24], vc[:, :24], ks, vs), (kc[0], vc[0], ks, vs),
                  (kc.transpose(2, 3).contiguous().transpose(2, 3), vc, ks, vs), (kc[:, :0], vc[:, :0], ks[:, :0], vs[:, :0])]
    for c in bad_caches:
        for call in (lambda: op.rope_kv_write8(q, k, v, pos, slots, *c, f), lambda: op.kv_read8(*c, slots), lambda: op.paged_attention8(q, *c, table, cu, seq, 1.0)):
            with pytest.raises(RuntimeError, match="exl3rocm: "):
                call()
    for bad in ((q.float(), k, v, pos, slots, *cache4, f), (q, k.half(), v, pos, slots, *cache4, f), (q[0], k, v, pos, slots, *cache4, f),
                (q, k[:4], v, pos, slots, *cache4, f), (q, k[:, :1], v[:, :1], pos, slots, *cache4, f), (q, k, v, pos[:4], slots, *cache4, f),
                (q, k, v, pos, slots.int(), *cache4, f), (q, k, v, pos, slots, *cache4, f.float()), (q, k, v, pos, slots, *wide, f),
                (q, k.transpose(1, 2).contiguous().transpose(1, 2), v, pos, slots, *cache4, f)):
        with pytest.raises(RuntimeError, match="rope_kv_write8"):
            op.rope_kv_write8(*bad)
    for bad in ((*cache4, slots.int()), (*cache4, slots, torch.float32)):
        with pytest.raises(RuntimeError, match="kv_read8"):
            op.kv_read8(*bad)
    for bad in ((q.float(), *cache4, table, cu, seq, 1.0), (q[0], *cache4, table, cu, seq, 1.0), (q[:, :3], *cache4, table, cu, seq, 1.0),
                (q, *wide, table, cu, seq, 1.0), (q, *cache4, table.long(), cu, seq, 1.0), (q, *cache4, table[:1], cu, seq, 1.0),
                (q, *cache4, table, cu[:2], seq, 1.0), (q, *cache4, table, cu, seq.long(), 1.0), (q, *cache4, table, cu, seq, 1.0, -1),
                (q, *cache4, table, cu, seq, 1.0, 1 << 31), (q[..., :32], *cache4, table, cu, seq, 1.0)):
        with pytest.raises(RuntimeError, match="paged_attention8"):
            op.paged_attention8(*bad)
    assert not called


def test_ops_refuse_cpu_tensors():
    q, k, v, pos, slots, *rest = args()
    op = torch.ops.exl3rocm
    with pytest.raises(RuntimeError, match="must be on a GPU"):
        op.rope_kv_write8(q, k, v, pos, slots, *rest)
    with pytest.raises(RuntimeError, match="must be on a GPU"):
        op.kv_read8(*rest[:4], slots)
    with pytest.raises(RuntimeError, match="must be on a GPU"):
        op.paged_attention8(q, *rest[:4], torch.zeros(1, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 1.0)


def test_schemas_say_what_is_written():
    op = torch.ops.exl3rocm
    written = lambda f: [a.name for a in f.default._schema.arguments if a.alias_info is not None and a.alias_info.is_write]  # noqa: E731
    assert written(op.rope_kv_write8) == ["k_cache", "v_cache", "k_scale", "v_scale"]
    assert written(op.kv_read8) == written(op.paged_attention8) == []


def test_fake_shapes():
    with torch._subclasses.FakeTensorMode():
        q, k, v, pos, slots, kc, vc, ks, vs, f = args()
        op = torch.ops.exl3rocm
        assert op.rope_kv_write8(q, k, v, pos, slots, kc, vc, ks, vs, f).shape == q.shape
        a, b = op.kv_read8(kc, vc, ks, vs, slots[:3], torch.bfloat16)
        assert a.shape == b.shape == (3, 2, 64) and a.dtype is torch.bfloat16
        o = op.paged_attention8(q, kc, vc, ks, vs, torch.zeros(3, 9, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), 0.1, 7)
        assert o.shape == q.shape and o.dtype is torch.bfloat16
