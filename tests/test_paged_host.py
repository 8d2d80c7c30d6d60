"""CPU tests of the paged attention step: the C entry points refuse before any launch, the rotary frequencies, the ops'
schemas and shapes.  No kernel runs here."""
import ctypes as C
import math

import pytest
import torch

from exl3rocm import _lib, paged

P = C.c_void_p(0x1000)
ODD = C.c_void_p(0x1008)


def attention(L, **k):
    a = dict(q=P, q_ldt=128, q_ldh=128, kc=P, k_ldp=2048, k_ldt=128, k_ldh=128, vc=P, v_ldp=2048, v_ldt=128, v_ldh=128, table=P, ld=4, cols=4,
             cu=P, seq=P, out=P, o_ldt=128, o_ldh=128, tokens=2, requests=1, hq=2, hkv=1, d=128, pages=8, page=16, scale=1.0, window=0, dtype=0,
             ws=P, nbytes=1 << 30, stream=None)
    a.update(k)
    return L.exl3_paged_attention(*a.values())


def test_attention_refusals():
    L = _lib.lib()
    assert attention(L, tokens=0) == _lib.OK                           # an empty batch launches nothing
    for bad in (dict(q=None), dict(kc=None), dict(vc=None), dict(table=None), dict(cu=None), dict(seq=None), dict(out=None), dict(q=ODD), dict(kc=ODD),
                dict(out=ODD), dict(q_ldt=4), dict(k_ldt=132), dict(v_ldp=2047), dict(k_ldt=1 << 27), dict(d=96), dict(d=80), dict(hq=3, hkv=2), dict(hkv=0),
                dict(page=8), dict(page=40), dict(page=0), dict(pages=-1), dict(pages=1 << 28), dict(ld=3), dict(cols=-1, ld=0), dict(window=-1),
                dict(window=(1 << 30) + 1), dict(dtype=2), dict(tokens=-1), dict(requests=20000), dict(hq=2048, hkv=2), dict(cols=1 << 27, ld=1 << 27)):
        assert attention(L, **bad) == _lib.EINVAL, bad
    assert attention(L, ws=None) == _lib.EWORKSPACE
    assert attention(L, ws=ODD) == _lib.EWORKSPACE
    assert attention(L, nbytes=L.exl3_paged_attention_workspace_size() - 1) == _lib.EWORKSPACE


def rope(L, **k):
    a = dict(q=P, q_ldt=128, q_ldh=128, k=P, k_ldt=128, k_ldh=128, v=P, v_ldt=128, v_ldh=128, pos=P, slots=P, out=P, kc=P, kc_ldp=4096, kc_ldt=256,
             kc_ldh=128, vc=P, vc_ldp=4096, vc_ldt=256, vc_ldh=128, inv=P, m=1.0, tokens=2, hq=4, hkv=2, d=128, rot=128, inter=0, pages=4, page=16, dtype=1,
             stream=None)
    a.update(k)
    return L.exl3_rope_kv_write(*a.values())


def test_rope_refusals():
    L = _lib.lib()
    assert rope(L, tokens=0) == _lib.OK
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(pos=None), dict(slots=None), dict(out=None), dict(kc=None), dict(vc=None), dict(inv=None),
                dict(q=ODD), dict(vc=ODD), dict(q_ldh=100), dict(k_ldt=-128), dict(kc_ldh=12), dict(rot=3), dict(rot=130), dict(rot=-2), dict(d=72),
                dict(hkv=0), dict(hq=1, hkv=2), dict(pages=1 << 27, page=32), dict(page=0), dict(dtype=5), dict(tokens=-1), dict(tokens=1 << 23)):
        assert rope(L, **bad) == _lib.EINVAL, bad


def plan(L, **k):
    a = dict(ctx=P, new=P, table=P, ld=4, cols=4, free=P, n_free=8, count=P, cu=P, seq=P, pos=P, slots=P, left=P, requests=2, page=16, tokens=4, stream=None)
    a.update(k)
    return L.exl3_batch_plan(*a.values())


def test_plan_refusals():
    L = _lib.lib()
    for bad in (dict(ctx=None), dict(new=None), dict(table=None), dict(free=None), dict(count=None), dict(cu=None), dict(seq=None), dict(pos=None),
                dict(slots=None), dict(left=None), dict(ld=3), dict(cols=-1), dict(n_free=-1), dict(requests=-1), dict(requests=16385), dict(page=0),
                dict(page=65537), dict(tokens=-1), dict(tokens=(1 << 22) + 1)):
        assert plan(L, **bad) == _lib.EINVAL, bad


def test_workspace_size_and_limits():
    L = _lib.lib()
    assert 2048 < L.exl3_paged_attention_workspace_size() < 80 << 20


def test_ops_refuse_cpu_tensors():
    q = torch.zeros(1, 2, 64, dtype=torch.float16)
    i = torch.zeros(1, dtype=torch.int32)
    kc = torch.zeros(2, 16, 1, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="must be on a GPU"):
        torch.ops.exl3rocm.paged_attention(q, kc, kc, i[None], torch.zeros(2, dtype=torch.int32), i, 1.0)
    with pytest.raises(RuntimeError, match="must be on a GPU"):
        torch.ops.exl3rocm.rope_kv_write(q, q[:, :1], q[:, :1], i.long(), i.long(), kc, kc, torch.zeros(32, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="must be on a GPU"):
        torch.ops.exl3rocm.batch_plan(i, i, i[None], i, i, 16, 1)


def test_schemas_say_what_is_written():
    s = torch.ops.exl3rocm.rope_kv_write.default._schema
    assert [a.name for a in s.arguments if a.alias_info is not None and a.alias_info.is_write] == ["k_cache", "v_cache"]
    s = torch.ops.exl3rocm.batch_plan.default._schema
    assert [a.name for a in s.arguments if a.alias_info is not None and a.alias_info.is_write] == ["block_table"]
    s = torch.ops.exl3rocm.paged_attention.default._schema
    assert not any(a.alias_info is not None for a in s.arguments)


def test_fake_shapes():
    with torch._subclasses.FakeTensorMode():
        i = torch.zeros(3, dtype=torch.int32)
        cu, seq, pos, slots, left = torch.ops.exl3rocm.batch_plan(i, i, torch.zeros(3, 9, dtype=torch.int32), i, i[:1], 16, 20)
        assert [tuple(t.shape) for t in (cu, seq, pos, slots, left)] == [(4,), (3,), (20,), (20,), (1,)]
        assert pos.dtype == slots.dtype == torch.int64 and cu.dtype == torch.int32
        q, kc = torch.zeros(20, 4, 64, dtype=torch.bfloat16), torch.zeros(5, 16, 2, 64, dtype=torch.bfloat16)
        k = torch.zeros(20, 2, 64, dtype=torch.bfloat16)
        r = torch.ops.exl3rocm.rope_kv_write(q, k, k, pos, slots, kc, kc.clone(), torch.zeros(32, dtype=torch.float64))
        o = torch.ops.exl3rocm.paged_attention(r, kc, kc, torch.zeros(3, 9, dtype=torch.int32), cu, seq, 0.1, 7)
        assert o.shape == q.shape and o.dtype == torch.bfloat16


def test_frequencies_refusals_and_defaults():
    for bad in (dict(rot_dim=7), dict(rot_dim=0), dict(rot_dim=8, base=1.0), dict(rot_dim=8, scaling={"rope_type": "dynamic"})):
        with pytest.raises(RuntimeError, match="rope_frequencies"):
            paged.rope_frequencies(**bad, device="cpu")
    f, m = paged.rope_frequencies(64, 1e4, {"type": "linear", "factor": 2.0}, device="cpu")
    assert m == 1.0 and f.dtype == torch.float64 and torch.allclose(f, 1e4 ** (-torch.arange(32).double() / 32) / 2)
    y, m = paged.rope_frequencies(64, 1e4, {"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 4096, "attention_factor": 1.25}, device="cpu")
    plain, _ = paged.rope_frequencies(64, 1e4, device="cpu")
    # the ramp's ends: pairs of 32 turns and of one in 4096 tokens
    low = math.floor(64 * math.log(4096 / (2 * math.pi * 32)) / (2 * math.log(1e4)))
    high = math.ceil(64 * math.log(4096 / (2 * math.pi)) / (2 * math.log(1e4)))
    assert m == 1.25 and torch.equal(y[:low + 1], plain[:low + 1]) and torch.allclose(y[high:], plain[high:] / 8)
