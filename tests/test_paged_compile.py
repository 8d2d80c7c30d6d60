"""The attention step's ops under torch.compile and PyTorch's check of an op against its schema.  Without a GPU the library's
entry points are replaced by plain ones on host memory, so that the Python side runs whole."""
import ctypes as C

import pytest
import torch

from exl3rocm import paged


def _ints(p, n, t=C.c_int32):
    return (t * n).from_address(p) if n else []


def _plan(ctx, new, table, ld, cols, free, n_free, count, cu, seq, pos, slots, left, R, page, T, stream):
    """exl3_batch_plan on host memory, where every position has its page already."""
    c, n, t, at = _ints(ctx, R), _ints(new, R), _ints(table, ld * R), 0
    out_cu, out_seq, p, s = _ints(cu, R + 1), _ints(seq, R), _ints(pos, T, C.c_int64), _ints(slots, T, C.c_int64)
    for r in range(R):
        out_cu[r], out_seq[r] = at, c[r] + n[r]
        for i in range(n[r]):
            p[at], s[at] = c[r] + i, t[r * ld + (c[r] + i) // page] * page + (c[r] + i) % page
            at += 1
    out_cu[R] = at
    for i in range(at, T):
        p[i], s[i] = 0, -1
    _ints(left, 1)[0] = _ints(count, 1)[0]
    return 0


@pytest.fixture(autouse=True)
def one_compiling_process():
    from torch._inductor import config
    with config.patch(compile_threads=1):
        yield
    torch._dynamo.reset()


@pytest.fixture
def host(monkeypatch):
    monkeypatch.setattr(paged, "_gpu", lambda t, what: t.get_device())
    monkeypatch.setattr(paged, "_raw_stream", lambda gpu: 0)
    monkeypatch.setattr(paged, "_entry", lambda name: {"exl3_batch_plan": _plan}[name])


def plan_args(R, T, device="cpu"):
    i = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    new = [1 + r % 2 for r in range(R)]
    return i([3 * r for r in range(R)]), i(new), i([[4 * r + c for c in range(4)] for r in range(R)]), i([0, 1, 2]), i([3]), 16, T or sum(new)


@pytest.mark.parametrize("R,T", [(1, 0), (4, 0), (5, 9), (3, 8)])
def test_plan_keeps_its_schema(host, R, T):
    """Outputs that share no storage, as the schema says; shapes, types and places in memory as the fake kernel promises."""
    a = plan_args(R, T)
    torch.library.opcheck(torch.ops.exl3rocm.batch_plan.default, a, test_utils=("test_schema", "test_faketensor"))
    out = torch.ops.exl3rocm.batch_plan(*a)
    assert len({t.untyped_storage().data_ptr() for t in out}) == 5
    assert all(t.storage_offset() == 0 and t.is_contiguous() for t in out)


def step(ctx, new, table, free, count, page, T):
    cu, seq, pos, slots, left = torch.ops.exl3rocm.batch_plan(ctx + 1, new + 0, table.clone(), free + 0, count + 0, page, T)
    return cu * 2, seq + 1, pos + slots, slots - 1, left + 5


@pytest.mark.parametrize("R,T", [(3, 9), (4, 9)])
def test_plan_compiles(host, R, T):
    """Through Inductor, with odd counts: its code takes every output of an op for aligned."""
    a = plan_args(R, T)
    want = step(*a)
    got = torch.compile(step, fullgraph=True)(*a)
    assert all(torch.equal(g, w) for g, w in zip(got, want))


# ---------------------------------------------------------------------------------------------
# on a GPU
# ---------------------------------------------------------------------------------------------
def attention_step(ctx, new, table, free, count, q, k, v, kc, vc, f):
    op = torch.ops.exl3rocm
    cu, seq, pos, slots, left = op.batch_plan(ctx, new, table, free, count, 16, q.shape[0])
    q = op.rope_kv_write(q, k, v, pos, slots, kc, vc, f, 1.25)
    return q, op.paged_attention(q, kc, vc, table, cu, seq, 0.125), cu, seq, pos, slots, left


def attention_args(R, T, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g).half()  # noqa: E731
    kc, vc = paged.new_cache(4 * R, 16, 2, 64)
    kc.copy_(randn(4 * R, 16, 2, 64)), vc.copy_(randn(4 * R, 16, 2, 64))
    rows = randn(T, 8 * 64)
    q, k, v = (rows[:, 64 * a:64 * b].view(T, -1, 64) for a, b in ((0, 4), (4, 6), (6, 8)))
    return *plan_args(R, T, "cuda")[:5], q, k, v, kc, vc, paged.rope_frequencies(64)[0]


@pytest.mark.gpu
@pytest.mark.parametrize("R,T", [(3, 5), (4, 7)])
def test_compiled_step_is_the_eager_one(R, T):
    """The three ops as nodes of one compiled graph: the same bits, and the same cache and table behind them."""
    eager, compiled = attention_args(R, T), attention_args(R, T)
    want = attention_step(*eager)
    got = torch.compile(attention_step, fullgraph=True)(*compiled)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(compiled, eager))


@pytest.mark.gpu
def test_ops_keep_their_schemas():
    ctx, new, table, free, count, q, k, v, kc, vc, f = attention_args(3, 5)
    check = lambda op, *a: torch.library.opcheck(op.default, a, test_utils=("test_schema", "test_faketensor"))  # noqa: E731
    check(torch.ops.exl3rocm.batch_plan, ctx, new, table, free, count, 16, 5)
    cu, seq, pos, slots, _ = paged.batch_plan(ctx, new, table, free, count, 16, 5)
    check(torch.ops.exl3rocm.rope_kv_write, q, k, v, pos, slots, kc, vc, f, 1.25)
    check(torch.ops.exl3rocm.paged_attention, q, kc, vc, table, cu, seq, 0.125)
