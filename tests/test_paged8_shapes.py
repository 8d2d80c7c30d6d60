"""CPU tests: shapes that the paged caches' ops take beside the documented ones, as the ops and their fake kernels (compiled code) see them."""
import pytest
import torch

from exl3rocm import paged, paged8
from test_paged8_host import args, called  # noqa: F401


@pytest.mark.parametrize("shape", [(5,), (2, 3), (2, 0), (1, 1, 4), ()])
def test_read_of_slots_of_any_shape(called, shape):  # noqa: F811
    """A row for each slot, in their order."""
    slots = torch.zeros(shape, dtype=torch.int64)
    cache = args()[5:9]
    a, b = torch.ops.exl3rocm.kv_read8(*cache, slots)
    assert a.shape == b.shape == (slots.numel(), 2, 64)
    (name, c), = called
    assert name == "exl3_kv_read8" and c[4] == slots.numel()
    with torch._subclasses.FakeTensorMode() as mode:
        a, b = torch.ops.exl3rocm.kv_read8(*(mode.from_tensor(t) for t in cache), mode.from_tensor(slots), torch.bfloat16)
        assert a.shape == b.shape == (slots.numel(), 2, 64) and a.dtype is b.dtype is torch.bfloat16
    assert len(called) == 1
    assert paged8.kv_read8(*cache, slots)[0].shape[0] == slots.numel()


@pytest.mark.parametrize("shape", [(6,), (2, 3), ()])
def test_plan_of_lengths_of_any_shape(called, monkeypatch, shape):  # noqa: F811
    """One request for each length, in their order."""
    monkeypatch.setattr(paged, "_entry", lambda name: lambda *a: 0)
    lens = torch.zeros(shape, dtype=torch.int32)
    R = lens.numel()
    a = (lens, lens.clone(), torch.zeros(R, 4, dtype=torch.int32), torch.zeros(9, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    want = [R + 1, R, 7, 7, 1]
    assert [t.shape for t in torch.ops.exl3rocm.batch_plan(*a, 16, 7)] == [(n,) for n in want]
    with torch._subclasses.FakeTensorMode() as mode:
        assert [t.shape for t in torch.ops.exl3rocm.batch_plan(*(mode.from_tensor(t) for t in a), 16, 7)] == [(n,) for n in want]
