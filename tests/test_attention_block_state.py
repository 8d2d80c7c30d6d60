"""The server's state of examples/attention_block.py when pages run out: on a GPU, and on host memory, where batch_plan's
library call is replaced by the same steps in Python."""
import ctypes as C
import os
import sys

import pytest
import torch

from exl3rocm import paged

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
PAGE, PAGES = 16, 6


def _view(p, n, t=C.c_int32):
    return (t * n).from_address(p) if n else []


def _plan(ctx, new, table, ld, cols, free, n_free, count, cu, seq, pos, slots, left, R, page, T, stream):
    c, n, rows, stack, have = _view(ctx, R), _view(new, R), _view(table, ld * R), _view(free, n_free), min(_view(count, 1)[0], n_free)
    at = taken = 0
    o_cu, o_seq, o_pos, o_slots = _view(cu, R + 1), _view(seq, R), _view(pos, T, C.c_int64), _view(slots, T, C.c_int64)
    for r in range(R):
        o_cu[r], o_seq[r] = at, c[r] + n[r]
        for col in range(-(-c[r] // page), -(-(c[r] + n[r]) // page) if n[r] else 0):
            rows[r * ld + col] = stack[have - 1 - taken] if have - 1 - taken >= 0 else -1
            taken += 1
        for p in range(c[r], c[r] + n[r]):
            held = rows[r * ld + p // page]
            o_pos[at], o_slots[at] = p, held * page + p % page if held >= 0 else -1
            at += 1
    o_cu[R] = at
    _view(left, 1)[0] = have - taken
    return 0


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def requests(request, monkeypatch):
    if request.param == "cpu":
        monkeypatch.setattr(paged, "_gpu", lambda t, what: t.get_device())
        monkeypatch.setattr(paged, "_raw_stream", lambda gpu: 0)
        monkeypatch.setattr(paged, "_entry", lambda name: {"exl3_batch_plan": _plan}[name])
    import attention_block
    return attention_block.Requests(3, PAGES, PAGE, 96, device=request.param)


def test_a_step_without_its_pages_does_not_take_place(requests):
    step = lambda *n: requests.step(torch.tensor(n, dtype=torch.int32, device=requests.lens.device), sum(n))  # noqa: E731

    def consistent():
        """Every page is free or held once, and what a request holds are pages."""
        count = int(requests.free_count)
        held = [requests.table[r, :-(-int(requests.lens[r]) // PAGE)].tolist() for r in range(3)]
        assert sorted(requests.free[:count].tolist() + sum(held, [])) == list(range(PAGES)), (count, held)

    step(33, 17, 5)                                                    # all six pages
    assert requests.lens.tolist() == [33, 17, 5] and int(requests.free_count) == 0 and int(requests.missing) == 0
    step(1, 1, 1)                                                      # the last pages' room
    assert requests.lens.tolist() == [34, 18, 6] and int(requests.missing) == 0
    consistent()
    for _ in range(2):                                                 # two pages short, twice
        plan = step(20, 1, 20)
        assert int(plan[4]) == -2 and int(requests.missing) == 2
        assert requests.lens.tolist() == [34, 18, 6] and int(requests.free_count) == 0
        consistent()
    requests.release(1)
    consistent()
    assert int(requests.free_count) == 2
    plan = step(20, 0, 20)
    assert requests.lens.tolist() == [54, 0, 26] and int(requests.free_count) == 0 and int(requests.missing) == 0
    assert bool((plan[3] >= 0).all())
    consistent()
    requests.release(0)
    requests.release(2)
    consistent()
    assert int(requests.free_count) == PAGES
