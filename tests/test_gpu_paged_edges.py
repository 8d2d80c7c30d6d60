"""GPU tests of the attention step at the ends of its ranges: lengths that pass 2^31 together."""
import pytest
import torch

paged = pytest.importorskip("exl3rocm.paged")
pytestmark = pytest.mark.gpu

MOST = 2 ** 31 - 1


def ints(v, dtype=torch.int32):
    return torch.tensor(v, device="cuda", dtype=dtype)


def plan(ctx, new, cols, stack, count, page, num_tokens):
    """batch_plan in Python's whole numbers, where a length and a count stop at 2^31 - 1; an empty table before."""
    table, taken, first = [[-1] * cols for _ in ctx], 0, 0
    cu, seq, pos, slots = [0], [], [0] * num_tokens, [-1] * num_tokens
    for r, (c, n) in enumerate(zip(ctx, new)):
        n = min(n, MOST - c)
        seq.append(c + n)
        had, have = min(-(-c // page), cols), min(-(-(c + n) // page), cols)
        for i, col in enumerate(range(had, have if n else had)):
            at = count - 1 - taken - i
            table[r][col] = stack[at] if at >= 0 else -1
        taken = min(taken + (have - had if n else 0), MOST)
        for t in range(first, min(first + n, num_tokens)):
            p = c + t - first
            pos[t] = p
            held = table[r][p // page] if p // page < cols else -1
            slots[t] = held * page + p % page if held >= 0 else -1
        first = min(first + n, MOST)
        cu.append(first)
    return cu, seq, pos, slots, count - taken, table


@pytest.mark.parametrize("ctx,new", [([0, 0], [MOST, MOST]), ([MOST, 0], [MOST, 40]), ([MOST - 3, 5, 0], [9, MOST, 7]), ([0, MOST], [3, 1]),
                                     ([0] * 300, [MOST // 2] * 300)])
@pytest.mark.parametrize("page,cols,tokens", [(16, 8, 8), (1, 5, 64), (65536, 3, 4200)])
def test_plan_of_lengths_beyond_32_bits(ctx, new, page, cols, tokens):
    """No index is formed from a sum that wrapped: outputs and table as the definition has them, and what lies around the
    table and the stack is untouched."""
    stack = list(range(100, 112))
    around = torch.full((len(ctx) + 2, cols + 4), -7, device="cuda", dtype=torch.int32)
    table = around[1:-1, 2:2 + cols]
    table.fill_(-1)
    free = ints([-7] * 64 + stack + [-7] * 64)[64:64 + len(stack)]
    cu, seq, pos, slots, left = paged.batch_plan(ints(ctx), ints(new), table, free, ints([len(stack)]), page, tokens)
    want = plan(ctx, new, cols, stack, len(stack), page, tokens)
    assert (cu.tolist(), seq.tolist(), pos.tolist(), slots.tolist(), left.item(), table.tolist()) == want
    around[1:-1, 2:2 + cols] = -7
    assert bool((around == -7).all())


@pytest.mark.parametrize("count", [-5, -(2 ** 31)])
def test_plan_with_a_stack_that_misses_pages(count):
    """A count below zero, as a step that ran out leaves it, holds no page."""
    table = torch.full((2, 4), -1, device="cuda", dtype=torch.int32)
    _, _, _, slots, left = paged.batch_plan(ints([0, 0]), ints([20, 1]), table, ints([1, 2, 3]), ints([count]), 16, 21)
    assert bool((slots == -1).all()) and bool((table == -1).all()) and left.item() == max(count - 3, -(2 ** 31))
