"""Every key counts once, however attention's work is shared: V marks each 32 keys by a column, so that an output is a weighted
count of keys and a step that is lost, doubled or weighted wrongly shows by a known amount.

Key j of a request has weight 2^-e(j // 32), e a whole number: its score is -e ln 2 by one column of K and a scale of ln 2
(weights are then powers of two to within fp32's error of the score and the exponential).  V[j] is 1 in column
(j // 32) mod D.  A row that sees n keys has out[c] = W_c / W with W_c the weights of column c's keys.

Bound, relative: the kernels' weights are off by at most 2^-20 (ln 2 and log2(e) rounded to fp32: 2^-23 of a score of at most 8;
the exponential: 2^-22), their fp16 or bf16 roundings by nothing more than that crosses (a power of two is exact, and
its neighbours' spacing is above 2^-12 of it), which moves a weight by one rounding u at most; sums of n positive terms in
fp32, of which at most 2^9 follow each other in one accumulator and its joins: 2^-15; the output's rounding u.  In all
2 u + 2^-14.
"""
import math

import pytest
import torch

from exl3rocm import paged

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F16, BF16 = torch.float16, torch.bfloat16


def bound_of(dtype):
    return 2 * U[dtype] + 2.0 ** -14


def exponents(steps, most, device="cpu"):
    g = torch.Generator().manual_seed(steps)
    return torch.randint(0, most + 1, (steps,), generator=g).to(device)


def columns(n, d, most, device="cpu"):
    """Running weights [n, d] of the columns over keys 0 .. j, in float64 (sums of few powers of two: exact)."""
    step = torch.arange(n, device=device) // 32
    w = torch.zeros(n, d, dtype=torch.float64, device=device)
    w[torch.arange(n, device=device), step % d] = torch.exp2(-exponents(-(-n // 32), most, device).double())[step]
    return w.cumsum(0)


CASES = [  # cached, new tokens, head width, type, largest exponent
    (131000, 1, 256, F16, 3), (60000, 1, 128, F16, 3), (30001, 1, 64, F16, 3), (40000, 1, 256, BF16, 0), (20000, 1, 128, BF16, 0),
    (50000, 3, 256, F16, 3), (40000, 40, 128, F16, 3), (70000, 30, 256, F16, 3), (15000, 200, 64, F16, 3), (10000, 130, 128, BF16, 0)]


@pytest.mark.parametrize("c,n,d,dtype,most", CASES)
def test_a_lost_step_is_out_of_bound(c, n, d, dtype, most):
    """The reference without any one step of 32 keys, or with it twice, is off by more than twice the bound in its column."""
    keys = c + n
    total = columns(keys, d, most)[-1]
    steps = keys // 32                                                 # whole ones
    w = 32 * torch.exp2(-exponents(-(-keys // 32), most).double())[:steps]
    col = total[torch.arange(steps) % d]
    lost = (col - w) / (total.sum() - w) / (col / total.sum()) - 1
    twice = (col + w) / (total.sum() + w) / (col / total.sum()) - 1
    assert min(lost.abs().min(), twice.abs().min()) > 2 * bound_of(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("c,n,d,dtype,most", CASES)
@pytest.mark.parametrize("group,hkv", [(5, 2), (1, 1)])
def test_every_key_counts_once(c, n, d, dtype, most, group, hkv):
    """Alone, and beside requests that shift the shares' boundaries."""
    page = 16
    for others in ([], [(700, 1), (0, n)], [(5, 1)] * 40):
        lens = others[:1] + [(c, n)] + others[1:]
        held = [-(-(a + b) // page) for a, b in lens]
        pages = sum(held)
        table = torch.full((len(lens), max(held)), -1, device="cuda", dtype=torch.int32)
        kc, vc = paged.new_cache(pages, page, hkv, d, dtype)
        at = 0
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(c)).int().cuda()
        for r, (a, b) in enumerate(lens):
            table[r, :held[r]] = order[at:at + held[r]]
            at += held[r]
            j = torch.arange(a + b, device="cuda")
            p = table[r].long()[j // page]
            kc[p, j % page, :, 7] = -exponents(-(-(a + b) // 32), most, "cuda")[j // 32].to(dtype)[:, None]
            vc[p, j % page, :, (j // 32) % d] = 1.0
        T = sum(b for _, b in lens)
        q = torch.zeros(T, group * hkv, d, device="cuda", dtype=dtype)
        q[..., 7] = 1.0
        cu = torch.tensor([0] + [sum(b for _, b in lens[:r + 1]) for r in range(len(lens))], device="cuda", dtype=torch.int32)
        seq = torch.tensor([a + b for a, b in lens], device="cuda", dtype=torch.int32)
        got = paged.paged_attention(q, kc, vc, table, cu, seq, math.log(2.0)).double()
        t0 = 0
        for a, b in lens:
            if b:
                w = columns(a + b, d, most, "cuda")[a:]
                want = w / w.sum(1, keepdim=True)
                off = (got[t0:t0 + b] - want[:, None]).abs() / want[:, None].clamp_min(1e-30)
                off = torch.where(want[:, None] > 0, off, got[t0:t0 + b].abs() * 1e30)
                worst = off.max().item()
                assert worst <= bound_of(dtype), (a, b, worst)
            t0 += b
