"""The attention block of examples/attention_block.py end to end: prompts, then single tokens, against the same block
computed from the oracle's decoded weights in float64 with a plain causal softmax."""
import math
import os
import sys

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

HID, HQ, HKV, D, BITS = 512, 8, 2, 64, 4


def dense(trellis, suh, svh):
    """float64 W with y = x W of one EXL3 tensor: rotations and scales around the oracle's decoded weights."""
    import cpu
    w = cpu.reconstruct(trellis.cpu().numpy().view(np.uint16), BITS, 2).astype(np.float64)
    h = np.ones((1, 1))
    while h.shape[0] < 128:
        h = np.block([[h, h], [h, -h]])
    h /= math.sqrt(128.0)
    k, n = w.shape
    w = (h @ w.reshape(k // 128, 128, n)).reshape(k, n)
    w = (w.reshape(k, n // 128, 128) @ h).reshape(k, n)
    return torch.from_numpy(suh.cpu().double().numpy()[:, None] * w * svh.cpu().double().numpy()[None])


def rotate(x, pos, f):
    ang = pos.double()[:, None] * f
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def test_block_prefill_and_decode():
    import attention_block as ab
    block = ab.AttentionBlock(HID, HQ, HKV, D, BITS, pages=64, page_size=16)
    prompts, steps = [37, 1, 100], 3
    reqs = ab.Requests(3, 64, 16, 160)
    g = torch.Generator(device="cuda").manual_seed(1)
    xs = [torch.randn(sum(prompts), HID, device="cuda", generator=g).half()] + \
         [torch.randn(3, HID, device="cuda", generator=g).half() for _ in range(steps)]
    got, new = [], [prompts] + [[1, 1, 1]] * steps
    for x, n in zip(xs, new):
        plan = reqs.step(torch.tensor(n, dtype=torch.int32, device="cuda"), sum(n))
        got.append(block(x, plan, reqs.table).cpu().double())
    assert reqs.lens.tolist() == [40, 4, 103] and int(reqs.free_count) == 64 - (3 + 1 + 7)
    reqs.release(2)
    assert int(reqs.free_count) == 64 - (3 + 1) and reqs.lens.tolist() == [40, 4, 0]

    w = [dense(*t) for t in block.qkv]
    wo, f = dense(*block.o), block.inv_freq.cpu()
    for r in range(3):
        rows, at = [], []                                              # the request's inputs, and where its outputs are
        for s, n in enumerate(new):
            i0 = sum(n[:r])
            rows.append(xs[s][i0:i0 + n[r]].cpu().double())
            at += [(s, i0 + i) for i in range(n[r])]
        x = torch.cat(rows)
        pos = torch.arange(len(x))
        q, k, v = (x @ m for m in w)
        q, k = rotate(q.view(-1, HQ, D), pos, f), rotate(k.view(-1, HKV, D), pos, f)
        v = v.view(-1, HKV, D)
        out = torch.empty(len(x), HQ, D, dtype=torch.float64)
        for h in range(HQ):
            s = q[:, h] @ k[:, h // (HQ // HKV)].T * D ** -0.5
            s = s.masked_fill(pos[None] > pos[:, None], -math.inf)
            out[:, h] = torch.softmax(s, -1) @ v[:, h // (HQ // HKV)]
        want = out.reshape(len(x), -1) @ wo
        have = torch.stack([got[s][i] for s, i in at])
        # each linear is within rel-L2 1e-3 of the oracle; scores of the order of 1 carry that to the probabilities, and the o
        # module's input roundings add theirs: 4e-3 in all
        rel = ((have - want).norm() / want.norm()).item()
        assert rel < 4e-3, (r, rel)
