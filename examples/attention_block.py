"""A decoder layer's attention block on this engine: EXL3 qkv and o modules around the paged attention step.

    x -> qkv (EXL3) -> rope_kv_write -> paged_attention -> o (EXL3) -> y

with the batch's bookkeeping (batch_plan) on the GPU, over a cache in 16 bits or, with `--cache-bits 8`, in 8.  `python examples/attention_block.py` prefills ragged prompts in
one step, then decodes: eagerly, and by replaying one captured HIP graph whose lengths grow on the GPU.  Weights are
seeded synthetic ones (exl3rocm.synth).
"""
import argparse
import os
import sys
import time

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen38-27b-exl3-rdna4_amd"))

from exl3rocm import ops, paged, paged8, synth  # noqa: E402,F401


class AttentionBlock:
    """qkv, attention over a paged cache (fp16, or int8 with a scale for each 16 tokens and head), o; mul1 codebook, fp16."""

    def __init__(self, hidden=5120, q_heads=40, kv_heads=8, head_dim=128, bits=4, rot_dim=None, base=1e6, scaling=None,
                 pages=4096, page_size=16, name="attention_block", cache_bits=16):
        self.q_heads, self.kv_heads, self.head_dim, self.bits = q_heads, kv_heads, head_dim, bits
        widths = [q_heads * head_dim, kv_heads * head_dim, kv_heads * head_dim]
        def load(part, k, n):
            tr, su, sv = synth.layer(name, part, k, n, bits)
            # outputs of the order of the inputs
            sv = (sv.astype(np.float32) * k ** -0.5).astype(np.float16)
            return tuple(torch.from_numpy(a).cuda() for a in (tr.view(np.int16), su, sv))
        self.qkv = [load(f"qkv{i}", hidden, n) for i, n in enumerate(widths)]
        self.o = load("o", widths[0], hidden)
        self.inv_freq, self.mscale = paged.rope_frequencies(rot_dim or head_dim, base, scaling)
        op = torch.ops.exl3rocm
        if cache_bits == 8:
            self.cache, self.write, self.attend = paged8.new_cache8(pages, page_size, kv_heads, head_dim), op.rope_kv_write8, op.paged_attention8
        else:
            self.cache, self.write, self.attend = paged.new_cache(pages, page_size, kv_heads, head_dim), op.rope_kv_write, op.paged_attention

    def __call__(self, x, step, block_table):
        """x [T, hidden] fp16; step: batch_plan's result."""
        cu_q, seq_lens, positions, slots, _ = step
        op, T, d = torch.ops.exl3rocm, x.shape[0], self.head_dim
        qkv = op.linear_groups(x, *(list(t) for t in zip(*self.qkv)), [self.bits] * 3, False, True)
        q, k, v = (t.view(T, -1, d) for t in qkv.split([self.q_heads * d, self.kv_heads * d, self.kv_heads * d], 1))
        q = self.write(q, k, v, positions, slots, *self.cache, self.inv_freq, self.mscale)
        a = self.attend(q, *self.cache, block_table, cu_q, seq_lens, d ** -0.5)
        return op.linear(a.view(T, -1), *self.o, self.bits, False, True)


class Requests:
    """A server's state on the GPU: lengths, block tables, free pages."""

    def __init__(self, count, pages, page_size, max_tokens, device="cuda"):
        self.page_size = page_size
        self.lens = torch.zeros(count, dtype=torch.int32, device=device)
        self.table = torch.full((count, -(-max_tokens // page_size)), -1, dtype=torch.int32, device=device)
        self.free = torch.arange(pages, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), pages, dtype=torch.int32, device=device)
        self.missing = torch.zeros(1, dtype=torch.int32, device=device)    # pages that the last step lacked

    def step(self, new_lens, num_tokens):
        """The plan of a step that adds new_lens tokens; the state moves on if every token has its page.  Otherwise it stays as it
        was and the step's outputs mean nothing: `missing` says so, to be read with the step's tokens; the server then
        releases a request (or leaves some out) and makes the step again."""
        plan = torch.ops.exl3rocm.batch_plan(self.lens, new_lens, self.table, self.free, self.free_count, self.page_size, num_tokens)
        fits = plan[4] >= 0
        self.lens.copy_(torch.where(fits, plan[1], self.lens))
        self.free_count.copy_(torch.where(fits, plan[4], self.free_count))
        self.missing.copy_((-plan[4]).clamp_min(0))
        return plan

    def release(self, request):
        """Returns a finished request's pages (its length is known to the host's scheduler)."""
        held, count = -(-int(self.lens[request]) // self.page_size), int(self.free_count)
        self.free[count:count + held] = self.table[request, :held]
        self.free_count += held
        self.table[request] = -1
        self.lens[request] = 0


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--prompts", type=int, nargs="*", default=[517, 64, 1200, 33, 2000, 801, 16, 290])
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--cache-bits", type=int, default=16, choices=(8, 16))
    a = ap.parse_args()
    R, total = len(a.prompts), sum(a.prompts)
    block = AttentionBlock(cache_bits=a.cache_bits)
    reqs = Requests(R, 4096, 16, max(a.prompts) + a.steps + 16)
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(total, 5120, device="cuda", generator=g).half()
    plan = reqs.step(torch.tensor(a.prompts, dtype=torch.int32, device="cuda"), total)
    y = block(x, plan, reqs.table)
    assert int(reqs.missing) == 0, "the cache is too small for these prompts"
    print(f"prefilled {total} tokens of {R} requests: output {tuple(y.shape)}, rms {y.float().square().mean().sqrt().item():.3f}")

    ones = torch.ones(R, dtype=torch.int32, device="cuda")
    x = torch.randn(R, 5120, device="cuda", generator=g).half()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                                      # an eager step first, as a server warms up
        block(x, reqs.step(ones, R), reqs.table)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = block(x, reqs.step(ones, R), reqs.table)
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(a.steps):
        graph.replay()
    torch.cuda.synchronize()
    assert int(reqs.missing) == 0, "the cache ran out of pages"
    print(f"decode step of {R} requests, one captured graph: {(time.perf_counter() - t) / a.steps * 1e6:.1f} us; lengths now {reqs.lens.tolist()}")
    reqs.release(0)
    print(f"free pages after the first request left: {int(reqs.free_count)}")


if __name__ == "__main__":
    main()
