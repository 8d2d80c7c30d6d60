"""GPU tests of the attention step over a paged cache (exl3rocm.paged) against plain computations: whole numbers in
Python, the rest in float64.

Bounds on the outputs are element by element, from the roundings that the kernels make (u: half an ulp of the element
type, 2^-11 in fp16, 2^-8 in bf16):
  rope       one rounding of a cos - b sin, formed in fp32 from values within 2^-22 of the exact ones:
             u |y| + 2^-21 (|a| + |b|) mscale
  attention  one rounding of the output, one of each probability, and fp32 scores: D products and sums of |q k| scale,
             each off by at most 2^-24 relative, move a probability by twice that relative to the sum, and the exponential
             and the sums by a few 2^-24: u |o| + (u + 2^-23 D scale max_j |q|.|k_j| + 2^-18) sum_j p_j |v_j|;
             subnormals of the element type: an absolute 2^-25 per key, and at the output
"""
import math
import random
from fractions import Fraction

import pytest
import torch

paged = pytest.importorskip("exl3rocm.paged")
pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F16, BF16 = torch.float16, torch.bfloat16


def ints(v, dtype=torch.int32):
    return torch.tensor(v, device="cuda", dtype=dtype)


# ---------------------------------------------------------------------------------------------
# batch_plan
# ---------------------------------------------------------------------------------------------
def plan_reference(ctx, new, table, free, count, page, num_tokens):
    table, stack = [list(r) for r in table], list(free[:count])
    cu, seq, pos, slots, want = [0], [], [], [], 0
    cols = len(table[0]) if table else 0
    for r, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(c, 0), max(n, 0)
        seq.append(c + n)
        if n:
            for col in range(min(-(-c // page), cols), min(-(-(c + n) // page), cols)):
                table[r][col] = stack.pop() if stack else -1
                want += 1
        for p in range(c, c + n):
            held = table[r][p // page] if p // page < cols else -1
            pos.append(p)
            slots.append(held * page + p % page if held >= 0 else -1)
        cu.append(cu[-1] + n)
    pos, slots = pos[:num_tokens], slots[:num_tokens]
    pad = num_tokens - len(pos)
    return cu, seq, pos + [0] * pad, slots + [-1] * pad, count - want, table


def check_plan(ctx, new, cols, pages, count, page, num_tokens, seed=0, ld=None):
    rng = random.Random(seed)
    ids = list(range(pages))
    rng.shuffle(ids)
    R = len(ctx)
    table = [[rng.randrange(max(pages, 1)) if col * page < c else -1 for col in range(cols)] for c in ctx]
    wide = torch.full((R, ld or cols), -7, device="cuda", dtype=torch.int32)
    t = wide[:, :cols]
    if R and cols:
        t.copy_(ints(table))
    free, cnt = ints(ids), ints([count])
    for _ in range(2):                              # the stack is only read: a second call gives the same
        cu, seq, pos, slots, left = paged.batch_plan(ints(ctx), ints(new), t, free, cnt, page, num_tokens)
        want = plan_reference(ctx, new, table, ids, count, page, num_tokens)
        got = (cu.tolist(), seq.tolist(), pos.tolist(), slots.tolist(), left.item(), t.tolist())
        assert got == want
    assert free.tolist() == ids and cnt.item() == count and bool((wide[:, cols:] == -7).all())


@pytest.mark.parametrize("page", [1, 7, 16, 48, 256])
def test_plan_lengths(page):
    ctx = [0, 1, page - 1, page, page + 1, 5 * page, 3, 0, 777, 0]
    new = [1, 1, 1, 1, 1, 0, 2 * page + 1, 0, 300, page]
    cols = 2 + max(-(-(a + b) // page) for a, b in zip(ctx, new))
    check_plan(ctx, new, cols, 2000, 1500, page, sum(new))
    check_plan(ctx, new, cols, 2000, 2000, page, sum(new) + 37, ld=cols + 5)


def test_plan_out_of_pages_and_out_of_columns():
    check_plan([0, 16, 3, 40], [33, 1, 60, 9], 12, 9, 5, 16, 103)      # the stack ends inside the third request
    check_plan([0, 16], [33, 1], 12, 9, 0, 16, 34)                     # empty from the start
    check_plan([10, 60, 200], [100, 10, 3], 4, 50, 50, 16, 113)        # rows of 4 pages: positions from 64 have no slot
    check_plan([5, 5], [20, 20], 0, 10, 10, 16, 40)                    # no columns at all


def test_plan_edges_of_the_batch():
    check_plan([], [], 3, 4, 4, 16, 5)                                 # no requests: padding alone
    check_plan([0, 0], [0, 0], 3, 4, 4, 16, 0)                         # no tokens
    check_plan([-3, 4], [2, -5], 3, 4, 4, 16, 6)                       # negative lengths count as 0
    check_plan([0, 9], [40, 30], 8, 20, 20, 16, 50)                    # a batch with fewer rows than tokens


def test_plan_many_requests_and_long_chunks():
    rng = random.Random(5)
    R = 1500
    ctx = [rng.choice([0, rng.randrange(400)]) for _ in range(R)]
    new = [rng.choice([0, 1, 1, 4]) for _ in range(R)]
    new[700] = 5001                                                    # three workgroups' share of tokens
    new[701] = 2048
    check_plan(ctx, new, 350, 20000, 19000, 16, sum(new) + 3000, seed=1)


# ---------------------------------------------------------------------------------------------
# rope_kv_write
# ---------------------------------------------------------------------------------------------
PI = Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803482534211706798")


def angles(pos, inv_freq):
    """pos x inv_freq less its whole turns.  A float64 product is off by 2^-53 of itself, so past 2^20 radians the
    turns are taken off in rational numbers."""
    if pos.numel() == 0 or pos.max().item() < 1 << 20:
        return pos.double()[:, None] * inv_freq
    per = [Fraction(v) / (2 * PI) for v in inv_freq.tolist()]
    return torch.tensor([[float((p * v) % 1 * 2 * PI) for v in per] for p in pos.tolist()], dtype=torch.float64, device=pos.device)


def rope_reference(x, pos, inv_freq, m, interleaved):
    """(rotated x, sum of the pair's magnitudes) in float64."""
    rot = 2 * inv_freq.numel()
    ang = angles(pos, inv_freq)
    cos, sin = ang.cos()[:, None], ang.sin()[:, None]
    x = x.double()
    y, mag = x.clone(), x.abs()
    ia = torch.arange(0, rot, 2) if interleaved else torch.arange(rot // 2)
    ib = ia + (1 if interleaved else rot // 2)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = (a * cos - b * sin) * m, (a * sin + b * cos) * m
    mag[..., ia] = mag[..., ib] = (a.abs() + b.abs()) * m
    return y, mag


def within(got, want, bound):
    off = (got.double() - want).abs()
    ok = bool((off <= bound).all())
    assert ok, f"off by {(off / bound).nan_to_num(1e9).max().item():.3g} of the bound"


def check_rope(T, hq, hkv, d, dtype, rot, interleaved, gated=False, page=16, m=1.0, pos_hi=5000, seed=0, flat_cache=False, skip=()):
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = -(-T // page) + 3
    wq = hq * d * (2 if gated else 1)
    rows = torch.randn(T, wq + 2 * hkv * d, device="cuda", generator=g).to(dtype)
    q = rows[:, :wq].view(T, hq, wq // hq)[:, :, :d]
    k = rows[:, wq:wq + hkv * d].view(T, hkv, d)
    v = rows[:, wq + hkv * d:].view(T, hkv, d)
    if flat_cache:
        kc, vc = (torch.full((pages, page, hkv, d), 7.0, device="cuda", dtype=dtype) for _ in range(2))
    else:
        kc, vc = paged.new_cache(pages, page, hkv, d, dtype)
        kc.fill_(7.0), vc.fill_(7.0)
    pos = torch.randint(0, pos_hi, (T,), device="cuda", generator=g)
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:T]
    for i, s in skip:
        slots[i] = s
    f, _ = paged.rope_frequencies(rot, 1e6) if rot else (torch.empty(0, device="cuda", dtype=torch.float64), 1.0)
    before = rows.clone()
    out = paged.rope_kv_write(q, k, v, pos, slots, kc, vc, f, m, interleaved)
    assert torch.equal(rows, before) and out.is_contiguous()
    live = (slots >= 0) & (slots < pages * page)
    sl = slots[live]
    u = U[dtype]
    want, mag = rope_reference(q, pos, f, m, interleaved)
    within(out, want, u * want.abs() + 2.0 ** -21 * mag + 2.0 ** -25)
    want, mag = rope_reference(k, pos, f, m, interleaved)
    within(kc[sl // page, sl % page], want[live], (u * want.abs() + 2.0 ** -21 * mag + 2.0 ** -25)[live])
    assert torch.equal(vc[sl // page, sl % page], v[live])
    rest = torch.ones(pages, page, dtype=torch.bool, device="cuda")
    rest[sl // page, sl % page] = False
    assert bool((kc[rest] == 7.0).all()) and bool((vc[rest] == 7.0).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_parts_of_the_head(dtype, d, interleaved):
    for rot in (d, d // 2, d // 4, 2, 10, d - 2, 0):
        check_rope(5, 6, 2, d, dtype, rot, interleaved, seed=rot)


@pytest.mark.parametrize("T", [1, 3, 33, 513, 2049])
def test_rope_token_counts_and_layouts(T):
    check_rope(T, 40, 8, 128, F16, 128, False)
    check_rope(T, 24, 4, 256, BF16, 64, False, gated=True, page=64, m=1.1386)
    check_rope(T, 7, 1, 64, F16, 64, True, page=5, flat_cache=True)


def test_rope_long_positions():
    check_rope(64, 4, 4, 128, F16, 128, False, pos_hi=1 << 40)


def test_rope_tokens_without_a_slot():
    check_rope(9, 4, 2, 64, F16, 64, False, skip=[(0, -1), (4, 10 ** 12), (8, -(1 << 40))])


def test_rope_empty_batch():
    check_rope(0, 4, 2, 64, F16, 64, False)


def test_rope_frequencies():
    f, m = paged.rope_frequencies(8, 100.0)
    assert m == 1.0 and torch.allclose(f.cpu(), torch.tensor([1, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64))
    assert torch.allclose(paged.rope_frequencies(8, 100.0, {"rope_type": "linear", "factor": 4.0})[0], f / 4)
    y, m = paged.rope_frequencies(128, 1e6, {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768})
    f, _ = paged.rope_frequencies(128, 1e6)
    assert torch.equal(y[:23], f[:23]) and torch.allclose(y[41:], f[41:] / 4) and abs(m - (0.1 * math.log(4) + 1)) < 1e-12
    assert bool((y[1:] < y[:-1]).all())
    z, _ = paged.rope_frequencies(128, 5e5, {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                                             "original_max_position_embeddings": 8192})
    f, _ = paged.rope_frequencies(128, 5e5)
    turns = 8192 * f / (2 * math.pi)
    assert torch.equal(z[turns > 4], f[turns > 4]) and torch.allclose(z[turns < 1], f[turns < 1] / 8)


# ---------------------------------------------------------------------------------------------
# paged_attention
# ---------------------------------------------------------------------------------------------
class Batch:
    """Requests of (cached, new) tokens over a cache whose unused slots hold NaN."""

    def __init__(self, lens, hq, hkv, d, dtype, page=16, seed=0, pad=0, q_scale=2.0, flat=False, fused_q=False, extra_pages=3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.hq, self.hkv, self.d, self.dtype, self.page = lens, hq, hkv, d, dtype, page
        held = [-(-(c + n) // page) for c, n in lens]
        pages = sum(held) + extra_pages
        order = torch.randperm(pages, generator=g, device="cuda")
        cols = max(held, default=0) + 2
        table = torch.full((len(lens), cols), -1, device="cuda", dtype=torch.int32)
        if flat:
            self.kc, self.vc = (torch.full((pages, page, hkv, d), math.nan, device="cuda", dtype=dtype) for _ in range(2))
        else:
            self.kc, self.vc = paged.new_cache(pages, page, hkv, d, dtype)
            self.kc.fill_(math.nan), self.vc.fill_(math.nan)
        self.k, self.v, at = [], [], 0
        for r, (c, n) in enumerate(lens):
            k, v = (torch.randn(c + n, hkv, d, device="cuda", generator=g).to(dtype) for _ in range(2))
            mine = order[at:at + held[r]]
            at += held[r]
            table[r, :held[r]] = mine.int()
            p = torch.arange(c + n, device="cuda")
            self.kc[mine[p // page], p % page], self.vc[mine[p // page], p % page] = k, v
            self.k.append(k), self.v.append(v)
        self.table = table
        T = sum(n for _, n in lens) + pad
        rows = (q_scale * torch.randn(T, hq, d * (2 if fused_q else 1), device="cuda", generator=g)).to(dtype)
        self.q = rows[:, :, :d]
        cu = [0]
        for _, n in lens:
            cu.append(cu[-1] + n)
        self.cu, self.seq = ints(cu), ints([c + n for c, n in lens])
        self.scale = d ** -0.5

    def run(self, window=0):
        return paged.paged_attention(self.q, self.kc, self.vc, self.table, self.cu, self.seq, self.scale, window)

    def reference(self, window=0, requests=None, rows=None):
        """(output, bound) in float64; requests: those to compute (default all); rows: of a request's new tokens."""
        T, g = self.q.shape[0], self.hq // self.hkv
        out = torch.zeros(T, self.hq, self.d, device="cuda", dtype=torch.float64)
        bound = torch.full_like(out, 2.0 ** -25)
        u, t0 = U[self.dtype], 0
        for r, (c, n) in enumerate(self.lens):
            if n and (requests is None or r in requests):
                q = self.q[t0:t0 + n].double()
                for h in range(self.hq):
                    k, v = self.k[r][:, h // g].double(), self.v[r][:, h // g].double()
                    s = q[:, h] @ k.T * self.scale
                    p, j = c + torch.arange(n, device="cuda")[:, None], torch.arange(c + n, device="cuda")
                    off = (j > p) | ((j <= p - window) if window else (j < 0))
                    w = torch.softmax(s.masked_fill(off, -math.inf), -1)
                    size = (q[:, h].abs() @ k.abs().T * abs(self.scale)).masked_fill(off, 0).amax(-1, keepdim=True)
                    o = w @ v
                    out[t0:t0 + n, h] = o
                    bound[t0:t0 + n, h] += (u * o.abs() + (u + 2.0 ** -23 * self.d * size + 2.0 ** -18) * (w @ v.abs())
                                            + 2.0 ** -25 * (~off).double() @ v.abs())
            t0 += n
        return out, bound

    def check(self, window=0):
        got = self.run(window)
        want, bound = self.reference(window)
        within(got, want, bound)
        assert torch.equal(got, self.run(window))                      # the same bits again
        return got


HEADS = [(40, 8), (24, 4), (8, 8), (5, 1), (12, 1), (28, 4), (3, 3), (17, 1)]
EDGE = [(0, 1), (1, 1), (14, 1), (15, 1), (16, 1), (31, 1), (62, 1), (63, 1), (64, 1), (127, 1), (128, 1), (300, 1), (1000, 1)]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_decode_lengths(d, dtype):
    for hq, hkv in HEADS:
        Batch(EDGE, hq, hkv, d, dtype, seed=hq).check()


@pytest.mark.parametrize("page", [16, 48, 64, 256])
@pytest.mark.parametrize("window", [0, 1, 16, 77, 1000])
def test_decode_pages_and_windows(page, window):
    Batch(EDGE + [(2000, 1)], 10, 2, 128, F16, page=page, seed=page).check(window)
    Batch([(517, 1), (33, 2), (0, 3), (90, 5)], 6, 1, 256, BF16, page=page, flat=True, fused_q=True).check(window)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new", [2, 4, 7, 13])
def test_drafts(d, new):
    Batch([(0, new), (61, new), (500, new), (1300, new - 1), (64, 1)], 24, 4, d, F16, seed=new).check()
    Batch([(0, new), (61, new), (500, new)], 5, 1, d, BF16, seed=new).check(window=40)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens", [[(0, 17)], [(0, 64)], [(0, 129)], [(1, 200)], [(100, 300)], [(63, 65), (0, 0), (5, 1), (700, 130)], [(0, 1025)]])
def test_chunks(d, dtype, lens):
    Batch(lens, 10, 2, d, dtype, seed=d).check()
    Batch(lens, 3, 3, d, dtype, page=48, seed=d).check(window=100)


@pytest.mark.parametrize("hq,hkv", HEADS)
def test_chunk_heads(hq, hkv):
    Batch([(40, 150), (0, 90), (333, 1)], hq, hkv, 128, F16, flat=True, fused_q=True).check()


def test_chunk_windows():
    for w in (1, 15, 64, 65, 128, 500, 4000):
        Batch([(300, 333), (2000, 1), (0, 70)], 8, 2, 64, BF16, seed=w).check(window=w)


def test_mixed_batch_with_empty_requests_and_padding():
    b = Batch([(0, 0), (900, 1), (0, 300), (5, 0), (64, 64), (3000, 1), (0, 0)], 40, 8, 128, F16, pad=9)
    got = b.check()
    assert bool((got[-9:] == 0).all())
    b = Batch([(0, 0), (90, 0)], 10, 2, 64, BF16, pad=3)
    assert bool((b.check() == 0).all())
    assert Batch([(7, 0)], 10, 2, 64, F16).check().shape == (0, 10, 64)
    b = Batch([], 10, 2, 64, F16, pad=2)
    assert bool((b.run() == 0).all())


def test_many_requests():
    rng = random.Random(3)
    Batch([(rng.randrange(200), rng.choice([0, 1, 1, 1, 2])) for _ in range(700)], 10, 2, 64, F16).check()


def test_long_context_is_split_and_joined():
    Batch([(60001, 1), (5, 1), (131000, 1)], 10, 2, 128, F16).check()
    Batch([(70000, 4)], 6, 1, 256, BF16, page=64).check()
    Batch([(40000, 100)], 4, 1, 128, F16).check()


def test_one_kv_head_and_one_head():
    for hq, hkv in ((64, 1), (40, 1), (1, 1)):
        Batch([(700, 1), (33, 2), (0, 1)], hq, hkv, 128, F16, seed=hq).check()
        Batch([(300, 50), (0, 7)], hq, hkv, 64, BF16, seed=hq).check(window=90)


def test_strides_that_address_nothing():
    """One token, one head, one page: torch leaves such strides at anything."""
    b = Batch([(9, 1)], 1, 1, 64, F16, extra_pages=0)
    want = b.check()
    odd = lambda t, shape, strides: t.as_strided(shape, strides)  # noqa: E731
    b.q = odd(b.q, (1, 1, 64), (3, 5, 1))
    b.kc, b.vc = (odd(c, (1, 16, 1, 64), (7, c.stride(1), 9, 1)) for c in (b.kc, b.vc))
    b.table = odd(b.table, (1, b.table.shape[1]), (1, 1))
    assert torch.equal(b.run(), want)
    f, _ = paged.rope_frequencies(64)
    k = torch.randn(1, 1, 64, device="cuda").half()
    q = paged.rope_kv_write(odd(k, (1, 1, 64), (3, 5, 1)), odd(k, (1, 1, 64), (11, 1, 1)), k, ints([0], torch.int64), ints([3], torch.int64), b.kc, b.vc, f)
    assert torch.equal(q, k) and torch.equal(b.kc[0, 3], k[0]) and torch.equal(b.vc[0, 3], k[0])


def test_large_scores():
    """Scores of hundreds: the running maximum carries them; keys far below it vanish."""
    Batch([(1000, 1), (700, 3), (0, 200)], 10, 2, 128, F16, q_scale=60.0).check()
    Batch([(1000, 1), (700, 3), (0, 200)], 10, 2, 128, BF16, q_scale=300.0).check()


@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-3, 2.0])
def test_scales(scale):
    for lens in ([(300, 1), (20, 3)], [(50, 200)]):
        b = Batch(lens, 6, 2, 64, F16)
        b.scale = scale
        b.check()


def test_rows_that_see_nothing():
    """More new tokens than the sequence holds: the first ones lie at negative positions."""
    b = Batch([(0, 20), (50, 1)], 10, 2, 64, F16)
    b.seq = ints([8, 0])
    got = b.run()
    assert bool((got[:12] == 0).all()) and bool((got[20] == 0).all()) and bool((got[12:20] != 0).all())


def test_pages_that_are_none():
    """Positions whose table entry is no page (-1, or past the cache) are not seen; nor are those past the row."""
    for d, new in ((128, 1), (64, 40)):
        b = Batch([(200, new)], 10, 2, d, F16)
        b.table[0, 3], b.table[0, 7] = -1, b.kc.shape[0]
        got = b.run()
        keep = torch.ones(200 + new, dtype=torch.bool, device="cuda")
        keep[48:64] = keep[112:128] = False
        want = _subset(b, keep)
        within(got, *want)
        b.table = b.table[:, :5]
        keep[80:] = False
        got = b.run()
        within(got, *_subset(b, keep))


def _subset(b, keep):
    """reference() of a one-request batch over the kept positions alone."""
    (c, n), g, u = b.lens[0], b.hq // b.hkv, U[b.dtype]
    out, bound = (torch.zeros(n, b.hq, b.d, device="cuda", dtype=torch.float64) for _ in range(2))
    for h in range(b.hq):
        q, k, v = b.q[:n, h].double(), b.k[0][:, h // g].double(), b.v[0][:, h // g].double()
        off = (torch.arange(c + n, device="cuda") > c + torch.arange(n, device="cuda")[:, None]) | ~keep
        w = torch.softmax((q @ k.T * b.scale).masked_fill(off, -math.inf), -1)
        size = (q.abs() @ k.abs().T * b.scale).amax(-1, keepdim=True)
        out[:, h] = w @ v
        bound[:, h] = (u * out[:, h].abs() + (u + 2.0 ** -23 * b.d * size + 2.0 ** -18) * (w @ v.abs())
                       + 2.0 ** -25 * (~off).double() @ v.abs() + 2.0 ** -25)
    return out, bound


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("d,lens,row", [(128, (100, 3), 1), (64, (30, 70), 20), (128, (0, 200), 63), (256, (5, 150), 100)])
def test_what_a_row_does_not_see_has_no_effect(bad, d, lens, row):
    """A later token of the chunk, and a key that left the window, hold NaN or infinities in K and V."""
    b = Batch([lens], 6, 2, d, F16)
    clean = b.run()
    p = lens[0] + row + 1                                              # the first position that `row` does not see
    page = b.table[0, p // 16].long()
    kc, vc = b.kc.clone(), b.vc.clone()
    b.kc, b.vc = b.kc.clone(), b.vc.clone()
    b.kc[page, p % 16] = bad
    b.vc[page, p % 16] = bad
    got = b.run()
    unseen, seen = torch.equal(got[:row + 1], clean[:row + 1]), bool(torch.isfinite(got[row + 1:]).any())
    assert unseen and not seen
    b.kc, b.vc = kc, vc
    if lens[0] + row > 20:
        clean = b.run(window=9)
        page = b.table[0, (lens[0] + row - 9) // 16].long()
        b.kc[page, (lens[0] + row - 9) % 16] = bad
        b.vc[page, (lens[0] + row - 9) % 16] = bad
        same = torch.equal(b.run(window=9)[row:], clean[row:])
        assert same


def test_infinite_scores():
    """A key whose score is minus infinity has weight 0; a row with one of plus infinity is NaN, as in the formula."""
    b = Batch([(40, 1)], 2, 1, 64, F16)
    b.q.fill_(1.0)
    page = b.table[0, 1].long()
    b.kc[page, 3] = -math.inf
    b.k[0][19] = -math.inf
    keep = torch.ones(41, dtype=torch.bool, device="cuda")
    keep[19] = False
    b.k[0][19] = 0
    within(b.run(), *_subset(b, keep))
    b.kc[page, 3] = math.inf
    nan = bool(torch.isnan(b.run()).all())
    assert nan


def test_offsets_beyond_32_bits():
    """A cache of more than 2^31 elements (4 GiB each for K and V): pages at its end."""
    b = Batch([(100, 1), (77, 40)], 10, 2, 128, F16, page=64)
    want, bound = b.reference()
    pages = (1 << 31) // (64 * 2 * 128) + 64
    kc, vc = (torch.empty(pages, 2, 64, 128, device="cuda", dtype=F16).transpose(1, 2) for _ in range(2))
    n = b.kc.shape[0]
    kc[pages - n:], vc[pages - n:] = b.kc, b.vc
    b.kc, b.vc = kc, vc
    b.table = torch.where(b.table >= 0, b.table + (pages - n), -1).int()
    within(b.run(), want, bound)
    # and the write
    q = torch.randn(2, 10, 128, device="cuda").half()
    k = torch.randn(2, 2, 128, device="cuda").half()
    f, _ = paged.rope_frequencies(128)
    slots = ints([pages * 64 - 1, pages * 64 - 64], torch.int64)
    paged.rope_kv_write(q, k, k, ints([0, 0], torch.int64), slots, kc, vc, f)
    assert torch.equal(kc[pages - 1, 63], k[0]) and torch.equal(vc[pages - 1, 0], k[1])


def test_another_stream_and_a_graph_with_growing_lengths():
    """The step is captured once and replayed as the requests grow: no length is baked into the graph."""
    hq, hkv, d, page = 10, 2, 128, 16
    R, steps = 5, 6
    g = torch.Generator(device="cuda").manual_seed(0)
    f, m = paged.rope_frequencies(d)
    start = [3, 15, 40, 100, 31]
    rows = torch.randn(steps, R, (hq + 2 * hkv) * d, device="cuda", generator=g).half()

    def fresh():
        kc, vc = paged.new_cache(64, page, hkv, d)
        gg = torch.Generator(device="cuda").manual_seed(1)
        kc.copy_(torch.randn(kc.shape, device="cuda", generator=gg)), vc.copy_(torch.randn(vc.shape, device="cuda", generator=gg))
        table = torch.full((R, 12), -1, device="cuda", dtype=torch.int32)
        at = 0
        for r, s in enumerate(start):
            n = -(-s // page)
            table[r, :n] = torch.arange(at, at + n, device="cuda")
            at += n
        free = torch.arange(64, device="cuda", dtype=torch.int32).roll(-at).contiguous()
        return dict(kc=kc, vc=vc, table=table, free=free, count=ints([64 - at]), ctx=ints(start), new=ints([1, 1, 1, 1, 0]),
                    x=rows[0].clone())

    def step(s):
        cu, seq, pos, slots, left = torch.ops.exl3rocm.batch_plan(s["ctx"], s["new"], s["table"], s["free"], s["count"], page, R)
        x = s["x"]
        q, k, v = (x[:, a * d:b * d].view(R, -1, d) for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv)))
        q = torch.ops.exl3rocm.rope_kv_write(q, k, v, pos, slots, s["kc"], s["vc"], f, m)
        o = torch.ops.exl3rocm.paged_attention(q, s["kc"], s["vc"], s["table"], cu, seq, d ** -0.5)
        s["ctx"].copy_(seq), s["count"].copy_(left)
        return o

    eager = fresh()
    want = []
    for i in range(steps):
        eager["x"].copy_(rows[i])
        want.append(step(eager).clone())
    side = torch.cuda.Stream()
    s = fresh()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = fresh()
        for i in range(2):
            warm["x"].copy_(rows[i])
            assert torch.equal(step(warm), want[i])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(s)
    for i in range(steps):
        s["x"].copy_(rows[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]), i
        torch.randn(100, device="cuda").sum().item()                   # eager work between replays
    assert torch.equal(s["table"], eager["table"]) and s["ctx"].tolist() == [9, 21, 46, 106, 31]


def test_refusals():
    b = Batch([(20, 1)], 10, 2, 64, F16)
    q, kc, vc, t, cu, seq = b.q, b.kc, b.vc, b.table, b.cu, b.seq
    ok = lambda **k: {**dict(q=q, k_cache=kc, v_cache=vc, block_table=t, cu_q=cu, seq_lens=seq, scale=1.0), **k}  # noqa: E731
    for bad in (dict(q=q.float()), dict(q=q.cpu()), dict(q=q[:, :, :32]), dict(q=q[:, :9]), dict(q=q.bfloat16()), dict(k_cache=kc[:, :8]),
                dict(k_cache=kc[:, :8], v_cache=vc[:, :8]), dict(v_cache=vc.bfloat16()), dict(block_table=t.long()), dict(block_table=t[:, None]),
                dict(cu_q=cu[:1]), dict(cu_q=cu.long()), dict(seq_lens=seq.long()), dict(seq_lens=seq.cpu()), dict(window=-1),
                dict(q=torch.zeros(1, 10, 65, device="cuda", dtype=F16)[:, :, 1:])):
        with pytest.raises(RuntimeError, match="exl3rocm"):
            paged.paged_attention(**ok(**bad))
    f, _ = paged.rope_frequencies(64)
    k = torch.zeros(1, 2, 64, device="cuda", dtype=F16)
    pos = ints([0], torch.int64)
    ok = lambda **n: {**dict(q=q, k=k, v=k, positions=pos, slots=pos, k_cache=kc, v_cache=vc, inv_freq=f), **n}  # noqa: E731
    for bad in (dict(k=k.float()), dict(v=k[:, :1]), dict(positions=pos.int()), dict(slots=pos.repeat(2)), dict(inv_freq=f.float()),
                dict(inv_freq=torch.ones(33, device="cuda", dtype=torch.float64)), dict(q=q.cpu()), dict(k_cache=kc[:, :, :1]),
                dict(k_cache=kc.bfloat16(), v_cache=vc.bfloat16()), dict(q=q[0])):
        with pytest.raises(RuntimeError, match="exl3rocm"):
            paged.rope_kv_write(**ok(**bad))
    free, one = ints([1, 2, 3]), ints([3])
    ok = lambda **n: {**dict(ctx_lens=ints([1]), new_lens=ints([1]), block_table=t, free_pages=free, free_count=one, page_size=16, num_tokens=1), **n}  # noqa: E731
    for bad in (dict(ctx_lens=ints([1, 2])), dict(new_lens=ints([1], torch.int64)), dict(block_table=t.T), dict(free_count=free),
                dict(page_size=0), dict(num_tokens=-1), dict(free_pages=free.cpu()), dict(page_size=1 << 20)):
        with pytest.raises(RuntimeError, match="exl3rocm"):
            paged.batch_plan(**ok(**bad))
    paged.batch_plan(**ok())
