"""GPU tests of the attention step over a cache in 8 bits (exl3rocm.paged8) against plain computations: codes and scales in
whole numbers and powers of two, the attention in float64.

Bounds, from the roundings that the kernels make:
  write      k and v that are not rotated have one right code and scale, to be met exactly.  A rotated k is a cos - b sin in fp32 from
             values within 2^-22 of the exact ones, so off by at most E = 2^-21 (|a| + |b|) mscale, and a scale may differ where E
             decides; a code that E would decide comes from float64, where positions below 2^18 leave an angle within 2^-35: it
             stands for a number within half a step and 2^-33 (|a| + |b|) mscale of the exact value
  attention  u |o| for the output's rounding (u: half an ulp, 2^-11 in fp16, 2^-8 in bf16); a probability's to fp16, 2^-11; fp32 scores:
             D products and sums of |q c| f (f = scale * the block's scale * log2 e), each off by 2^-24 relative, and four roundings of
             exponents up to S + L + 8 (largest score and logarithm of a scale, base 2), move a probability by 2 ln 2 times as much
             relative to the sum; sums over n keys, 2^-24 (n / 16 + 64); subnormal probabilities: 2^-33 of the row's
             largest p_j sv_j for each key, times its code
"""
import math
import random

import pytest
import torch

paged8 = pytest.importorskip("exl3rocm.paged8")
from exl3rocm import paged  # noqa: E402

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F16, BF16 = torch.float16, torch.bfloat16
BLOCK = 16


def ints(v, dtype=torch.int32):
    return torch.tensor(v, device="cuda", dtype=dtype)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def spread(g, *shape):
    """Values whose channels and rows have different sizes."""
    x = torch.randn(*shape, device="cuda", generator=g)
    return x * torch.exp(0.7 * torch.randn(*shape[1:], device="cuda", generator=g)) * torch.exp(torch.randn(shape[0], *[1] * (len(shape) - 1), device="cuda", generator=g))


LAYOUTS = ["new", "tokens", "gaps"]


def make_cache(layout, pages, page, hkv, d, fill=None):
    """A cache in one of several memory orders; fill: a generator of codes and scales (else zeros)."""
    if layout == "new":
        c = paged8.new_cache8(pages, page, hkv, d)
    elif layout == "tokens":                            # a token's heads together; scales likewise
        c = (*(torch.zeros(pages, page, hkv, d, device="cuda", dtype=torch.int8) for _ in range(2)),
             *(torch.zeros(pages, page // BLOCK, hkv, device="cuda") for _ in range(2)))
    else:                                               # k and v (and their scales) in one allocation, padded rows
        both = torch.zeros(pages, 2, page, hkv, d + 16, device="cuda", dtype=torch.int8)
        s = torch.zeros(2, hkv + 1, pages, page // BLOCK + 3, device="cuda")
        c = (both[:, 0, :, :, :d], both[:, 1, :, :, :d], s[0, :hkv, :, :page // BLOCK].permute(1, 2, 0), s[1, 1:, :, 2:2 + page // BLOCK].permute(1, 2, 0))
    if fill is not None:
        for t in c[:2]:
            t.copy_(torch.randint(-127, 128, t.shape, device="cuda", generator=fill))
        for t in c[2:]:
            t.copy_(2.0 ** torch.randint(-9, -3, t.shape, device="cuda", generator=fill).cpu().double())
    return c


# ---------------------------------------------------------------------------------------------
# rope_kv_write8
# ---------------------------------------------------------------------------------------------
def least_scale(most):
    """The least power of two, 2^-40 to 2^40, of which 127 reach `most`."""
    e = -40
    while e < 40 and 127.0 * 2.0 ** e < most:
        e += 1
    return 2.0 ** e


def write_reference(codes, scales, x, slots, page):
    """codes [slots, hkv, d] (float64) and scales [slots / 16, hkv] after x [T, hkv, d] (float64) went to its slots: plain host
    tensors, block by block in the order of the batch."""
    runs, last = [], None
    for t, s in enumerate(slots):
        b = s // BLOCK if 0 <= s < codes.shape[0] else None
        if b is not None:
            if b != last:
                runs.append((b, {}))
            runs[-1][1][s % BLOCK] = t
        last = b
    for b, rows in runs:
        at, t = torch.tensor(sorted(rows)), torch.tensor([rows[r] for r in sorted(rows)])
        new = x[t]
        for h in range(x.shape[1]):
            fin = new[:, h].abs()
            fin = fin[fin < math.inf]
            need = least_scale(fin.max().item() if fin.numel() else 0.0)
            old = scales[b, h].item()
            old = 2.0 ** -40 if math.isnan(old) else min(max(old, 2.0 ** -40), 2.0 ** 40)
            block = codes[b * BLOCK:(b + 1) * BLOCK, h]
            if 0 in rows:
                block.zero_()
                scales[b, h] = s = need
            elif need > old:
                block.copy_(torch.round(block * (old / need)))
                scales[b, h] = s = need
            else:
                s = old
            block[at] = torch.nan_to_num(torch.round(new[:, h] / s), 0.0, 127.0, -127.0).clamp(-127, 127)


def flat(t, page):
    return t.reshape(-1, *t.shape[2:]).cpu().double()


def inputs(g, T, hq, hkv, d, dtype, how="rows"):
    if how == "rows":                                   # columns of one projection's output
        w = (hq + 2 * hkv) * d
        rows = spread(g, T, w).to(dtype)
        q, k, v = rows.split([hq * d, hkv * d, hkv * d], 1)
        return q.view(T, hq, d), k.view(T, hkv, d), v.view(T, hkv, d)
    q = spread(g, T, hq, 2 * d).to(dtype)[..., :d]      # gated heads; heads outermost
    k, v = (spread(g, hkv, T, d + 8).to(dtype)[..., :d].transpose(0, 1) for _ in range(2))
    return q, k, v


def check_write(T, slots, *, hq=4, hkv=2, d=64, dtype=F16, page=16, pages=12, layout="new", how="rows", seed=0, change=None, scales=None):
    """Without a rotation every code and scale is exact, k's and v's."""
    g = gen(seed)
    c = make_cache(layout, pages, page, hkv, d, fill=g)
    if scales is not None:
        scales(c)
    q, k, v = inputs(g, T, hq, hkv, d, dtype, how)
    if change is not None:
        change(k, v)
    want = [(flat(c[i], page), flat(c[i + 2], page)) for i in (0, 1)]
    for (codes, sc), x in zip(want, (k, v)):
        write_reference(codes, sc, x.cpu().double(), slots, page)
    out = paged8.rope_kv_write8(q, k, v, ints([0] * T, torch.int64), ints(slots, torch.int64), *c, torch.zeros(0, device="cuda", dtype=torch.float64))
    assert torch.equal(out, q.contiguous())
    for i, name in ((0, "k"), (1, "v")):
        sc = flat(c[i + 2], page)
        same = (sc == want[i][1]) | (sc.isnan() & want[i][1].isnan())
        assert bool(same.all()), (name, "scales", same.logical_not().nonzero()[:4].tolist())
        assert torch.equal(flat(c[i], page), want[i][0]), (name, "codes", (flat(c[i], page) != want[i][0]).nonzero()[:4].tolist())
    return c


def run_of(start, n):
    return list(range(start, start + n))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("layout,how", [("new", "rows"), ("tokens", "heads"), ("gaps", "rows")])
def test_write_whole_and_partial_blocks(d, dtype, layout, how):
    # a block that begins, one that goes on, single tokens at a block's first, middle and last slot, rows that go nowhere
    slots = run_of(64, 37) + [3] + run_of(41, 7) + [-1, 48, -1, 31, 10 ** 9, 191, 176] + run_of(113, 40)
    check_write(len(slots), slots, d=d, dtype=dtype, layout=layout, how=how, seed=d)


@pytest.mark.parametrize("page", [16, 48, 256])
@pytest.mark.parametrize("hq,hkv", [(3, 3), (12, 1), (40, 8)])
def test_write_heads_and_pages(page, hq, hkv):
    pages = 1024 // page
    slots = run_of(2 * page + 5, page + 9) + [page - 1, 0] + run_of(900, 3)
    check_write(len(slots), slots, hq=hq, hkv=hkv, d=128, page=page, pages=pages, seed=page + hkv)


@pytest.mark.parametrize("T", [1, 16, 511, 512, 513, 1500])
def test_write_counts(T):
    """Either form of the launch; blocks that begin anywhere in a workgroup's rows, and a batch that ends inside one."""
    rng, slots, at = random.Random(T), [], 5
    while len(slots) < T:
        n = rng.choice([1, 1, 2, 5, 16, 17, 40, 200])
        slots += run_of(at, n)
        at += n + rng.randrange(16, 40)                 # the next run begins in another block
        if rng.random() < 0.2:
            slots += [-1] * rng.randrange(1, 20)
    check_write(T, slots[:T], pages=at // 16 + 2, seed=T)


def test_write_order_of_blocks_is_free():
    """A later block before an earlier one, and neighbouring blocks of different requests."""
    slots = run_of(80, 16) + run_of(64, 16) + run_of(17, 3) + run_of(5, 11) + run_of(96, 1) + run_of(32, 1)
    check_write(len(slots), slots)
    check_write(16 * len(slots), [s + 128 * i for i in range(16) for s in slots], pages=16 * 8 + 8)


@pytest.mark.parametrize("T", [6, 700])
def test_write_same_slot_twice(T):
    """The last row counts; so it does where a block's rows are more than 64."""
    slots = [21, 22, 21, 23, 22, 22] + [16 * 3 + i % 5 for i in range(T - 6)]
    check_write(T, slots)


def test_write_special_values():
    def change(k, v):
        k[0, 0, 3], k[0, 1, 5] = math.inf, -math.inf    # a row of large values, the scale from the others
        k[1, 0, 0] = math.nan
        v[2] = 0                                        # nothing but zeros: the least scale
        v[3, 0], v[3, 1] = math.nan, math.inf
        k[4] = 2.0 ** -24
        k[5, 0, 0] = 65504.0
    check_write(6, [0, 1, 32, 48, 64, 80], change=change)
    check_write(6, [3, 18, 33, 49, 66, 82], change=change)

    def wide(k, v):
        k[0] = 3e38                                     # past 127 * 2^40: saturated
        k[1] = 1e-30                                    # below half of 2^-40: 0
        v[0, 0, :2] = torch.tensor([127.0 * 2 ** 40, 1e14], device="cuda")
        v[1, 0] = 2.0 ** -41
        v[1, 0, 0] = -126.0 * 2.0 ** -40
    check_write(2, [0, 16], dtype=BF16, change=wide)
    check_write(2, [5, 23], dtype=BF16, change=wide, seed=1)


@pytest.mark.parametrize("m", [127.0, 127.5, 128.0, 126.0, 63.5, 64.0, 254.0, 1.0, 2.0 ** -14])
def test_write_scale_at_its_limits(m):
    """127 of a scale, exactly and just above; ties of the rounding go to even."""
    def change(k, v):
        k[:], v[:] = 0, 0
        k[:, 0, 0] = -m
        k[:, 0, 1:33] = (torch.arange(32, device="cuda") - 16) * m / 256     # halves of steps
        v[:, 1, 5] = torch.nextafter(torch.tensor(m, dtype=BF16), torch.tensor(math.inf, dtype=BF16)).cuda()
    check_write(3, [0, 21, 40], dtype=BF16, change=change)


@pytest.mark.parametrize("bad", [0.0, -1.0, math.nan, math.inf, 3e38, 1e-44, 0.3])
def test_write_over_any_scale(bad):
    """What a scale's memory held before counts as the nearest of 2^-40 .. 2^40; a block that begins does not read it."""
    def scales(c):
        c[2].fill_(bad), c[3].fill_(bad)
        if bad == 0.3:                                  # rows rounded anew from a scale that is no power of two
            c[0][0], c[1][0] = 0, 0
            c[0][2:], c[1][2:] = 0, 0

    def change(k, v):
        if bad == 0.3:                                  # products with such a scale are not exact: whole multiples of it only
            k[:], v[:] = 0.0, 0.0
            k[0, :, 0], v[1, :, 3] = 600.0, 19200.0
    check_write(3, [16, 37, 101], scales=scales, change=change)


def test_write_block_by_block_over_many_steps():
    """Tokens one at a time with growing values: every doubling rounds the rows before anew, as the reference does."""
    c = make_cache("new", 3, 16, 2, 64)
    g = gen(5)
    codes, sc = flat(c[0], 16), flat(c[2], 16)
    for i in range(37):
        k = (torch.randn(1, 2, 64, device="cuda", generator=g) * 1.3 ** i).half()
        paged8.rope_kv_write8(k, k, k, ints([i], torch.int64), ints([i], torch.int64), *c, torch.zeros(0, device="cuda", dtype=torch.float64))
        write_reference(codes, sc, k.cpu().double(), [i], 16)
        assert torch.equal(flat(c[0], 16), codes) and torch.equal(flat(c[2], 16), sc) and torch.equal(c[0], c[1])


def test_write_rejected_drafts_are_written_over():
    c = make_cache("new", 2, 16, 1, 64)
    g = gen(6)
    codes, sc = flat(c[1], 16), flat(c[3], 16)
    f = torch.zeros(0, device="cuda", dtype=torch.float64)
    for start, n in ((0, 9), (9, 4), (10, 4), (11, 4), (15, 4), (16, 2)):
        v = torch.randn(n, 1, 64, device="cuda", generator=g).half()
        paged8.rope_kv_write8(v, v, v, ints([0] * n, torch.int64), ints(run_of(start, n), torch.int64), *c, f)
        write_reference(codes, sc, v.cpu().double(), run_of(start, n), 16)
        assert torch.equal(flat(c[1], 16), codes) and torch.equal(flat(c[3], 16), sc)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d,rot,interleaved", [(64, 64, False), (128, 128, False), (128, 128, True), (256, 64, False), (256, 256, True), (128, 22, False), (64, 2, True)])
@pytest.mark.parametrize("T", [23, 530, 5000])
def test_write_rotated(d, rot, interleaved, dtype, T):
    hq, hkv, page = 6, 2, 32
    g = gen(rot + T)
    q, k, v = inputs(g, T, hq, hkv, d, dtype)
    pos = torch.randint(0, 1 << 18, (T,), device="cuda", generator=g)
    inv, mscale = paged.rope_frequencies(rot, 1e6)[0], torch.tensor(1.3).item()         # the entry point takes a float
    slots = run_of(0, T)
    c = make_cache("new", T // page + 1, page, hkv, d)
    out = paged8.rope_kv_write8(q, k, v, pos, ints(slots, torch.int64), *c, inv, mscale, interleaved)
    # q: the bits of the 16-bit cache's op
    kc, vc = paged.new_cache(T // page + 1, page, hkv, d, dtype)
    assert torch.equal(out, paged.rope_kv_write(q, k, v, pos, ints(slots, torch.int64), kc, vc, inv, mscale, interleaved))
    a = pos.double()[:, None] * inv
    cos, sin = a.cos()[:, None] * mscale, a.sin()[:, None] * mscale
    x = k.double()
    lo, hi = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    y, err = x.clone(), torch.zeros_like(x)
    y[..., lo], y[..., hi] = x[..., lo] * cos - x[..., hi] * sin, x[..., lo] * sin + x[..., hi] * cos
    err[..., lo] = err[..., hi] = 2.0 ** -21 * (x[..., lo].abs() + x[..., hi].abs()) * mscale
    codes, sc = (flat(t, page).cuda()[:T] if i == 0 else flat(t, page).cuda() for i, t in enumerate((c[0], c[2])))
    s = sc.repeat_interleave(BLOCK, 0)[:T, :, None]
    assert bool(((codes * s - y).abs() <= s / 2 + err * 2.0 ** -12).all())
    pad = -T % BLOCK
    most, e = (torch.nn.functional.pad(t, (0, 0, 0, 0, 0, pad)).view(-1, BLOCK, hkv, d).amax((1, 3)) for t in (y.abs(), err))
    sc = sc[:most.shape[0]]
    assert bool((127 * sc >= most - e).all()) and bool((127 * sc / 2 < most + e).all())
    codes, sc = flat(c[1], page), flat(c[3], page)
    want = torch.zeros_like(codes), torch.zeros_like(sc)
    write_reference(*want, v.cpu().double(), slots, page)
    assert torch.equal(codes, want[0]) and torch.equal(sc, want[1])


def test_write_nothing():
    c = make_cache("new", 2, 16, 1, 64, fill=gen(0))
    before = [t.clone() for t in c]
    z = torch.zeros(0, 1, 64, device="cuda", dtype=F16)
    e = ints([], torch.int64)
    f = torch.zeros(32, device="cuda", dtype=torch.float64)
    assert paged8.rope_kv_write8(z, z, z, e, e, *c, f).shape == (0, 1, 64)
    k = torch.ones(3, 1, 64, device="cuda", dtype=F16)
    paged8.rope_kv_write8(k, k, k, ints([0, 1, 2], torch.int64), ints([-1, 32, 1 << 40], torch.int64), *c, f)
    empty = make_cache("new", 0, 16, 1, 64)
    paged8.rope_kv_write8(k, k, k, ints([0, 1, 2], torch.int64), ints([-1, 0, 5], torch.int64), *empty, f)
    assert all(torch.equal(a, b) for a, b in zip(before, c))


# ---------------------------------------------------------------------------------------------
# kv_read8
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("T,page,hkv", [(1, 16, 1), (77, 48, 3), (1300, 16, 8)])
def test_read(T, page, hkv, d, layout, dtype):
    g = gen(T + d)
    pages = 700 // page
    c = make_cache(layout, pages, page, hkv, d, fill=g)
    c[0][-1, -1, -1, -1] = -128
    slots = torch.randint(-2, pages * page, (T,), device="cuda", generator=g)
    slots[0] = pages * page if T > 1 else 5
    for i, got in enumerate(paged8.kv_read8(*c, slots, dtype)):
        values = flat(c[i], page) * flat(c[i + 2], page).repeat_interleave(BLOCK, 0)[..., None]
        s = slots.cpu()
        held = (s >= 0) & (s < pages * page)
        want = torch.where(held[:, None, None], values[s.clamp(0, pages * page - 1)], 0.0).to(dtype)
        assert got.dtype is dtype and torch.equal(got.cpu(), want)


def test_read_rounds_once_and_clamps_scales():
    c = make_cache("new", 1, 48, 1, 64, fill=gen(1))
    c[2].copy_(torch.tensor([2.0 ** -26, 2.0 ** 12, 0.3], device="cuda").view(1, 3, 1))
    c[3].copy_(torch.tensor([math.nan, math.inf, 0.0], device="cuda").view(1, 3, 1))
    k, v = paged8.kv_read8(*c, ints(run_of(0, 48), torch.int64))
    s = torch.tensor([2.0 ** -26, 2.0 ** 12, torch.tensor(0.3).item()], dtype=torch.float64).repeat_interleave(16)
    want = (flat(c[0], 48)[:, 0] * s[:, None])
    assert torch.equal(k[:32, 0].cpu(), want[:32].half())                   # subnormals and infinities of fp16
    assert torch.equal(k[32:, 0].cpu(), want[32:].float().half())           # the product in fp32, then fp16
    s = torch.tensor([2.0 ** -40, 2.0 ** 40, 2.0 ** -40], dtype=torch.float64).repeat_interleave(16)
    assert torch.equal(v[:, 0].cpu(), (flat(c[1], 48)[:, 0] * s[:, None]).half())


def test_write_then_read_gives_the_values_within_half_a_step():
    g = gen(9)
    c = make_cache("new", 8, 16, 2, 128)
    q, k, v = inputs(g, 100, 2, 2, 128, BF16)
    slots = ints(run_of(0, 100), torch.int64)
    paged8.rope_kv_write8(q, k, v, slots, slots, *c, torch.zeros(0, device="cuda", dtype=torch.float64))
    for x, y, s in zip((k, v), paged8.kv_read8(*c, slots, BF16), c[2:]):
        step = flat(s, 16).cuda().repeat_interleave(BLOCK, 0)[:100, :, None]
        assert bool(((x.double() - y.double()).abs() <= step / 2).all())


# ---------------------------------------------------------------------------------------------
# paged_attention8
# ---------------------------------------------------------------------------------------------
def batch(ctx, new, page, pages=None, seed=0, spare=2):
    """(cu_q, seq_lens, block table, pages) of requests whose pages lie in random order."""
    rng = random.Random(seed)
    held = [-(-(a + b) // page) for a, b in zip(ctx, new)]
    n = pages or sum(held) + spare
    ids = list(range(n))
    rng.shuffle(ids)
    cols = max(held, default=0) + 1
    table = []
    for h in held:
        table.append([ids.pop() for _ in range(h)] + [-1] * (cols - h))
    cu = [0]
    for b in new:
        cu.append(cu[-1] + b)
    return ints(cu), ints([a + b for a, b in zip(ctx, new)]), ints(table).view(len(ctx), cols), n


def reference(q, c, table, cu, seq, scale, window, dtype):
    """(out, tolerance) in float64, from the codes and scales that the cache holds."""
    kc, vc, ks, vs = c
    T, hq, d = q.shape
    page, hkv = kc.shape[1], kc.shape[2]
    out, tol = torch.zeros(T, hq, d, device="cuda", dtype=torch.float64), torch.zeros(T, hq, d, device="cuda", dtype=torch.float64)
    cu, seq = cu.tolist(), seq.tolist()
    log2e = 1.4426950408889634
    for r in range(len(seq)):
        n, cap = cu[r + 1] - cu[r], table.shape[1] * page
        if n <= 0:
            continue
        end = min(seq[r], cap)
        key = torch.arange(max(end, 0), device="cuda")
        held = table[r, key // page].long()
        real = (held >= 0) & (held < kc.shape[0])
        held = held.clamp(0, max(kc.shape[0] - 1, 0))
        pos = (seq[r] - n + torch.arange(n, device="cuda"))[:, None]
        seen = (key <= pos) & real
        if window:
            seen &= key > pos - window
        for h in range(hkv):
            heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            qq = q[cu[r]:cu[r + 1], heads].double()
            sk, sv = (s[held, key % page // BLOCK, h].double().nan_to_num(0.0).clamp(2.0 ** -40, 2.0 ** 40) for s in (ks, vs))
            k, v = kc[held, key % page, h].double() * sk[:, None], vc[held, key % page, h].double() * sv[:, None]
            # what nobody sees may be anything
            any_seen = seen.any(0)[:, None]
            k, v = torch.where(any_seen, k, 0.0), torch.where(any_seen, v, 0.0)
            s = (qq @ k.T) * scale
            mask = ~seen[:, None]
            s = s.masked_fill(mask, -math.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0)
            out[cu[r]:cu[r + 1], heads] = p @ v
            if key.numel() == 0:
                continue
            size = ((qq.abs() @ k.abs().T) * abs(scale) * log2e).masked_fill(mask, 0.0).amax(-1, keepdim=True)
            big = s.masked_fill(mask, 0.0).abs().amax(-1, keepdim=True) * log2e
            lv = torch.where(any_seen[:, 0], torch.log2(sv), 0.0).abs().max()
            psv = (p * sv).amax(-1, keepdim=True)
            rel = 2.0 ** -11 + 2 * math.log(2) * (d * 2.0 ** -24 * size + 4 * 2.0 ** -24 * (big + lv + 8)) + 2.0 ** -24 * (key.numel() / 16 + 64)
            tol[cu[r]:cu[r + 1], heads] = rel * (p @ v.abs()) + key.numel() * 2.0 ** -33 * psv * 127
    return out, tol + U[dtype] * out.abs() + (2.0 ** -25 if dtype is F16 else 0.0)


def check_attention(ctx, new, *, hq=10, hkv=2, d=128, dtype=F16, page=16, window=0, layout="new", seed=0, scale=None, pad=0, q_size=1.0, change=None, cache=None):
    g = gen(seed + 77)
    cu, seq, table, pages = batch(ctx, new, page, seed=seed)
    c = cache(pages) if cache else filled_cache(g, layout, pages, page, hkv, d)
    T = sum(new) + pad
    q = (q_size * torch.randn(T, hq, 2 * d, device="cuda", generator=g)).to(dtype)[..., :d]
    scale = d ** -0.5 if scale is None else scale
    if change is not None:
        change(q, c, table)
    got = paged8.paged_attention8(q, *c, table, cu, seq, scale, window)
    want, tol = reference(q, c, table, cu, seq, scale, window, dtype)
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), (off / tol.clamp_min(1e-300)).max().item()
    assert bool((got[sum(new):] == 0).all())
    again = paged8.paged_attention8(q, *c, table, cu, seq, scale, window)
    assert torch.equal(got, again)
    return got, (q, c, table, cu, seq, scale, window)


def filled_cache(g, layout, pages, page, hkv, d):
    """Values as a writer leaves them: each block's largest code between 64 and 127."""
    c = make_cache(layout, pages, page, hkv, d)
    for codes, s in ((c[0], c[2]), (c[1], c[3])):
        x = torch.randn(pages, page, hkv, d, device="cuda", generator=g) * torch.exp(torch.randn(1, 1, hkv, d, device="cuda", generator=g) * 0.7)
        x = x.view(pages, page // BLOCK, BLOCK, hkv, d)
        x = x * torch.exp(torch.randn(pages, page // BLOCK, 1, hkv, 1, device="cuda", generator=g))
        m, e = torch.frexp(x.abs().amax((2, 4)))
        step = ((e - torch.where(m > 127 / 128, 6, 7) + 127) << 23).int().view(torch.float32)
        s.copy_(step)
        codes.copy_((x / step[:, :, None, :, None]).round().clamp(-127, 127).view(pages, page, hkv, d))
    return c


HEADS = [(10, 2, 128), (12, 2, 256), (8, 2, 64), (3, 3, 128), (14, 1, 64), (28, 4, 128), (17, 1, 256)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_decode_lengths(hq, hkv, d, dtype):
    """Contexts around the edges of blocks, steps and pages, one token each."""
    check_attention([0, 1, 14, 15, 16, 31, 62, 63, 64, 65, 127, 128, 200, 511, 1000, 2047], [1] * 16, hq=hq, hkv=hkv, d=d, dtype=dtype)


@pytest.mark.parametrize("page", [16, 32, 48, 80, 256])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_pages_and_layouts(page, layout):
    check_attention([1, 90, 333, 1025], [1, 3, 1, 2], page=page, layout=layout, seed=page)
    check_attention([100, 0], [40, 300], hkv=1, hq=3, page=page, layout=layout, seed=page)


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 64, 100, 1000])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_windows(window, d):
    check_attention([0, 5, 40, 300, 900], [1, 2, 4, 1, 3], hq=4, hkv=2, d=d, window=window, seed=window)
    check_attention([0, 70, 500], [130, 33, 65], hq=4, hkv=2, d=d, window=window, dtype=BF16, seed=window)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_chunks(hq, hkv, d, dtype):
    """Prompts and chunks behind cached tokens, odd lengths, beside decodes."""
    check_attention([0, 129, 0, 700, 33], [1, 77, 300, 63, 1], hq=hq, hkv=hkv, d=d, dtype=dtype, page=32)
    check_attention([0], [513], hq=hq, hkv=hkv, d=d, dtype=dtype)


@pytest.mark.parametrize("hq,hkv,d", [(40, 8, 128), (24, 4, 256), (32, 8, 64)])
def test_long_contexts(hq, hkv, d):
    """Tiles that many workgroups share and join, in both kernels."""
    check_attention([30000, 7, 4001], [1, 1, 1], hq=hq, hkv=hkv, d=d, seed=1)
    check_attention([9000], [100], hq=hq, hkv=hkv, d=d, dtype=BF16, seed=2)
    check_attention([20000, 100], [4, 4], hq=hq, hkv=hkv, d=d, seed=3)


@pytest.mark.parametrize("ctx,new,hq,hkv,d,dtype", [([140000], [1], 40, 1, 128, F16), ([140000], [1], 40, 1, 256, BF16), ([70000], [1], 40, 1, 64, F16),
                                                   ([30000], [9], 12, 2, 128, BF16), ([20000, 3000], [7, 7], 24, 4, 256, F16), ([8000], [110], 40, 1, 128, F16)])
def test_chunks_in_many_parts(ctx, new, hq, hkv, d, dtype):
    """Tiles of prompt chunks that 13 to 512 workgroups share, in every size of the groups that are joined first."""
    check_attention(ctx, new, hq=hq, hkv=hkv, d=d, dtype=dtype, seed=4)


def test_many_requests():
    check_attention([(37 * i) % 300 for i in range(700)], [i % 2 for i in range(700)], hq=2, hkv=1, d=64, pad=5)
    check_attention([(37 * i) % 90 for i in range(600)], [17 + i % 3 for i in range(600)], hq=2, hkv=2, d=64)


def test_padding_and_empty_batches():
    check_attention([10, 0, 0, 4], [1, 0, 0, 2], pad=3)
    check_attention([10, 600], [1, 200], pad=300)
    check_attention([0, 0], [0, 0], pad=4)
    g = gen(0)
    c = filled_cache(g, "new", 3, 16, 2, 128)
    q = torch.randn(2, 4, 128, device="cuda", generator=g).half()
    none, one = torch.zeros(0, 3, device="cuda", dtype=torch.int32), ints([0])
    assert paged8.paged_attention8(q, *c, none, one, ints([]), 0.1).eq(0).all()
    assert paged8.paged_attention8(q[:0], *c, none, one, ints([]), 0.1).shape == (0, 4, 128)
    # no columns in the table, no pages in the cache: nobody sees anything
    cu, seq = ints([0, 2]), ints([9])
    assert paged8.paged_attention8(q, *c, torch.zeros(1, 0, device="cuda", dtype=torch.int32), cu, seq, 0.1).eq(0).all()
    assert paged8.paged_attention8(q, *paged8.new_cache8(0, 16, 2, 128), torch.zeros(1, 3, device="cuda", dtype=torch.int32), cu, seq, 0.1).eq(0).all()


@pytest.mark.parametrize("new", [1, 90])
def test_scale_of_scores(new):
    for scale in (-0.2, 0.0, 1e-6):
        check_attention([300], [new], hq=6, hkv=2, scale=scale)
        check_attention([300], [new], hq=6, hkv=2, scale=scale, dtype=BF16)
    check_attention([300], [new], hq=6, hkv=2, q_size=40.0)                     # one key takes nearly all


@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("size", [1e-30, 1e-8, 1e4, 1e30])
def test_bf16_rows_of_any_size(size, new):
    """Rows of q whose sizes fp16 does not hold, each its own, beside each other; scale undoes it."""
    def change(q, c, table):
        q.mul_(size)
        q[::2] *= 0.01
        q[0, 0] = 0
        q[-1, 0, 1:] *= 2.0 ** -20
    check_attention([200, 64], [new, new], dtype=BF16, scale=0.1 / size, change=change)


@pytest.mark.parametrize("new", [1, 3, 70])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_infinities_and_nan_in_q_stay_in_their_rows(new, dtype):
    def change(q, c, table):
        change.clean = q.clone()
        q[0, 1, 5], q[0, 3, 0], q[-1, 0, 7] = math.nan, math.inf, -math.inf
    g = gen(3)
    cu, seq, table, pages = batch([100, 37], [new, new], 16)
    c = filled_cache(g, "new", pages, 16, 2, 128)
    q = torch.randn(2 * new, 10, 128, device="cuda", generator=g).to(dtype)
    clean = paged8.paged_attention8(q, *c, table, cu, seq, 0.09)
    change(q, c, table)
    got = paged8.paged_attention8(q, *c, table, cu, seq, 0.09)
    bad = torch.zeros(2 * new, 10, dtype=torch.bool, device="cuda")
    bad[0, 1] = bad[0, 3] = bad[-1, 0] = True
    assert torch.equal(got[~bad], clean[~bad]) and bool(got[0, 1].isnan().all())


@pytest.mark.parametrize("new", [1, 4, 90])
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_what_nobody_sees_may_be_anything(new, window, d):
    """Any bytes and scales after a request's last token, before its window, in unused pages, and table entries that are no
    page: the same bits."""
    page, ctx = 32, [70, 201, 5]
    g = gen(new + d)
    cu, seq, table, pages = batch(ctx, [new] * 3, page, spare=3)
    c = filled_cache(g, "new", pages, page, 2, d)
    q = torch.randn(3 * new, 8, d, device="cuda", generator=g).half()
    clean = paged8.paged_attention8(q, *c, table, cu, seq, d ** -0.5, window)
    seen = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    for r, a in enumerate(ctx):
        for p in range(max(0, a + 1 - window) if window else 0, a + new):
            seen[table[r, p // page].item(), p % page] = True
    blocks = seen.view(pages, page // BLOCK, BLOCK).any(-1)
    for codes in c[:2]:
        codes[~seen] = torch.randint(-128, 128, codes[~seen].shape, device="cuda", generator=g, dtype=torch.int8)
    for bad in (math.nan, math.inf, -math.inf, 0.0, -3.0, 3e38):
        for s in c[2:]:
            s[~blocks] = bad
        assert torch.equal(paged8.paged_attention8(q, *c, table, cu, seq, d ** -0.5, window), clean), bad
    for entry in (-1, pages, 2 ** 31 - 1, -2 ** 31):
        t = table.clone()
        for r, a in enumerate(ctx):
            t[r, -(-(a + new) // page):] = entry
            if window:
                t[r, :max(0, a + 1 - window) // page] = entry
        assert torch.equal(paged8.paged_attention8(q, *c, t, cu, seq, d ** -0.5, window), clean), entry


@pytest.mark.parametrize("new", [1, 40])
def test_missing_pages_and_short_tables(new):
    """Positions without a page, or past the table's columns, are left out; a request without any page gives zeros."""
    def change(q, c, table):
        table[0, 2], table[0, 4] = -1, 10 ** 6
        table[1] = -1
    check_attention([100, 30], [new, new], change=change)
    g = gen(4)
    cu, seq, table, pages = batch([300], [new], 16)
    c = filled_cache(g, "new", pages, 16, 2, 128)
    q = torch.randn(new, 4, 128, device="cuda", generator=g).half()
    got = paged8.paged_attention8(q, *c, table[:, :7], cu, seq, 0.1)
    want, tol = reference(q, c, table[:, :7], cu, seq, 0.1, 0, F16)
    assert bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("new", [1, 50])
def test_scales_of_very_different_sizes(new):
    """Blocks of v from 2^-40 to 2^40 and zero: keys that take the weight while their v is next to nothing count in the sum."""
    def change(q, c, table):
        for t, s in ((c[2], 0.002), (c[3], None)):
            e = torch.randint(-40, 41, t.shape, device="cuda", generator=gen(8)) if s is None else None
            t.copy_(torch.ldexp(torch.ones(t.shape, dtype=torch.float64), e.cpu()) if s is None else torch.full_like(t, s))
        c[1][::3] = 0
        c[3][::3] = 2.0 ** -40
    check_attention([400, 77], [new, new], dtype=BF16, change=change)
    check_attention([400, 77], [new, new], dtype=BF16, change=change, hq=4, hkv=2, d=256)


def test_scales_that_are_no_powers_of_two():
    def change(q, c, table):
        c[2].uniform_(0.01, 0.03)
        c[3].uniform_(0.001, 0.3)
    check_attention([300, 20], [1, 1], change=change)
    check_attention([300, 20], [70, 5], change=change)


def test_all_codes_once():
    """Every code from -128 to 127 in k and v, in every column."""
    c = make_cache("new", 16, 16, 1, 64)
    codes = (torch.arange(256, device="cuda")[:, None] + 5 * torch.arange(64, device="cuda")).remainder(256).sub(128).to(torch.int8).view(16, 16, 1, 64)
    c[0].copy_(codes), c[1].copy_(codes.flip(0))
    c[2].fill_(2.0 ** -9), c[3].fill_(2.0 ** -3)
    for new in (1, 60):
        table, cu, seq = ints([list(range(16))]), ints([0, new]), ints([256])
        q = torch.randn(new, 4, 64, device="cuda", generator=gen(new)).half()
        got = paged8.paged_attention8(q, *c, table, cu, seq, 0.05)
        want, tol = reference(q, c, table, cu, seq, 0.05, 0, F16)
        assert bool(((got.double() - want).abs() <= tol).all())


def test_every_key_counts_once():
    """v is 1 in one key's column alone: the output is that key's probability, for equal scores 1 / n."""
    n = 1000
    c = make_cache("new", 64, 16, 1, 64)
    c[2].fill_(1.0), c[3].fill_(1.0)
    for base in range(0, n, 64):
        c[1].zero_()
        for j in range(64):
            if base + j < n:
                c[1][(base + j) // 16, (base + j) % 16, 0, j] = 100
        q = torch.zeros(1, 2, 64, device="cuda", dtype=F16)
        got = paged8.paged_attention8(q, *c, ints([list(range(64))]), ints([0, 1]), ints([n]), 1.0)
        live = min(64, n - base)
        assert torch.allclose(got[0, :, :live].float(), torch.full((2, live), 0.1, device="cuda"), rtol=2.0 ** -10, atol=0)
        assert bool((got[0, :, live:] == 0).all())


def test_the_same_as_the_16_bit_cache():
    """A 16-bit cache that holds the values of this one: outputs within both kernels' roundings of each other."""
    for ctx, new in (([500, 33], [1, 1]), ([500, 33], [60, 7])):
        got, (q, c, table, cu, seq, scale, window) = check_attention(ctx, new, hq=8, hkv=2, d=128)
        slots = torch.arange(c[0].shape[0] * 16, device="cuda")
        k, v = (t.view(-1, 16, 2, 128) for t in paged8.kv_read8(*c, slots, F16))
        other = paged.paged_attention(q, k, v, table, cu, seq, scale, window)
        _, tol = reference(q, c, table, cu, seq, scale, window, F16)
        assert bool(((got.double() - other.double()).abs() <= 2 * tol).all())


def test_offsets_past_32_bits():
    """A cache of more than 4 GiB, whose last pages are used."""
    pages, page, hkv, d = 70000, 64, 8, 128
    c = paged8.new_cache8(pages, page, hkv, d)
    assert c[0].numel() > 1 << 32
    g = gen(1)
    T = 100
    k = torch.randn(T, hkv, d, device="cuda", generator=g).half()
    q = torch.randn(T, 16, d, device="cuda", generator=g).half()
    table = ints([[pages - 1, 3, pages - 2]])
    pos = torch.arange(T, device="cuda")
    slots = table[0, pos // page].long() * page + pos % page
    f = torch.zeros(0, device="cuda", dtype=torch.float64)
    paged8.rope_kv_write8(q, k, k, pos, slots, *c, f)
    rk, rv = paged8.kv_read8(*c, slots)
    step = c[2][slots // page, slots % page // BLOCK][..., None]
    assert bool(((rk.float() - k.float()).abs() <= step / 2).all()) and torch.equal(rk, rv)
    for new in (1, 40):
        cu, seq = ints([0, new]), ints([T])
        got = paged8.paged_attention8(q[:new], *c, table, cu, seq, 0.1)
        want, tol = reference(q[:new], c, table, cu, seq, 0.1, 0, F16)
        assert bool(((got.double() - want).abs() <= tol).all())
    # wide token strides: [pages, page, heads, d] views of a larger allocation
    wide = torch.zeros(40, page, 1 << 20, device="cuda", dtype=torch.int8)[..., :hkv * d].view(40, page, hkv, d)
    wide.copy_(c[0][-40:])
    t = table - (pages - 40)
    t[0, 1] = 0
    small = (wide, wide, c[2][-40:], c[2][-40:])
    got = paged8.paged_attention8(q[:1], *small, t, ints([0, 1]), ints([T]), 0.1)
    want, tol = reference(q[:1], small, t, ints([0, 1]), ints([T]), 0.1, 0, F16)
    assert bool(((got.double() - want).abs() <= tol).all())


# ---------------------------------------------------------------------------------------------
# streams, graphs, a whole step
# ---------------------------------------------------------------------------------------------
def step(x, lens, new, table, free, count, c, inv, d):
    cu, seq, pos, slots, left = paged.batch_plan(lens, new, table, free, count, c[0].shape[1], x.shape[0])
    q, k, v = (t.reshape(x.shape[0], -1, d) for t in x.split([8 * d, 2 * d, 2 * d], 1))
    q = paged8.rope_kv_write8(q, k, v, pos, slots, *c, inv)
    return paged8.paged_attention8(q, *c, table, cu, seq, d ** -0.5), seq, left, slots


@pytest.mark.parametrize("d", [64, 128, 256])
def test_steps_of_a_server_eager_and_captured(d):
    """Prompts, then decode steps: eager ones, and one graph replayed with eager work between, bit for bit the same; the
    attention against the cache's values at the end."""
    R, page, pages = 3, 16, 40
    inv = paged.rope_frequencies(d)[0]
    g = gen(d)
    prompt = torch.randn(60, 12 * d, device="cuda", generator=g).half()
    xs = [torch.randn(R + 1, 12 * d, device="cuda", generator=g).half() for _ in range(20)]          # a padding row

    def start():
        c = paged8.new_cache8(pages, page, 2, d)
        st = dict(c=c, table=torch.full((R, 12), -1, device="cuda", dtype=torch.int32), free=torch.arange(pages, device="cuda", dtype=torch.int32))
        _, seq, left, _ = step(prompt, ints([0] * R), ints([33, 1, 26]), st["table"], st["free"], ints([pages]), c, inv, d)
        return dict(st, lens=seq, count=left)

    one = ints([1] * R)
    eager, outs = start(), []
    for x in xs:
        o, eager["lens"], eager["count"], slots = step(x, eager["lens"], one, eager["table"], eager["free"], eager["count"], eager["c"], inv, d)
        outs.append(o)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        warm = start()
        step(xs[0], warm["lens"], one, warm["table"], warm["free"], warm["count"], warm["c"], inv, d)
        st, x = start(), xs[0].clone()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            o, seq, left, _ = step(x, st["lens"], one, st["table"], st["free"], st["count"], st["c"], inv, d)
            st["lens"].copy_(seq), st["count"].copy_(left)
    torch.cuda.synchronize()
    for i, xi in enumerate(xs):
        x.copy_(xi)
        graph.replay()
        if i % 3 == 0:                                  # eager work of its own between replays
            check_attention([50], [1], seed=i)
        torch.cuda.synchronize()
        assert torch.equal(o, outs[i]), i
    for a, b in zip((*st["c"], st["table"], st["lens"], st["count"]), (*eager["c"], eager["table"], eager["lens"], eager["count"])):
        assert torch.equal(a, b)
    assert eager["lens"].tolist() == [53, 21, 46] and bool((outs[-1][R] == 0).all())
    q, k, v = (t.reshape(R + 1, -1, d) for t in xs[-1].split([8 * d, 2 * d, 2 * d], 1))
    rot = torch.zeros(R + 1, dtype=torch.int64, device="cuda")
    rot[:R] = eager["lens"].long() - 1
    q = paged8.rope_kv_write8(q, k, v, rot, torch.full_like(rot, -1), *eager["c"], inv)
    want, tol = reference(q, eager["c"], eager["table"], ints([0, 1, 2, 3]), eager["lens"], d ** -0.5, 0, F16)
    assert bool(((outs[-1].double() - want).abs() <= tol).all())


def test_two_streams_at_once():
    """Calls of two streams overlap, each with its own workspace."""
    _, a = check_attention([5000, 900], [1, 1], hq=40, hkv=8, seed=1)
    _, b = check_attention([3000], [80], hq=40, hkv=8, seed=2)
    want = [paged8.paged_attention8(x[0], *x[1], *x[2:]) for x in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (s, x) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(s):
                got[i].append(paged8.paged_attention8(x[0], *x[1], *x[2:]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in (0, 1) for y in got[i])


def test_captured_read():
    c = make_cache("new", 20, 16, 2, 128, fill=gen(0))
    slots = torch.randint(-1, 320, (200,), device="cuda", generator=gen(1))
    want = paged8.kv_read8(*c, slots, BF16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = paged8.kv_read8(*c, slots, BF16)
    for shift in (0, 3, 7):
        slots.copy_((slots + shift).clamp(max=319))
        graph.replay()
        want = paged8.kv_read8(*c, slots, BF16)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_ops_keep_their_schemas_and_compile():
    g = gen(2)
    c = make_cache("new", 9, 16, 2, 64)
    q, k, v = inputs(g, 5, 4, 2, 64, F16)
    pos, slots = ints(run_of(3, 5), torch.int64), ints([4, 5, 6, -1, 40], torch.int64)
    inv = paged.rope_frequencies(64)[0]
    table, cu, seq = ints([[0, 1, 2], [2, 3, 4]]), ints([0, 3, 5]), ints([7, 41])
    op = torch.ops.exl3rocm
    check = lambda o, *a: torch.library.opcheck(o.default, a, test_utils=("test_schema", "test_faketensor"))  # noqa: E731
    check(op.rope_kv_write8, q, k, v, pos, slots, *c, inv, 1.25)
    check(op.kv_read8, *c, slots, BF16)
    check(op.paged_attention8, q, *c, table, cu, seq, 0.125)

    def whole(q, k, v, pos, slots, kc, vc, ks, vs, table, cu, seq):
        q = op.rope_kv_write8(q, k, v, pos, slots, kc, vc, ks, vs, inv, 1.25)
        return op.paged_attention8(q, kc, vc, ks, vs, table, cu, seq, 0.125), *op.kv_read8(kc, vc, ks, vs, slots)

    from torch._inductor import config
    a, b = make_cache("new", 9, 16, 2, 64), make_cache("new", 9, 16, 2, 64)
    want = whole(q, k, v, pos, slots, *a, table, cu, seq)
    with config.patch(compile_threads=1):
        got = torch.compile(whole, fullgraph=True)(q, k, v, pos, slots, *b, table, cu, seq)
    torch._dynamo.reset()
    assert all(torch.equal(x, y) for x, y in zip((*want, *a), (*got, *b)))


def test_a_stream_without_a_workspace_cannot_capture():
    _, x = check_attention([40], [1])
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="no eager call"):
        with torch.cuda.graph(graph, stream=side):
            paged8.paged_attention8(x[0], *x[1], *x[2:])
