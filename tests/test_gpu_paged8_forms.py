"""GPU tests of forms of the 8-bit cache's kernels that only large calls take: prompt tiles of 256 rows, decodes whose tiles many workgroups share, and
writes whose workgroups have many heads.  Bounds as in test_gpu_paged8.py."""
import math

import pytest
import torch

pytest.importorskip("exl3rocm.paged8")
from exl3rocm import paged8  # noqa: E402
from test_gpu_paged8 import BF16, F16, check_attention, check_write, flat, gen, inputs, ints, make_cache, reference, run_of  # noqa: E402

pytestmark = pytest.mark.gpu


# ---- chunks of heads of 128 with more than 4096 rows a request and kv head: tiles of 256 rows ----
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("ctx,new", [([0], [103]), ([0], [128]), ([333], [131]), ([17, 500], [150, 107]), ([1000, 0, 5], [1, 330, 2])])
def test_wide_tiles(ctx, new, dtype):
    """Rows that end inside a tile, a fresh prompt, requests beside each other, decodes beside a prompt."""
    check_attention(ctx, new, hq=40, hkv=1, dtype=dtype, page=32)


@pytest.mark.parametrize("window", [1, 16, 100, 700])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_wide_tiles_with_a_window(window, dtype):
    check_attention([70, 900], [120, 111], hq=40, hkv=1, dtype=dtype, window=window, seed=window)


@pytest.mark.parametrize("layout", ["new", "tokens", "gaps"])
@pytest.mark.parametrize("page", [16, 48, 80, 256])
def test_wide_tiles_pages_and_layouts(page, layout):
    """Pages that end inside a step, padding rows."""
    check_attention([200, 0], [110, 141], hq=80, hkv=2, dtype=BF16, page=page, layout=layout, pad=37, seed=page)


@pytest.mark.parametrize("window", [0, 90])
def test_wide_tiles_without_some_pages(window):
    def change(q, c, table):
        table[0, 1], table[0, 3], table[0, 6] = -1, 10 ** 6, -1
        table[1, 4:] = -1
    check_attention([100, 30], [130, 120], hq=40, hkv=1, window=window, change=change)


@pytest.mark.parametrize("scale,dtype", [(-0.1, F16), (0.0, BF16), (2.0, BF16)])
def test_wide_tiles_scale_of_scores(scale, dtype):
    check_attention([50], [115], hq=40, hkv=1, dtype=dtype, scale=scale)


@pytest.mark.parametrize("ctx,new", [([9000], [104]), ([30000], [105]), ([2500, 12000], [104, 106])])
def test_wide_tiles_in_many_parts(ctx, new):
    check_attention(ctx, new, hq=40, hkv=1, dtype=BF16, seed=5)


@pytest.mark.parametrize("hq,hkv,d", [(40, 8, 128), (12, 2, 256), (8, 2, 64)])
def test_many_decodes_beside_a_chunk_in_one_call_and_in_two(hq, hkv, d):
    """One call takes the decode kernel for all; of two, the second takes the prompt kernel."""
    R = 60
    ctx, new = [(53 * i) % 700 for i in range(R)] + [900], [1] * R + [120]
    got, (q, c, table, cu, seq, scale, window) = check_attention(ctx, new, hq=hq, hkv=hkv, d=d)
    want, tol = reference(q, c, table, cu, seq, scale, window, F16)
    for rows, reqs in ((slice(0, R), slice(0, R)), (slice(R, R + 120), slice(R, R + 1))):
        part = paged8.paged_attention8(q[rows], *c, table[reqs], cu[reqs.start:reqs.stop + 1] - cu[reqs.start], seq[reqs], scale, window)
        assert bool(((part.double() - want[rows]).abs() <= tol[rows]).all())


# ---- decodes and drafts over tiles that more than 64 and more than 256 workgroups share ----
@pytest.mark.parametrize("ctx,new,hq,hkv,d,dtype", [
    ([140000], [1], 12, 1, 128, F16), ([140000], [1], 12, 1, 64, BF16), ([140000], [1], 16, 1, 256, BF16),              # 438, 438 and 244 workgroups
    ([35000], [1], 5, 1, 128, BF16), ([100000, 39000], [1, 1], 7, 1, 128, F16), ([90000, 11, 60000], [1, 1, 1], 6, 1, 64, F16),
    ([70000], [2], 16, 2, 128, F16), ([140000], [1], 24, 1, 128, BF16), ([140000], [2], 12, 1, 256, F16), ([50000, 80000], [3, 3], 8, 1, 64, BF16)])
def test_decodes_in_many_parts(ctx, new, hq, hkv, d, dtype):
    check_attention(ctx, new, hq=hq, hkv=hkv, d=d, dtype=dtype, page=64, seed=6)


def test_decodes_in_many_parts_with_a_window():
    check_attention([150000], [1], hq=12, hkv=1, page=64, window=100001, seed=7)


# ---- writes of many tokens: up to all heads a workgroup ----
@pytest.mark.parametrize("T,hkv,d", [(1300, 8, 128), (1300, 8, 64), (2900, 8, 128), (4100, 8, 64), (4100, 5, 256), (4200, 16, 64)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_writes_of_several_heads_a_workgroup(T, hkv, d, dtype):
    """Blocks that begin and blocks that go on, whose rows are rounded anew under a larger scale; parts of 3, 3 and 2 heads, 6 and 2, and all."""
    slots, at = [], 5
    while len(slots) < T:
        n = (200, 1, 33, 16, 7, 500)[len(slots) % 6]
        slots += run_of(at, n)
        at += n + 17 + n % 13
    slots = slots[:T]

    def scales(c):
        for s in c[2:]:
            s.copy_(2.0 ** torch.randint(-14, -2, s.shape, device="cuda", generator=gen(T)).cpu().double())
    check_write(T, slots, hq=hkv, hkv=hkv, d=d, dtype=dtype, pages=at // 16 + 2, seed=T, scales=scales)


@pytest.mark.parametrize("d,rot,interleaved", [(128, 128, False), (64, 32, True), (128, 22, False)])
def test_rotated_writes_of_several_heads_a_workgroup(d, rot, interleaved):
    """Every head as in a call of its own: one kv head, whose workgroups have that head alone."""
    T, hkv = 4100, 8
    g = gen(rot)
    q, k, v = inputs(g, T, hkv, hkv, d, BF16)
    pos = torch.randint(0, 1 << 18, (T,), device="cuda", generator=g)
    slots = ints([s + 16 * (s // 600) for s in run_of(5, T)], torch.int64)
    inv = 10000.0 ** (-torch.arange(rot // 2, device="cuda", dtype=torch.float64) * 2 / rot)
    c = make_cache("new", 290, 16, hkv, d, fill=g)
    one = [[t[:, :, h:h + 1].clone() for t in c] for h in range(hkv)]
    out = paged8.rope_kv_write8(q, k, v, pos, slots, *c, inv, 1.0, interleaved)
    for h in range(hkv):
        o = paged8.rope_kv_write8(q[:, h:h + 1], k[:, h:h + 1], v[:, h:h + 1], pos, slots, *one[h], inv, 1.0, interleaved)
        assert torch.equal(o, out[:, h:h + 1])
        assert all(torch.equal(a, b[:, :, h:h + 1]) for a, b in zip(one[h], c)), h
    codes, sc = flat(c[1], 16), flat(c[3], 16)
    assert math.isfinite(sc.sum().item()) and bool((codes.abs() <= 127).all())
