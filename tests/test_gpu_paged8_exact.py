"""GPU tests of rope_kv_write8 where a rotated key lies next to a border, by less than 32 bits tell: 127 steps of a scale, or the middle
between two codes.  Every scale and code is that of the exact value.

A pair (a, b) = r (cos p, sin p) turned by t has the first element r cos(p + t).  At position 1 the angle is the frequency, any float64 number, so
t = acos(x / r) - p puts the element at any x below r; what float64 loses of it (2^-50) is far below the distances 2^-30 and 2^-40 from the
border, and those far below what fp32 resolves (2^-24).  r is at most 1.3 |x|, so the second element is below 0.84 |x|.
"""
import math
import random

import pytest
import torch

pytest.importorskip("exl3rocm.paged8")
from exl3rocm import paged8  # noqa: E402
from test_gpu_paged8 import BF16, F16, flat, gen, ints, least_scale, make_cache, write_reference  # noqa: E402

pytestmark = pytest.mark.gpu

NEAR = [2.0 ** -30, -2.0 ** -30, 2.0 ** -40, -2.0 ** -40]
LAYOUTS = [(64, 64, False), (128, 128, False), (256, 64, False), (128, 22, False), (64, 6, False), (64, 64, True), (256, 256, True)]


def pair_at(rng, x, dtype):
    """(a, b, angle): a pair of dtype's numbers whose first element, turned by the angle, is x."""
    while True:
        r = abs(x) * rng.uniform(1.03, 1.28)
        p = rng.uniform(0, 2 * math.pi)
        a, b = torch.tensor([r * math.cos(p), r * math.sin(p)]).to(dtype).double().tolist()
        r, p = math.hypot(a, b), math.atan2(b, a)
        if 1.02 * abs(x) < r < 1.3 * abs(x):
            t = (rng.choice((1, -1)) * math.acos(x / r) - p) % (2 * math.pi)
            assert abs((a * math.cos(t) - b * math.sin(t)) / x - 1) < 2.0 ** -48
            return a, b, t


def columns(rot, interleaved, j):
    return (2 * j, 2 * j + 1) if interleaved else (j, j + rot // 2)


def turned(k, freq, rot, interleaved, mscale):
    """k [T, heads, d] (float64) at position 1."""
    y = k.clone()
    for j, f in enumerate(freq):
        lo, hi = columns(rot, interleaved, j)
        c, s = math.cos(f), math.sin(f)
        y[..., lo], y[..., hi] = (k[..., lo] * c - k[..., hi] * s) * mscale, (k[..., lo] * s + k[..., hi] * c) * mscale
    return y


def check(k, freq, rot, interleaved, mscale, slots, dtype, seed):
    """k [T, 2, d], float64 numbers of dtype; the cache's blocks hold small values of a small scale."""
    T, hkv, d = k.shape
    c = make_cache("new", max(slots) // 16 + 1, 16, hkv, d, fill=gen(seed))
    for s in c[2:]:
        s.fill_(2.0 ** -12)
    codes, scales = flat(c[0], 16), flat(c[2], 16)
    write_reference(codes, scales, turned(k, freq, rot, interleaved, mscale), slots, 16)
    kt = k.to(dtype).cuda()
    assert torch.equal(kt.cpu().double().nan_to_num(7.0), k.nan_to_num(7.0))
    paged8.rope_kv_write8(kt, kt, kt, ints([1] * T, torch.int64), ints(slots, torch.int64), *c, torch.tensor(freq, dtype=torch.float64, device="cuda"),
                          mscale, interleaved)
    got = flat(c[2], 16)
    assert torch.equal(got, scales), ("scales", (got != scales).nonzero()[:4].tolist())
    got = flat(c[0], 16)
    assert torch.equal(got, codes), ("codes", (got != codes).nonzero()[:4].tolist())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("mscale", [1.0, 1.25])
@pytest.mark.parametrize("d,rot,interleaved", LAYOUTS)
def test_scale_of_a_rotated_key_is_that_of_the_exact_largest(d, rot, interleaved, mscale, dtype):
    """Each token's largest element is 127 steps, or next to nothing more or less, in a block that begins or goes on."""
    rng = random.Random(d + rot)
    for turn in range(3):
        T = rot // 2
        k, freq, slots = torch.zeros(T, 2, d, dtype=torch.float64), [], []
        for j in range(T):
            x = rng.choice((1, -1)) * 127.0 * 2.0 ** rng.randint(-6, 3) * (1 + NEAR[(j + turn) % 4])
            a, b, t = pair_at(rng, x / mscale, dtype)
            lo, hi = columns(rot, interleaved, j)
            k[j, 0, lo], k[j, 0, hi] = a, b
            k[j, 1, lo], k[j, 1, hi] = a / 4, b / 4
            freq.append(t)
            slots.append(16 * j + rng.choice((0, 5)))
        check(k, freq, rot, interleaved, mscale, slots, dtype, turn)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("beside", [0.0, math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("d,rot,interleaved", LAYOUTS[:4] + LAYOUTS[5:])
def test_code_of_a_rotated_key_is_that_of_its_exact_value(d, rot, interleaved, beside, dtype):
    """An element next to the middle between two codes; a neighbour that is infinite or no number changes nothing but its own pair.  The last pair
    (100, 0) is not turned and makes the scale 1."""
    rng = random.Random(d + rot)
    for turn in range(4):
        pairs = list(range(0, 8, 2))
        k, freq = torch.zeros(len(pairs), 2, d, dtype=torch.float64), [1.0] * (rot // 2)
        freq[-1] = 0.0
        lo, hi = columns(rot, interleaved, rot // 2 - 1)
        k[..., lo] = 100.0
        for i, j in enumerate(pairs):
            x = rng.choice((1, -1)) * (rng.randint(1, 60) + 0.5) * (1 + NEAR[(i + turn) % 4])
            a, b, freq[j] = pair_at(rng, x, dtype)
            lo, hi = columns(rot, interleaved, j)
            k[i, 0, lo], k[i, 0, hi] = a, b
            k[i, 1, lo], k[i, 1, hi] = -a, -b
            lo, hi = columns(rot, interleaved, j + 1)
            k[i, 0, lo], k[i, 1, hi] = beside, beside
        check(k, freq, rot, interleaved, 1.0, [16 * i + rng.choice((0, 5)) for i in range(len(pairs))], dtype, turn)


def near_middles(rng, dtype, n):
    """(values of dtype, scales): quotients that are the middle between two codes, or next to it by a unit of a scale's last place."""
    x, s = [], []
    for i in range(n):
        v = torch.tensor(rng.uniform(0.3, 3.0)).to(dtype).float()
        scale = v / (rng.randint(0, 125) + 0.5)
        for _ in range(i % 3):
            scale = torch.nextafter(scale, scale * (2.0 if i % 2 else 0.5))
        x.append(v.item() * rng.choice((1, -1))), s.append(scale.item())
    return torch.tensor(x, dtype=torch.float64), torch.tensor(s)


def check_quotients(got, quotients):
    """Codes of quotients in float64: the nearest, and either one within 2^-16 of the middle between two (127.5 steps, by a reciprocal and a product
    that are each off by 2^-24)."""
    q = quotients.clamp(-127, 127)
    open_ = (q.abs().frac() - 0.5).abs() <= 2.0 ** -16
    ok = torch.where(open_, (got - q).abs() <= 0.5 + 2.0 ** -16, got == q.round())
    assert bool(ok.all()), ok.logical_not().nonzero()[:4].tolist()
    assert bool(open_.any())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_quotients_by_a_scale_that_is_no_power_of_two(d, dtype):
    """A scale that someone else put there stays where it is large enough: v, and k turned and not turned."""
    rng, host, T, hkv, rot = random.Random(d), torch.Generator().manual_seed(d), 600, 2, 16
    x, s = near_middles(rng, dtype, T * hkv)
    c = make_cache("new", T, 16, hkv, d, fill=gen(d))
    for sc in c[2:]:
        sc.copy_(s.view(T, 1, hkv))
    k = torch.zeros(T, hkv, d, dtype=torch.float64)
    for i in range(rot, d):
        k[:, :, i] = x.view(T, hkv) if i % 7 == 0 else torch.randn(T, hkv, dtype=torch.float64, generator=host) * x.view(T, hkv).abs().clamp_max(0.3) / 4
    k = k.to(dtype).double()
    freq = [rng.uniform(0, 6) for _ in range(rot // 2)]
    for j in range(rot // 2):
        a, b, freq[j] = pair_at(rng, x[2 * j].item(), dtype)
        k[j, 0, j], k[j, 0, j + rot // 2] = a, b
    v = k.roll(1, -1)
    slots = [16 * t + 5 for t in range(T)]
    y = turned(k, freq, rot, False, 1.0)
    kt, vt = k.to(dtype).cuda(), v.to(dtype).cuda()
    paged8.rope_kv_write8(kt, kt, vt, ints([1] * T, torch.int64), ints(slots, torch.int64), *c, torch.tensor(freq, dtype=torch.float64, device="cuda"))
    for i, new in ((0, y), (1, v)):
        scales = flat(c[i + 2], 16)
        need = torch.tensor([[least_scale(m) for m in row] for row in new.abs().amax(-1).tolist()], dtype=torch.float64)
        assert torch.equal(scales, torch.maximum(s.double().view(T, hkv), need)) and bool((scales > need).any())
        check_quotients(flat(c[i], 16)[slots], new / scales[:, :, None])


def test_rows_rounded_anew_from_a_scale_that_is_no_power_of_two():
    """Codes c of a scale that makes c * scale the middle between two steps of the new scale, or next to it."""
    rng, T = random.Random(1), 500
    c = make_cache("new", T, 16, 1, 64)
    for t in range(T):
        code = rng.choice([i for i in range(-127, 128) if i])
        s = torch.tensor(4.0 * (rng.randint(0, max(abs(code) // 4 - 1, 0)) + 0.5) / abs(code))       # the new scale is 4
        for _ in range(t % 3):
            s = torch.nextafter(s, s * (2.0 if t % 2 else 0.5))
        c[0][t, :, 0, :] = code
        c[2][t] = s.cuda()
    k = torch.full((T, 1, 64), 500.0, device="cuda", dtype=F16)
    new = [16 * t + t % 15 + 1 for t in range(T)]
    old = flat(c[0], 16) * flat(c[2], 16).repeat_interleave(16, 0)[:, :, None]
    paged8.rope_kv_write8(k, k, k, ints([0] * T, torch.int64), ints(new, torch.int64), *c, torch.zeros(0, device="cuda", dtype=torch.float64))
    assert bool((c[2] == 4.0).all())
    old[new] = 500.0
    check_quotients(flat(c[0], 16), old / 4.0)


def test_a_value_is_off_by_up_to_a_127th_of_its_blocks_largest():
    """63.6 needs a scale of 1, so 0.5 is stored as 0: more than a 128th of the largest off."""
    c = make_cache("new", 1, 16, 1, 64)
    k = torch.full((1, 1, 64), 0.5, device="cuda", dtype=F16)
    k[..., 0] = 63.59375
    paged8.rope_kv_write8(k, k, k, ints([0], torch.int64), ints([0], torch.int64), *c, torch.zeros(0, device="cuda", dtype=torch.float64))
    got = paged8.kv_read8(*c, ints([0], torch.int64))[0]
    off = (got - k).abs().max().item()
    assert c[2].flatten().tolist() == [1.0] and 63.59375 / 128 < off <= 63.59375 / 127
