"""GPU tests of rope_kv_write8 where a rotated key lies next to a border, by less than 32 bits tell: 127 steps of a scale.  Every scale and code is
that of the exact value.

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
from test_gpu_paged8 import BF16, F16, flat, gen, ints, make_cache, write_reference  # noqa: E402

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
