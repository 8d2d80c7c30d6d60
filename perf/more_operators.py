"""The attention step over a paged cache that is held in 8 bits: the cache's write, its reading back and the attention over
it, in their plain form and through exl3rocm's ops.

The cache: whole numbers from -127 to 127 and, for every 16 tokens of a page and kv head, a scale that is a power of two; a
value is their product.  A call that writes a block's first token starts the block anew (its scale is the smallest
that holds what the call writes, its other rows 0); otherwise the scale stays, or grows to what the new rows need, and
then the block's other rows are rounded to the new step.

A case names one operator ("op") and its sizes:
  write  rotary embedding of q and k, with k and v quantised into the cache; then every block that it touched, read back
  read   a batch's cached tokens, read back into the element type
  attn   attention of each request's new tokens over its cached ones, causal, with or without a window
Requests' lengths follow from the case alone (`ragged` seeds them); tensors' values from the seed.

  reqs          requests of the batch; ctx_lo, ctx_hi: range of their cached tokens (spread over the logarithm)
  new_lo, new_hi  range of the new tokens of a request; big: one more request with that many
                (0: none) after big_ctx cached ones
  page          tokens of a cache page
  hq, hkv, d    query heads, key/value heads, head width; dtype "float16" or "bfloat16"
  rot, interleaved   rotated part of a head, pair layout
  gated         q comes as [q | gate] per head, so its heads lie 2 d apart
  window        keys a token sees, itself included (0: all)
"""
import math
import os
import random
import sys

import torch

own = False

_REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PKG = os.path.join(_REPO, "qwen38-27b-exl3-rdna4_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

BLOCK = 16
GQA = dict(hq=40, hkv=8, d=128)        # the heads of the 5120-wide decoder with 1024-wide k and v
GATED = dict(hq=24, hkv=4, d=256)      # the checkpoint's attention: 6144 of q (and as much gate), 1024 of k and v


def listed():
    return [
        # a decode step of 32 sequences: latency, every token inside a block of its own
        dict(name="write_decode_t32", op="write", reqs=32, ctx_lo=1, ctx_hi=16384, new_lo=1, new_hi=1, big=0, page=16, **GQA,
             dtype="float16", rot=128, interleaved=False, gated=False, ragged=3),
        # ragged prompts behind cached tokens, so their first blocks are partly filled; a quarter of each head rotated
        dict(name="write_ragged_t894", op="write", reqs=6, ctx_lo=500, ctx_hi=60000, new_lo=9, new_hi=190, big=333, page=64, **GATED,
             dtype="bfloat16", rot=64, interleaved=False, gated=True, ragged=4),
        # a large prefill step, pairs side by side
        dict(name="write_prefill_t8192", op="write", reqs=0, ctx_lo=0, ctx_hi=0, new_lo=0, new_hi=0, big=8192, page=16, **GQA,
             dtype="float16", rot=128, interleaved=True, gated=False, ragged=5),
        # a short conversation's cache, handed to another server
        dict(name="read_r1", op="read", reqs=1, ctx_lo=700, ctx_hi=700, new_lo=0, new_hi=0, big=0, page=16, **GQA,
             dtype="float16", ragged=6),
        # a shared prefix of many requests and two long documents
        dict(name="read_long", op="read", reqs=9, ctx_lo=900, ctx_hi=120000, new_lo=0, new_hi=0, big=0, page=64, **GATED,
             dtype="bfloat16", ragged=7),
        # a single stream's decode at a short context: latency
        dict(name="attn8_decode_r1", op="attn", reqs=1, ctx_lo=1500, ctx_hi=1500, new_lo=1, new_hi=1, big=0, page=16, **GQA,
             dtype="float16", window=0, ragged=8),
        # a server's decode step: 96 sequences of very different lengths, as half the bytes a token let it hold
        dict(name="attn8_decode_r96", op="attn", reqs=96, ctx_lo=100, ctx_hi=16000, new_lo=1, new_hi=1, big=0, page=16, **GQA,
             dtype="float16", window=0, ragged=9),
        # two streams deep in a long document
        dict(name="attn8_decode_long", op="attn", reqs=2, ctx_lo=120000, ctx_hi=262143, new_lo=1, new_hi=1, big=0, page=64, **GATED,
             dtype="bfloat16", window=0, ragged=10),
        # speculative decoding's verification: twelve streams of one token and three drafts
        dict(name="attn8_verify_r12", op="attn", reqs=12, ctx_lo=1000, ctx_hi=32000, new_lo=4, new_hi=4, big=0, page=16, **GATED,
             dtype="float16", window=0, ragged=11),
        # a chunk in the middle of a long prompt
        dict(name="attn8_chunk_long", op="attn", reqs=0, ctx_lo=0, ctx_hi=0, new_lo=0, new_hi=0, big=2048, big_ctx=12000, page=16, **GQA,
             dtype="bfloat16", window=0, ragged=12),
        # a long prompt's later chunk with wide heads, an odd number of tokens
        dict(name="attn8_chunk_wide", op="attn", reqs=0, ctx_lo=0, ctx_hi=0, new_lo=0, new_hi=0, big=1501, big_ctx=9001, page=48, **GATED,
             dtype="float16", window=0, ragged=13),
        # decodes beside a prompt's chunk, small heads, sliding window
        dict(name="attn8_mixed_window", op="attn", reqs=7, ctx_lo=10, ctx_hi=6000, new_lo=1, new_hi=1, big=509, big_ctx=1777, page=32,
             hq=32, hkv=8, d=64, dtype="bfloat16", window=1024, ragged=14),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "write", "read", "attn", "attn", "attn"])
    c = dict(op=op, page=rng.choice([16, 16, 32, 48, 64, 128]), ragged=rng.randrange(1 << 20), ctx_lo=1, big=0, new_lo=0, new_hi=0)
    c.update(rng.choice([GQA, GATED, dict(hq=32, hkv=8, d=64), dict(hq=16, hkv=16, d=128), dict(hq=28, hkv=4, d=128),
                         dict(hq=12, hkv=1, d=128), dict(hq=rng.randint(1, 9) * 3, hkv=3, d=64)]), dtype=rng.choice(["float16", "bfloat16"]))
    most = 230_000_000                   # cached values of either kind that the requests' longest lengths would take
    if op == "write":
        t = _log_int(rng, 1, 8000)
        c["reqs"] = rng.randint(1, min(t, 64))
        c.update(ctx_hi=_log_int(rng, 16, max(16, min(250000, most // (c["reqs"] * c["hkv"] * c["d"])))),
                 rot=rng.choice([c["d"], c["d"], c["d"] // 2, c["d"] // 4, 2 * rng.randint(1, c["d"] // 2)]),
                 interleaved=rng.random() < 0.4, gated=rng.random() < 0.3)
        c["new_lo"] = c["new_hi"] = t // c["reqs"]
        return c
    if op == "read":
        c["ctx_hi"] = _log_int(rng, 16, 100000)
        c["ctx_lo"] = rng.choice([1, c["ctx_hi"]])
        c["reqs"] = max(1, min(_log_int(rng, 1, 32), most // (c["ctx_hi"] * c["hkv"] * c["d"])))
        return c
    kind = rng.choice(["decode", "decode", "verify", "chunk", "mixed"])
    longest = 16384 if kind != "decode" else 131072
    c.update(window=rng.choice([0, 0, 0, _log_int(rng, 1, 8192)]), big_ctx=0, reqs=0, ctx_hi=0)
    if kind in ("decode", "verify", "mixed"):
        c["ctx_hi"] = _log_int(rng, 16, longest)
        c["ctx_lo"] = rng.choice([1, max(1, c["ctx_hi"] // 4), c["ctx_hi"]])
        c["reqs"] = max(1, min(_log_int(rng, 1, 128), most // (c["ctx_hi"] * c["hkv"] * c["d"])))
        c["new_lo"] = 1
        c["new_hi"] = 1 if kind != "verify" else rng.randint(2, 8)
    if kind in ("chunk", "mixed"):
        if kind == "mixed":
            c["reqs"], c["ctx_hi"] = min(c["reqs"], 7), min(c["ctx_hi"], 6000)
            c["ctx_lo"] = min(c["ctx_lo"], c["ctx_hi"])
        c["big"] = _log_int(rng, 16, 2000 if kind == "chunk" else 512)
        c["big_ctx"] = rng.choice([0, _log_int(rng, 1, 12000 if kind == "chunk" else 5000)])
    return c


# ---------------------------------------------------------------------------------------------
# lengths, and what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def _lengths(c):
    """(cached tokens, new tokens) of every request, from the case alone."""
    rng = random.Random(c["ragged"])
    ctx = [_log_int(rng, max(1, c["ctx_lo"]), max(1, c["ctx_hi"])) for _ in range(c["reqs"])]
    new = [rng.randint(c["new_lo"], c["new_hi"]) for _ in range(c["reqs"])]
    if c["big"]:
        at = rng.randint(0, c["reqs"])
        ctx.insert(at, c.get("big_ctx", 0))
        new.insert(at, c["big"])
    return ctx, new


def _up(a, b):
    return -(-a // b)


def _visible(ctx, new, window):
    """(token, key) pairs of one request, and the keys that any of its tokens sees."""
    if not window:
        return new * ctx + new * (new + 1) // 2, ctx + new if new else 0
    pairs = sum(min(ctx + i + 1, window) for i in range(new))
    return pairs, ctx + new - max(0, ctx + 1 - window) if new else 0


def work(case):
    ctx, new = _lengths(case)
    total, hq, hkv, d = sum(new), case["hq"], case["hkv"], case["d"]
    row = 2 * hkv * d                      # a token's k and v, values
    scales = 8 * hkv                       # a block's, bytes
    if case["op"] == "write":
        blocks = sum(_up(a + b, BLOCK) - a // BLOCK for a, b in zip(ctx, new) if b)
        write = total * (4 * hq * d + 2 * row + 16 + row) + 2 * blocks * scales
        return {"bytes": write + blocks * BLOCK * (3 * row + 8) + blocks * scales + 4 * case["rot"],
                "flops": 3 * total * (hq + hkv) * case["rot"] + 4 * total * row + blocks * BLOCK * row}
    if case["op"] == "read":
        t = sum(ctx)
        return {"bytes": t * (3 * row + 8) + sum(_up(a, BLOCK) for a in ctx) * scales, "flops": t * row}
    seen = [_visible(a, b, case["window"]) for a, b in zip(ctx, new)]
    keys = sum(k for _, k in seen)
    return {"bytes": keys * row + _up(keys, BLOCK) * scales + 4 * total * hq * d, "flops": 4 * d * hq * sum(p for p, _ in seen)}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _scale_of(amax):
    """The smallest power of two (2^-40 to 2^40) of which 127 reach amax."""
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, e - torch.where(m > 127 / 128, 6, 7), -40)
    return ((e.clamp(-40, 40) + 127) << 23).int().view(torch.float32)    # by its bits: a computed power can be off by one


def _spread(g, *shape):
    """Values of k or v as a head has them: some channels several times as large as others, tokens of different norms."""
    x = torch.randn(*shape, device="cuda", generator=g)
    x *= torch.exp(0.7 * torch.randn(shape[1], 1, shape[-1], device="cuda", generator=g))
    return x.mul_(torch.exp(0.3 * torch.randn(*shape[:-1], 1, device="cuda", generator=g)))


def _cache(g, pages, page, hkv, d):
    """(codes [pages, page, hkv, d], scales [pages, page / 16, hkv]); a page holds each head's tokens together."""
    x = _spread(g, pages, hkv, page, d).view(pages, hkv, page // BLOCK, BLOCK, d)
    s = _scale_of(x.abs().amax((-1, -2)))
    codes = (x / s[..., None, None]).round_().clamp_(-127, 127).to(torch.int8)
    return codes.view(pages, hkv, page, d).transpose(1, 2), s.transpose(1, 2)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 29)
    ctx, new = _lengths(case)
    page, total, n = case["page"], sum(new), len(ctx)
    held = [_up(a + b, page) for a, b in zip(ctx, new)]
    pages = sum(held) + 3 + sum(held) // 8
    order = torch.randperm(pages, device="cuda", generator=g).int()
    ints = lambda v, t=torch.int32: torch.tensor(v, device="cuda", dtype=t)  # noqa: E731
    hq, hkv, d, dtype = case["hq"], case["hkv"], case["d"], getattr(torch, case["dtype"])
    first = ints([sum(held[:i]) for i in range(n)])
    col = torch.arange(max(held), device="cuda", dtype=torch.int32)
    table = torch.where(col < ints(held)[:, None], order[(first[:, None] + col).clamp_max(pages - 1).long()], -1).contiguous()
    (kc, ks), (vc, vs) = (_cache(g, pages, page, hkv, d) for _ in range(2))
    st = dict(op=case["op"], page=page, total=total, reqs=n, kc=kc, vc=vc, ks=ks, vs=vs, dtype=dtype)

    def tokens(lo, hi):
        """(request, position) of the tokens [lo, hi) of every request."""
        count = ints([b - a for a, b in zip(lo, hi)]).long()
        size = sum(hi) - sum(lo)
        req = torch.repeat_interleave(torch.arange(n, device="cuda"), count, output_size=size)
        return req, ints(lo).long()[req] + torch.arange(size, device="cuda") - (torch.cumsum(count, 0) - count)[req]

    def slots(req, pos):
        return table[req, pos // page].long() * page + pos % page

    if case["op"] == "read":
        st["slots"] = slots(*tokens([0] * n, ctx))
        return st
    if case["op"] == "write":
        # q, k and v as columns of the fused projection's output rows
        wq = hq * d * (2 if case["gated"] else 1)
        rows = torch.empty(total, wq + 2 * hkv * d, device="cuda", dtype=dtype)
        rows[:, :wq] = torch.randn(total, wq, device="cuda", generator=g)
        kv = _spread(g, total, 2 * hkv, 1, d)
        rows[:, wq:] = kv.view(total, -1)
        q = rows[:, :wq].view(total, hq, -1)[:, :, :d]
        k, v = (rows[:, wq + i * hkv * d:wq + (i + 1) * hkv * d].view(total, hkv, d) for i in range(2))
        req, pos = tokens(ctx, [a + b for a, b in zip(ctx, new)])
        f = 1e6 ** (-torch.arange(case["rot"] // 2, dtype=torch.float64) * 2.0 / case["rot"])
        # the blocks that the new tokens touch, and every slot of them
        begin, end = [a // BLOCK * BLOCK for a in ctx], [_up(a + b, BLOCK) * BLOCK if b else a // BLOCK * BLOCK for a, b in zip(ctx, new)]
        look = slots(*tokens(begin, end))
        st.update(q=q, k=k, v=v, pos=pos, slots=slots(req, pos), look=look, blocks=look[::BLOCK] // BLOCK, f=f.cuda(), rot=case["rot"],
                  interleaved=case["interleaved"])
        return st
    cu = ints([0] + [sum(new[:i + 1]) for i in range(n)])
    longest, most = max(a + b for a, b in zip(ctx, new)), max(new)
    span = min(longest, case["window"] + most - 1) if case["window"] else longest
    # queries such that a softmax is over some tens of keys, as trained heads have it
    q = torch.randn(total, hq, d, device="cuda", generator=g).to(dtype)
    st.update(q=q, table=table, cu=cu, new=ints(new), seq=ints(ctx) + ints(new), scale=d ** -0.5, window=case["window"], span=span, most_new=most)
    return st


# ---------------------------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------------------------
def _turn(x, cos, sin, rot, interleaved):
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    a, b = a * cos - b * sin, a * sin + b * cos
    head = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([head, x[..., rot:]], -1)


def _into(codes, scales, x, st):
    """x [tokens, hkv, d] (fp32) quantised into its slots."""
    page, slots, blocks = st["page"], st["slots"], st["blocks"]
    per = page // BLOCK
    most = torch.zeros(scales.shape[0] * per, x.shape[1], device="cuda")
    most.index_reduce_(0, slots // BLOCK, x.abs().amax(-1), "amax")
    anew = torch.zeros(scales.shape[0] * per, device="cuda").index_reduce_(0, slots // BLOCK, (slots % BLOCK == 0).float(), "amax")
    where = (blocks // per, blocks % per)
    old, need = scales[where], _scale_of(most[blocks])
    keep = anew[blocks][:, None] == 0
    now = torch.where(keep, torch.maximum(old, need), need)
    scales[where] = now
    at = blocks[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")
    at = (at // page, at % page)
    kept = codes[at].float() * torch.where(keep, old / now, 0.0)[:, None, :, None]
    codes[at] = kept.round_().to(torch.int8)
    step = scales[slots // page, slots % page // BLOCK]
    codes[slots // page, slots % page] = (x / step[..., None]).round_().clamp_(-127, 127).to(torch.int8)


def _read_plain(codes, scales, slots, page, dtype):
    return (codes[slots // page, slots % page].float() * scales[slots // page, slots % page // BLOCK][..., None]).to(dtype)


def _write_plain(st):
    angle = torch.remainder(st["pos"].double()[:, None] * st["f"], 2 * math.pi).float()[:, None]
    cos, sin = angle.cos(), angle.sin()
    q, k = (_turn(x.float(), cos, sin, st["rot"], st["interleaved"]) for x in (st["q"], st["k"]))
    _into(st["kc"], st["ks"], k, st)
    _into(st["vc"], st["vs"], st["v"].float(), st)
    return dict(q=q.to(st["dtype"]), k=_read_plain(st["kc"], st["ks"], st["look"], st["page"], st["dtype"]),
                v=_read_plain(st["vc"], st["vs"], st["look"], st["page"], st["dtype"]))


def _attn_plain(st):
    q, page, span, most = st["q"], st["page"], st["span"], st["most_new"]
    total, hq, d = q.shape
    hkv = st["kc"].shape[2]
    i = torch.arange(most, device="cuda")
    j = (st["seq"] - span).clamp_min(0).long()[:, None] + torch.arange(span, device="cuda")   # the keys that a token may see
    p, o = st["table"].gather(1, j // page).clamp_min(0).long(), j % page
    # [reqs, hkv, span, d]
    k, v = (c[p, o].float().mul_(s[p, o // BLOCK][..., None]).transpose(1, 2) for c, s in ((st["kc"], st["ks"]), (st["vc"], st["vs"])))
    live = i < st["new"][:, None]
    rows = torch.where(live, st["cu"][:-1, None] + i, total)
    qs = torch.nn.functional.pad(q, (0, 0, 0, 0, 0, 1))[rows].float()                     # [reqs, most, hq, d]
    qs = qs.view(-1, most, hkv, hq // hkv, d).transpose(1, 2).flatten(2, 3)
    s = (qs @ k.transpose(-1, -2)).mul_(st["scale"]).view(-1, hkv, most, hq // hkv, span)
    at = (st["seq"] - st["new"])[:, None] + i
    seen = (j[:, None] <= at[..., None]) & live[..., None]
    if st["window"]:
        seen &= j[:, None] > at[..., None] - st["window"]
    s.masked_fill_(~seen[:, None, :, None], -math.inf)
    e = s.sub_(s.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    r = (e.flatten(2, 3) @ v) / e.sum(-1).flatten(2, 3).clamp_min(1e-30)[..., None]
    r = r.view(-1, hkv, most, hq // hkv, d).transpose(1, 2).reshape(-1, most, hq, d)
    out = torch.zeros(total + 1, hq, d, device="cuda", dtype=q.dtype)
    out[rows] = r.to(q.dtype)
    return out[:total]


def run(state):
    st = state
    if not own:
        if st["op"] == "read":
            return dict(k=_read_plain(st["kc"], st["ks"], st["slots"], st["page"], st["dtype"]),
                        v=_read_plain(st["vc"], st["vs"], st["slots"], st["page"], st["dtype"]))
        return _write_plain(st) if st["op"] == "write" else _attn_plain(st)
    from exl3rocm import paged8
    cache = (st["kc"], st["vc"], st["ks"], st["vs"])
    if st["op"] == "read":
        k, v = paged8.kv_read8(*cache, st["slots"], st["dtype"])
        return dict(k=k, v=v)
    if st["op"] == "write":
        q = paged8.rope_kv_write8(st["q"], st["k"], st["v"], st["pos"], st["slots"], *cache, st["f"], 1.0, st["interleaved"])
        k, v = paged8.kv_read8(*cache, st["look"], st["dtype"])
        return dict(q=q, k=k, v=v)
    return paged8.paged_attention8(st["q"], *cache, st["table"], st["cu"], st["seq"], st["scale"], st["window"])


# ---------------------------------------------------------------------------------------------
# the same in 64 bits, block by block and request by request
# ---------------------------------------------------------------------------------------------
def _exact_blocks(codes, scales, x, st):
    """The touched blocks' values [blocks * 16, hkv, d] after x [tokens, hkv, d] (64 bits) went into their slots."""
    page, hkv, d = st["page"], x.shape[1], x.shape[2]
    powers = torch.tensor([math.ldexp(1.0, e) for e in range(-40, 41)], device="cuda", dtype=torch.float64)
    of_block = {}
    for t, s in enumerate(st["slots"].tolist()):
        of_block.setdefault(s // BLOCK, []).append((t, s % BLOCK))
    out = []
    for b in st["blocks"].tolist():
        p, o = b * BLOCK // page, b * BLOCK % page
        old = codes[p, o:o + BLOCK].double() * scales[p, o // BLOCK].double()[None, :, None]
        t, r = (torch.tensor(v, device="cuda") for v in zip(*of_block[b]))
        most = x[t].abs().amax((0, 2))
        step = powers[(127.0 * powers[:, None] < most).sum(0).clamp_max(80)]
        if of_block[b][0][1] == 0:
            old = torch.zeros_like(old)
        else:
            step = torch.maximum(step, scales[p, o // BLOCK].double())
        old[r] = x[t]
        out.append(torch.clamp(torch.round(old / step[None, :, None]), -127, 127) * step[None, :, None])
    return torch.cat(out).view(-1, hkv, d)


def exact(case, seed):
    st = prepare(case, seed)
    page = st["page"]
    if case["op"] == "read":
        s = st["slots"]
        return {n: c.flatten(0, 1)[s].double() * sc.repeat_interleave(BLOCK, 1).flatten(0, 1)[s].double()[..., None]
                for n, c, sc in (("k", st["kc"], st["ks"]), ("v", st["vc"], st["vs"]))}
    if case["op"] == "write":
        # the pair (a, b) as a complex number, times e^(i position frequency)
        angle = st["pos"].double()[:, None] * st["f"]
        turn = torch.polar(torch.ones_like(angle), angle)
        rot, out = st["rot"], []
        lo, hi = ((slice(0, rot, 2), slice(1, rot, 2)) if st["interleaved"] else (slice(0, rot // 2), slice(rot // 2, rot)))
        for x in (st["q"], st["k"]):
            y = x.double().clone()
            z = torch.complex(y[..., lo], y[..., hi]) * turn[:, None]
            y[..., lo], y[..., hi] = z.real, z.imag
            out.append(y)
        return dict(q=out[0], k=_exact_blocks(st["kc"], st["ks"], out[1], st), v=_exact_blocks(st["vc"], st["vs"], st["v"].double(), st))
    ctx, new = _lengths(case)
    hq, hkv, d, w = case["hq"], case["hkv"], case["d"], case["window"]
    out, t0 = torch.zeros(st["total"], hq, d, device="cuda", dtype=torch.float64), 0
    for r, (a, b) in enumerate(zip(ctx, new)):
        if not b:
            continue
        n = a + b
        held = st["table"][r, :_up(n, page)].long()
        key = torch.arange(n, device="cuda")
        for h in range(hkv):
            kk, vv = ((c[held, :, h].double() * s[held, :, h].double().repeat_interleave(BLOCK, 1)[..., None]).reshape(-1, d)[:n]
                      for c, s in ((st["kc"], st["ks"]), (st["vc"], st["vs"])))
            heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            # queries in pieces: 64-bit scores of at most about a gigabyte
            step = max(1, 134_000_000 // (n * (hq // hkv)))
            for i in range(0, b, step):
                qq = st["q"][t0 + i:t0 + min(b, i + step), heads].double()
                at = a + i + torch.arange(qq.shape[0], device="cuda")[:, None]
                s = (qq.reshape(-1, d) @ kk.T).view(qq.shape[0], -1, n) * st["scale"]
                off = (key > at) | (key <= at - w) if w else key > at
                s = s.masked_fill(off[:, None], -math.inf)
                out[t0 + i:t0 + i + qq.shape[0], heads] = torch.softmax(s, -1) @ vv
        t0 += b
    return out
