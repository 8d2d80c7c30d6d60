"""The attention step of a decoder layer that a server runs between its q/k/v and o projections, over a paged
key/value cache: three operators, in their plain form and through exl3rocm's ops.

A case names one operator ("op") and its sizes:
  plan   the batch's block-table growth, token positions and cache slots, from the requests' lengths
  rope   rotary embedding of q and k, with k and v written into the cache
  attn   attention of each request's new tokens over its cached ones, causal, with or without a window
Requests' lengths follow from the case alone (`ragged` seeds them); tensors' values from the seed.

  reqs          requests of the batch; ctx_lo, ctx_hi: range of their cached tokens (spread over the logarithm)
  new_lo, new_hi  range of the new tokens of a request; big: one more request with that many
                (0: none) after big_ctx cached ones
  page          tokens of a cache page
  hq, hkv, d    query heads, key/value heads, head width; dtype "float16" or "bfloat16"
  rot, interleaved, scaling, factor   rotated part of a head, pair layout, long-context scaling
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

GQA = dict(hq=40, hkv=8, d=128)        # the heads of the 5120-wide decoder with 1024-wide k and v
GATED = dict(hq=24, hkv=4, d=256)      # the checkpoint's attention: 6144 of q (and as much gate), 1024 of k and v


def listed():
    return [
        # one decode step's bookkeeping for a small server batch: latency alone
        dict(name="plan_decode_r48", op="plan", reqs=48, ctx_lo=1, ctx_hi=32768, new_lo=1, new_hi=1, big=0, page=16, ragged=1),
        # continuous batching with chunked prefill: decodes, draft tokens and prompts in one step
        dict(name="plan_mixed_r300", op="plan", reqs=300, ctx_lo=1, ctx_hi=16384, new_lo=1, new_hi=40, big=4096, page=32, ragged=2),
        # a decode step of 32 sequences
        dict(name="rope_decode_t32", op="rope", reqs=32, ctx_lo=1, ctx_hi=16384, new_lo=1, new_hi=1, big=0, page=16, **GQA,
             dtype="float16", rot=128, interleaved=False, scaling="none", factor=1.0, gated=False, ragged=3),
        # ragged prompts, a quarter of each head rotated, positions stretched for a long context
        dict(name="rope_partial_ragged", op="rope", reqs=6, ctx_lo=500, ctx_hi=60000, new_lo=9, new_hi=190, big=333, page=64, **GATED,
             dtype="bfloat16", rot=64, interleaved=False, scaling="yarn", factor=4.0, gated=True, ragged=4),
        # a large prefill step, pairs side by side
        dict(name="rope_prefill_t8192", op="rope", reqs=0, ctx_lo=0, ctx_hi=0, new_lo=0, new_hi=0, big=8192, page=16, **GQA,
             dtype="float16", rot=128, interleaved=True, scaling="linear", factor=2.0, gated=False, ragged=5),
        # a single stream's decode at a short context: latency
        dict(name="attn_decode_r1", op="attn", reqs=1, ctx_lo=1500, ctx_hi=1500, new_lo=1, new_hi=1, big=0, page=16, **GQA,
             dtype="float16", window=0, ragged=6),
        # a server's decode step: 48 sequences of very different lengths
        dict(name="attn_decode_r48", op="attn", reqs=48, ctx_lo=100, ctx_hi=16000, new_lo=1, new_hi=1, big=0, page=16, **GQA,
             dtype="float16", window=0, ragged=7),
        # two streams deep in a long document
        dict(name="attn_decode_long", op="attn", reqs=2, ctx_lo=90000, ctx_hi=131071, new_lo=1, new_hi=1, big=0, page=64, **GATED,
             dtype="bfloat16", window=0, ragged=8),
        # speculative decoding's verification: eight streams of one token and three drafts
        dict(name="attn_verify_r8", op="attn", reqs=8, ctx_lo=1000, ctx_hi=32000, new_lo=4, new_hi=4, big=0, page=16, **GATED,
             dtype="float16", window=0, ragged=9),
        # a fresh prompt of one prefill chunk
        dict(name="attn_prefill_t2048", op="attn", reqs=0, ctx_lo=0, ctx_hi=0, new_lo=0, new_hi=0, big=2048, big_ctx=0, page=16, **GQA,
             dtype="float16", window=0, ragged=10),
        # a later chunk of a long prompt
        dict(name="attn_chunk_long", op="attn", reqs=0, ctx_lo=0, ctx_hi=0, new_lo=0, new_hi=0, big=2048, big_ctx=14000, page=16, **GQA,
             dtype="bfloat16", window=0, ragged=11),
        # decodes beside a prompt's chunk, small heads, sliding window
        dict(name="attn_mixed_window", op="attn", reqs=7, ctx_lo=10, ctx_hi=6000, new_lo=1, new_hi=1, big=509, big_ctx=1777, page=32,
             hq=32, hkv=8, d=64, dtype="bfloat16", window=1024, ragged=12),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "rope", "attn", "attn", "attn"])
    c = dict(op=op, page=rng.choice([16, 16, 32, 48, 64, 128]), ragged=rng.randrange(1 << 20), ctx_lo=1)
    if op == "plan":
        c.update(reqs=_log_int(rng, 1, 512), ctx_hi=_log_int(rng, 16, 32768), big=rng.choice([0, _log_int(rng, 2, 4096)]))
        c["new_lo"] = rng.choice([0, 1]) if c["big"] else 1
        c["new_hi"] = max(1, min(_log_int(rng, 1, 64), 4096 // c["reqs"]))
        return c
    heads = rng.choice([GQA, GATED, dict(hq=32, hkv=8, d=64), dict(hq=16, hkv=16, d=128), dict(hq=28, hkv=4, d=128),
                        dict(hq=12, hkv=1, d=128), dict(hq=rng.randint(1, 9) * 3, hkv=3, d=64)])
    c.update(heads, dtype=rng.choice(["float16", "float16", "bfloat16"]))
    if op == "rope":
        t = _log_int(rng, 1, 8000)
        c["reqs"] = rng.randint(1, min(t, 64))
        c.update(ctx_hi=_log_int(rng, 16, max(16, min(250000, 150_000_000 // (c["reqs"] * c["hkv"] * c["d"])))), big=0, rot=rng.choice([c["d"], c["d"], c["d"] // 2, c["d"] // 4, 2 * rng.randint(1, c["d"] // 2)]),
                 interleaved=rng.random() < 0.4, scaling=rng.choice(["none", "none", "linear", "yarn"]), factor=rng.choice([2.0, 4.0, 8.0]),
                 gated=rng.random() < 0.3)
        c["new_lo"] = c["new_hi"] = t // c["reqs"]
        return c
    kind = rng.choice(["decode", "decode", "verify", "chunk", "mixed"])
    longest = 16384 if kind != "decode" else 131072
    most = 230_000_000                   # cached values of either kind that the requests' longest lengths would take
    c.update(window=rng.choice([0, 0, 0, _log_int(rng, 1, 8192)]), big=0, big_ctx=0, reqs=0, ctx_hi=0, new_lo=0, new_hi=0)
    if kind in ("decode", "verify", "mixed"):
        c["ctx_hi"] = _log_int(rng, 16, longest)
        c["ctx_lo"] = rng.choice([1, max(1, c["ctx_hi"] // 4), c["ctx_hi"]])
        c["reqs"] = max(1, min(_log_int(rng, 1, 96), most // (c["ctx_hi"] * c["hkv"] * c["d"])))
        c["new_lo"] = 1
        c["new_hi"] = 1 if kind != "verify" else rng.randint(2, 8)
    if kind in ("chunk", "mixed"):
        if kind == "mixed":
            c["reqs"], c["ctx_hi"] = min(c["reqs"], 7), min(c["ctx_hi"], 6000)
            c["ctx_lo"] = min(c["ctx_lo"], c["ctx_hi"])
        c["big"] = _log_int(rng, 16, 2048 if kind == "chunk" else 512)
        c["big_ctx"] = rng.choice([0, _log_int(rng, 1, 13000 if kind == "chunk" else 5000)])
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


def _pages(tokens, page):
    return -(-tokens // page)


def _visible(ctx, new, window):
    """(token, key) pairs of one request, and the keys that any of its tokens sees."""
    if not window:
        return new * ctx + new * (new + 1) // 2, ctx + new if new else 0
    pairs = sum(min(ctx + i + 1, window) for i in range(new))
    return pairs, ctx + new - max(0, ctx + 1 - window) if new else 0


def work(case):
    ctx, new = _lengths(case)
    total, page = sum(new), case["page"]
    if case["op"] == "plan":
        grown = sum(_pages(a + b, page) - _pages(a, page) if b else 0 for a, b in zip(ctx, new))
        partly = sum(1 for a, b in zip(ctx, new) if b and a % page)
        return {"bytes": 8 * len(ctx) + 4 * partly + 4 * grown + 4 + 16 * total + 4 * grown + 8 * len(ctx) + 8, "flops": 0}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "rope":
        return {"bytes": 4 * total * (hq + 2 * hkv) * d + 16 * total + 4 * case["rot"], "flops": 3 * total * (hq + hkv) * case["rot"]}
    seen = [_visible(a, b, case["window"]) for a, b in zip(ctx, new)]
    return {"bytes": 4 * hkv * d * sum(k for _, k in seen) + 4 * total * hq * d, "flops": 4 * d * hq * sum(p for p, _ in seen)}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _inv_freq(c):
    """Radians a position adds to each rotated pair, and the factor on cosine and sine: base 10^6, positions divided
    ("linear"), or by frequency ("yarn": divided below 1 turn in the original context of 32768 tokens, kept above 32)."""
    half = c["rot"] // 2
    f = 1e6 ** (-torch.arange(half, dtype=torch.float64) * 2.0 / c["rot"])
    if c["scaling"] == "linear":
        return (f / c["factor"]).cuda(), 1.0
    if c["scaling"] == "yarn":
        turns = 32768.0 * f / (2 * math.pi)
        keep = ((turns.log() - math.log(1.0)) / math.log(32.0)).clamp(0, 1)
        return (f * keep + f / c["factor"] * (1 - keep)).cuda(), 0.1 * math.log(c["factor"]) + 1.0
    return f.cuda(), 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 23)
    ctx, new = _lengths(case)
    page, total, n = case["page"], sum(new), len(ctx)
    held = [_pages(a + b, page) for a, b in zip(ctx, new)]
    spare = 3 + sum(held) // 8
    pages = sum(held) + spare
    order = torch.randperm(pages, device="cuda", generator=g).int()
    ints = lambda v, t=torch.int32: torch.tensor(v, device="cuda", dtype=t)  # noqa: E731
    st = dict(op=case["op"], page=page, total=total, reqs=n, ctx=ints(ctx), new=ints(new))
    if case["op"] == "plan":
        # the table as the last step left it (rows wide enough for the longest request a server admits), and the pages
        # that no request holds
        had = [_pages(a, page) for a in ctx]
        width = max(held) + 5
        first = ints([sum(had[:i]) for i in range(n)])
        col = torch.arange(width, device="cuda", dtype=torch.int32)
        held_at = (first[:, None] + col).clamp_max(pages - 1)
        st["table"] = torch.where(col < ints(had)[:, None], order[held_at.long()], -1).contiguous()
        st["free"], st["count"] = order.roll(-sum(had)).contiguous(), ints([pages - sum(had)])
        return st
    hq, hkv, d, dtype = case["hq"], case["hkv"], case["d"], getattr(torch, case["dtype"])
    first = [sum(held[:i]) for i in range(n)]
    width = max(held)
    col = torch.arange(width, device="cuda", dtype=torch.int32)
    at = (ints(first)[:, None] + col).clamp_max(pages - 1)
    table = torch.where(col < ints(held)[:, None], order[at.long()], -1).contiguous()

    def randn(*s):
        return torch.randn(*s, device="cuda", generator=g, dtype=dtype)

    # a page holds each head's tokens together
    kc, vc = (randn(pages, hkv, page, d).transpose(1, 2) for _ in range(2))
    st.update(kc=kc, vc=vc)
    if case["op"] == "rope":
        f, m = _inv_freq(case)
        # q, k and v as columns of the fused projection's output rows
        wq = hq * d * (2 if case["gated"] else 1)
        rows = randn(total, wq + 2 * hkv * d)
        q = rows[:, :wq].view(total, hq, -1)[:, :, :d]
        k, v = (rows[:, wq + i * hkv * d:wq + (i + 1) * hkv * d].view(total, hkv, d) for i in range(2))
        req = torch.repeat_interleave(torch.arange(n, device="cuda"), st["new"].long(), output_size=total)
        start = torch.cumsum(st["new"], 0) - st["new"]
        pos = st["ctx"][req].long() + torch.arange(total, device="cuda") - start[req]
        slots = table[req, pos // page].long() * page + pos % page
        st.update(q=q, k=k, v=v, pos=pos, slots=slots, f=f, m=m, rot=case["rot"], interleaved=case["interleaved"])
        return st
    cu = ints([0] + [sum(new[:i + 1]) for i in range(n)])
    longest, most = max(a + b for a, b in zip(ctx, new)), max(new)
    span = min(longest, case["window"] + most - 1) if case["window"] else longest
    # queries of twice the keys' spread: a softmax over some tens of keys, as trained heads have it
    st.update(q=2.0 * randn(total, hq, d), table=table, cu=cu, seq=st["ctx"] + st["new"], scale=d ** -0.5, window=case["window"],
              span=span, most_new=most)
    return st


# ---------------------------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------------------------
def _plan_plain(st):
    ctx, new, table, page, total = st["ctx"].long(), st["new"].long(), st["table"], st["page"], st["total"]
    had = (ctx + page - 1) // page
    need = torch.where(new > 0, (ctx + new + page - 1) // page - had, 0)
    end = torch.cumsum(need, 0)
    col = torch.arange(table.shape[1], device="cuda")[None]
    grown = (col >= had[:, None]) & (col < (had + need)[:, None])
    at = st["count"].long() - 1 - (end - need)[:, None] - (col - had[:, None])
    fresh = torch.where(at >= 0, st["free"][at.clamp(0, st["free"].shape[0] - 1)], -1)
    table = torch.where(grown, fresh, table)
    upto = torch.cumsum(new, 0)
    req = torch.repeat_interleave(torch.arange(st["reqs"], device="cuda"), new, output_size=total)
    pos = ctx[req] + torch.arange(total, device="cuda") - (upto - new)[req]
    held = table[req, pos // page].long()
    slots = torch.where(held >= 0, held * page + pos % page, -1)
    cu = torch.nn.functional.pad(upto, (1, 0)).int()
    return dict(table=table, cu=cu, seq=(ctx + new).int(), pos=pos, slots=slots, left=(st["count"] - end[-1]).int())


def _turn(x, cos, sin, rot, interleaved):
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    a, b = a * cos - b * sin, a * sin + b * cos
    head = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([head, x[..., rot:]], -1)


def _rope_plain(st):
    angle = torch.remainder(st["pos"].double()[:, None] * st["f"], 2 * math.pi).float()[:, None]
    cos, sin = angle.cos() * st["m"], angle.sin() * st["m"]
    q, k = (_turn(x.float(), cos, sin, st["rot"], st["interleaved"]).to(x.dtype) for x in (st["q"], st["k"]))
    where = (st["slots"] // st["page"], st["slots"] % st["page"])
    st["kc"][where] = k
    st["vc"][where] = st["v"]
    return dict(q=q, k_cache=st["kc"], v_cache=st["vc"])


def _attn_plain(st):
    q, page, span, most = st["q"], st["page"], st["span"], st["most_new"]
    total, hq, d = q.shape
    hkv = st["kc"].shape[2]
    i = torch.arange(most, device="cuda")
    j = (st["seq"] - span).clamp_min(0).long()[:, None] + torch.arange(span, device="cuda")   # the keys that a token may see
    at = (st["table"].gather(1, j // page).clamp_min(0).long(), j % page)
    k, v = (c[at].float().transpose(1, 2) for c in (st["kc"], st["vc"]))                  # [reqs, hkv, span, d]
    live = i < st["new"][:, None]
    rows = torch.where(live, st["cu"][:-1, None] + i, total)
    qs = torch.nn.functional.pad(q, (0, 0, 0, 0, 0, 1))[rows].float()                     # [reqs, most, hq, d]
    qs = qs.view(-1, most, hkv, hq // hkv, d).transpose(1, 2).flatten(2, 3)
    s = (qs @ k.transpose(-1, -2)).mul_(st["scale"]).view(-1, hkv, most, hq // hkv, span)
    p = (st["seq"] - st["new"])[:, None] + i
    seen = (j[:, None] <= p[..., None]) & live[..., None]
    if st["window"]:
        seen &= j[:, None] > p[..., None] - st["window"]
    s.masked_fill_(~seen[:, None, :, None], -math.inf)
    e = s.sub_(s.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    o = (e.flatten(2, 3) @ v) / e.sum(-1).flatten(2, 3).clamp_min(1e-30)[..., None]
    o = o.view(-1, hkv, most, hq // hkv, d).transpose(1, 2).reshape(-1, most, hq, d)
    out = torch.zeros(total + 1, hq, d, device="cuda", dtype=q.dtype)
    out[rows] = o.to(q.dtype)
    return out[:total]


def run(state):
    if not own:
        return {"plan": _plan_plain, "rope": _rope_plain, "attn": _attn_plain}[state["op"]](state)
    from exl3rocm import paged
    if state["op"] == "plan":
        cu, seq, pos, slots, left = paged.batch_plan(state["ctx"], state["new"], state["table"], state["free"], state["count"],
                                                     state["page"], state["total"])
        return dict(table=state["table"], cu=cu, seq=seq, pos=pos, slots=slots, left=left)
    if state["op"] == "rope":
        q = paged.rope_kv_write(state["q"], state["k"], state["v"], state["pos"], state["slots"], state["kc"], state["vc"],
                                state["f"], state["m"], state["interleaved"])
        return dict(q=q, k_cache=state["kc"], v_cache=state["vc"])
    return paged.paged_attention(state["q"], state["kc"], state["vc"], state["table"], state["cu"], state["seq"],
                                 state["scale"], state["window"])


# ---------------------------------------------------------------------------------------------
# the same in 64 bits, token by token and request by request
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "plan":
        return None
    st = prepare(case, seed)
    if case["op"] == "rope":
        # the pair (a, b) as a complex number, times m e^(i position frequency)
        turn = torch.polar(torch.full_like(st["f"], st["m"]).expand(st["total"], -1).contiguous(), st["pos"].double()[:, None] * st["f"])
        rot, out = st["rot"], []
        lo, hi = ((slice(0, rot, 2), slice(1, rot, 2)) if st["interleaved"] else (slice(0, rot // 2), slice(rot // 2, rot)))
        for x in (st["q"], st["k"]):
            y = x.double().clone()
            z = torch.complex(y[..., lo], y[..., hi]) * turn[:, None]
            y[..., lo], y[..., hi] = z.real, z.imag
            out.append(y)
        kc, vc = st["kc"].double(), st["vc"].double()
        where = (st["slots"] // st["page"], st["slots"] % st["page"])
        kc[where], vc[where] = out[1], st["v"].double()
        return dict(q=out[0], k_cache=kc, v_cache=vc)
    ctx, new = _lengths(case)
    hq, hkv, d, w = case["hq"], case["hkv"], case["d"], case["window"]
    out, t0 = torch.zeros(st["total"], hq, d, device="cuda", dtype=torch.float64), 0
    for r, (a, b) in enumerate(zip(ctx, new)):
        if not b:
            continue
        n = a + b
        held = st["table"][r, :_pages(n, case["page"])].long()
        key = torch.arange(n, device="cuda")
        for h in range(hkv):
            kk, vv = (c[held, :, h].reshape(-1, d)[:n].double() for c in (st["kc"], st["vc"]))
            heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            # queries in pieces: 64-bit scores of at most about a gigabyte
            step = max(1, 134_000_000 // (n * (hq // hkv)))
            for i in range(0, b, step):
                qq = st["q"][t0 + i:t0 + min(b, i + step), heads].double()
                p = a + i + torch.arange(qq.shape[0], device="cuda")[:, None]
                s = (qq.reshape(-1, d) @ kk.T).view(qq.shape[0], -1, n) * st["scale"]
                off = (key > p) | (key <= p - w) if w else key > p
                s = s.masked_fill(off[:, None], -math.inf)
                out[t0 + i:t0 + i + qq.shape[0], heads] = torch.softmax(s, -1) @ vv
        t0 += b
    return out
