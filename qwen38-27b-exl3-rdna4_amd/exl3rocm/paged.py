"""
The attention step of a decoder layer over a paged key/value cache, between the q/k/v and o modules:

  batch_plan       block-table growth, token positions and cache slots of one step, from the requests' lengths
  rope_kv_write    rotary embedding of q and k, with k and v written into the cache
  paged_attention  causal attention of every request's new tokens (decodes, drafts and prompt chunks in one call)

The lengths stay on the GPU: no call reads them back, so a step's calls can be captured in a HIP graph and replayed
as the lengths grow.  Each function is also the torch op of its name (torch.ops.exl3rocm.*), one opaque node for
torch.compile.  Inference only: no gradients.  `rope_frequencies` makes the rotary frequencies, `new_cache` a
cache in the layout that the kernels read fastest.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _lib as L
from .kernels import _need

_DTYPES = {torch.float16: 0, torch.bfloat16: 1}
HEAD_DIMS = (64, 128, 256)


def new_cache(pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=torch.float16, device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """(k_cache, v_cache), each [pages, page_size, kv_heads, head_dim] of a memory order in which a page holds every head's
    tokens together."""
    return tuple(torch.zeros(pages, kv_heads, page_size, head_dim, dtype=dtype, device=device).transpose(1, 2) for _ in range(2))


# what rope_frequencies reads of each kind's `rope_scaling`
_ROPE_KEYS = {
    "default": (),
    "linear": ("factor",),
    "yarn": ("factor", "original_max_position_embeddings", "attention_factor", "mscale", "mscale_all_dim", "beta_fast", "beta_slow", "truncate"),
    "llama3": ("factor", "original_max_position_embeddings", "low_freq_factor", "high_freq_factor"),
}
# what lies beside it and changes nothing here: names, what the caller gives elsewhere (base, rot_dim), what a kind does
# not use, and the sections of a position of several coordinates, which agree where a token has one position
_ROPE_BESIDE = ("rope_type", "type", "rope_theta", "partial_rotary_factor", "original_max_position_embeddings", "finetuned",
                "mrope_section", "mrope_interleaved")


def rope_frequencies(rot_dim: int, base: float = 10000.0, scaling: Optional[dict] = None, device="cuda") -> Tuple[torch.Tensor, float]:
    """(inv_freq, mscale) for rope_kv_write: radians a position adds to each of the rot_dim / 2 pairs (float64), and the
    factor on cosine and sine.  scaling (the keys of a model's `rope_scaling`):
      None or rope_type "default"   base ** (-2 i / rot_dim)
      "linear"   every frequency divided by factor
      "yarn"     divided by factor where a pair makes fewer than beta_slow (1) turns in
                 original_max_position_embeddings tokens, kept above beta_fast (32), a ramp over the pair's index
                 between, whose ends are whole pairs unless truncate is False; mscale = attention_factor, or
                 0.1 ln(factor) + 1, or with mscale and mscale_all_dim the quotient (0.1 mscale ln(factor) + 1) /
                 (0.1 mscale_all_dim ln(factor) + 1): such a model also scales its scores, which is paged_attention's `scale`
      "llama3"   divided by factor where its wavelength exceeds original / low_freq_factor, kept below original /
                 high_freq_factor, blended between
    A key that is None counts as absent; one that would change the result and is not read here is refused."""
    _need(rot_dim >= 2 and rot_dim % 2 == 0, f"rope_frequencies: rot_dim must be even, got {rot_dim}")
    _need(base > 1, f"rope_frequencies: base must be above 1, got {base}")
    i = torch.arange(rot_dim // 2, dtype=torch.float64)
    f = base ** (-2.0 * i / rot_dim)
    s = {key: v for key, v in (scaling or {}).items() if v is not None}
    kind, mscale = s.get("rope_type", s.get("type", "default")), 1.0
    _need(kind in _ROPE_KEYS, f"rope_frequencies: unknown rope_type {kind!r}")
    unread = sorted(set(s) - set(_ROPE_KEYS[kind]) - set(_ROPE_BESIDE))
    _need(not unread, f"rope_frequencies: rope_type {kind!r} with keys that are not read: {', '.join(unread)}")
    _need(s.get("rope_theta", base) == base, f"rope_frequencies: base is {base}, rope_theta {s.get('rope_theta')}")
    if kind == "linear":
        f = f / s["factor"]
    elif kind == "yarn":
        factor, orig = float(s["factor"]), float(s["original_max_position_embeddings"])
        # the pair index that makes b turns in the original context
        at = lambda b: rot_dim * math.log(orig / (2 * math.pi * b)) / (2 * math.log(base))  # noqa: E731
        low, high = at(s.get("beta_fast", 32)), at(s.get("beta_slow", 1))
        if s.get("truncate", True):
            low, high = math.floor(low), math.ceil(high)
        low, high = max(low, 0), min(high, rot_dim - 1)
        slow = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        f = f / factor * slow + f * (1 - slow)
        grown = lambda m: 0.1 * m * math.log(factor) + 1.0 if factor > 1 else 1.0  # noqa: E731
        _need(("mscale" in s) == ("mscale_all_dim" in s), "rope_frequencies: mscale and mscale_all_dim go together")
        if "attention_factor" in s:
            mscale = float(s["attention_factor"])
        elif "mscale" in s:
            mscale = grown(s["mscale"]) / grown(s["mscale_all_dim"])
        else:
            mscale = grown(1.0)
    elif kind == "llama3":
        lo, hi = s["low_freq_factor"], s["high_freq_factor"]
        turns = s["original_max_position_embeddings"] * f / (2 * math.pi)
        keep = ((turns - lo) / (hi - lo)).clamp(0, 1)
        f = f * keep + f / s["factor"] * (1 - keep)
    return f.to(device), mscale


# An eager call's host time is what bounds a decode step's small launches, so the checks below read each attribute
# once (get_device is half the time of device), and the library's entry points are looked up once.
_fn: dict = {}


def _entry(name: str):
    f = _fn.get(name)
    if f is None:
        f = _fn[name] = getattr(L.lib(), name)
    return f


def _raw_stream(gpu: int) -> int:
    """The current stream's handle on a GPU (looked up at the call: a torch without a GPU backend has no such function)."""
    return torch._C._cuda_getCurrentRawStream(gpu)


def _ints(name: str, t: torch.Tensor, gpu: int, dtype, numel: Optional[int] = None):
    if t.dtype is not dtype or t.get_device() != gpu or not t.is_contiguous() or (numel is not None and t.numel() != numel):
        _need(False, f"{name} must be a contiguous {dtype} tensor on GPU {gpu}" + (f" of {numel} elements" if numel is not None else ""))


def _gpu(t: torch.Tensor, what: str) -> int:
    i = t.get_device()
    _need(i >= 0, f"{what}: tensors must be on a GPU (no CPU path)")
    return i


def _table(what: str, t: torch.Tensor, gpu: int, requests: int):
    """(columns, row stride) of a block table."""
    shape = t.shape
    if t.dtype is not torch.int32 or t.get_device() != gpu or len(shape) != 2 or shape[0] != requests:
        _need(False, f"{what}: block_table must be int32 [{requests}, columns] on GPU {gpu}")
    cols = shape[1]
    ld, one = t.stride()
    _need(one == 1 or cols <= 1, f"{what}: block_table needs unit column stride")
    return cols, ld if requests > 1 else cols


def batch_plan(ctx_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
               free_count: torch.Tensor, page_size: int, num_tokens: int
               ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(cu_q, seq_lens, positions, slots, free_left) of a step in which request r, with ctx_lens[r] tokens in the cache,
    adds new_lens[r] (int32 [R]).  block_table (int32 [R, columns], rows any stride apart) gets the pages that the new
    tokens need, popped from the stack free_pages[:free_count] (int32; its top first, in the order of the requests).
    num_tokens: rows of the step's batch; rows past the last request get position 0 and slot -1, as a batch
    padded for a captured graph has them.  free_left [1] is the next free_count; negative: that many pages were missing,
    and the tokens without one have slot -1 (nothing is written for them).  The stack and its count are only read:
    a repeated call gives the same result, and a step that lacks pages is undone by keeping ctx_lens and free_count as they
    were.  It is not to be kept: a later plan counts the pages of ctx_lens as held and never fills them in."""
    gpu, i32 = _gpu(ctx_lens, "batch_plan"), torch.int32
    R = ctx_lens.numel()
    _ints("batch_plan: ctx_lens", ctx_lens, gpu, i32)
    _ints("batch_plan: new_lens", new_lens, gpu, i32, R)
    _ints("batch_plan: free_pages", free_pages, gpu, i32)
    _ints("batch_plan: free_count", free_count, gpu, i32, 1)
    cols, ld = _table("batch_plan", block_table, gpu, R)
    _need(page_size >= 1 and num_tokens >= 0, "batch_plan: page_size from 1, num_tokens from 0")
    dev = ctx_lens.device
    # an allocation each: slices of one would share storage, against the schema, and start where compiled code, which takes
    # an op's outputs for aligned to 16 bytes, cannot read them
    cu_q, seq, left = (torch.empty(n, dtype=i32, device=dev) for n in (R + 1, R, 1))
    pos, slots = (torch.empty(num_tokens, dtype=torch.int64, device=dev) for _ in range(2))
    L.check(_entry("exl3_batch_plan")(ctx_lens.data_ptr(), new_lens.data_ptr(), block_table.data_ptr(), ld, cols, free_pages.data_ptr(),
                                      free_pages.numel(), free_count.data_ptr(), cu_q.data_ptr(), seq.data_ptr(),
                                      pos.data_ptr(), slots.data_ptr(), left.data_ptr(), R, page_size, num_tokens, _raw_stream(gpu)),
            "batch_plan")
    return cu_q, seq, pos, slots, left


def _cache(what: str, k_cache: torch.Tensor, v_cache: torch.Tensor, dtype, gpu: int, d: int):
    """Checks a cache against the heads that use it; its (pages, page size, kv heads)."""
    shape = k_cache.shape
    if not (len(shape) == 4 and shape == v_cache.shape and k_cache.dtype is dtype and v_cache.dtype is dtype
            and k_cache.get_device() == gpu and v_cache.get_device() == gpu and shape[3] == d
            and k_cache.stride(3) == 1 and v_cache.stride(3) == 1):
        _need(False, f"{what}: k_cache and v_cache must be {dtype} [pages, page_size, kv_heads, {d}] on GPU {gpu} with unit last stride, "
                     f"got {tuple(shape)} {k_cache.dtype} and {tuple(v_cache.shape)} {v_cache.dtype}")
    return shape[0], shape[1], shape[2]


def rope_kv_write(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
                  k_cache: torch.Tensor, v_cache: torch.Tensor, inv_freq: torch.Tensor, mscale: float = 1.0,
                  interleaved: bool = False) -> torch.Tensor:
    """Rotated q [T, q_heads, D]; the rotated k and v [T, kv_heads, D] are written to their tokens' slots of the cache
    [pages, page_size, kv_heads, D].  q, k and v may be slices (any token and head strides that are multiples of
    8, unit last stride), e.g. columns of the fused q/k/v module's output.  positions, slots: int64 [T]; a slot
    outside the cache (-1) writes nothing.  inv_freq: float64 [rot_dim / 2], mscale: rope_frequencies; interleaved:
    pairs (2 i, 2 i + 1) instead of (i, i + rot_dim / 2).  fp16 or bf16, D of 64, 128 or 256."""
    gpu, dt = _gpu(q, "rope_kv_write"), q.dtype
    qs, ks = q.shape, k.shape
    _need(len(qs) == 3 and len(ks) == 3 and v.shape == ks and qs[0] == ks[0] and qs[2] == ks[2],
          "rope_kv_write: q must be [T, q_heads, D], k and v [T, kv_heads, D]")
    T, hq, d = qs
    hkv = ks[1]
    _need(dt in _DTYPES and k.dtype is dt and v.dtype is dt and k.get_device() == gpu and v.get_device() == gpu and d in HEAD_DIMS,
          "rope_kv_write: q, k and v must be fp16 or bf16, all alike, on one GPU, with heads of 64, 128 or 256")
    qt, qh, q1 = q.stride()
    kt, kh, k1 = k.stride()
    vt, vh, v1 = v.stride()
    _need(q1 == 1 and k1 == 1 and v1 == 1 or T == 0, "rope_kv_write: q, k and v need unit last stride")
    pages, page, heads = _cache("rope_kv_write", k_cache, v_cache, dt, gpu, d)
    _need(heads == hkv, f"rope_kv_write: a cache of {heads} kv heads, k of {hkv}")
    _ints("rope_kv_write: positions", positions, gpu, torch.int64, T)
    _ints("rope_kv_write: slots", slots, gpu, torch.int64, T)
    _ints("rope_kv_write: inv_freq", inv_freq, gpu, torch.float64)
    out = torch.empty(qs, dtype=dt, device=q.device)
    kcp, kct, kch, _ = k_cache.stride()
    vcp, vct, vch, _ = v_cache.stride()
    L.check(_entry("exl3_rope_kv_write")(q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, positions.data_ptr(), slots.data_ptr(),
                                         out.data_ptr(), k_cache.data_ptr(), kcp, kct, kch, v_cache.data_ptr(), vcp, vct, vch,
                                         inv_freq.data_ptr(), mscale, T, hq, hkv, d, 2 * inv_freq.numel(), interleaved, pages, page,
                                         _DTYPES[dt], _raw_stream(gpu)), "rope_kv_write")
    return out


_workspaces: dict = {}      # (GPU, stream) -> zeroed workspace of paged_attention


def _workspace(device: torch.device, stream: int) -> torch.Tensor:
    """The stream's workspace: one size serves every shape, so a stream that made one eager call can capture any."""
    _need(not torch.cuda.is_current_stream_capturing(), "paged_attention: this stream made no eager call before graph capture")
    ws = _workspaces[(device.index, stream)] = torch.zeros(int(L.lib().exl3_paged_attention_workspace_size()), dtype=torch.uint8, device=device)
    return ws


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, cu_q: torch.Tensor,
                    seq_lens: torch.Tensor, scale: float, window: int = 0) -> torch.Tensor:
    """Causal attention [T, q_heads, D] of the rows of q [T, q_heads, D] (any token and head strides that are multiples of
    8) over a paged cache [pages, page_size, kv_heads, D], page_size a multiple of 16.  Rows [cu_q[r], cu_q[r + 1])
    belong to request r and are the last of its seq_lens[r] tokens, whose pages block_table[r] lists (int32, as batch_plan
    makes them).  window: keys that a token sees, itself included (0: all).  A row that sees no key is 0; what a row
    does not see has no effect on it, NaN included."""
    gpu, dt = _gpu(q, "paged_attention"), q.dtype
    qs = q.shape
    _need(len(qs) == 3 and dt in _DTYPES and qs[2] in HEAD_DIMS, "paged_attention: q must be fp16 or bf16 [T, q_heads, D] with D of 64, 128 or 256")
    T, hq, d = qs
    pages, page, hkv = _cache("paged_attention", k_cache, v_cache, dt, gpu, d)
    _need(hkv > 0 and hq > 0 and hq % hkv == 0, f"paged_attention: {hq} query heads are no multiple of {hkv} kv heads")
    _need(page >= 16 and page % 16 == 0, f"paged_attention: page_size must be a multiple of 16, got {page}")
    qt, qh, q1 = q.stride()
    _need(q1 == 1 or T == 0, "paged_attention: q needs unit last stride")
    R = seq_lens.numel()
    _ints("paged_attention: seq_lens", seq_lens, gpu, torch.int32)
    _ints("paged_attention: cu_q", cu_q, gpu, torch.int32, R + 1)
    cols, ld = _table("paged_attention", block_table, gpu, R)
    _need(0 <= window <= 1 << 30, "paged_attention: window from 0 (none) to 2 ** 30")
    dev = q.device
    out = torch.empty(qs, dtype=dt, device=dev)
    st = _raw_stream(gpu)
    ws = _workspaces.get((gpu, st))
    if ws is None:
        ws = _workspace(dev, st)
    kcp, kct, kch, _ = k_cache.stride()
    vcp, vct, vch, _ = v_cache.stride()
    L.check(_entry("exl3_paged_attention")(q.data_ptr(), qt, qh, k_cache.data_ptr(), kcp, kct, kch, v_cache.data_ptr(), vcp, vct, vch,
                                           block_table.data_ptr(), ld, cols, cu_q.data_ptr(), seq_lens.data_ptr(), out.data_ptr(), hq * d, d,
                                           T, R, hq, hkv, d, pages, page, scale, window, _DTYPES[dt], ws.data_ptr(), ws.numel(), st), "paged_attention")
    return out


# The ops are registered with their schemas and the functions above as their GPU kernels: torch.library.custom_op's
# wrapper takes an eager call 14 us of host time (18 where the op changes an input), this way 5.
_ops = torch.library.Library("exl3rocm", "FRAGMENT")
_ops.define("batch_plan(Tensor ctx_lens, Tensor new_lens, Tensor(a!) block_table, Tensor free_pages, Tensor free_count, int page_size, "
            "int num_tokens) -> (Tensor, Tensor, Tensor, Tensor, Tensor)")
_ops.define("rope_kv_write(Tensor q, Tensor k, Tensor v, Tensor positions, Tensor slots, Tensor(a!) k_cache, Tensor(b!) v_cache, "
            "Tensor inv_freq, float mscale=1.0, bool interleaved=False) -> Tensor")
_ops.define("paged_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor cu_q, Tensor seq_lens, float scale, "
            "int window=0) -> Tensor")
for _f in (batch_plan, rope_kv_write, paged_attention):
    _ops.impl(_f.__name__, _f, "CompositeExplicitAutograd")


@torch.library.register_fake("exl3rocm::batch_plan")
def _(ctx_lens, new_lens, block_table, free_pages, free_count, page_size, num_tokens):
    R = ctx_lens.numel()
    return (ctx_lens.new_empty(R + 1), ctx_lens.new_empty(R), ctx_lens.new_empty(num_tokens, dtype=torch.int64),
            ctx_lens.new_empty(num_tokens, dtype=torch.int64), ctx_lens.new_empty(1))


@torch.library.register_fake("exl3rocm::rope_kv_write")
def _(q, k, v, positions, slots, k_cache, v_cache, inv_freq, mscale=1.0, interleaved=False):
    return q.new_empty(q.shape)


@torch.library.register_fake("exl3rocm::paged_attention")
def _(q, k_cache, v_cache, block_table, cu_q, seq_lens, scale, window=0):
    return q.new_empty(q.shape)
