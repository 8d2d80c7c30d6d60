"""
The attention step over a paged key/value cache held in 8 bits: half the bytes of the cache of exl3rocm.paged, so half the
reading of a decode step and twice the tokens in memory.  batch_plan and rope_frequencies are the same; the cache is made by
`new_cache8` and written, read back and attended over by

  rope_kv_write8    rotary embedding of q and k, with k and v quantised into the cache
  kv_read8          tokens of the cache as fp16 or bf16 values
  paged_attention8  causal attention of every request's new tokens (decodes, drafts and prompt chunks in one call)

A value is code * scale: int8 codes, and an fp32 scale for each block of 16 tokens of a page and kv head.  A call that writes a
block's first token starts the block anew: its scale becomes the least power of two (2 ** -40 to 2 ** 40) of which 127 reach
the largest absolute value that the call writes there, and rows that the call does not write become 0.  A call that writes later tokens keeps
the scale or doubles it as often as they need, and then rounds the block's other rows to the new step.  So a value is off by at
most half a step (1 / 254 to 1 / 127 of its block's largest), and by as much again for each later doubling, the steps before it
being half as large.

Each function is also the torch op of its name (torch.ops.exl3rocm.*).  Lengths stay on the GPU and a step's calls can be
captured in a HIP graph, as in exl3rocm.paged.  Inference only: no gradients.
"""
from __future__ import annotations

from struct import Struct
from typing import Tuple

import torch

from . import _lib as L
from . import paged
from .kernels import _need
from .paged import _DTYPES, HEAD_DIMS, _entry, _gpu, _ints, _table

BLOCK = 16

Cache8 = Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]


def new_cache8(pages: int, page_size: int, kv_heads: int, head_dim: int, device="cuda") -> Cache8:
    """(k_cache, v_cache, k_scale, v_scale): int8 [pages, page_size, kv_heads, head_dim] of a memory order in which a page
    holds every head's tokens together, and float32 [pages, page_size / 16, kv_heads].  page_size: a multiple of 16."""
    _need(page_size >= BLOCK and page_size % BLOCK == 0, f"new_cache8: page_size must be a multiple of 16, got {page_size}")
    codes = (torch.zeros(pages, kv_heads, page_size, head_dim, dtype=torch.int8, device=device).transpose(1, 2) for _ in range(2))
    scales = (torch.zeros(pages, kv_heads, page_size // BLOCK, dtype=torch.float32, device=device).transpose(1, 2) for _ in range(2))
    return (*codes, *scales)


_pack = Struct("=16q4i").pack           # exl3_cache8 of the C interface
# torch.empty with a type and a device takes an eager call twice the host time of empty_like
_like, _contiguous = torch.empty_like, torch.contiguous_format


def _cache8(what: str, kc: torch.Tensor, vc: torch.Tensor, ks: torch.Tensor, vs: torch.Tensor, gpu: int):
    """Checks a cache; (its C struct, kv heads, head width)."""
    shape, sshape, i8, f32 = kc.shape, ks.shape, torch.int8, torch.float32
    if not (len(shape) == 4 and shape == vc.shape and kc.dtype is i8 and vc.dtype is i8 and kc.get_device() == gpu and vc.get_device() == gpu):
        _need(False, f"{what}: k_cache and v_cache must be int8 [pages, page_size, kv_heads, head_dim] on GPU {gpu}, "
                     f"got {tuple(shape)} {kc.dtype} and {tuple(vc.shape)} {vc.dtype}")
    pages, page, heads, d = shape
    if page < BLOCK or page % BLOCK or d not in HEAD_DIMS:
        _need(False, f"{what}: page_size must be a multiple of 16 and heads of 64, 128 or 256, got {page} and {d}")
    if not (sshape == (pages, page // BLOCK, heads) and sshape == vs.shape and ks.dtype is f32 and vs.dtype is f32
            and ks.get_device() == gpu and vs.get_device() == gpu):
        _need(False, f"{what}: k_scale and v_scale must be float32 [{pages}, {page // BLOCK}, {heads}] on GPU {gpu}, "
                     f"got {tuple(sshape)} {ks.dtype} and {tuple(vs.shape)} {vs.dtype}")
    kp, kt, kh, k1 = kc.stride()
    vp, vt, vh, v1 = vc.stride()
    _need(k1 == 1 and v1 == 1, f"{what}: k_cache and v_cache need unit last stride")
    return _pack(kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), kp, kt, kh, vp, vt, vh, *ks.stride(), *vs.stride(),
                 pages, page, heads, d), heads, d


def _launch(what: str, gpu: int, name: str, *args):
    """The entry point on the current stream of the tensors' GPU, which need not be the current one."""
    st = paged._raw_stream(gpu)
    if torch._C._cuda_getDevice() == gpu:
        L.check(_entry(name)(*args, st), what)
    else:
        with torch.cuda.device(gpu):
            L.check(_entry(name)(*args, st), what)


def rope_kv_write8(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
                   k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                   inv_freq: torch.Tensor, mscale: float = 1.0, interleaved: bool = False) -> torch.Tensor:
    """Rotated q [T, q_heads, D]; the rotated k and v [T, kv_heads, D] are quantised into their tokens' slots of the cache.
    Arguments as rope_kv_write.  Rows of one block of 16 slots have to be consecutive in the batch, as a request's tokens are (else
    they race); of a slot that comes twice in them the last row counts.  Infinities and NaN do not count for a
    scale; an infinity is stored as 127 steps, NaN as 0."""
    gpu, dt = _gpu(q, "rope_kv_write8"), q.dtype
    qs, ks = q.shape, k.shape
    _need(len(qs) == 3 and len(ks) == 3 and v.shape == ks and qs[0] == ks[0] and qs[2] == ks[2],
          "rope_kv_write8: q must be [T, q_heads, D], k and v [T, kv_heads, D]")
    T, hq, d = qs
    _need(dt in _DTYPES and k.dtype is dt and v.dtype is dt and k.get_device() == gpu and v.get_device() == gpu,
          "rope_kv_write8: q, k and v must be fp16 or bf16, all alike, on one GPU")
    cache, heads, cd = _cache8("rope_kv_write8", k_cache, v_cache, k_scale, v_scale, gpu)
    _need(heads == ks[1] and cd == d, f"rope_kv_write8: a cache of {heads} kv heads of {cd}, k of {ks[1]} of {d}")
    qt, qh, q1 = q.stride()
    kt, kh, k1 = k.stride()
    vt, vh, v1 = v.stride()
    _need(q1 == 1 and k1 == 1 and v1 == 1 or T == 0, "rope_kv_write8: q, k and v need unit last stride")
    _ints("rope_kv_write8: positions", positions, gpu, torch.int64, T)
    _ints("rope_kv_write8: slots", slots, gpu, torch.int64, T)
    _ints("rope_kv_write8: inv_freq", inv_freq, gpu, torch.float64)
    out = _like(q, memory_format=_contiguous)
    _launch("rope_kv_write8", gpu, "exl3_rope_kv_write8", q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, positions.data_ptr(),
            slots.data_ptr(), out.data_ptr(), cache, inv_freq.data_ptr(), mscale, T, hq, 2 * inv_freq.numel(), interleaved, _DTYPES[dt])
    return out


def kv_read8(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, slots: torch.Tensor,
             dtype: torch.dtype = torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v), each [T, kv_heads, D] of dtype (fp16 or bf16): the values that the T slots (int64, contiguous) hold.  A slot outside the
    cache (-1) gives zeros."""
    gpu = _gpu(k_cache, "kv_read8")
    cache, heads, d = _cache8("kv_read8", k_cache, v_cache, k_scale, v_scale, gpu)
    _need(dtype in _DTYPES, f"kv_read8: dtype must be fp16 or bf16, got {dtype}")
    _ints("kv_read8: slots", slots, gpu, torch.int64)
    T = slots.numel()
    k = torch.empty(T, heads, d, dtype=dtype, device=k_cache.device)
    v = _like(k)
    _launch("kv_read8", gpu, "exl3_kv_read8", cache, slots.data_ptr(), k.data_ptr(), v.data_ptr(), T, _DTYPES[dtype])
    return k, v


def paged_attention8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                     block_table: torch.Tensor, cu_q: torch.Tensor, seq_lens: torch.Tensor, scale: float, window: int = 0) -> torch.Tensor:
    """Causal attention [T, q_heads, D] of the rows of q [T, q_heads, D] over the cache; arguments as paged_attention, and
    as there a row that sees no key is 0 and what a row does not see has no effect on it.  Shares paged_attention's workspace of the
    stream, so a stream that captures a graph needs one eager call of either before."""
    gpu, dt = _gpu(q, "paged_attention8"), q.dtype
    qs = q.shape
    _need(len(qs) == 3 and dt in _DTYPES, "paged_attention8: q must be fp16 or bf16 [T, q_heads, D]")
    T, hq, d = qs
    cache, hkv, cd = _cache8("paged_attention8", k_cache, v_cache, k_scale, v_scale, gpu)
    _need(hkv > 0 and hq > 0 and hq % hkv == 0 and cd == d, f"paged_attention8: {hq} query heads of {d} over {hkv} kv heads of {cd}")
    qt, qh, q1 = q.stride()
    _need(q1 == 1 or T == 0, "paged_attention8: q needs unit last stride")
    R = seq_lens.numel()
    _ints("paged_attention8: seq_lens", seq_lens, gpu, torch.int32)
    _ints("paged_attention8: cu_q", cu_q, gpu, torch.int32, R + 1)
    cols, ld = _table("paged_attention8", block_table, gpu, R)
    _need(0 <= window <= 1 << 30, "paged_attention8: window from 0 (none) to 2 ** 30")
    out = _like(q, memory_format=_contiguous)
    st = paged._raw_stream(gpu)
    ws = paged._workspaces.get((gpu, st))
    if ws is None:
        ws = paged._workspace(q.device, st)
    _launch("paged_attention8", gpu, "exl3_paged_attention8", q.data_ptr(), qt, qh, cache, block_table.data_ptr(), ld, cols, cu_q.data_ptr(),
            seq_lens.data_ptr(), out.data_ptr(), hq * d, d, T, R, hq, scale, window, _DTYPES[dt], ws.data_ptr(), ws.numel())
    return out


# registered as the ops of exl3rocm.paged are, for the same reason
_ops = torch.library.Library("exl3rocm", "FRAGMENT")
_ops.define("rope_kv_write8(Tensor q, Tensor k, Tensor v, Tensor positions, Tensor slots, Tensor(a!) k_cache, Tensor(b!) v_cache, "
            "Tensor(c!) k_scale, Tensor(d!) v_scale, Tensor inv_freq, float mscale=1.0, bool interleaved=False) -> Tensor")
_ops.define("kv_read8(Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, Tensor slots, ScalarType dtype=half) -> (Tensor, Tensor)")
_ops.define("paged_attention8(Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, Tensor block_table, Tensor cu_q, "
            "Tensor seq_lens, float scale, int window=0) -> Tensor")
for _f in (rope_kv_write8, kv_read8, paged_attention8):
    _ops.impl(_f.__name__, _f, "CompositeExplicitAutograd")


@torch.library.register_fake("exl3rocm::rope_kv_write8")
def _(q, k, v, positions, slots, k_cache, v_cache, k_scale, v_scale, inv_freq, mscale=1.0, interleaved=False):
    return q.new_empty(q.shape)


@torch.library.register_fake("exl3rocm::kv_read8")
def _(k_cache, v_cache, k_scale, v_scale, slots, dtype=torch.float16):
    shape = (slots.numel(), *k_cache.shape[2:])
    return k_cache.new_empty(shape, dtype=dtype), k_cache.new_empty(shape, dtype=dtype)


@torch.library.register_fake("exl3rocm::paged_attention8")
def _(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_q, seq_lens, scale, window=0):
    return q.new_empty(q.shape)
