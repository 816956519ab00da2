"""Shared-prompt decode operators on torch CUDA tensors (include/mm_latent.h).

The pieces of a decode step whose rows share stored prompts, keep their latent cache in 8
bits and check drafted tokens:

``alloc_cache`` / ``cache_write`` / ``cache_read``
    an 8-bit compressed (MLA) cache: e4m3 latents with one fp32 scale per position and a
    16-bit rope key;
``shared_prefix_attention``
    absorbed latent attention of one or more query tokens per row over the prompt its group
    shares (stored and read once) and over the row's own suffix;
``verify_drafts``
    acceptance of drafted tokens against the target's probabilities.

The reference decodes one request at a time over its own fp32 cache
(src/infer/inference.cpp:47-174, 469-579). A 16-bit cache is a plain tensor ``[rows,
positions, kv + rope]`` (the layout of the context's own cache), an 8-bit one a
:class:`LatentCache`. Calls enqueue on the current stream of the tensors' device and do not
wait; outputs and scratch come from torch's allocator. Failures raise :class:`EngineError`.

A small call's time is this module's own (a launch takes a few microseconds), so the calls
look at each tensor once and hand the C entries packed descriptions.
"""
from __future__ import annotations

import ctypes
import struct
from typing import NamedTuple

import torch

from .engine import EngineError, lib

MM_F32, MM_F16, MM_BF16, MM_E4M3 = range(4)
_KIND = {torch.float32: MM_F32, torch.float16: MM_F16, torch.bfloat16: MM_BF16}
_HALF = (torch.float16, torch.bfloat16)
_E4M3 = torch.float8_e4m3fn

# mm_latent_cache and mm_shared_prefix_desc, field by field
_CACHE = struct.Struct("=3Q5q6i")
_DESC = struct.Struct("=Q3q4i3Q4ifi2Q")

_stream = torch._C._cuda_getCurrentRawStream
_device = torch._C._cuda_getDevice


class LatentCache(NamedTuple):
    """An 8-bit cache: latent [rows, positions, kv] float8_e4m3fn, rope [rows, positions, rope]
    fp16 or bf16, scale [rows, positions] fp32; value = latent * scale."""
    latent: torch.Tensor
    rope: torch.Tensor
    scale: torch.Tensor


_bound = None


def _lib():
    global _bound
    if _bound is None:
        L = lib()
        vp, i64, i32, text = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_char_p
        for name, res, args in (
                ("mm_latent_last_error", ctypes.c_size_t, [text, ctypes.c_size_t]),
                ("mm_latent_cache_write", i32, [text, vp, i64, vp, i64, i32, vp, i64, vp]),
                ("mm_latent_cache_read", i32, [text, vp, i64, vp, i64, i32, vp]),
                ("mm_shared_prefix_attention_workspace", i64, [text, text, text]),
                ("mm_shared_prefix_attention", i32, [text, text, text, vp, ctypes.c_size_t, vp]),
                ("mm_verify_drafts", i32, [vp, vp, i32, vp, vp, vp, vp, i32, i32, i32, vp, vp, vp])):
            f = getattr(L, name)
            f.restype, f.argtypes = res, args
        _bound = L
    return _bound


def _bad(message: str):
    raise EngineError(1, message)


def _fail(rc: int):
    buf = ctypes.create_string_buffer(512)
    _lib().mm_latent_last_error(buf, 512)
    raise EngineError(rc, buf.value.decode(errors="replace"))


def _index(t: torch.Tensor) -> int:
    """The CUDA device a call runs on: that of its first tensor."""
    i = t.get_device()
    if i < 0:
        _bad(f"a CUDA tensor is needed, got one on {t.device}")
    return i


def _on(dev: int, *tensors):
    for t in tensors:
        if t.get_device() != dev:
            _bad(f"tensors must be on one CUDA device: got {t.device} beside cuda:{dev}")


def _on_device(call):
    """Runs a call with its first tensor's device current (kernels launch on the current one)."""
    def run(first, *args, **kwargs):
        t = first[0] if isinstance(first, tuple) else first
        dev = t.get_device()
        if dev < 0 or dev == _device():
            return call(first, *args, **kwargs)
        with torch.cuda.device(dev):
            return call(first, *args, **kwargs)
    run.__name__, run.__doc__, run.__wrapped__ = call.__name__, call.__doc__, call
    return run


def _pack(c, dev: int, kv) -> tuple:
    """A cache as (mm_latent_cache, positions, kv + rope width, kv, rope width)."""
    if isinstance(c, torch.Tensor):
        if kv is None:
            _bad("an 8-bit cache (LatentCache) is needed")
        kind = _KIND.get(c.dtype, 0)
        if c.dim() != 3 or kind == 0:
            _bad("a 16-bit cache is fp16 or bf16 [rows, positions, kv + rope] with adjacent values")
        n, p, w = c.shape
        sr, sp, s1 = c.stride()
        if s1 != 1 and w > 1:
            _bad("a 16-bit cache is fp16 or bf16 [rows, positions, kv + rope] with adjacent values")
        if c.get_device() != dev:
            _on(dev, c)
        return _CACHE.pack(c.data_ptr(), 0, 0, sr, sp, 0, 0, 0, n, p, kv, w - kv, kind, kind), p, w, kv, w - kv
    if not isinstance(c, tuple) or len(c) != 3:
        _bad("a cache is a tensor or a LatentCache")
    lat, rope, scale = c
    shape = lat.shape
    if len(shape) != 3 or rope.dim() != 3 or rope.shape[:2] != shape[:2] or scale.shape != shape[:2]:
        _bad("an 8-bit cache is latent [rows, positions, kv], rope [rows, positions, rope], scale [rows, positions]")
    kind = _KIND.get(rope.dtype, 0)
    if lat.dtype is not _E4M3 or kind == 0 or scale.dtype is not torch.float32:
        _bad("an 8-bit cache is float8_e4m3fn latents, fp16 or bf16 rope keys and fp32 scales")
    n, p, w = shape
    r = rope.shape[2]
    sr, sp, s1 = lat.stride()
    rr, rp, r1 = rope.stride()
    cr, c1 = scale.stride()
    if (s1 != 1 and w > 1) or (r1 != 1 and r > 1) or (c1 != 1 and p > 1):
        _bad("the last dimension of a cache must be contiguous")
    if kv is not None and kv != w:
        _bad("cache width differs from kv_rank")
    if lat.get_device() != dev or rope.get_device() != dev or scale.get_device() != dev:
        _on(dev, lat, rope, scale)
    return (_CACHE.pack(lat.data_ptr(), rope.data_ptr(), scale.data_ptr(), sr, sp, rr, rp, cr, n, p, w, r, MM_E4M3, kind),
            p, w + r, w, r)


def alloc_cache(rows: int, positions: int, kv: int, rope: int, dtype=torch.float16, device="cuda") -> LatentCache:
    """An 8-bit cache of zeros; `dtype` is the rope key's (and the queries')."""
    if dtype not in _HALF:
        _bad("rope keys are fp16 or bf16")
    return LatentCache(torch.zeros(rows, positions, kv, dtype=torch.uint8, device=device).view(_E4M3),
                       torch.zeros(rows, positions, rope, dtype=dtype, device=device),
                       torch.zeros(rows, positions, dtype=torch.float32, device=device))


def _slots(slots, dev: int) -> int:
    if slots.dim() != 1 or slots.dtype is not torch.int64 or not slots.is_contiguous():
        _bad("slots is a contiguous int64 vector (row * positions + position)")
    if slots.get_device() != dev:
        _on(dev, slots)
    return slots.shape[0]


@_on_device
def cache_write(cache: LatentCache, latent: torch.Tensor, rope: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantises new positions into an 8-bit cache in place: latent [n, kv] and rope [n, rope] of
    one type (fp32, fp16 or bf16), position i into slots[i] = row * positions + position; slots
    outside the cache are skipped (free rows of a step pass -1)."""
    dev = _index(latent)
    packed, _, _, kv, rd = _pack(cache, dev, None)
    kind = _KIND.get(latent.dtype, -1)
    if latent.dim() != 2 or rope.dim() != 2 or rope.dtype is not latent.dtype or kind < 0:
        _bad("latent [n, kv] and rope [n, rope] share one floating type")
    n = _slots(slots, dev)
    if latent.shape != (n, kv) or rope.shape != (n, rd):
        _bad("latent, rope and slots do not match the cache")
    sl, l1 = latent.stride()
    sr, r1 = rope.stride()
    if (l1 != 1 and kv > 1) or (r1 != 1 and rd > 1):
        _bad("the last dimension must be contiguous")
    if rope.get_device() != dev:
        _on(dev, rope)
    rc = _lib().mm_latent_cache_write(packed, latent.data_ptr(), sl, rope.data_ptr(), sr, kind, slots.data_ptr(), n,
                                      _stream(dev))
    if rc:
        _fail(rc)


@_on_device
def cache_read(cache: LatentCache, slots: torch.Tensor, dtype=None) -> torch.Tensor:
    """Positions `slots` of an 8-bit cache as rows [n, kv + rope] of `dtype` (default: the rope
    key's); rows of slots outside the cache are zeros."""
    dev = _index(slots)
    packed, _, w, _, _ = _pack(cache, dev, None)
    n = _slots(slots, dev)
    kind = _KIND.get(dtype or cache[1].dtype, -1)
    if kind < 0:
        _bad("cache_read writes fp32, fp16 or bf16")
    out = slots.new_empty((n, w), dtype=dtype or cache[1].dtype)
    rc = _lib().mm_latent_cache_read(packed, slots.data_ptr(), n, out.data_ptr(), w, kind, _stream(dev))
    if rc:
        _fail(rc)
    return out


def _ints(t, dev: int, n: int, what: str) -> int:
    if t is None or t.dtype is not torch.int32 or t.shape != (n,) or not t.is_contiguous():
        _bad(f"{what} is a contiguous int32 vector of {n}")
    if t.get_device() != dev:
        _on(dev, t)
    return t.data_ptr()


@_on_device
def shared_prefix_attention(q: torch.Tensor, prefix, suffix, group_start, prefix_len, suffix_len, scale: float, *,
                            kv_rank: int, max_group: int | None = None, max_prefix: int | None = None,
                            max_suffix: int | None = None, return_lse: bool = False):
    """Absorbed latent attention over a shared prefix and each row's own suffix.

    q [rows, tokens, heads, kv + rope] fp16 or bf16 (any strides, adjacent values); prefix a
    cache of one row per group, suffix a cache of one row per query row (either may be None);
    rows [group_start[g], group_start[g + 1]) attend over prefix row g, positions
    [0, prefix_len[g]), and row b over suffix row b, whose last `tokens` positions are the query
    tokens' own: token t sees [0, suffix_len[b] - (tokens - 1 - t)). max_* are host-side bounds
    (default: the tensors' sizes) that size the launch and clamp the lengths. Returns the
    latent context [rows, tokens, heads, kv] in q's type (zeros for a query that sees nothing)
    and, with return_lse, the natural log-sum-exp [rows, tokens, heads] fp32."""
    dev = _index(q)
    kind = _KIND.get(q.dtype, 0)
    if q.dim() != 4 or kind == 0:
        _bad("q is fp16 or bf16 [rows, tokens, heads, kv + rope] with adjacent values")
    B, T, H, W = q.shape
    qr, qt, qh, q1 = q.stride()
    if q1 != 1 and W > 1:
        _bad("q is fp16 or bf16 [rows, tokens, heads, kv + rope] with adjacent values")
    if not 0 < kv_rank <= W or T < 1 or H < 1:
        _bad("kv_rank must be in (0, q's width]")
    pre = suf = None
    starts = plen = slen = groups = group = maxp = maxs = 0
    if prefix is not None:
        pre, positions, w, _, _ = _pack(prefix, dev, kv_rank)
        if w != W:
            _bad("prefix width differs from q's")
        if group_start is None or prefix_len is None or group_start.dim() != 1 or group_start.shape[0] < 1:
            _bad("a prefix needs group_start [groups + 1] and prefix_len [groups]")
        groups = group_start.shape[0] - 1
        starts = _ints(group_start, dev, groups + 1, "group_start")
        plen = _ints(prefix_len, dev, groups, "prefix_len")
        group = B if max_group is None else max_group
        maxp = positions if max_prefix is None else max_prefix
    if suffix is not None:
        suf, positions, w, _, _ = _pack(suffix, dev, kv_rank)
        if w != W:
            _bad("suffix width differs from q's")
        slen = _ints(suffix_len, dev, B, "suffix_len")
        maxs = positions if max_suffix is None else max_suffix
    out = q.new_empty((B, T, H, kv_rank))
    lse = q.new_empty((B, T, H), dtype=torch.float32) if return_lse else None
    d = _DESC.pack(q.data_ptr(), qr, qt, qh, kind, B, T, H, starts, plen, slen, groups, group, maxp, maxs, scale, 0,
                   out.data_ptr(), lse.data_ptr() if return_lse else 0)
    L = _lib()
    n = L.mm_shared_prefix_attention_workspace(d, pre, suf)
    if n < 0:
        _fail(-n)
    work = q.new_empty((n,), dtype=torch.uint8) if n else None
    rc = L.mm_shared_prefix_attention(d, pre, suf, work.data_ptr() if n else None, n, _stream(dev))
    if rc:
        _fail(rc)
    return (out, lse) if return_lse else out


@_on_device
def verify_drafts(target_probs: torch.Tensor, draft_tokens: torch.Tensor, draft_len: torch.Tensor,
                  u_accept: torch.Tensor, u_sample: torch.Tensor, *, draft_probs: torch.Tensor | None = None):
    """Accepts drafted tokens against the target's probabilities (speculative sampling).

    target_probs [rows, drafts + 1, vocab] and draft_probs [rows, drafts, vocab] (None:
    deterministic drafts) share one type (fp32, fp16 or bf16); draft_tokens [rows, drafts] and
    draft_len [rows] int32; u_accept [rows, drafts] and u_sample [rows] fp32 in [0, 1). Returns
    int32 (tokens [rows, drafts + 1], accepted [rows]): the accepted tokens, one more sampled
    from the residual at the first rejection (from the target when all were accepted), then -1."""
    dev = _index(target_probs)
    kind = _KIND.get(target_probs.dtype, -1)
    if target_probs.dim() != 3 or kind < 0 or not target_probs.is_contiguous():
        _bad("target_probs is contiguous [rows, drafts + 1, vocab]")
    B, K1, V = target_probs.shape
    K = K1 - 1
    if draft_tokens.shape != (B, K) or draft_tokens.dtype is not torch.int32 or not draft_tokens.is_contiguous():
        _bad("draft_tokens is contiguous int32 [rows, drafts]")
    if u_accept.shape != (B, K) or u_accept.dtype is not torch.float32 or not u_accept.is_contiguous() or \
            u_sample.shape != (B,) or u_sample.dtype is not torch.float32 or not u_sample.is_contiguous():
        _bad("u_accept is contiguous fp32 [rows, drafts], u_sample fp32 [rows]")
    _on(dev, draft_tokens, u_accept, u_sample)
    draft = None
    if draft_probs is not None:
        if draft_probs.shape != (B, K, V) or draft_probs.dtype is not target_probs.dtype or \
                not draft_probs.is_contiguous():
            _bad("draft_probs is contiguous [rows, drafts, vocab] of target_probs' type")
        _on(dev, draft_probs)
        draft = draft_probs.data_ptr()
    lens = _ints(draft_len, dev, B, "draft_len")
    tokens = draft_tokens.new_empty((B, K1))
    accepted = draft_tokens.new_empty((B,))
    rc = _lib().mm_verify_drafts(target_probs.data_ptr(), draft, kind, draft_tokens.data_ptr(), lens, u_accept.data_ptr(),
                                 u_sample.data_ptr(), B, K, V, tokens.data_ptr(), accepted.data_ptr(), _stream(dev))
    if rc:
        _fail(rc)
    return tokens, accepted
