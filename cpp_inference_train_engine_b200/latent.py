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
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from .engine import EngineError, lib

MM_F32, MM_F16, MM_BF16, MM_E4M3 = range(4)
_KIND = {torch.float32: MM_F32, torch.float16: MM_F16, torch.bfloat16: MM_BF16}
_HALF = (torch.float16, torch.bfloat16)

_vp, _i64, _i32, _f32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_float


class LatentCache(NamedTuple):
    """An 8-bit cache: latent [rows, positions, kv] float8_e4m3fn, rope [rows, positions, rope]
    fp16 or bf16, scale [rows, positions] fp32; value = latent * scale."""
    latent: torch.Tensor
    rope: torch.Tensor
    scale: torch.Tensor


class _Cache(ctypes.Structure):
    _fields_ = [("latent", _vp), ("rope", _vp), ("scale", _vp), ("row_stride", _i64), ("pos_stride", _i64),
                ("rope_row_stride", _i64), ("rope_pos_stride", _i64), ("scale_row_stride", _i64), ("rows", _i32),
                ("positions", _i32), ("kv", _i32), ("rope_dim", _i32), ("kind", _i32), ("rope_kind", _i32)]


class _Desc(ctypes.Structure):
    _fields_ = [("q", _vp), ("q_row_stride", _i64), ("q_token_stride", _i64), ("q_head_stride", _i64),
                ("dtype", _i32), ("rows", _i32), ("tokens", _i32), ("heads", _i32),
                ("prefix", ctypes.POINTER(_Cache)), ("suffix", ctypes.POINTER(_Cache)), ("group_start", _vp),
                ("prefix_len", _vp), ("suffix_len", _vp), ("groups", _i32), ("max_group", _i32),
                ("max_prefix", _i32), ("max_suffix", _i32), ("scale", _f32), ("reserved", _i32), ("out", _vp),
                ("lse", _vp)]


_bound = None


def _lib():
    global _bound
    if _bound is None:
        L = lib()
        pc, pd = ctypes.POINTER(_Cache), ctypes.POINTER(_Desc)
        for name, res, args in (
                ("mm_latent_last_error", ctypes.c_size_t, [ctypes.c_char_p, ctypes.c_size_t]),
                ("mm_latent_cache_write", ctypes.c_int, [pc, _vp, _i64, _vp, _i64, ctypes.c_int, _vp, _i64, _vp]),
                ("mm_latent_cache_read", ctypes.c_int, [pc, _vp, _i64, _vp, _i64, ctypes.c_int, _vp]),
                ("mm_shared_prefix_attention_workspace", _i64, [pd]),
                ("mm_shared_prefix_attention", ctypes.c_int, [pd, _vp, ctypes.c_size_t, _vp]),
                ("mm_verify_drafts", ctypes.c_int, [_vp, _vp, ctypes.c_int, _vp, _vp, _vp, _vp, ctypes.c_int,
                                                    ctypes.c_int, ctypes.c_int, _vp, _vp, _vp])):
            f = getattr(L, name)
            f.restype, f.argtypes = res, args
        _bound = L
    return _bound


def _fail(rc: int):
    buf = ctypes.create_string_buffer(512)
    _bound.mm_latent_last_error(buf, 512)
    raise EngineError(rc, buf.value.decode(errors="replace"))


def _require(ok, message: str):
    if not ok:
        raise EngineError(1, message)


def _on(device, *tensors):
    for t in tensors:
        if t.device != device:
            raise EngineError(1, f"tensors must be on one CUDA device: got {t.device} beside {device}")


class _Device:
    """Makes a tensor's device current for a call when it is not (kernels launch there)."""

    def __init__(self, device):
        if device.type != "cuda":
            raise EngineError(1, f"a CUDA tensor is needed, got one on {device}")
        self.index, self.back = device.index, torch.cuda.current_device()

    def __enter__(self):
        if self.index != self.back:
            torch.cuda.set_device(self.index)
        return torch.cuda.current_stream(self.index).cuda_stream

    def __exit__(self, *exc):
        if self.index != self.back:
            torch.cuda.set_device(self.back)


def _cache(c, device, kv) -> _Cache:
    if isinstance(c, torch.Tensor):
        _require(c.dim() == 3 and c.dtype in _HALF and (c.shape[2] <= 1 or c.stride(2) == 1),
                 "a 16-bit cache is fp16 or bf16 [rows, positions, kv + rope] with adjacent values")
        _require(kv is not None, "an 8-bit cache (LatentCache) is needed")
        _on(device, c)
        s = c.stride()
        kind = _KIND[c.dtype]
        return _Cache(c.data_ptr(), None, None, s[0], s[1], 0, 0, 0, c.shape[0], c.shape[1], kv, c.shape[2] - kv, kind,
                      kind)
    _require(isinstance(c, tuple) and len(c) == 3, "a cache is a tensor or a LatentCache")
    lat, rope, scale = c
    _require(lat.dim() == 3 and rope.dim() == 3 and scale.dim() == 2 and lat.shape[:2] == rope.shape[:2] == scale.shape,
             "an 8-bit cache is latent [rows, positions, kv], rope [rows, positions, rope], scale [rows, positions]")
    _require(lat.dtype == torch.float8_e4m3fn and rope.dtype in _HALF and scale.dtype == torch.float32,
             "an 8-bit cache is float8_e4m3fn latents, fp16 or bf16 rope keys and fp32 scales")
    _require((lat.shape[2] <= 1 or lat.stride(2) == 1) and (rope.shape[2] <= 1 or rope.stride(2) == 1) and
             (scale.shape[1] <= 1 or scale.stride(1) == 1), "the last dimension of a cache must be contiguous")
    _require(kv is None or lat.shape[2] == kv, "cache width differs from kv_rank")
    _on(device, lat, rope, scale)
    s, r = lat.stride(), rope.stride()
    return _Cache(lat.data_ptr(), rope.data_ptr(), scale.data_ptr(), s[0], s[1], r[0], r[1], scale.stride(0),
                  lat.shape[0], lat.shape[1], lat.shape[2], rope.shape[2], MM_E4M3, _KIND[rope.dtype])


def alloc_cache(rows: int, positions: int, kv: int, rope: int, dtype=torch.float16, device="cuda") -> LatentCache:
    """An 8-bit cache of zeros; `dtype` is the rope key's (and the queries')."""
    _require(dtype in _HALF, "rope keys are fp16 or bf16")
    return LatentCache(torch.zeros(rows, positions, kv, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
                       torch.zeros(rows, positions, rope, dtype=dtype, device=device),
                       torch.zeros(rows, positions, dtype=torch.float32, device=device))


def _slots(slots, device):
    _require(slots.dim() == 1 and slots.dtype == torch.int64 and slots.is_contiguous(),
             "slots is a contiguous int64 vector (row * positions + position)")
    _on(device, slots)


def cache_write(cache: LatentCache, latent: torch.Tensor, rope: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantises new positions into an 8-bit cache in place: latent [n, kv] and rope [n, rope] of
    one type (fp32, fp16 or bf16), position i into slots[i] = row * positions + position; slots
    outside the cache are skipped (free rows of a step pass -1)."""
    device = latent.device
    with _Device(device) as stream:
        c = _cache(cache, device, None)
        _require(latent.dim() == 2 and rope.dim() == 2 and latent.dtype == rope.dtype and latent.dtype in _KIND,
                 "latent [n, kv] and rope [n, rope] share one floating type")
        n = latent.shape[0]
        _require(latent.shape[1] == c.kv and rope.shape == (n, c.rope_dim) and slots.shape == (n,),
                 "latent, rope and slots do not match the cache")
        _require((c.kv <= 1 or latent.stride(1) == 1) and (c.rope_dim <= 1 or rope.stride(1) == 1),
                 "the last dimension must be contiguous")
        _on(device, rope)
        _slots(slots, device)
        rc = _lib().mm_latent_cache_write(ctypes.byref(c), latent.data_ptr(), latent.stride(0), rope.data_ptr(),
                                          rope.stride(0), _KIND[latent.dtype], slots.data_ptr(), n, stream)
        if rc:
            _fail(rc)


def cache_read(cache: LatentCache, slots: torch.Tensor, dtype=None) -> torch.Tensor:
    """Positions `slots` of an 8-bit cache as rows [n, kv + rope] of `dtype` (default: the rope
    key's); rows of slots outside the cache are zeros."""
    device = slots.device
    with _Device(device) as stream:
        c = _cache(cache, device, None)
        _slots(slots, device)
        dtype = dtype or cache[1].dtype
        _require(dtype in _KIND, "cache_read writes fp32, fp16 or bf16")
        out = torch.empty(slots.shape[0], c.kv + c.rope_dim, dtype=dtype, device=device)
        rc = _lib().mm_latent_cache_read(ctypes.byref(c), slots.data_ptr(), slots.shape[0], out.data_ptr(),
                                         c.kv + c.rope_dim, _KIND[dtype], stream)
        if rc:
            _fail(rc)
    return out


def _index(t, device, n, what):
    _require(t.dtype == torch.int32 and t.dim() == 1 and t.shape[0] == n and t.is_contiguous(),
             f"{what} is a contiguous int32 vector of {n}")
    _on(device, t)
    return t.data_ptr()


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
    device = q.device
    with _Device(device) as stream:
        _require(q.dim() == 4 and q.dtype in _HALF and (q.shape[3] <= 1 or q.stride(3) == 1),
                 "q is fp16 or bf16 [rows, tokens, heads, kv + rope] with adjacent values")
        B, T, H, W = q.shape
        _require(0 < kv_rank <= W and T > 0 and H > 0, "kv_rank must be in (0, q's width]")
        d = _Desc()
        d.q, (d.q_row_stride, d.q_token_stride, d.q_head_stride, _) = q.data_ptr(), q.stride()
        d.dtype, d.rows, d.tokens, d.heads, d.scale = _KIND[q.dtype], B, T, H, scale
        if prefix is not None:
            c = _cache(prefix, device, kv_rank)
            _require(c.kv + c.rope_dim == W, "prefix width differs from q's")
            _require(group_start is not None and prefix_len is not None and group_start.dim() == 1 and
                     group_start.shape[0] > 0, "a prefix needs group_start [groups + 1] and prefix_len [groups]")
            G = group_start.shape[0] - 1
            d.prefix = ctypes.pointer(c)
            d.groups = G
            d.group_start = _index(group_start, device, G + 1, "group_start")
            d.prefix_len = _index(prefix_len, device, G, "prefix_len")
            d.max_group = B if max_group is None else max_group
            d.max_prefix = c.positions if max_prefix is None else max_prefix
        if suffix is not None:
            c = _cache(suffix, device, kv_rank)
            _require(c.kv + c.rope_dim == W, "suffix width differs from q's")
            _require(suffix_len is not None, "a suffix needs suffix_len [rows]")
            d.suffix = ctypes.pointer(c)
            d.suffix_len = _index(suffix_len, device, B, "suffix_len")
            d.max_suffix = c.positions if max_suffix is None else max_suffix
        out = torch.empty(B, T, H, kv_rank, dtype=q.dtype, device=device)
        d.out = out.data_ptr()
        lse = None
        if return_lse:
            lse = torch.empty(B, T, H, dtype=torch.float32, device=device)
            d.lse = lse.data_ptr()
        L = _lib()
        n = L.mm_shared_prefix_attention_workspace(ctypes.byref(d))
        if n < 0:
            _fail(-n)
        work = torch.empty(n, dtype=torch.uint8, device=device) if n else None
        rc = L.mm_shared_prefix_attention(ctypes.byref(d), work.data_ptr() if n else None, n, stream)
        if rc:
            _fail(rc)
    return (out, lse) if return_lse else out


def verify_drafts(target_probs: torch.Tensor, draft_tokens: torch.Tensor, draft_len: torch.Tensor,
                  u_accept: torch.Tensor, u_sample: torch.Tensor, *, draft_probs: torch.Tensor | None = None):
    """Accepts drafted tokens against the target's probabilities (speculative sampling).

    target_probs [rows, drafts + 1, vocab] and draft_probs [rows, drafts, vocab] (None:
    deterministic drafts) share one type (fp32, fp16 or bf16); draft_tokens [rows, drafts] and
    draft_len [rows] int32; u_accept [rows, drafts] and u_sample [rows] fp32 in [0, 1). Returns
    int32 (tokens [rows, drafts + 1], accepted [rows]): the accepted tokens, one more sampled
    from the residual at the first rejection (from the target when all were accepted), then -1."""
    device = target_probs.device
    with _Device(device) as stream:
        _require(target_probs.dim() == 3 and target_probs.dtype in _KIND and target_probs.is_contiguous(),
                 "target_probs is contiguous [rows, drafts + 1, vocab]")
        B, K1, V = target_probs.shape
        K = K1 - 1
        _require(K >= 0 and draft_tokens.shape == (B, K) and draft_tokens.dtype == torch.int32 and
                 draft_tokens.is_contiguous(), "draft_tokens is contiguous int32 [rows, drafts]")
        _require(u_accept.shape == (B, K) and u_accept.dtype == torch.float32 and u_accept.is_contiguous() and
                 u_sample.shape == (B,) and u_sample.dtype == torch.float32 and u_sample.is_contiguous(),
                 "u_accept is contiguous fp32 [rows, drafts], u_sample fp32 [rows]")
        _on(device, draft_tokens, u_accept, u_sample)
        if draft_probs is not None:
            _require(draft_probs.shape == (B, K, V) and draft_probs.dtype == target_probs.dtype and
                     draft_probs.is_contiguous(), "draft_probs is contiguous [rows, drafts, vocab] of target_probs' type")
            _on(device, draft_probs)
        lens = _index(draft_len, device, B, "draft_len")
        tokens = torch.empty(B, K1, dtype=torch.int32, device=device)
        accepted = torch.empty(B, dtype=torch.int32, device=device)
        rc = _lib().mm_verify_drafts(target_probs.data_ptr(), None if draft_probs is None else draft_probs.data_ptr(),
                                     _KIND[target_probs.dtype], draft_tokens.data_ptr(), lens, u_accept.data_ptr(),
                                     u_sample.data_ptr(), B, K, V, tokens.data_ptr(), accepted.data_ptr(), stream)
        if rc:
            _fail(rc)
    return tokens, accepted
