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
wait; outputs and scratch come from torch's allocator. No gradient flows through them: a tensor
that requires one is refused while gradients are recorded. Failures raise :class:`EngineError`
(what only the device knows: ``check_status``).

The checks, allocations and C calls are in csrc/latent_torch.cpp (a small call's time is its
host path); this module names the arguments and documents them.
"""
from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import os
from typing import NamedTuple

import torch

from .engine import EngineError, lib

_EXT_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_latent_torch.so")


def _load():
    lib()  # reports a library that was not built
    if not os.path.exists(_EXT_PATH):
        raise EngineError(3, f"torch binding not built: {_EXT_PATH} "
                             "(run python -m cpp_inference_train_engine_b200.build)")
    loader = importlib.machinery.ExtensionFileLoader("_latent_torch", _EXT_PATH)
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_latent_torch", loader))
    loader.exec_module(module)
    return module


_ext = _load()
_attention, _write, _read, _verify = (_ext.shared_prefix_attention, _ext.cache_write, _ext.cache_read,
                                      _ext.verify_drafts)


def check_status(device=None) -> None:
    """Waits for the current stream and raises EngineError when a kernel of these operators gave up on
    a wait on `device` since the last check (the results it concerns are NaN)."""
    with torch.cuda.device(device):
        rc = lib().mm_latent_status(torch.cuda.current_stream().cuda_stream)
    if rc:
        text = ctypes.create_string_buffer(512)
        lib().mm_latent_last_error(text, len(text))
        raise EngineError(rc, text.value.decode())


class LatentCache(NamedTuple):
    """An 8-bit cache: latent [rows, positions, kv] float8_e4m3fn, rope [rows, positions, rope]
    fp16 or bf16, scale [rows, positions] fp32; value = latent * scale."""
    latent: torch.Tensor
    rope: torch.Tensor
    scale: torch.Tensor


def alloc_cache(rows: int, positions: int, kv: int, rope: int, dtype=torch.float16, device="cuda") -> LatentCache:
    """An 8-bit cache of zeros; `dtype` is the rope key's (and the queries')."""
    if dtype not in (torch.float16, torch.bfloat16):
        raise EngineError(1, "rope keys are fp16 or bf16")
    return LatentCache(torch.zeros(rows, positions, kv, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
                       torch.zeros(rows, positions, rope, dtype=dtype, device=device),
                       torch.zeros(rows, positions, dtype=torch.float32, device=device))


def cache_write(cache: LatentCache, latent: torch.Tensor, rope: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantises new positions into an 8-bit cache in place: latent [n, kv] and rope [n, rope] of
    one type (fp32, fp16 or bf16), position i into slots[i] = row * positions + position; slots
    outside the cache are skipped (free rows of a step pass -1), the others must be distinct (a
    position given twice ends as a mix of both)."""
    _write(cache, latent, rope, slots)


def cache_read(cache: LatentCache, slots: torch.Tensor, dtype=None) -> torch.Tensor:
    """Positions `slots` of an 8-bit cache as rows [n, kv + rope] of `dtype` (default: the rope
    key's); rows of slots outside the cache are zeros."""
    return _read(cache, slots, dtype)


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
    return _attention(q, prefix, suffix, group_start, prefix_len, suffix_len, scale, kv_rank, max_group, max_prefix,
                      max_suffix, return_lse)


def verify_drafts(target_probs: torch.Tensor, draft_tokens: torch.Tensor, draft_len: torch.Tensor,
                  u_accept: torch.Tensor, u_sample: torch.Tensor, *, draft_probs: torch.Tensor | None = None):
    """Accepts drafted tokens against the target's probabilities (speculative sampling).

    target_probs [rows, drafts + 1, vocab] and draft_probs [rows, drafts, vocab] (None:
    deterministic drafts) share one type (fp32, fp16 or bf16); draft_tokens [rows, drafts] and
    draft_len [rows] int32; u_accept [rows, drafts] and u_sample [rows] fp32 in [0, 1). Returns
    int32 (tokens [rows, drafts + 1], accepted [rows]): the accepted tokens, one more sampled
    from the residual at the first rejection (from the target when all were accepted), then -1."""
    return _verify(target_probs, draft_tokens, draft_len, u_accept, u_sample, draft_probs)
