"""Paged latent caches and beam search on torch CUDA tensors (include/mm_paged.h).

A paged cache is a pool of pages and a table: position t of row r is entry ``t % page_size`` of page
``table[r, t // page_size]``, so rows of any length share one pool, long rows need no contiguous
memory, and rows may share pages. A 16-bit pool is a plain tensor ``[pages, page_size, kv + rope]``,
an 8-bit one a :class:`latent.LatentCache` whose rows are pages; ``alloc_pages`` makes both, with one
such pool per layer.

``append``
    stores new positions: latents normalised, keys rotated, in 16 or 8 bits;
``attention``
    absorbed latent attention of one new token per row over its pages, over all of them or through
    a sliding window with a few first positions that stay visible;
``beam_select`` / ``beam_reorder``
    a beam search's best continuations, and the page tables that follow the chosen parents.

The reference keeps one contiguous cache per request and decodes it greedily or by sampling
(src/infer/inference.cpp:47-174, 345-426). Calls enqueue on the current stream of the tensors'
device and do not wait; outputs and scratch come from torch's allocator. No gradient flows through
them: a tensor that requires one is refused while gradients are recorded. Failures raise
:class:`EngineError` (what only the device knows: ``check_status``).

The checks, allocations and C calls are in csrc/paged_torch.cpp; this module names the arguments
and documents them.
"""
from __future__ import annotations

import ctypes

import torch

from .engine import EngineError, lib
from .latent import LatentCache, _ext


def check_status(device=None) -> None:
    """Waits for the current stream and raises EngineError when a kernel of these operators gave up on
    a wait on `device` since the last check (the results it concerns are NaN)."""
    with torch.cuda.device(device):
        rc = lib().mm_paged_status(torch.cuda.current_stream().cuda_stream)
    if rc:
        text = ctypes.create_string_buffer(512)
        lib().mm_latent_last_error(text, len(text))
        raise EngineError(rc, text.value.decode())


def alloc_pages(layers: int, pages: int, page_size: int, kv: int, rope: int, dtype=torch.float16, bits: int = 16,
                device="cuda"):
    """The pools of `layers` layers, zeros: a tensor [layers, pages, page_size, kv + rope] of `dtype`
    (fp16 or bf16), or with bits = 8 a LatentCache whose tensors have the layers ahead and whose rope keys
    are of `dtype`. The fast forms of the operators need 128 + 16 or 512 + 32 values and pages of a
    multiple of 16 positions."""
    if dtype not in (torch.float16, torch.bfloat16):
        raise EngineError(1, "pages hold fp16 or bf16 (with bits = 8: rope keys)")
    if bits not in (8, 16):
        raise EngineError(1, "bits must be 8 or 16")
    if bits == 16:
        return torch.zeros(layers, pages, page_size, kv + rope, dtype=dtype, device=device)
    return LatentCache(torch.zeros(layers, pages, page_size, kv, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
                       torch.zeros(layers, pages, page_size, rope, dtype=dtype, device=device),
                       torch.zeros(layers, pages, page_size, dtype=torch.float32, device=device))


def layer(cache, index: int):
    """One layer's pool of an ``alloc_pages`` cache."""
    return cache[index] if torch.is_tensor(cache) else LatentCache(*(t[index] for t in cache))


def append(cache, values: torch.Tensor, table: torch.Tensor, positions: torch.Tensor, *, kv_rank: int,
           rows: torch.Tensor | None = None, theta: float = 10000.0, norm: torch.Tensor | None = None,
           eps: float = 1e-5) -> None:
    """Stores new positions in a pool in place: values [tokens, kv + rope] fp32, fp16 or bf16 (a
    projection's result: latents, then keys before their rotation), token i at positions[i] of table row
    rows[i] (None: token i is row i's). The latents are RMS-normalised with `norm` (fp32 [kv]; None: as they
    are), the keys' adjacent pairs rotated by position * theta^(-2 j / rope). positions and rows are int32
    [tokens]; a token with a negative position (a free row of a step), or whose position has no page, is
    skipped; two tokens of one call do not share a position."""
    _ext.paged_append(cache, values, table, positions, kv_rank, rows, theta, norm, eps)


def attention(q: torch.Tensor, cache, table: torch.Tensor, lengths: torch.Tensor, scale: float, *, kv_rank: int,
              window: int | None = None, sinks: int = 0, max_length: int | None = None, return_lse: bool = False):
    """Absorbed latent attention of one new token per row over its pages.

    q [rows, heads, kv + rope] fp16 or bf16 (any strides, adjacent values); table [rows, columns] and
    lengths [rows] int32. Row b sees positions [0, lengths[b]), with a `window` only its last `window` ones and
    the first `sinks`; entries of pages that it does not see may hold anything (positions of pages outside the
    pool are not seen either). `max_length` is what the host knows of the lengths (default: the table's
    columns); a tight one makes smaller launches. Returns the latent context [rows, heads, kv] in q's type
    (zeros for a row that sees nothing) and, with return_lse, the natural log-sum-exp [rows, heads] fp32."""
    return _ext.paged_attention(q, cache, table, lengths, scale, kv_rank, window, sinks, max_length, return_lse)


def beam_select(logits: torch.Tensor, scores: torch.Tensor, *, beams: int | None = None,
                finished: torch.Tensor | None = None, eos: int | None = None):
    """The best continuations of a beam search: (scores, parents, tokens) [batch, beams], best first.

    logits [batch, k, vocab] fp32, fp16 or bf16 (any strides, adjacent tokens), scores fp32 [batch, k]: the
    beams' log-probabilities so far (-infinity: a dead beam). A continuation's score is its beam's plus the
    token's log-probability; a finished beam (bool [batch, k]) has one, `eos` at its own score. `beams`
    (default k) are taken, ties by the lowest beam, then token. Entries for which there is no continuation
    are (-infinity, min(entry, k - 1), -1)."""
    return _ext.beam_select(logits, scores, beams, finished, eos)


def beam_reorder(cache, table: torch.Tensor, spare: torch.Tensor, lengths: torch.Tensor, parents: torch.Tensor):
    """Lets every row take over its parent's cache: new (table, spare, lengths), the pools changed in place.

    cache has its layers ahead (``alloc_pages``); table [rows, columns], spare, lengths and parents [rows]
    int32, parents as row numbers. Full pages are shared through the table. A row whose parent is another one
    gets the positions of its last, partly filled page in its own spare page, in every layer, and its own page at
    its length becomes its spare. Every row needs a page of its own for each column that it may grow into and a spare
    one, none of them another row's; a row that fills its table and then takes over a shorter one is left without a
    spare page (-1). A row that takes over one shorter by a page or more, and grows again, lacks pages: its entries up
    to its old length are others' too. They become -1, at the latest in the call after which the row begins them: put a
    page of its own there before it stores (a position without a page is not stored), and store no further than to
    the end of its last page between two calls (see include/mm_paged.h)."""
    return _ext.beam_reorder(cache, table, spare, lengths, parents)
