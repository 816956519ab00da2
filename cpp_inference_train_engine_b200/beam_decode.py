"""Beam search over paged latent caches.

The reference decodes one hypothesis per request, greedily or by sampling
(src/infer/inference.cpp:345-426, 469-579). Here every request keeps `beams` of them, and a step runs on
the operators of :mod:`paged`: each beam's position is stored through the page table (normalised and
rotated on the way, in 16 or 8 bits), one query token per beam attends over its pages, the best
continuations over beams and vocabulary are selected, and the page tables follow the chosen parents:
full pages, the prompt's among them, are shared by all beams that descend from them, and only a
beam's last, partly filled page is copied.

    python -m cpp_inference_train_engine_b200.beam_decode --model mla36m --requests 4 --beams 4 \\
        --prompt 128 --new 64

With `window`, a beam sees its last `window` positions and the first `sinks` ones. The projections and the
feed-forward blocks are plain torch products in fp16 with the residual in fp32.
"""
from __future__ import annotations

import argparse
import math

import numpy as np
import torch

from . import latent, paged
from .config import MLA36M, TINY, ModelConfig
from .engine import EngineError, init_params
from .group_decode import _rmsnorm, check_parameters, decode_weights, rotate


class BeamDecoder:
    """`prompts`: one token list per request; `beams` hypotheses each; `new_tokens` bounds a completion.
    `cache_bits` 8 or 16 is the storage of all positions, `page_size` the positions of a page."""

    def __init__(self, cfg: ModelConfig, params, prompts, beams: int, new_tokens: int, page_size: int = 16,
                 cache_bits: int = 16, window: int | None = None, sinks: int = 0, device="cuda"):
        if cache_bits not in (8, 16):
            raise EngineError(1, "cache_bits must be 8 or 16")
        if new_tokens < 1 or not prompts or any(len(p) < 1 for p in prompts):
            raise EngineError(1, "prompts of one token or more and new_tokens >= 1 are needed")
        if not 1 <= beams <= 32 or beams > cfg.vocab_size:
            raise EngineError(1, "beams must be between 1 and 32 and no more than the vocabulary")
        if page_size < 1 or (window is not None and window < 1) or sinks < 0:
            raise EngineError(1, "page_size and window must be positive, sinks not negative")
        if max(len(p) for p in prompts) + new_tokens > cfg.max_sequence_length:
            raise EngineError(1, "Prompt plus requested tokens exceeds context")
        prompts = [list(map(int, p)) for p in prompts]
        if any(not 0 <= t < cfg.vocab_size for p in prompts for t in p):
            raise EngineError(1, "a prompt's token is outside the vocabulary")
        params = check_parameters(cfg, params)
        self.cfg, self.beams, self.new_tokens, self.page, self.device = cfg, beams, new_tokens, page_size, device
        self.window, self.sinks = window, sinks
        self.embedding, self.final_norm, self.layers = decode_weights(cfg, params, device)
        G, R, P = len(prompts), len(prompts) * beams, page_size
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
        self.prompt_len = i32([len(p) for p in prompts])
        self.max_prompt = max(len(p) for p in prompts)
        # Pages: every request's prompt in line (so that its rows are a contiguous cache too), then each beam's own
        # for the columns it may write, and its spare one. The prompts are rows of their own behind the beams', from
        # which a search's first beams descend.
        held = -(-self.max_prompt // P)                       # pages of a prompt's stretch
        columns = -(-(self.max_prompt + new_tokens) // P)
        table = torch.full((R + G, columns), -1, dtype=torch.int32)
        spare, lengths, free = torch.full((R + G,), -1, dtype=torch.int32), torch.zeros(R + G, dtype=torch.int32), G * held
        for g, p in enumerate(prompts):
            table[R + g, :-(-len(p) // P)] = g * held + torch.arange(-(-len(p) // P))
            lengths[R + g] = len(p)
            begin, end = len(p) // P, -(-(len(p) + new_tokens) // P)
            for r in range(g * beams, (g + 1) * beams):
                table[r, begin:end] = free + torch.arange(end - begin)
                spare[r], lengths[r] = free + end - begin, begin * P
                free += end - begin + 1
        self.cache = paged.alloc_pages(cfg.n_layers, free, P, cfg.kv_lora_rank, cfg.head_dim_rope, torch.float16, cache_bits, device)
        self.start = (table.to(device), spare.to(device), lengths.to(device))
        self.prompt_rows = torch.arange(R, R + G, dtype=torch.int32, device=device)
        self.base = (torch.arange(G, dtype=torch.int32, device=device) * beams)[:, None]  # a request's first row
        padded = torch.zeros(G, self.max_prompt, dtype=torch.int32, device=device)
        for g, p in enumerate(prompts):
            padded[g, self.max_prompt - len(p):] = i32(p)  # aligned at the end: the positions before the first are negative
        self.prompt_logits = self._prefill(padded, held)
        self._check_status()

    def _check_status(self):
        """Waits, and raises EngineError where a kernel gave up on a wait: of the prompts' attention (latent) or of the
        beams' (paged)."""
        latent.check_status(self.device)
        paged.check_status(self.device)

    def _layer(self, l, x, w, positions, table, rows, attend):
        """One block over hidden rows x [n, T, d] whose tokens stand at `positions` [n, T] (negative: none)."""
        c = self.cfg
        n, T = positions.shape
        h = _rmsnorm(x, w["attn_norm"], c.norm_epsilon).half()
        cq = _rmsnorm(h @ w["w_dq"], w["q_norm"], c.norm_epsilon).half()
        q = (cq @ w["w_uq"]).view(n, T, c.n_heads, c.qk_dim)
        paged.append(paged.layer(self.cache, l), (h @ w["w_dkv"]).view(n * T, c.kv_width), table, positions.reshape(-1),
                     kv_rank=c.kv_lora_rank, rows=rows, theta=c.rope_theta, norm=w["kv_norm"], eps=c.norm_epsilon)
        absorbed = torch.einsum("bthd,hdk->bthk", q[..., :c.head_dim_nope], w["uk"])
        turned = rotate(q[..., c.head_dim_nope:], positions.clamp_min(0)[..., None], c.rope_theta).half()
        context = attend(l, torch.cat([absorbed, turned], -1))
        heads = torch.einsum("bthk,hkd->bthd", context, w["uv"]).reshape(n, T, c.attn_width)
        x = x + (heads @ w["w_o"]).float()
        h = _rmsnorm(x, w["ffn_norm"], c.norm_epsilon).half()
        return x + ((torch.nn.functional.silu(h @ w["w_gate"]) * (h @ w["w_up"])) @ w["w_down"]).float()

    def _hidden(self, tokens, positions, table, rows, attend):
        # what only the device knows is kept inside the table instead of checked
        x = self.embedding[tokens.long().clamp(0, self.cfg.vocab_size - 1)].float()
        for l, w in enumerate(self.layers):
            x = self._layer(l, x, w, positions, table, rows, attend)
        return _rmsnorm(x, self.final_norm, self.cfg.norm_epsilon).half()

    @property
    def scale(self):
        return 1.0 / math.sqrt(self.cfg.qk_dim)

    def _prefill(self, padded, held):
        """Every prompt once: its tokens are the last of its stretch of pages, each seeing those before it."""
        G, T = padded.shape
        P, c = self.page, self.cfg
        positions = torch.arange(T, dtype=torch.int32, device=self.device)[None] - (T - self.prompt_len[:, None])
        rows = torch.repeat_interleave(self.prompt_rows, T)

        def attend(l, q):
            pool = paged.layer(self.cache, l)
            stretch = lambda t, *w: t[:G * held].view(G, held * P, *w)  # noqa: E731
            stored = stretch(pool, c.kv_width) if torch.is_tensor(pool) else latent.LatentCache(
                stretch(pool.latent, c.kv_lora_rank), stretch(pool.rope, c.head_dim_rope), stretch(pool.scale))
            if self.window is None:
                return latent.shared_prefix_attention(q, None, stored, None, None, self.prompt_len, self.scale, kv_rank=c.kv_lora_rank)
            # with a window a prompt's tokens go one at a time: token t of every prompt is a row
            context = torch.zeros(*q.shape[:3], c.kv_lora_rank, dtype=q.dtype, device=q.device)
            table = self.start[0][G * self.beams:]
            for t in range(T):
                context[:, t] = paged.attention(q[:, t], pool, table, positions[:, t].clamp_min(-1) + 1, self.scale,
                                                kv_rank=c.kv_lora_rank, window=self.window, sinks=self.sinks)
            return context

        hidden = self._hidden(padded, positions, self.start[0], rows, attend)
        return (hidden[:, -1] @ self.embedding.T).float()

    def step_logits(self, tokens, positions, table):
        """Logits [requests, beams, vocab] of the beams' last tokens [rows], which are stored at `positions` [rows]
        of their tables (negative: a finished beam, which stores nothing and whose logits mean nothing)."""
        lengths = positions + 1

        def attend(l, q):
            return paged.attention(q[:, 0], paged.layer(self.cache, l), table, lengths, self.scale, kv_rank=self.cfg.kv_lora_rank,
                                   window=self.window, sinks=self.sinks)[:, None]

        hidden = self._hidden(tokens[:, None], positions[:, None], table, None, attend)
        return (hidden[:, 0] @ self.embedding.T).float().view(-1, self.beams, self.cfg.vocab_size)

    def search(self, length_penalty: float = 0.0):
        """The beams of every request, best first: lists of (tokens, log-probability). A completion ends with the
        end-of-sequence token or after `new_tokens`; hypotheses are ranked by log-probability / length ^
        length_penalty at the end (the search itself compares log-probabilities). Raises EngineError where a
        request has no continuation left (its logits hold a NaN)."""
        c, K, N = self.cfg, self.beams, self.new_tokens
        G = self.base.shape[0]
        R = G * K
        zero = torch.zeros(G, 1, device=self.device)
        scores, _, tokens = paged.beam_select(self.prompt_logits[:, None].contiguous(), zero, beams=K)
        table, spare, lengths = (t[:R] for t in paged.beam_reorder(
            self.cache, *self.start, torch.cat([torch.repeat_interleave(self.prompt_rows, K), self.prompt_rows])))
        history = torch.full((G, K, N), -1, dtype=torch.int32, device=self.device)
        history[:, :, 0] = tokens
        finished = tokens == c.eos_id
        count = torch.ones_like(tokens)
        for step in range(1, N + 1):
            failed = torch.isneginf(scores[:, 0]).any()
            stop, none = torch.stack([finished.all(), failed]).tolist()
            if none:
                self._check_status()  # results of a kernel that gave up are NaN too
                raise EngineError(6, "a request has no continuation with a probability (its logits hold a NaN)")
            if stop or step == N:
                break
            live = ~finished.view(-1)
            positions = torch.where(live, lengths, -1)
            logits = self.step_logits(tokens.view(-1), positions, table)
            lengths = lengths + live.int()
            scores, chosen, tokens = paged.beam_select(logits, scores, finished=finished, eos=c.eos_id)
            at = chosen.long()
            follow = lambda t: t.gather(1, at)  # noqa: E731
            was = follow(finished)
            history = history.gather(1, at[:, :, None].expand(-1, -1, N))
            history[:, :, step] = torch.where(was, -1, tokens)
            count = follow(count) + ~was
            finished = was | (tokens == c.eos_id) | (tokens < 0)
            table, spare, lengths = paged.beam_reorder(self.cache, table, spare, lengths, (chosen + self.base).view(-1))
        self._check_status()
        ranked = (scores / count.float().pow(length_penalty)).nan_to_num(nan=-math.inf, neginf=-math.inf)
        order = ranked.sort(dim=1, descending=True, stable=True).indices.cpu()
        history, count, scores = history.cpu(), count.cpu(), scores.cpu()
        return [[([t for t in history[g, k, :count[g, k]].tolist() if t >= 0], float(scores[g, k]))
                 for k in order[g].tolist() if scores[g, k] > -math.inf] for g in range(G)]


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--model", choices=("tiny", "mla36m"), default="mla36m")
    ap.add_argument("--requests", type=int, default=4)
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=128)
    ap.add_argument("--new", type=int, default=64)
    ap.add_argument("--page", type=int, default=16)
    ap.add_argument("--cache-bits", type=int, choices=(8, 16), default=16)
    ap.add_argument("--window", type=int, default=None)
    ap.add_argument("--sinks", type=int, default=0)
    ap.add_argument("--length-penalty", type=float, default=0.0)
    ap.add_argument("--seed", type=int, default=1)
    args = ap.parse_args(argv)
    cfg = {"tiny": TINY, "mla36m": MLA36M}[args.model]
    rng = np.random.default_rng(args.seed)
    prompts = [rng.integers(0, cfg.vocab_size - 8, args.prompt).tolist() for _ in range(args.requests)]
    params = init_params(cfg, args.seed)

    def run():
        d = BeamDecoder(cfg, params, prompts, args.beams, args.new, args.page, args.cache_bits, args.window, args.sinks)
        begin, end = torch.cuda.Event(True), torch.cuda.Event(True)
        begin.record()
        out = d.search(args.length_penalty)
        end.record()
        end.synchronize()
        return out, begin.elapsed_time(end)

    run()  # first launches and allocations
    out, ms = run()
    tokens = sum(len(t) for beams in out for t, _ in beams)
    print(f"{args.requests} requests x {args.beams} beams, {tokens} tokens in {ms:.1f} ms ({tokens / ms * 1e3:.0f} tokens/s), "
          f"best scores {', '.join(f'{beams[0][1]:.2f}' for beams in out[:4])}")


if __name__ == "__main__":
    main()
