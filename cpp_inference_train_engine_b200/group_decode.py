"""Decoding groups of completions that share their prompts, with drafted tokens.

One decode step of the MLA decoder (src/infer/inference.cpp:47-174) on the operators of
:mod:`latent`: every prompt's latent rows are stored once for its group of rows, each row keeps
its own completion in an 8-bit (or 16-bit) cache, a step decodes the row's last token together
with up to `drafts` proposed ones, and the proposals are accepted against the model's
probabilities. The rollout of a GRPO group (several completions of one prompt,
src/train/trainer.cpp:187-213) and requests with a common system prompt have this form; the
rollout of the context (``CudaExecution.rollout``) keeps a copy of the prompt in every row.

    python -m cpp_inference_train_engine_b200.group_decode --model mla36m --groups 4 --rows 8 \\
        --prompt 128 --new 64 --drafts 4

Proposals come from the row's own history (the tokens that followed the latest earlier
occurrence of its last token), so they need no second model. The operators are those of
latent.py; the projections and the feed-forward blocks are plain torch products in fp16 with
the residual in fp32.
"""
from __future__ import annotations

import argparse
import math

import numpy as np
import torch

from . import latent
from .config import MLA36M, TINY, ModelConfig
from .engine import EngineError, init_params

_NAMES = ("attn_norm", "w_dq", "q_norm", "w_uq", "w_dkv", "kv_norm", "w_uk", "w_uv", "w_o", "ffn_norm", "w_gate",
          "w_up", "w_down")


def _rmsnorm(x, w, eps):
    x = x.float()
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w


def check_parameters(cfg: ModelConfig, params):
    """The model's parameters as one flat fp32 array; another model's are refused."""
    params = np.ascontiguousarray(params, np.float32).reshape(-1)
    if params.size != cfg.parameter_count():
        raise EngineError(1, f"the model has {cfg.parameter_count()} parameters, got {params.size}")
    return params


def decode_weights(cfg: ModelConfig, params, device):
    """(embedding, final norm, layers) of a flat parameter array as decode uses them: matrices in fp16, norms
    in fp32, and per head `uk` [heads, nope, kv], which queries absorb, and `uv` [heads, kv, value], which
    expands the latent context."""
    flat = torch.from_numpy(params).to(device)
    tensors, at = [], 0
    for _, (r, c), _ in cfg.parameter_shapes():
        tensors.append(flat[at:at + r * c].view(r, c))
        at += r * c
    layers = []
    for l in range(cfg.n_layers):
        w = dict(zip(_NAMES, tensors[2 + 13 * l:15 + 13 * l]))
        w = {k: v.view(-1) if k.endswith("norm") else v.half() for k, v in w.items()}
        w["uk"] = w["w_uk"].view(cfg.kv_lora_rank, cfg.n_heads, cfg.head_dim_nope).permute(1, 2, 0).contiguous()
        w["uv"] = w["w_uv"].view(cfg.kv_lora_rank, cfg.n_heads, cfg.head_dim_value).permute(1, 0, 2).contiguous()
        layers.append(w)
    return tensors[0].half(), tensors[1].view(-1), layers


def rotate(x, positions, theta: float):
    """Adjacent pairs rotated by position * theta^(-j / width) (src/model/ops.cpp:88-108)."""
    w = x.shape[-1]
    j = torch.arange(0, w, 2, device=x.device, dtype=torch.float32)
    angle = positions.float()[..., None] * torch.pow(theta, -j / w)
    cos, sin = angle.cos(), angle.sin()
    a, b = x[..., 0::2].float(), x[..., 1::2].float()
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)


class GroupDecoder:
    """`prompts`: one token list per group; `rows`: completions per group (a number, or one per
    group); `new_tokens` bounds every completion. `cache_bits` 8 or 16 is the storage of the
    prompts and the completions."""

    def __init__(self, cfg: ModelConfig, params, prompts, rows, new_tokens: int, drafts: int = 0,
                 cache_bits: int = 8, device="cuda"):
        if cache_bits not in (8, 16):
            raise EngineError(1, "cache_bits must be 8 or 16")
        if drafts < 0 or new_tokens < 1 or not prompts or any(len(p) < 1 for p in prompts):
            raise EngineError(1, "prompts of one token or more, new_tokens >= 1 and drafts >= 0 are needed")
        if max(len(p) for p in prompts) + new_tokens > cfg.max_sequence_length:
            raise EngineError(1, "Prompt plus requested tokens exceeds context")
        rows = [rows] * len(prompts) if isinstance(rows, int) else list(rows)
        if len(rows) != len(prompts) or min(rows) < 1:
            raise EngineError(1, "rows: one positive number per group")
        prompts = [list(map(int, p)) for p in prompts]
        if any(not 0 <= t < cfg.vocab_size for p in prompts for t in p):
            raise EngineError(1, "a prompt's token is outside the vocabulary")
        params = check_parameters(cfg, params)
        self.cfg, self.drafts, self.new_tokens, self.bits = cfg, drafts, new_tokens, cache_bits
        self.device = device
        self.embedding, self.final_norm, self.layers = decode_weights(cfg, params, device)
        G, B = len(prompts), sum(rows)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
        self.max_prompt, self.max_group = max(len(p) for p in prompts), max(rows)
        self.group_start = i32(np.concatenate([[0], np.cumsum(rows)]))
        self.prompt_len = i32([len(p) for p in prompts])
        self.row_group = torch.repeat_interleave(torch.arange(G, device=device), torch.tensor(rows, device=device))
        self.row_prompt = self.prompt_len[self.row_group].long()
        # a row's completion, and what a step writes past its end
        self.capacity = new_tokens + drafts
        self.prefix = [self._cache(G, self.max_prompt) for _ in self.layers]
        self.suffix = [self._cache(B, self.capacity) for _ in self.layers]
        self.history = torch.full((B, self.max_prompt + self.capacity + 1), -1, dtype=torch.int32, device=device)
        padded = torch.zeros(G, self.max_prompt, dtype=torch.int32, device=device)
        for i, p in enumerate(prompts):
            tokens = i32(p)
            padded[i, self.max_prompt - len(p):] = tokens  # aligned at the end: the positions before the first are negative
            self.history[self.row_group == i, :len(p)] = tokens
        self.count = torch.zeros(B, dtype=torch.int64, device=device)  # generated tokens per row
        self.prompt_logits = self._prefill(padded)

    def _cache(self, rows, positions):
        c = self.cfg
        if self.bits == 8:
            return latent.alloc_cache(rows, positions, c.kv_lora_rank, c.head_dim_rope, torch.float16, self.device)
        return torch.zeros(rows, positions, c.kv_width, dtype=torch.float16, device=self.device)

    def _write(self, cache, values, key, slots):
        if self.bits == 8:
            latent.cache_write(cache, values, key, slots)
        else:
            keep = slots >= 0
            cache.view(-1, cache.shape[-1])[slots[keep]] = torch.cat([values, key], -1)[keep].half()

    def stored(self, layer: int, group: int):
        """The stored prompt of a group as fp16 rows [latent | rope]."""
        n = int(self.prompt_len[group])
        if self.bits == 16:
            return self.prefix[layer][group, :n]
        slots = group * self.max_prompt + torch.arange(n, device=self.device)
        return latent.cache_read(self.prefix[layer], slots)

    def cache_bytes(self):
        tensors = [t for c in self.prefix + self.suffix for t in (c if self.bits == 8 else (c,))]
        return sum(t.numel() * t.element_size() for t in tensors)

    def _rope(self, x, positions):
        return rotate(x, positions, self.cfg.rope_theta)

    def _blocks(self, tokens, positions, slots, stores, attend):
        """The decoder over tokens [n, T] at `positions`; writes each position's latent row into
        stores[layer] at `slots`, attends with attend(layer, q) and returns the final hidden rows."""
        c = self.cfg
        n, T = tokens.shape
        # what only the device knows is kept inside the table instead of checked
        x = self.embedding[tokens.long().clamp(0, c.vocab_size - 1)].float()
        for l, w in enumerate(self.layers):
            h = _rmsnorm(x, w["attn_norm"], c.norm_epsilon).half()
            cq = _rmsnorm(h @ w["w_dq"], w["q_norm"], c.norm_epsilon).half()
            q = (cq @ w["w_uq"]).view(n, T, c.n_heads, c.qk_dim)
            kv = h @ w["w_dkv"]
            values = _rmsnorm(kv[..., :c.kv_lora_rank], w["kv_norm"], c.norm_epsilon)
            key = self._rope(kv[..., c.kv_lora_rank:], positions)
            self._write(stores[l], values.view(n * T, -1), key.view(n * T, -1), slots.view(-1))
            absorbed = torch.einsum("bthd,hdk->bthk", q[..., :c.head_dim_nope], w["uk"])
            turned = self._rope(q[..., c.head_dim_nope:], positions[..., None]).half()
            context = attend(l, torch.cat([absorbed, turned], -1))
            heads = torch.einsum("bthk,hkd->bthd", context, w["uv"]).reshape(n, T, c.attn_width)
            x = x + (heads @ w["w_o"]).float()
            h = _rmsnorm(x, w["ffn_norm"], c.norm_epsilon).half()
            x = x + ((torch.nn.functional.silu(h @ w["w_gate"]) * (h @ w["w_up"])) @ w["w_down"]).float()
        return _rmsnorm(x, self.final_norm, c.norm_epsilon).half()

    def _attend(self, layer, q, prefix, suffix, suffix_len):
        return latent.shared_prefix_attention(
            q, prefix[layer] if prefix else None, suffix[layer], self.group_start if prefix else None,
            self.prompt_len if prefix else None, suffix_len, 1.0 / math.sqrt(self.cfg.qk_dim),
            kv_rank=self.cfg.kv_lora_rank, max_group=self.max_group if prefix else None)

    def _prefill(self, padded):
        """Every prompt once: its tokens are the last of its stored row, each seeing those before it."""
        G, P = padded.shape
        positions = torch.arange(P, device=self.device)[None] - (P - self.prompt_len[:, None])
        slots = torch.where(positions >= 0, torch.arange(G, device=self.device)[:, None] * P + positions, -1)
        hidden = self._blocks(padded, positions.clamp_min(0), slots, self.prefix,
                              lambda l, q: self._attend(l, q, None, self.prefix, self.prompt_len))
        return (hidden[:, -1] @ self.embedding.T).float()

    def step_logits(self, tokens):
        """Logits [rows, T, vocab] of the tokens [rows, T] that follow what the caches hold (the
        completions' first count - 1 tokens)."""
        B, T = tokens.shape
        done = (self.count - 1).clamp_min(0)
        # a generating row has room for its last token and `drafts` more; only for others is the count waited for
        if T > self.drafts + 1 and int(done.max()) + T > self.capacity:
            raise EngineError(1, "a row's completion has no room for that many tokens")
        at = done[:, None] + torch.arange(T, device=self.device)
        slots = torch.where(at < self.capacity, torch.arange(B, device=self.device)[:, None] * self.capacity + at, -1)
        suffix_len = (done + T).clamp_max(self.capacity).int()
        hidden = self._blocks(tokens, self.row_prompt[:, None] + at, slots, self.suffix,
                              lambda l, q: self._attend(l, q, self.prefix, self.suffix, suffix_len))
        return (hidden @ self.embedding.T).float()

    def _propose(self):
        """Proposals [rows, drafts] and how many each row has: what followed the latest earlier
        occurrence of the row's last token."""
        B, L = self.history.shape
        end = self.row_prompt + self.count  # tokens the row has
        place = torch.arange(L, device=self.device)
        last = self.history.gather(1, (end - 1)[:, None])
        earlier = (self.history == last) & (place[None] < (end - 1)[:, None])
        found = torch.where(earlier, place[None], -1).amax(1)
        at = (found[:, None] + 1 + place[None, :self.drafts]).clamp_max(L - 1)
        tokens = self.history.gather(1, at)
        number = torch.where(found >= 0, (end - 1 - found).clamp_max(self.drafts), 0)
        # the last token's place in the completion leaves room for this many more
        number = torch.minimum(number, (self.new_tokens - self.count - 1).clamp_min(0))
        return tokens.clamp_min(0), number.int()

    def _append(self, tokens, number):
        """Appends the first number[b] of tokens [rows, k] to every row."""
        k = tokens.shape[1]
        place = torch.arange(k, device=self.device)[None]
        at = ((self.row_prompt + self.count)[:, None] + place).clamp_max(self.history.shape[1] - 1)
        keep = place < number[:, None]
        self.history.scatter_(1, at, torch.where(keep, tokens, self.history.gather(1, at)))
        self.count += number

    def _probabilities(self, logits, temperature):
        if temperature > 0:
            return torch.softmax(logits / temperature, -1)
        best = torch.nn.functional.one_hot(logits.argmax(-1), logits.shape[-1]).float()
        return best.masked_fill_(logits.isnan().any(-1, keepdim=True), 0)  # argmax would pick the NaN

    def generate(self, temperature: float = 0.0, seed: int = 0):
        """Completes every row from its prompt: (tokens as one list per row, statistics). A completion
        ends with the end-of-sequence token or after `new_tokens`. Raises EngineError when a row's
        logits leave no token to pick (a NaN)."""
        c, B = self.cfg, self.row_group.numel()
        self.count.zero_()
        self.history.masked_fill_(torch.arange(self.history.shape[1], device=self.device) >= self.row_prompt[:, None], -1)
        g = torch.Generator(device=self.device).manual_seed(seed)
        uniform = lambda *shape: torch.rand(*shape, generator=g, device=self.device)  # noqa: E731

        def accept(logits, proposals, number):
            return latent.verify_drafts(self._probabilities(logits, temperature), proposals, number,
                                        uniform(B, proposals.shape[1]), uniform(B))

        none = torch.zeros(B, 0, dtype=torch.int32, device=self.device)
        zero = torch.zeros(B, dtype=torch.int32, device=self.device)
        first, _ = accept(self.prompt_logits[self.row_group][:, None], none, zero)
        self._append(first, torch.ones_like(self.count))
        open_rows = (first[:, 0] != c.eos_id) & (self.count < self.new_tokens)
        steps = kept = proposed = 0
        failed = (first[:, 0] < 0).any()
        while True:
            go_on, no_token = torch.stack([open_rows.any(), failed]).tolist()
            if no_token:
                raise EngineError(6, "no token has a probability (the logits hold a NaN)")
            if not go_on:
                break
            last = self.history.gather(1, (self.row_prompt + self.count - 1)[:, None])
            tokens, number = self._propose() if self.drafts else (none, zero)
            number = torch.where(open_rows, number, 0).int()
            picked, accepted = accept(self.step_logits(torch.cat([last, tokens], 1)), tokens.contiguous(), number)
            failed = (open_rows & (picked.gather(1, accepted.long()[:, None])[:, 0] < 0)).any()
            # nothing after an end-of-sequence token, nothing for the rows that are done
            take = accepted.long() + 1
            stop = (picked == c.eos_id) & (torch.arange(picked.shape[1], device=self.device)[None] < take[:, None])
            take = torch.where(stop.any(1), stop.int().argmax(1) + 1, take) * open_rows
            self._append(picked, take)
            open_rows &= ~stop.any(1) & (self.count < self.new_tokens)
            steps += 1
            kept += int((accepted * (number > 0)).sum())
            proposed += int(number.sum())
        latent.check_status(self.device)
        history, count, start = self.history.cpu(), self.count.cpu(), self.row_prompt.cpu()
        out = [history[b, start[b]:start[b] + count[b]].tolist() for b in range(B)]
        return out, {"steps": steps, "tokens": int(count.sum()), "proposed": proposed, "accepted": kept}


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--model", choices=("tiny", "mla36m"), default="mla36m")
    ap.add_argument("--groups", type=int, default=4)
    ap.add_argument("--rows", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=128)
    ap.add_argument("--new", type=int, default=64)
    ap.add_argument("--drafts", type=int, default=4)
    ap.add_argument("--cache-bits", type=int, choices=(8, 16), default=8)
    ap.add_argument("--temperature", type=float, default=0.0)
    ap.add_argument("--seed", type=int, default=1)
    args = ap.parse_args(argv)
    cfg = {"tiny": TINY, "mla36m": MLA36M}[args.model]
    rng = np.random.default_rng(args.seed)
    prompts = [rng.integers(0, cfg.vocab_size - 8, args.prompt).tolist() for _ in range(args.groups)]
    params = init_params(cfg, args.seed)

    def run():
        d = GroupDecoder(cfg, params, prompts, args.rows, args.new, args.drafts, args.cache_bits)
        begin, end = torch.cuda.Event(True), torch.cuda.Event(True)
        begin.record()
        _, stats = d.generate(args.temperature, args.seed)
        end.record()
        end.synchronize()
        return d, stats, begin.elapsed_time(end)

    run()  # first launches and allocations
    d, stats, ms = run()
    copies = args.groups * args.rows * (args.prompt + d.capacity) * cfg.kv_width * 2 * cfg.n_layers
    print(f"{stats['tokens']} tokens in {ms:.1f} ms ({stats['tokens'] / ms * 1e3:.0f} tokens/s), {stats['steps']} steps, "
          f"{stats['accepted']} of {stats['proposed']} drafted tokens accepted; cache {d.cache_bytes() / 1e6:.2f} MB "
          f"({copies / 1e6:.2f} MB as 16-bit rows that each hold their prompt)")


if __name__ == "__main__":
    main()
