"""The latent-cache decode operators at the sizes they are used at: inputs, plain form, work.

Four operators of one decode step over a compressed (MLA) cache whose rows share prompts:
``cache_write`` and ``cache_read`` (8-bit latent cache), ``shared_prefix_attention`` (the
prompt of a group stored and read once) and ``verify_drafts`` (acceptance of drafted tokens).
A case is plain sizes; ``prepare`` makes its inputs on the GPU from a seed; ``run`` is one
call of the operator (``own``) or its plain form in elementary torch operations in 32 bits;
``exact`` is the definition in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
E4M3_MAX = 448.0
SCALE_FLOOR = 2.0 ** -100


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # one group of eight rollouts of a short prompt, early in the completion: latency
        _att("group_of_8", groups=1, rows=8, heads=8, kv=128, rope=16, prefix=128, suffix=9),
        # the 2,048-row rollout (256 prompts x 8) of the 35.8M model late in its completions
        _att("rollout_2048_rows", groups=256, rows=8, heads=8, kv=128, rope=16, prefix=128, suffix=193),
        # requests that share system prompts of many lengths, bf16, groups of 1 to 16
        _att("system_prompts_ragged", groups=48, rows=16, heads=8, kv=128, rope=16, prefix=4099,
             suffix=771, dtype="bf16", ragged=True),
        # the scaled model's rollout: 16 prompts x 16, completions of up to 1,536
        _att("wide_rollout", groups=16, rows=16, heads=16, kv=512, rope=32, prefix=512, suffix=1536,
             ragged=True),
        # the same over the 8-bit cache
        _att("wide_rollout_fp8", groups=16, rows=16, heads=16, kv=512, rope=32, prefix=512, suffix=1536,
             ragged=True, cache="fp8"),
        # drafted tokens of 32 requests over one long document, 8-bit suffixes and prefix in bf16
        _att("long_prefix_drafts", groups=1, rows=32, tokens=4, heads=16, kv=512, rope=32, prefix=32768,
             suffix=513, dtype="bf16"),
        # one decode step's new positions
        _write("write_step", tokens=61, kv=128, rope=16, dtype="bf16", rows=64, positions=2048),
        # a prefill chunk of the scaled model
        _write("write_prefill", tokens=196608, kv=512, rope=32, dtype="fp16", rows=512, positions=512),
        # one request's prompt read back
        _read("read_prompt", tokens=517, kv=128, rope=16, dtype="fp16", rows=64, positions=2048),
        # a batch's prompts read back
        _read("read_batch", tokens=131072, kv=512, rope=32, dtype="bf16", rows=256, positions=1024),
        # a small server's step with four drafted tokens
        _verify("verify_8", rows=8, drafts=4, vocab=16384),
        # a large batch with seven drafted tokens each
        _verify("verify_1024", rows=1024, drafts=7, vocab=32768),
    ]


def _att(name=None, groups=1, rows=8, tokens=1, heads=8, kv=128, rope=16, prefix=128, suffix=16,
         dtype="fp16", cache="same", ragged=False):
    c = dict(op="attention", groups=groups, rows=rows, tokens=tokens, heads=heads, kv=kv, rope=rope,
             prefix=prefix, suffix=suffix, dtype=dtype, cache=cache, ragged=ragged)
    return dict(c, name=name) if name else c


def _write(name=None, tokens=1, kv=128, rope=16, dtype="fp16", rows=1, positions=128):
    c = dict(op="write", tokens=tokens, kv=kv, rope=rope, dtype=dtype, rows=rows, positions=positions)
    return dict(c, name=name) if name else c


def _read(name=None, tokens=1, kv=128, rope=16, dtype="fp16", rows=1, positions=128):
    c = dict(op="read", tokens=tokens, kv=kv, rope=rope, dtype=dtype, rows=rows, positions=positions)
    return dict(c, name=name) if name else c


def _verify(name=None, rows=1, drafts=4, vocab=16384, dtype="fp32", draft_probs=True):
    c = dict(op="verify", rows=rows, drafts=drafts, vocab=vocab, dtype=dtype, draft_probs=draft_probs)
    return dict(c, name=name) if name else c


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {"attention": work(listed()[5]), "write": work(listed()[7]), "read": work(listed()[9]),
            "verify": work(listed()[11])}
    while True:
        op = rng.choice(["attention", "attention", "attention", "write", "read", "verify"])
        wide = rng.random() < 0.5
        kv, rope = (512, 32) if wide else (128, 16)
        if op == "attention":
            c = _att(groups=_log(rng, 1, 256), rows=_log(rng, 1, 48), tokens=rng.choice([1, 1, 1, 2, 3, 4, 5, 8]),
                     heads=rng.choice([16, 16, 12, 5] if wide else [8, 8, 16, 3]), kv=kv, rope=rope,
                     prefix=_log(rng, 1, 16384), suffix=_log(rng, 9, 2048), dtype=rng.choice(["fp16", "bf16"]),
                     cache=rng.choice(["same", "fp8"]), ragged=rng.random() < 0.7)
            fits = c["groups"] * c["rows"] * (c["suffix"] + c["tokens"] * c["heads"]) * (kv + rope) < 6e8 and \
                c["groups"] * c["prefix"] * (kv + rope) < 3e8 and \
                c["groups"] * c["rows"] * c["tokens"] * c["heads"] * (c["prefix"] + c["suffix"]) < 1.2e8
        elif op == "verify":
            c = _verify(rows=_log(rng, 1, 1024), drafts=rng.randint(1, 8), vocab=_log(rng, 257, 50001),
                        dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]), draft_probs=rng.random() < 0.7)
            fits = c["rows"] * (c["drafts"] + 1) * c["vocab"] < 2.4e8
        else:
            make = _write if op == "write" else _read
            rows = _log(rng, 1, 512)
            c = make(tokens=_log(rng, 1, 130000), kv=kv, rope=rope, dtype=rng.choice(["fp16", "bf16", "fp32"]),
                     rows=rows, positions=_log(rng, 16, 2048))
            fits = c["tokens"] <= c["rows"] * c["positions"] <= 300000
        w = work(c)
        if fits and w["bytes"] <= most[op]["bytes"] * 4 and w["flops"] <= most["attention"]["flops"] \
                and w["bytes"] <= 8e8:
            return c


# --------------------------------------------------------------------------- sizes of a case
def _sizes(c):
    """Rows of each group, prefix length of each group, suffix length of each row: a fixed
    pattern of the case (ragged: spread over the range, odd lengths among them)."""
    G, R, P, S, T = c["groups"], c["rows"], c["prefix"], c["suffix"], c["tokens"]
    if not c["ragged"]:
        return [R] * G, [P] * G, [max(S, T)] * (G * R)
    rows = [1 + (g * 7919 + 5) % R for g in range(G)]
    plen = [P - (g * 613) % (P // 2 + 1) for g in range(G)]
    slen = [T + (b * 40503 + 77) % (max(S, T) - T + 1) for b in range(sum(rows))]
    return rows, plen, slen


def work(c):
    if c["op"] == "attention":
        rows, plen, slen = _sizes(c)
        kv, rope, T, H = c["kv"], c["rope"], c["tokens"], c["heads"]
        pos = kv + 2 * rope + 4 if c["cache"] == "fp8" else 2 * (kv + rope)
        qrows = len(slen) * T * H
        pairs = sum(r * p for r, p in zip(rows, plen)) * T * H + \
            sum(sum(n - (T - 1 - t) for t in range(T)) for n in slen) * H
        return {"bytes": (sum(plen) + sum(slen)) * pos + qrows * 2 * (2 * kv + rope) + qrows * 4,
                "flops": 2 * (2 * kv + rope) * pairs}
    if c["op"] in ("write", "read"):
        n, e = c["tokens"], BYTES[c["dtype"]]
        return {"bytes": n * ((c["kv"] + c["rope"]) * e + c["kv"] + 2 * c["rope"] + 4 + 8),
                "flops": 4 * n * c["kv"]}
    # one row of the target's probabilities for each sequence, and the draft's where one was rejected
    e = BYTES[c["dtype"]]
    rejected = 1 - 0.8 ** c["drafts"] if c["draft_probs"] else 0.0
    return {"bytes": c["rows"] * (c["vocab"] * e * (1 + rejected) + c["drafts"] * 16 + 16),
            "flops": 3 * c["rows"] * c["vocab"]}


# --------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g, dtype=dtype)


def _quantised(x, kv, dtype):
    """An 8-bit cache holding the rows x [..., kv + rope] (plain arithmetic)."""
    lat = x[..., :kv].float()
    s = (lat.abs().amax(-1) / E4M3_MAX).clamp_min(SCALE_FLOOR)
    return (lat / s[..., None]).to(torch.float8_e4m3fn), x[..., kv:].to(dtype).contiguous(), s


def _cache(g, c, batch, positions, dtype):
    # normalised latent rows (unit RMS) and rotated keys
    x = _randn(g, batch, positions, c["kv"] + c["rope"], dtype=dtype)
    return _quantised(x, c["kv"], dtype) if c["cache"] == "fp8" else x


def prepare(c, seed):
    g = _gen(seed)
    if c["op"] == "attention":
        rows, plen, slen = _sizes(c)
        dt = DTYPES[c["dtype"]]
        B, G = len(slen), c["groups"]
        start = [0]
        for r in rows:
            start.append(start[-1] + r)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        return dict(case=c, q=_randn(g, B, c["tokens"], c["heads"], c["kv"] + c["rope"], dtype=dt),
                    prefix=_cache(g, c, G, c["prefix"], dt), suffix=_cache(g, c, B, max(slen), dt),
                    group_start=i32(start), prefix_len=i32(plen), suffix_len=i32(slen),
                    # what the program that holds the requests knows on the host
                    max_group=max(rows), scale=1.0 / math.sqrt(64 if c["kv"] == 128 else 128))
    if c["op"] in ("write", "read"):
        dt, n = DTYPES[c["dtype"]], c["tokens"]
        half = torch.bfloat16 if c["dtype"] == "bf16" else torch.float16
        x = _randn(g, c["rows"], c["positions"], c["kv"] + c["rope"], dtype=half)
        cache = _quantised(x, c["kv"], half)
        slots = torch.randperm(c["rows"] * c["positions"], device="cuda", generator=g)[:n]
        if n > 4:  # a step's rows that are free write and read nothing
            slots[3] = -1
        s = dict(case=c, cache=cache, slots=slots)
        if c["op"] == "write":
            s.update(latent=_randn(g, n, c["kv"], dtype=dt), rope=_randn(g, n, c["rope"], dtype=dt))
        return s
    B, K, V, dt = c["rows"], c["drafts"], c["vocab"], DTYPES[c["dtype"]]
    p = torch.empty(B, K + 1, V, dtype=dt, device="cuda")
    q = torch.empty(B, K, V, dtype=dt, device="cuda") if c["draft_probs"] else None
    tokens = torch.empty(B, K, dtype=torch.int32, device="cuda")
    step = max(1, int(3e7) // ((K + 1) * V))
    for b in range(0, B, step):  # logits of both models: the draft's are the target's plus noise
        n = min(step, B - b)
        z = _randn(g, n, K + 1, V) * 2.0
        p[b:b + n] = torch.softmax(z, -1).to(dt)
        d = torch.softmax(z[:, :K] + 0.4 * _randn(g, n, K, V), -1)
        e = torch.empty(n, K, V, device="cuda").exponential_(generator=g)
        tokens[b:b + n] = (d / e).argmax(-1).int()
        if q is not None:
            q[b:b + n] = d.to(dt)
        else:  # drafts looked up: right with probability 0.8
            best = p[b:b + n, :K].float().argmax(-1).int()
            keep = torch.rand(n, K, device="cuda", generator=g) < 0.8
            tokens[b:b + n] = torch.where(keep, best, tokens[b:b + n])
    lens = torch.full((B,), K, dtype=torch.int32, device="cuda")
    lens[1::3] = K // 2  # requests with fewer drafts
    return dict(case=c, target_probs=p, draft_probs=q, draft_tokens=tokens, draft_len=lens,
                u_accept=torch.rand(B, K, device="cuda", generator=g),
                u_sample=torch.rand(B, device="cuda", generator=g))


# --------------------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    if own:
        from cpp_inference_train_engine_b200 import latent
        if c["op"] == "attention":
            return latent.shared_prefix_attention(
                s["q"], s["prefix"], s["suffix"], s["group_start"], s["prefix_len"], s["suffix_len"],
                s["scale"], kv_rank=c["kv"], max_group=s["max_group"], return_lse=True)
        if c["op"] == "write":
            latent.cache_write(s["cache"], s["latent"], s["rope"], s["slots"])
            return s["cache"]
        if c["op"] == "read":
            return latent.cache_read(s["cache"], s["slots"], DTYPES[c["dtype"]])
        return latent.verify_drafts(s["target_probs"], s["draft_tokens"], s["draft_len"], s["u_accept"],
                                    s["u_sample"], draft_probs=s["draft_probs"])
    return {"attention": _plain_attention, "write": _plain_write, "read": _plain_read,
            "verify": _plain_verify}[c["op"]](s)


def _values(cache):
    if isinstance(cache, tuple):
        return torch.cat([cache[0].float() * cache[2][..., None], cache[1].float()], -1)
    return cache.float()


def _plain_attention(s):
    c = s["case"]
    kv, T = c["kv"], c["tokens"]
    q = s["q"].float() * s["scale"]
    prefix, suffix = _values(s["prefix"]), _values(s["suffix"])
    B, _, H, W = q.shape
    G, P, S, R = prefix.shape[0], prefix.shape[1], suffix.shape[1], s["max_group"]
    start = s["group_start"].long()
    row = torch.arange(B, device=q.device)
    group = (row[:, None] >= start[None, 1:]).sum(1)
    at = group * R + (row - start[group])  # the row's place among padded groups
    # scores over the prefix, each group's queries in one product, and over each row's own suffix
    qg = q.new_zeros(G * R, T * H, W)
    qg[at] = q.reshape(B, T * H, W)
    sp = torch.bmm(qg.reshape(G, R * T * H, W), prefix.transpose(1, 2)).reshape(G * R, T, H, P)[at]
    ss = torch.bmm(q.reshape(B, T * H, W), suffix.transpose(1, 2)).reshape(B, T, H, S)
    seen = s["suffix_len"].long()[:, None] - (T - 1 - torch.arange(T, device=q.device))[None, :]
    ok_p = (torch.arange(P, device=q.device)[None, :] < s["prefix_len"].long()[group][:, None])[:, None, None, :]
    ok_s = (torch.arange(S, device=q.device)[None, None, :] < seen[:, :, None])[:, :, None, :]
    sp = torch.where(ok_p, sp, float("-inf"))
    ss = torch.where(ok_s, ss, float("-inf"))
    top = torch.maximum(sp.amax(-1), ss.amax(-1))
    base = torch.where(torch.isfinite(top), top, torch.zeros_like(top))[..., None]
    sp, ss = torch.exp(sp - base), torch.exp(ss - base)
    total = sp.sum(-1) + ss.sum(-1)
    inv = torch.where(total > 0, 1.0 / total, torch.zeros_like(total))[..., None]
    pg = q.new_zeros(G * R, T * H, P)
    pg[at] = sp.reshape(B, T * H, P)
    o = torch.bmm(pg.reshape(G, R * T * H, P), prefix[..., :kv]).reshape(G * R, T, H, kv)[at]
    o = o + torch.bmm(ss.reshape(B, T * H, S), suffix[..., :kv]).reshape(B, T, H, kv)
    return (o * inv).to(s["q"].dtype), base[..., 0] + torch.log(total)


def _plain_write(s):
    lat8, rope, scale = s["cache"]
    keep = s["slots"] >= 0
    slots = s["slots"][keep]
    x = s["latent"].float()[keep]
    sc = (x.abs().amax(-1) / E4M3_MAX).clamp_min(SCALE_FLOOR)
    lat8.view(torch.uint8).view(-1, x.shape[1])[slots] = (x / sc[:, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    rope.view(-1, rope.shape[-1])[slots] = s["rope"].float()[keep].to(rope.dtype)
    scale.view(-1)[slots] = sc
    return s["cache"]


def _plain_read(s):
    lat8, rope, scale = s["cache"]
    keep = s["slots"] >= 0
    slots = s["slots"].clamp_min(0)
    x = lat8.view(torch.uint8).view(-1, lat8.shape[-1])[slots].view(torch.float8_e4m3fn).float()
    x = torch.cat([x * scale.view(-1)[slots][:, None], rope.view(-1, rope.shape[-1])[slots].float()], -1)
    return torch.where(keep[:, None], x, torch.zeros_like(x)).to(DTYPES[s["case"]["dtype"]])


def _plain_verify(s):
    p, q, x = s["target_probs"], s["draft_probs"], s["draft_tokens"].long()
    B, K, V = p.shape[0], x.shape[1], p.shape[2]
    lens = s["draft_len"].long()
    px = torch.gather(p[:, :K], 2, x[..., None])[..., 0].float()
    qx = torch.gather(q, 2, x[..., None])[..., 0].float() if q is not None else torch.ones_like(px)
    ok = (s["u_accept"] * qx < px) & (torch.arange(K, device=p.device)[None] < lens[:, None])
    n = ok.long().cumprod(1).sum(1)  # drafts accepted
    row = torch.arange(B, device=p.device)
    pj = p[row, n].float()
    at = n.clamp_max(K - 1)
    qj = q[row, at].float() if q is not None else \
        (torch.arange(V, device=p.device)[None] == x[row, at][:, None]).float()
    rest = torch.where((n < lens)[:, None], (pj - qj).clamp_min(0), pj)
    weigh = lambda v: (v.clamp(0, 1) * 2.0 ** 38).long()  # noqa: E731
    w = weigh(rest)
    w = torch.where((w.sum(1) > 0)[:, None], w, weigh(pj))
    cum = w.cumsum(1)
    total = cum[:, -1]
    k = (s["u_sample"] * 2.0 ** 24).long().clamp(0, 2 ** 24 - 1)
    t = (total >> 24) * k + (((total & (2 ** 24 - 1)) * k) >> 24)
    y = (cum <= t[:, None]).sum(1)
    y = torch.where(total > 0, y, torch.full_like(y, -1))
    col = torch.arange(K + 1, device=p.device)[None]
    padded = torch.cat([x, x[:, :1]], 1)
    tokens = torch.where(col < n[:, None], padded, torch.where(col == n[:, None], y[:, None], torch.full_like(padded, -1)))
    return tokens.int(), n.int()


# --------------------------------------------------------------------------- 64 bits
def exact(c, seed):
    if c["op"] == "verify":
        return None  # whole numbers
    s = prepare(c, seed)
    return {"attention": _exact_attention, "write": _exact_write, "read": _exact_read}[c["op"]](c, s)


def _values64(cache, index, n, kv):
    """Rows [0, n) of batch entry `index` of a cache as 64-bit values."""
    if isinstance(cache, tuple):
        lat = cache[0][index, :n].to(torch.float32).double() * cache[2][index, :n].double()[:, None]
        return torch.cat([lat, cache[1][index, :n].double()], 1)
    return cache[index, :n].double()


def _exact_attention(c, s):
    rows, plen, slen = _sizes(c)
    T, H, kv = c["tokens"], c["heads"], c["kv"]
    if work(c)["flops"] > 4e11:
        return None
    out = torch.zeros(len(slen), T, H, kv, dtype=torch.float64, device="cuda")
    lse = torch.zeros(len(slen), T, H, dtype=torch.float64, device="cuda")
    b = 0
    for g, r in enumerate(rows):
        pre = _values64(s["prefix"], g, plen[g], kv)
        for b in range(b, b + r):
            keys = torch.cat([pre, _values64(s["suffix"], b, slen[b], kv)])
            z = s["q"][b].double().reshape(T * H, -1) @ keys.T * s["scale"]
            z = z.reshape(T, H, -1)
            for t in range(T - 1):  # the later query tokens' own positions
                z[t, :, plen[g] + max(0, slen[b] - (T - 1 - t)):] = float("-inf")
            lse[b] = torch.logsumexp(z, -1)
            out[b] = (torch.softmax(z, -1).reshape(T * H, -1) @ keys[:, :kv]).reshape(T, H, kv)
        b += 1
    return out, lse


def _e4m3_64(v):
    """The nearest e4m3 value of |v| <= 448 (ties to even), in 64 bits."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), torch.clamp(e - 1, min=-6) - 3)
    return torch.clamp(torch.round(v / step) * step, -E4M3_MAX, E4M3_MAX)


def _exact_write(c, s):
    lat, rope, scale = (t.to(torch.float32).double() for t in s["cache"])
    keep = (s["slots"] >= 0).nonzero()[:, 0]
    slots = s["slots"][keep]
    x = s["latent"][keep].double()
    sc = torch.clamp(x.abs().max(1).values / E4M3_MAX, min=SCALE_FLOOR)
    lat.view(-1, c["kv"]).index_copy_(0, slots, _e4m3_64(x / sc[:, None]))
    rope.view(-1, c["rope"]).index_copy_(0, slots, s["rope"][keep].double())
    scale.view(-1).index_copy_(0, slots, sc)
    return lat, rope, scale


def _exact_read(c, s):
    lat, rope, scale = (t.to(torch.float32).double() for t in s["cache"])
    rows = torch.cat([lat.view(-1, c["kv"]) * scale.view(-1, 1), rope.view(-1, c["rope"])], 1)
    out = torch.zeros(c["tokens"], c["kv"] + c["rope"], dtype=torch.float64, device="cuda")
    keep = s["slots"] >= 0
    out[keep] = rows[s["slots"][keep]]
    return out
