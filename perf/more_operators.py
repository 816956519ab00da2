"""Paged latent-cache decode and beam search at the sizes they are used at: inputs, plain form, work.

Four operators of a decode step over a paged (MLA) cache: ``append`` (new positions normalised,
rotated and stored through the page table), ``attention`` (one new token a row over its pages,
whole or through a sliding window with a few first positions), ``beam_select`` (the best
continuations over beams and vocabulary) and ``beam_reorder`` (page tables follow the chosen
parents). A case is plain sizes; ``prepare`` makes its inputs on the GPU from a seed; ``run`` is
one call of the operator (``own``) or its plain form in elementary torch operations; ``exact`` is
the definition in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
E4M3_MAX = 448.0
SCALE_FLOOR = 2.0 ** -100
THETA, EPS = 10000.0, 1e-5


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of a small server: every row's new position, latency
        _append("append_step", tokens=61, rows=61, kv=128, rope=16, dtype="bf16", page=64, length=2048),
        # a prefill chunk of the scaled model's prompts into 8-bit pages
        _append("append_prefill", tokens=131072, rows=320, kv=512, rope=32, dtype="fp16", page=32, length=512, cache="fp8"),
        # four requests early in their answers: latency
        _att("few_rows", rows=4, heads=8, kv=128, rope=16, length=197, page=64),
        # a full server of the 35.8M model, requests of all ages
        _att("server_512_rows", rows=512, heads=8, kv=128, rope=16, length=2048, page=64, ragged=True),
        # the scaled model's server over long contexts, bf16
        _att("wide_server", rows=96, heads=16, kv=512, rope=32, length=8192, page=64, dtype="bf16", ragged=True),
        # one request over a very long document
        _att("one_long_row", rows=1, heads=16, kv=512, rope=32, length=131072, page=128),
        # 8-bit pages
        _att("wide_server_fp8", rows=120, heads=16, kv=512, rope=32, length=6001, page=32, cache="fp8", ragged=True),
        # endless sessions: a window and four first positions, the pages between them given back
        _att("sliding_window", rows=190, heads=16, kv=512, rope=32, length=16384, page=16, dtype="bf16", ragged=True,
             window=1024, sinks=4),
        # one request's beams
        _select("select_4_beams", batch=1, beams=4, vocab=16384),
        # a batch of requests with eight beams each
        _select("select_64x8", batch=64, beams=8, vocab=32768),
        # one request's beams follow their parents through ten layers
        _reorder("reorder_4_beams", batch=1, beams=4, layers=10, kv=128, rope=16, page=64, length=173, dtype="bf16"),
        # 256 beams through 24 layers
        _reorder("reorder_256_rows", batch=32, beams=8, layers=24, kv=512, rope=32, page=32, length=87),
    ]


def _named(c, name):
    return dict(c, name=name) if name else c


def _append(name=None, tokens=1, rows=1, kv=128, rope=16, dtype="fp16", page=64, length=128, cache="same", norm=True):
    return _named(dict(op="append", tokens=tokens, rows=rows, kv=kv, rope=rope, dtype=dtype, page=page, length=length,
                       cache=cache, norm=norm), name)


def _att(name=None, rows=1, heads=8, kv=128, rope=16, length=128, page=64, dtype="fp16", cache="same", ragged=False,
         window=0, sinks=0):
    return _named(dict(op="attention", rows=rows, heads=heads, kv=kv, rope=rope, length=length, page=page, dtype=dtype,
                       cache=cache, ragged=ragged, window=window, sinks=sinks), name)


def _select(name=None, batch=1, beams=4, vocab=16384, dtype="fp32"):
    return _named(dict(op="select", batch=batch, beams=beams, vocab=vocab, dtype=dtype), name)


def _reorder(name=None, batch=1, beams=4, layers=2, kv=128, rope=16, page=64, length=100, dtype="fp16", cache="same"):
    return _named(dict(op="reorder", batch=batch, beams=beams, layers=layers, kv=kv, rope=rope, page=page, length=length,
                       dtype=dtype, cache=cache), name)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        m = most.setdefault(c["op"], {"bytes": 0, "flops": 0})
        for k in m:
            m[k] = max(m[k], w[k])
    while True:
        op = rng.choice(["attention", "attention", "attention", "append", "select", "reorder"])
        wide = rng.random() < 0.5
        kv, rope = (512, 32) if wide else (128, 16)
        page, dtype = rng.choice([16, 32, 64, 128]), rng.choice(["fp16", "bf16"])
        cache = rng.choice(["same", "same", "fp8"])
        if op == "attention":
            windowed = rng.random() < 0.4
            c = _att(rows=_log(rng, 1, 700), heads=rng.choice([16, 16, 12, 5, 24] if wide else [8, 8, 16, 3]), kv=kv,
                     rope=rope, length=_log(rng, 1, 100000), page=page, dtype=dtype, cache=cache,
                     ragged=rng.random() < 0.7, window=_log(rng, 1, 4096) if windowed else 0,
                     sinks=rng.choice([0, 1, 4, 37]) if windowed else 0)
            fits = c["rows"] * c["length"] * (kv + rope) < 2.4e9
        elif op == "append":
            c = _append(tokens=_log(rng, 1, 131072), rows=_log(rng, 1, 300), kv=kv, rope=rope,
                        dtype=rng.choice(["fp16", "bf16", "fp32"]), page=page, length=_log(rng, 16, 100000), cache=cache,
                        norm=rng.random() < 0.7)
            fits = c["tokens"] <= c["rows"] * c["length"]
        elif op == "select":
            c = _select(batch=_log(rng, 1, 200), beams=rng.randint(2, 16), vocab=_log(rng, 257, 50001),
                        dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]))
            fits = True
        else:
            c = _reorder(batch=_log(rng, 1, 64), beams=rng.randint(2, 16), layers=rng.choice([2, 10, 24]), kv=kv,
                         rope=rope, page=page, length=_log(rng, 1, 700), dtype=dtype, cache=cache)
            pages = c["batch"] * c["beams"] * (c["length"] // page + 3)
            fits = c["layers"] * pages * page * (kv + rope) < 5e8
        w = work(c)
        if fits and all(w[k] <= most[op][k] for k in w):
            return c


# --------------------------------------------------------------------------- sizes of a case
def _lengths(c):
    """Length of each row: a fixed pattern of the case (ragged: spread over the range, odd ones among them)."""
    n = c["length"]
    if not c["ragged"]:
        return [n] * c["rows"]
    return [1 + (b * 40503 + 77 + n // 2) % n for b in range(c["rows"])]


def _places(c):
    """Row and first position of each run of appended tokens, and its length: every row gets the same
    number (one fewer in the last rows), somewhere in its range."""
    n, r = c["tokens"], c["rows"]
    runs = []
    for b in range(r):
        k = n // r + (1 if b < n % r else 0)
        k = min(k, c["length"])
        if k:
            runs.append((b, (b * 7919 + c["length"] // 2) % (c["length"] - k + 1), k))
    return runs


def _parents(c):
    """Parent of each row within its batch entry: a fixed pattern in which the leading beams have several children."""
    k = c["beams"]
    return [b * k + (((b * 31 + i * 17 + 5) * 2654435761 >> 7) % k) * (i % 3 != 0) for b in range(c["batch"]) for i in range(k)]


def _position_bytes(c):
    return c["kv"] + 2 * c["rope"] + 4 if c["cache"] == "fp8" else 2 * (c["kv"] + c["rope"])


def work(c):
    if c["op"] == "attention":
        w, s = c["window"], c["sinks"]
        seen = sum(n if not w else min(n, w + min(s, max(n - w, 0))) for n in _lengths(c))
        return {"bytes": seen * _position_bytes(c) + c["rows"] * c["heads"] * (2 * (2 * c["kv"] + c["rope"]) + 4),
                "flops": 2 * (2 * c["kv"] + c["rope"]) * c["heads"] * seen}
    if c["op"] == "append":
        n = sum(k for _, _, k in _places(c))
        return {"bytes": n * ((c["kv"] + c["rope"]) * BYTES[c["dtype"]] + _position_bytes(c) + 8),
                "flops": 8 * n * (c["kv"] + c["rope"])}
    if c["op"] == "select":
        n = c["batch"] * c["beams"]
        return {"bytes": n * (c["vocab"] * BYTES[c["dtype"]] + 4 + 12), "flops": 8 * n * c["vocab"]}
    moved = sum(i != p for i, p in enumerate(_parents(c))) * (c["length"] % c["page"]) * c["layers"]
    rows = c["batch"] * c["beams"]
    return {"bytes": 2 * moved * _position_bytes(c) + rows * (8 * _columns(c) + 24), "flops": 0}


# --------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g, dtype=dtype)


def _half(c):
    return torch.bfloat16 if c["dtype"] == "bf16" else torch.float16


def _quantised(x, kv):
    """An 8-bit cache holding the rows x [..., kv + rope] (plain arithmetic)."""
    lat = x[..., :kv].float()
    s = (lat.abs().amax(-1) / E4M3_MAX).clamp_min(SCALE_FLOOR)
    return (lat / s[..., None]).to(torch.float8_e4m3fn), x[..., kv:].contiguous(), s


def _pages(g, c, *shape):
    # normalised latent rows (unit RMS) and rotated keys
    x = _randn(g, *shape, c["page"], c["kv"] + c["rope"], dtype=_half(c))
    return _quantised(x, c["kv"]) if c["cache"] == "fp8" else x


def _table(g, c, used, rows, columns):
    """A page table whose used [(row, column)] entries are pages of a shuffled pool, -1 elsewhere; the pool's size."""
    n = len(used) + 3
    table = torch.full((rows, columns), -1, dtype=torch.int32, device="cuda")
    at = torch.tensor([r * columns + j for r, j in used], dtype=torch.int64, device="cuda")
    table.view(-1)[at] = torch.randperm(n, device="cuda", generator=g)[:len(used)].int()
    return table, n


def _columns(c):
    """Pages of a reordered row: its positions' and one to grow into."""
    return c["length"] // c["page"] + 2


def prepare(c, seed):
    g = _gen(seed)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if c["op"] == "attention":
        lengths, P = _lengths(c), c["page"]
        used = []
        for b, n in enumerate(lengths):
            if not c["window"]:
                used += [(b, j) for j in range((n + P - 1) // P)]
            else:  # pages that neither the window nor the first positions need were given back
                first, sinks = max(n - c["window"], 0), min(c["sinks"], n)
                used += [(b, j) for j in range((n + P - 1) // P) if (j + 1) * P > first or j * P < sinks]
        table, pool = _table(g, c, used, c["rows"], (max(lengths) + P - 1) // P)
        return dict(case=c, q=_randn(g, c["rows"], c["heads"], c["kv"] + c["rope"], dtype=_half(c)),
                    cache=_pages(g, c, pool), table=table, lengths=i32(lengths),
                    scale=1.0 / math.sqrt(64 if c["kv"] == 128 else 128))
    if c["op"] == "append":
        runs, P = _places(c), c["page"]
        used = [(b, j) for b, p, k in runs for j in range(p // P, (p + k - 1) // P + 1)]
        table, pool = _table(g, c, used, c["rows"], (c["length"] + P - 1) // P)
        rows = torch.cat([torch.full((k,), b, dtype=torch.int32) for b, _, k in runs]).cuda()
        positions = torch.cat([torch.arange(p, p + k, dtype=torch.int32) for _, p, k in runs]).cuda()
        if positions.numel() > 4:  # a step's free rows store nothing
            positions[3] = -1
        # the projection's result: latents of any size, keys before their rotation
        values = 1.7 * _randn(g, positions.numel(), c["kv"] + c["rope"], dtype=DTYPES[c["dtype"]])
        norm = 1 + 0.1 * _randn(g, c["kv"]) if c["norm"] else None
        return dict(case=c, cache=_pages(g, c, pool), values=values, table=table, rows=rows, positions=positions, norm=norm)
    if c["op"] == "select":
        B, K, V = c["batch"], c["beams"], c["vocab"]
        logits = torch.empty(B, K, V, dtype=DTYPES[c["dtype"]], device="cuda")
        for b in range(B):
            logits[b] = 2.0 * _randn(g, K, V)
        scores = (-20.0 - 0.7 * _randn(g, B, K).abs().cumsum(1)).contiguous()
        finished = torch.zeros(B, K, dtype=torch.bool, device="cuda")
        finished[1::3, K // 2] = True  # some answers have ended
        return dict(case=c, logits=logits, scores=scores, finished=finished, eos=V - 6)
    rows, cols = c["batch"] * c["beams"], _columns(c)
    pages = torch.randperm(rows * (cols + 1), device="cuda", generator=g).int()
    return dict(case=c, cache=_pages(g, c, c["layers"], rows * (cols + 1)), table=pages[:rows * cols].view(rows, cols),
                spare=pages[rows * cols:].clone(), lengths=torch.full((rows,), c["length"], dtype=torch.int32, device="cuda"),
                parents=i32(_parents(c)))


# --------------------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    if own:
        from cpp_inference_train_engine_b200 import paged
        if c["op"] == "attention":
            return paged.attention(s["q"], s["cache"], s["table"], s["lengths"], s["scale"], kv_rank=c["kv"],
                                   window=c["window"] or None, sinks=c["sinks"], return_lse=True)
        if c["op"] == "append":
            paged.append(s["cache"], s["values"], s["table"], s["positions"], kv_rank=c["kv"], rows=s["rows"], theta=THETA,
                         norm=s["norm"], eps=EPS)
            return s["cache"]
        if c["op"] == "select":
            return paged.beam_select(s["logits"], s["scores"], finished=s["finished"], eos=s["eos"])
        return s["cache"], paged.beam_reorder(s["cache"], s["table"], s["spare"], s["lengths"], s["parents"])
    return {"attention": _plain_attention, "append": _plain_append, "select": _plain_select,
            "reorder": _plain_reorder}[c["op"]](s)


def _plain_attention(s):
    c, table = s["case"], s["table"].long().clamp_min(0)
    rows, n = table.shape[0], table.shape[1] * c["page"]
    if isinstance(s["cache"], tuple):
        codes, rope, scale = s["cache"]
        lat = codes.view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * scale[table][..., None]
        keys = torch.cat([lat, rope[table].float()], -1).view(rows, n, -1)
    else:
        keys = s["cache"][table].float().view(rows, n, -1)
    z = torch.bmm(s["q"].float() * s["scale"], keys.transpose(1, 2))
    j, length = torch.arange(n, device=z.device)[None], s["lengths"][:, None]
    seen = j < length
    if c["window"]:
        seen &= (j < c["sinks"]) | (j >= length - c["window"])
    z = torch.where(seen[:, None], z, float("-inf"))
    top = z.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    p = torch.exp(z - top)
    total = p.sum(-1, keepdim=True)
    values = torch.where(seen[..., None], keys[..., :c["kv"]], 0)
    o = torch.bmm(p, values) / torch.where(total > 0, total, torch.ones_like(total))
    return o.to(s["q"].dtype), (top + torch.log(total))[..., 0]


def _turned(key, positions):
    """Adjacent pairs rotated by position * theta^(-2 j / width); the angles in 64 bits."""
    w = key.shape[-1]
    j = torch.arange(0, w, 2, device=key.device, dtype=torch.float64)
    angle = positions.double()[:, None] * THETA ** (-j / w)
    cos, sin = angle.cos().to(key.dtype), angle.sin().to(key.dtype)
    a, b = key[:, 0::2], key[:, 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(1)


def _entries(s):
    """Kept tokens and where they go in the pool."""
    P = s["case"]["page"]
    keep = (s["positions"] >= 0).nonzero()[:, 0]
    position, row = s["positions"][keep].long(), s["rows"][keep].long()
    return keep, position, s["table"][row, position // P].long() * P + position % P


def _plain_append(s):
    c = s["case"]
    keep, position, at = _entries(s)
    x = s["values"][keep].float()
    lat, key = x[:, :c["kv"]], _turned(x[:, c["kv"]:], position)
    if s["norm"] is not None:
        lat = lat / torch.sqrt((lat * lat).mean(-1, keepdim=True) + EPS) * s["norm"]
    if not isinstance(s["cache"], tuple):
        s["cache"].view(-1, x.shape[1])[at] = torch.cat([lat, key], 1).to(s["cache"].dtype)
        return s["cache"]
    codes, rope, scale = s["cache"]
    sc = (lat.abs().amax(-1) / E4M3_MAX).clamp_min(SCALE_FLOOR)
    codes.view(torch.uint8).view(-1, c["kv"])[at] = (lat / sc[:, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    rope.view(-1, c["rope"])[at] = key.to(rope.dtype)
    scale.view(-1)[at] = sc
    return s["cache"]


def _plain_select(s):
    # candidates in 64 bits: which of two near ones is taken depends on them
    x, eos = s["logits"], s["eos"]
    B, K, V = x.shape
    top = x.float().amax(-1, keepdim=True).double()
    lse = top + torch.log(torch.exp((x.float() - top.float())).sum(-1, keepdim=True, dtype=torch.float64))
    cand = s["scores"].double()[..., None] + (x.double() - lse)
    ended = s["finished"][..., None]
    only = torch.arange(V, device=x.device) == eos
    cand = torch.where(ended, torch.where(only, s["scores"].double()[..., None], float("-inf")), cand).view(B, K * V)
    best, at = torch.sort(cand, dim=1, descending=True, stable=True)
    best, at = best[:, :K], at[:, :K]
    return best.float(), (at // V).int(), (at % V).int()


def _plain_reorder(s):
    P = s["case"]["page"]
    table, lengths, parent = s["table"].long(), s["lengths"].long(), s["parents"].long()
    rows, cols = table.shape
    row = torch.arange(rows, device=table.device)
    n = lengths[parent]
    full, part = n // P, n % P
    moves = (parent != row) & (part > 0)
    col = torch.arange(cols, device=table.device)[None]
    new = torch.where(col < full[:, None], table[parent], table)
    at = full.clamp_max(cols - 1)
    source = table[parent, at]
    new[row, at] = torch.where(moves, s["spare"].long(), new[row, at])
    own_tail = table[row, (lengths // P).clamp_max(cols - 1)]
    spare = torch.where(moves, own_tail, s["spare"].long())
    who = moves.nonzero()[:, 0]
    tensors = s["cache"] if isinstance(s["cache"], tuple) else (s["cache"],)
    place = torch.arange(P, device=table.device)[None] < part[who][:, None]
    for t in tensors:
        t = t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
        for layer in t:
            target = s["spare"].long()[who]
            keep = place[..., None] if layer.dim() == 3 else place
            layer[target] = torch.where(keep, layer[source[who]], layer[target])
    return s["cache"], (new.int(), spare.int(), n.int())


# --------------------------------------------------------------------------- 64 bits
def exact(c, seed):
    if c["op"] == "reorder":
        return None  # copies and whole numbers
    s = prepare(c, seed)
    return {"attention": _exact_attention, "append": _exact_append, "select": _exact_select}[c["op"]](c, s)


def _exact_attention(c, s):
    P, kv = c["page"], c["kv"]
    out = torch.zeros(c["rows"], c["heads"], kv, dtype=torch.float64, device="cuda")
    lse = torch.full((c["rows"], c["heads"]), float("-inf"), dtype=torch.float64, device="cuda")
    table = s["table"].cpu()
    for b, n in enumerate(_lengths(c)):
        first = max(n - c["window"], 0) if c["window"] else 0
        position = sorted(set(range(min(c["sinks"], n))) | set(range(first, n))) if c["window"] else list(range(n))
        position = torch.tensor(position)
        page, at = table[b, position // P].long().cuda(), (position % P).cuda()
        if isinstance(s["cache"], tuple):
            codes, rope, scale = s["cache"]
            lat = codes.view(torch.uint8)[page, at].view(torch.float8_e4m3fn).float().double() * scale[page, at].double()[:, None]
            keys = torch.cat([lat, rope[page, at].double()], 1)
        else:
            keys = s["cache"][page, at].double()
        z = s["q"][b].double() @ keys.T * s["scale"]
        lse[b] = torch.logsumexp(z, -1)
        out[b] = torch.softmax(z, -1) @ keys[:, :kv]
    return out, lse


def _exact_append(c, s):
    """The stored values; 8-bit codes as the quotients that they stand for."""
    keep, position, at = _entries(s)
    x = s["values"][keep].double()
    lat, key = x[:, :c["kv"]], x[:, c["kv"]:]
    phase = torch.outer(position.double(), torch.pow(torch.tensor(THETA, dtype=torch.float64, device="cuda"),
                                                     -torch.arange(0, c["rope"], 2, device="cuda").double() / c["rope"]))
    turned = torch.view_as_real(torch.view_as_complex(key.reshape(len(keep), -1, 2).contiguous()) *
                                torch.polar(torch.ones_like(phase), phase)).flatten(1)
    if s["norm"] is not None:
        lat = lat * torch.rsqrt(lat.square().sum(-1, keepdim=True) / c["kv"] + EPS) * s["norm"].double()
    if not isinstance(s["cache"], tuple):
        out = s["cache"].double()
        out.view(-1, x.shape[1]).index_copy_(0, at, torch.cat([lat, turned], 1))
        return out
    codes, rope, scale = (t.to(torch.float32).double() for t in s["cache"])
    sc = torch.clamp(lat.abs().max(1).values / E4M3_MAX, min=SCALE_FLOOR)
    codes.view(-1, c["kv"]).index_copy_(0, at, lat / sc[:, None])
    rope.view(-1, c["rope"]).index_copy_(0, at, turned)
    scale.view(-1).index_copy_(0, at, sc)
    return codes, rope, scale


def _exact_select(c, s):
    B, K, V = c["batch"], c["beams"], c["vocab"]
    if B * K * V > 1.2e8:
        return None
    out = torch.empty(B, K, dtype=torch.float64, device="cuda")
    for b in range(B):
        cand = s["scores"][b].double()[:, None] + torch.log_softmax(s["logits"][b].double(), -1)
        for k in s["finished"][b].nonzero()[:, 0].tolist():
            cand[k] = float("-inf")
            cand[k, s["eos"]] = s["scores"][b, k].double()
        out[b] = cand.view(-1).topk(K).values
    return out, None, None
