"""Attention over shared prompts (latent.py) where its numbers are easy to lose: cache values far from one,
keys that weigh little, masked and lowest scores, positions that hold a NaN or an infinity, and many query
tokens a row. Against the definition in 64 bits."""
import pytest

from tests.test_gpu_latent import NAN, make_cache, mods, reference

pytestmark = pytest.mark.gpu

# (latent width, rope width, heads, tokens): blocks of 16 and of 64 queries at both tensor-core widths, and a
# width without that form
FORMS = [(128, 16, 8, 1), (512, 32, 5, 3), (128, 16, 8, 9), (512, 32, 16, 5), (40, 6, 3, 2)]
TENSOR_CORE = FORMS[:4]


def stored(torch, x, kv, dtype, fp8):
    """Rows x as a cache: (what the call takes, its values in 64 bits, one unit per position): 16-bit values
    have the unit 1, codes their scale."""
    if not fp8:
        c = x.to(dtype)
        return c, c.double(), torch.ones(x.shape[:2], dtype=torch.float64, device="cuda")
    s = (x[..., :kv].float().abs().amax(-1) / 448).clamp_min(2.0 ** -100)
    codes = (x[..., :kv].float() / s[..., None]).to(torch.float8_e4m3fn)
    rk = x[..., kv:].to(dtype)
    return (codes, rk, s), torch.cat([codes.float().double() * s.double()[..., None], rk.double()], -1), s.double()


def run(torch, latent, q, pre, suf, starts, plen, slen, kv, scale):
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return latent.shared_prefix_attention(
        q, pre, suf, i32(starts) if pre is not None else None, i32(plen) if pre is not None else None,
        i32(slen) if suf is not None else None, scale, kv_rank=kv, return_lse=True)


def bound(torch, q, pre, suf, starts, plen, slen, kv, scale, fp8):
    """(out, lse, tolerance of out, tolerance of lse) of the definition. The tolerance of a result counts
    - two roundings of weights and results to 16 bits, relative 2^-11 (fp16) or 2^-8 (bf16) each,
    - the scores' fp32 sums of W products in steps of 16, 2^-23 of their magnitude each, as a change of the
      weights (twice: above and below the line),
    - fp16 weights below its normal range: they are held relative to the largest weight of a part, which is
      stored as 2^6 or more, so each is off by at most 2^-25 / 2^6 of that one,
    - an fp16 result below the normal range: 2^-25."""
    values = lambda c: None if c is None else c[1]  # noqa: E731
    want, lse, size, mag = reference(torch, q, values(pre), values(suf), starts, plen, slen, scale, kv)
    half = q.dtype == torch.float16
    u = 2.0 ** -11 if half else 2.0 ** -8
    es = (q.shape[-1] / 16 + 2) * 2.0 ** -23 * mag
    tol = size * (2 * u + 2 * es[..., None]) + 1e-30
    if half:
        # weights are probabilities times the positions' units
        top = torch.zeros_like(lse)
        for cache, lens, row in ((pre, plen, False), (suf, slen, True)):
            if cache is None:
                continue
            _, v, unit = cache
            for b in range(q.shape[0]):
                g = b if row else max([i for i in range(len(starts) - 1) if starts[i] <= b < starts[i + 1]], default=-1)
                if g < 0 or lens[g] <= 0:
                    continue
                k = v[g, :lens[g]]
                p = torch.exp(torch.einsum("thw,kw->thk", q[b].double(), k) * scale - lse[b][..., None]).clamp_max(1)
                top[b] = torch.maximum(top[b], torch.nan_to_num((p * unit[g, :lens[g]]).amax(-1)))
        keys = max(plen, default=0) + max(slen, default=0)
        code = 448.0 if fp8 else max(c[1][..., :kv].abs().amax().item() for c in (pre, suf) if c is not None)
        tol = tol + keys * code * top[..., None] * 2.0 ** -31 + 2.0 ** -25
    keys = max(plen, default=0) + max(slen, default=0)
    return want, lse, tol, es + keys * 2.0 ** -24 + 2.0 ** -20 * (1 + lse.abs())


def agree(torch, got, want, where=None):
    out, lse = got
    wo, wl, to, tl = want
    where = torch.ones_like(wl, dtype=torch.bool) if where is None else where
    err = (out.double() - wo).abs() / to
    # a result past the type's largest value is its infinity
    most = torch.finfo(out.dtype).max
    past = torch.isinf(out) & (out.double().sign() == wo.sign()) & (wo.abs() + to >= most)
    err = torch.where(past, 0.0, err)[where]
    assert torch.all(err <= 1), float(torch.nan_to_num(err, nan=1e9).max())
    el = (lse.double() - wl)[where].abs()
    assert torch.all(el <= tl[where]), float((el / tl[where]).max())

def test_no_wait_ran_out():
    """The device's note of waits that ran out stays empty over calls of every form, and can be read on
    any stream."""
    torch, latent = mods()
    for kv, rope, H, T in FORMS:
        for fp8 in (False, True):
            g = torch.Generator(device="cuda").manual_seed(36)
            pre = make_cache(torch, g, [300], 300, kv, rope, torch.float16, fp8)
            suf = make_cache(torch, g, [200, 20], 200, kv, rope, torch.float16, fp8)
            q = torch.randn(2, T, H, kv + rope, generator=g, device="cuda").half()
            run(torch, latent, q, pre[0], suf[0], [0, 2], [300], [200, 20], kv, 0.1)
            latent.check_status()
    with torch.cuda.stream(torch.cuda.Stream()):
        latent.check_status("cuda")


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("dtype,rms", [("float16", 1.0), ("float16", 1e-2), ("float16", 1e-3), ("float16", 1e-5),
                                       ("float16", 3e4), ("float16", "mixed"), ("bfloat16", 1e-20), ("bfloat16", 1e-3),
                                       ("bfloat16", 1e10), ("bfloat16", "mixed")])
def test_8_bit_values_of_any_size(form, dtype, rms):
    """An e4m3 cache's values are codes times any scale: small ones, large ones, and both side by side."""
    torch, latent = mods()
    kv, rope, H, T = form
    dtype = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(31)
    starts, plen, slen = [0, 2, 3], [700, 130], [40, 300, 9]
    if rms == "mixed":
        size = lambda *s: 10.0 ** (-5 * torch.rand(*s, 1, generator=g, device="cuda"))  # noqa: E731
    else:
        size = lambda *s: torch.full((*s, 1), rms, device="cuda")  # noqa: E731

    def cache(lens):
        s = (len(lens), max(lens))
        x = torch.randn(*s, kv + rope, generator=g, device="cuda")
        x[..., :kv] = (x[..., :kv] + 0.25) * size(*s)  # a mean that the average does not lose
        return stored(torch, x, kv, dtype, True)

    pre, suf = cache(plen), cache(slen)
    q = torch.randn(3, T, H, kv + rope, generator=g, device="cuda")
    q[..., :kv] *= min(1.0 if rms == "mixed" else 1 / rms, 10.0)
    q = q.to(dtype)
    args = (starts, plen, slen, kv, 0.08)
    agree(torch, run(torch, latent, q, pre[0], suf[0], *args), bound(torch, q, pre, suf, *args, True))


@pytest.mark.parametrize("form", TENSOR_CORE, ids=str)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("nats", [8, 15])
def test_many_weak_keys_beside_a_dominant_one(form, fp8, nats):
    """One position without a value takes nearly all of the weight: the result is what thousands of others,
    each of little weight, add up to."""
    torch, latent = mods()
    kv, rope, H, T = form
    g = torch.Generator(device="cuda").manual_seed(32)
    n, scale = 9000, 0.125
    x = 0.01 * (1 + 0.3 * torch.randn(1, n, kv + rope, generator=g, device="cuda"))
    x[..., kv:] = 0
    x[0, 5, :kv] = 0
    x[0, 5, kv] = nats / scale
    pre = stored(torch, x, kv, torch.float16, fp8)
    suf = stored(torch, x[:, :20].expand(2, 20, kv + rope).contiguous(), kv, torch.float16, fp8)
    q = torch.zeros(2, T, H, kv + rope, device="cuda").half()
    q[..., kv] = 1
    args = ([0, 2], [n], [0, 20], kv, scale)
    agree(torch, run(torch, latent, q, pre[0], suf[0], *args), bound(torch, q, pre, suf, *args, fp8))


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("low", ["lowest", "-inf"])
def test_positions_masked_by_their_rope_key(form, dtype, fp8, low):
    """Keys whose scores are the type's lowest value or minus infinity weigh nothing beside others, wherever
    they lie; where all are lowest they weigh the same, where all are -infinity the sum is zero."""
    torch, latent = mods()
    kv, rope, H, T = form
    dtype = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(33)
    bottom = float("-inf") if low == "-inf" else torch.finfo(dtype).min
    x = torch.randn(1, 700, kv + rope, generator=g, device="cuda")
    y = torch.randn(4, 300, kv + rope, generator=g, device="cuda")
    x[..., kv], y[..., kv] = 0, 0
    masked = torch.zeros(700, dtype=torch.bool, device="cuda")
    masked[:300] = True      # the first tiles
    masked[400:450] = True
    q = torch.randn(4, T, H, kv + rope, generator=g, device="cuda").to(dtype)
    q[..., kv] = 1.0
    plen, slen, starts = [700], [300, 40, 0, 300], [0, 3]
    kept = stored(torch, x[:, ~masked], kv, dtype, fp8)
    x[0, masked, kv] = bottom
    y[0, :290, kv] = bottom  # a row of one suffix range, masked but for its end
    y[3, :, kv] = bottom     # a row without a prefix, masked altogether
    pre, suf = stored(torch, x, kv, dtype, fp8), stored(torch, y, kv, dtype, fp8)
    got = run(torch, latent, q, pre[0], suf[0], starts, plen, slen, kv, 0.1)
    # row 0 keeps its last positions, of which its tokens see all but the last T - 1 - t
    want = bound(torch, q, kept, tuple(t for t in stored(torch, y[:, 290:], kv, dtype, fp8)), starts,
                 [int((~masked).sum())], [10, 0, 0, 0], kv, 0.1, fp8)
    rows = torch.zeros(4, T, H, dtype=torch.bool, device="cuda")
    rows[0] = True
    agree(torch, got, want, rows)
    want = bound(torch, q, kept, stored(torch, y[:, :40], kv, dtype, fp8), starts, [int((~masked).sum())], [0, 40, 0, 0], kv, 0.1, fp8)
    rows[0], rows[1:3] = False, True
    agree(torch, got, want, rows)
    if low == "-inf":
        assert torch.all(got[0][3] == 0) and torch.all(got[1][3] == float("-inf"))
    else:
        # the differences of such scores are below what fp32 (and the product's sums) resolve, or above what a
        # weight can hold: a mean of the values, whatever the weights
        assert torch.isfinite(got[0][3]).all() and torch.isfinite(got[1][3]).all()
        top = suf[1][3, :, :kv].abs().amax()
        assert torch.all(got[0][3].double().abs() <= top * (1 + 2.0 ** -6)) and torch.any(got[0][3] != 0)


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("low", ["lowest", "-inf"])
@pytest.mark.parametrize("level", [-400.0, 900.0])
def test_scores_far_from_zero_beside_masked_ones(form, dtype, low, level):
    """All scores that count lie far below or above zero, after key tiles that are masked altogether, in rows
    that are not divided (there are more of them than multiprocessors)."""
    torch, latent = mods()
    kv, rope, H, T = form
    dtype = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(37)
    B, n = 400, 600
    x = 0.5 * torch.randn(B, n, kv + rope, generator=g, device="cuda")
    x[..., kv], x[..., kv + 1] = 0, level
    x[:, :290, kv] = float("-inf") if low == "-inf" else torch.finfo(dtype).min
    suf = stored(torch, x, kv, dtype, False)
    q = torch.randn(B, T, H, kv + rope, generator=g, device="cuda").to(dtype)
    q[..., kv], q[..., kv + 1] = 1.0, 1.0
    slen = [n - b % 3 for b in range(B)]
    out, lse = run(torch, latent, q, None, suf[0], [0], [], slen, kv, 1.0)
    rows = [0, 1, 2, B - 1]
    kept = stored(torch, x[rows, 290:], kv, dtype, False)
    agree(torch, (out[rows], lse[rows]),
          bound(torch, q[rows], None, kept, [0], [], [slen[b] - 290 for b in rows], kv, 1.0, False))


BAD = {False: ["latent nan", "latent inf", "latent -inf", "rope nan"],
       True: ["latent nan", "rope nan", "scale nan", "scale inf"]}


@pytest.mark.parametrize("form", [f for f in FORMS if f[3] > 1] + [(128, 16, 3, 4), (512, 32, 1, 9), (128, 16, 64, 2)], ids=str)
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("bad", [(k, b) for k in BAD for b in BAD[k]], ids=str)
def test_a_bad_position_reaches_the_tokens_that_see_it_alone(form, dtype, bad):
    """A later token's own position holds a NaN or an infinity: the tokens before it do not notice."""
    torch, latent = mods()
    kv, rope, H, T = form
    fp8, what = bad
    dtype = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(34)
    # last positions inside a tile, across tiles of 64 and 128 and across key ranges, and nothing but them
    slen = [50, 66, 130, 129, 385, 700, T, 258, 257, 50]
    back = [(3 * b) % T for b in range(len(slen))]
    back[0], back[1], back[-1] = 0, T - 1, None  # how many positions from the last; the last row is sound
    starts, plen = [0, 7], [90]
    pre = make_cache(torch, g, plen, 90, kv, rope, dtype, fp8)
    suf = make_cache(torch, g, slen, max(slen), kv, rope, dtype, fp8)
    q = torch.randn(len(slen), T, H, kv + rope, generator=g, device="cuda").to(dtype)
    clean = (suf[0] if not fp8 else None, suf[1].clone(), None)
    raw = suf[0] if not fp8 else tuple(t.clone() for t in suf[0])
    raw = raw.clone() if not fp8 else raw
    sees = torch.zeros(len(slen), T, dtype=torch.bool, device="cuda")
    for b, d in enumerate(back):
        if d is None:
            continue
        j = slen[b] - 1 - d
        sees[b, T - 1 - d:] = True
        value = {"nan": NAN, "inf": float("inf"), "-inf": float("-inf")}[what.split()[1]]
        if what.startswith("scale"):
            raw[2][b, j] = value
        elif what.startswith("rope"):
            (raw[1][b, j] if fp8 else raw[b, j, kv:])[rope // 2] = value
        elif fp8:
            raw[0].view(torch.uint8)[b, j, kv // 3] = 0x7F
        else:
            raw[b, j, kv // 3] = value
    out, lse = run(torch, latent, q, pre[0], raw, starts, plen, slen, kv, 0.11)
    want, wl, size, mag = reference(torch, q, pre[1], clean[1], starts, plen, slen, 0.11, kv)
    u = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    es = (q.shape[-1] / 16 + 2) * 2.0 ** -23 * mag
    ok = ~sees[..., None].expand(-1, -1, H)
    # fp16 weights: at most 2^-25 of 2^6 off each, for at most 800 values of up to 6
    tol = size * (3 * u + 2 * es[..., None]) + 800 * 6 * 2.0 ** -31 + 1e-7
    assert torch.isfinite(out[ok]).all() and torch.isfinite(lse[ok]).all()
    assert torch.all(((out.double() - want).abs() <= tol)[ok])
    assert torch.all(((lse.double() - wl).abs() <= es + 800 * 2.0 ** -24 + 2.0 ** -20 * (1 + wl.abs()))[ok])
    # who sees it has a NaN in its result
    assert torch.isnan(out[~ok]).any(-1).all()


@pytest.mark.parametrize("form", [(128, 16, 8), (512, 32, 16), (512, 32, 5), (128, 16, 1), (40, 6, 2)], ids=str)
@pytest.mark.parametrize("kind", ["fp16", "bf16", "fp8/fp16"])
@pytest.mark.parametrize("tokens", [70, 333])
def test_every_position_of_a_prompt_is_a_query(form, kind, tokens):
    """The prompt form: rows of different lengths whose positions are their own query tokens, aligned at the
    end (a short row's first tokens see nothing), one of them with a NaN inside."""
    torch, latent = mods()
    kv, rope, H = form
    dtype = torch.bfloat16 if "bf16" in kind else torch.float16
    fp8 = "fp8" in kind
    g = torch.Generator(device="cuda").manual_seed(35)
    slen = [tokens, 1, tokens // 2 + 3, 0, tokens]
    suf = make_cache(torch, g, slen, tokens, kv, rope, dtype, fp8)
    q = torch.randn(len(slen), tokens, H, kv + rope, generator=g, device="cuda").to(dtype)
    at = tokens // 2 + 2  # the last row's bad position
    values = suf[1].clone()
    if fp8:
        suf[0][0].view(torch.uint8)[4, at, 3] = 0x7F
    else:
        suf[0][4, at, 3] = NAN
        values[4, at, 3] = 0
    out, lse = run(torch, latent, q, None, suf[0], [0], [], slen, kv, 0.11)
    want, wl, size, mag = reference(torch, q, None, values, [0], [], slen, 0.11, kv)
    u = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    es = (q.shape[-1] / 16 + 2) * 2.0 ** -23 * mag
    tol = size * (3 * u + 2 * es[..., None]) + tokens * 6 * 2.0 ** -31 + 1e-7
    ok = torch.ones_like(wl, dtype=torch.bool)
    ok[4, at:] = False
    seen = torch.isfinite(wl)
    assert torch.all(out[~seen] == 0) and torch.all(lse[~seen] == float("-inf"))
    assert torch.all(((out.double() - want).abs() <= tol)[ok])
    assert torch.all(((lse.double() - wl).abs() <= es + tokens * 2.0 ** -24 + 2.0 ** -20 * (1 + wl.abs()))[ok & seen])
    assert torch.isnan(out[~ok]).all()


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("fp8", [False, True])
def test_caches_whose_rows_share_their_storage(form, fp8):
    """Groups that share one stored prompt, and rows one suffix: strides of zero. And a cache of one row."""
    torch, latent = mods()
    kv, rope, H, T = form
    g = torch.Generator(device="cuda").manual_seed(38)

    def shared(n, positions):
        c, v, unit = stored(torch, torch.randn(1, positions, kv + rope, generator=g, device="cuda"), kv, torch.float16, fp8)
        e = lambda t: t.expand(n, *t.shape[1:])  # noqa: E731
        return (tuple(map(e, c)) if fp8 else e(c)), e(v), e(unit)

    pre, suf = shared(2, 300), shared(5, 210)
    q = torch.randn(5, T, H, kv + rope, generator=g, device="cuda").half()
    args = ([0, 3, 5], [300, 141], [210, 9, 0, 64, 130], kv, 0.1)
    agree(torch, run(torch, latent, q, pre[0], suf[0], *args), bound(torch, q, pre, suf, *args, fp8))
    pre, suf = shared(1, 130), shared(1, 90)
    args = ([0, 1], [130], [90], kv, 0.1)
    agree(torch, run(torch, latent, q[:1], pre[0], suf[0], *args), bound(torch, q[:1], pre, suf, *args, fp8))


def test_no_argument_may_require_a_gradient():
    torch, latent = mods()
    from cpp_inference_train_engine_b200 import EngineError
    half = dict(dtype=torch.float16, device="cuda")
    q, pre, suf = torch.zeros(2, 1, 8, 144, **half), torch.zeros(1, 16, 144, **half), torch.zeros(2, 16, 144, **half)
    for t in (q, pre, suf):
        t.requires_grad_()
        with pytest.raises(EngineError, match="gradient"):
            run(torch, latent, q, pre, suf, [0, 2], [4], [1, 2], 128, 0.1)
        with torch.no_grad():
            run(torch, latent, q, pre, suf, [0, 2], [4], [1, 2], 128, 0.1)
        t.requires_grad_(False)
    c = latent.alloc_cache(2, 16, 128, 16)
    x, r, s = torch.zeros(3, 128, **half), torch.zeros(3, 16, **half), torch.arange(3, device="cuda")
    for t in (x, r, c.rope, c.scale):
        t.requires_grad_()
        with pytest.raises(EngineError, match="gradient"):
            latent.cache_write(c, x, r, s)
        t.requires_grad_(False)
    c.scale.requires_grad_()
    with pytest.raises(EngineError, match="gradient"):
        latent.cache_read(c, s)


def test_a_write_counts_as_one():
    """autograd notices that a tensor which it keeps was written."""
    torch, latent = mods()
    c = latent.alloc_cache(2, 16, 128, 16)
    w = torch.ones_like(c.scale, requires_grad=True)
    loss = (c.scale * w).sum()  # keeps the scales for w's gradient
    x, r, s = torch.ones(3, 128, device="cuda"), torch.ones(3, 16, device="cuda"), torch.arange(3, device="cuda")
    before = [t._version for t in c]
    latent.cache_write(c, x, r, s)
    assert all(t._version > v for t, v in zip(c, before))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        latent.cache_write(latent.alloc_cache(2, 16, 128, 16), x, r, s)
