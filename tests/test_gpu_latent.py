"""Shared-prompt decode operators (latent.py / include/mm_latent.h) against their definitions in
64 bits: attention over a shared prefix and per-row suffixes, the 8-bit latent cache, and the
verification of drafted tokens."""
import itertools

import pytest

from tests.gpu_util import require_gpu

pytestmark = pytest.mark.gpu

WIDTHS = [(128, 16, 8), (512, 32, 16), (128, 16, 3), (512, 32, 5), (8, 4, 2), (40, 6, 3)]
NAN = float("nan")


def mods():
    require_gpu()
    import torch

    from cpp_inference_train_engine_b200 import latent
    return torch, latent


# ------------------------------------------------------------------ attention
def make_cache(torch, g, lens, positions, kv, rope, dtype, fp8):
    """A cache of len(lens) rows whose positions at or past the length hold NaN."""
    n = len(lens)
    x = torch.randn(n, positions, kv + rope, generator=g, device="cuda")
    past = (torch.arange(positions, device="cuda")[None] >= torch.tensor(lens, device="cuda")[:, None])
    if not fp8:
        x = x.to(dtype)
        x[past] = NAN
        return x, x.double()
    s = (x[..., :kv].abs().amax(-1) / 448).clamp_min(2.0 ** -100)
    codes = (x[..., :kv] / s[..., None]).to(torch.float8_e4m3fn)
    rk = x[..., kv:].to(dtype)
    values = torch.cat([codes.float().double() * s.double()[..., None], rk.double()], -1)
    raw = codes.view(torch.uint8)
    raw[past] = 0x7F  # NaN code
    rk[past] = NAN
    s[past] = NAN
    return (codes, rk, s), values


def reference(torch, q, prefix, suffix, starts, plen, slen, scale, kv):
    """out, lse, elementwise bound of |out|'s error per unit of relative error, score magnitude."""
    B, T, H, W = q.shape
    out = torch.zeros(B, T, H, kv, dtype=torch.float64, device="cuda")
    lse = torch.full((B, T, H), float("-inf"), dtype=torch.float64, device="cuda")
    size = torch.zeros_like(out)
    mag = torch.zeros_like(lse)
    group = [-1] * B
    for i in range(len(starts) - 1):
        for b in range(starts[i], starts[i + 1]):
            group[b] = i
    for b, t in itertools.product(range(B), range(T)):
        keys = []
        if group[b] >= 0:
            keys.append(prefix[group[b], :plen[group[b]]])
        if suffix is not None:
            keys.append(suffix[b, :max(0, slen[b] - (T - 1 - t))])
        k = torch.cat(keys) if keys else q.new_zeros(0, W, dtype=torch.float64)
        if k.shape[0] == 0:
            continue
        qd = q[b, t].double()
        z = qd @ k.T * scale
        lse[b, t] = torch.logsumexp(z, -1)
        p = torch.softmax(z, -1)
        out[b, t] = p @ k[:, :kv]
        size[b, t] = p @ k[:, :kv].abs()
        mag[b, t] = (qd.abs() @ k.abs().T * abs(scale)).amax(-1)
    return out, lse, size, mag


def check_attention(torch, latent, q, pre, suf, starts, plen, slen, kv, scale, **hints):
    (pc, pv), (sc, sv) = pre, suf
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    out, lse = latent.shared_prefix_attention(
        q, pc, sc, i32(starts) if pc is not None else None, i32(plen) if pc is not None else None,
        i32(slen) if sc is not None else None, scale, kv_rank=kv, return_lse=True, **hints)
    want, wl, size, mag = reference(torch, q, pv, sv, starts, plen, slen, scale, kv)
    assert out.dtype == q.dtype and out.shape == want.shape and lse.dtype == torch.float32
    # unit roundoff of the 16-bit type: probabilities and the result are each rounded to it once
    # (three with the shared scale of an 8-bit value folded into the probability)
    u = 2.0 ** -11 if q.dtype == torch.float16 else 2.0 ** -8
    W = q.shape[-1]
    # fp32 accumulation of W products in steps of 16, each losing at most 2^-23 of the magnitude
    es = (W / 16 + 2) * 2.0 ** -23 * mag
    keys = max(plen, default=0) + max(slen, default=0)
    sub = keys * 2.0 ** -25 * 8  # probabilities below the normal range of fp16
    tol = size * (3 * u + 2 * es[..., None]) + sub + 1e-7
    seen = torch.isfinite(wl)
    assert torch.equal(torch.isfinite(lse), seen)
    assert torch.all(out[~seen] == 0) and torch.all(lse[~seen] == float("-inf"))
    err = (out.double() - want).abs()
    assert torch.all(err <= tol), float((err / tol).max())
    el = (lse.double() - wl)[seen].abs()
    assert torch.all(el <= (es + keys * 2.0 ** -24 + 2.0 ** -20 * (1 + wl.abs()))[seen]), float(el.max())
    return out, lse


CASES = [
    # (rows per group, prefix lengths, suffix lengths pattern, tokens)
    ([1], [1], [1], 1),
    ([8], [128], [9], 1),
    ([3, 0, 5, 1], [0, 7, 129, 300], [0, 1, 64, 65, 2, 0, 16, 17, 33], 1),
    ([16, 2, 9], [127, 513, 1], [31, 128, 129, 5], 1),
    ([4, 3], [200, 65], [0, 1, 2, 5, 70, 3, 130], 3),
    ([11], [257], [8, 40, 7], 8),
]


@pytest.mark.parametrize("width", WIDTHS, ids=str)
@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("kind", ["fp16", "bf16", "fp8/fp16", "fp8/bf16", "mixed"])
def test_attention(width, case, kind):
    torch, latent = mods()
    kv, rope, H = width
    groups, plen, pattern, T = CASES[case]
    dtype = torch.bfloat16 if "bf16" in kind else torch.float16
    g = torch.Generator(device="cuda").manual_seed(100 * case + kv)
    B = sum(groups)
    starts = [sum(groups[:i]) for i in range(len(groups) + 1)]
    slen = [pattern[i % len(pattern)] for i in range(B)]
    pre = make_cache(torch, g, plen, max(plen) + 3, kv, rope, dtype, "fp8" in kind or kind == "mixed")
    suf = make_cache(torch, g, slen, max(slen) + 5, kv, rope, dtype, "fp8" in kind)
    q = (torch.randn(B, T, H, kv + rope, generator=g, device="cuda") * 1.5).to(dtype)
    check_attention(torch, latent, q, pre, suf, starts, plen, slen, kv, 0.11)


@pytest.mark.parametrize("width", WIDTHS[:2], ids=str)
@pytest.mark.parametrize("fp8", [False, True])
def test_attention_long_prefix_split_over_the_grid(width, fp8):
    """One group, few rows, a prefix long enough that its positions are divided and joined."""
    torch, latent = mods()
    kv, rope, H = width
    g = torch.Generator(device="cuda").manual_seed(5)
    plen, slen = [9001], [700, 0, 1023]
    pre = make_cache(torch, g, plen, 9001, kv, rope, torch.float16, fp8)
    suf = make_cache(torch, g, slen, 1024, kv, rope, torch.float16, fp8)
    q = torch.randn(3, 2, H, kv + rope, generator=g, device="cuda").half()
    check_attention(torch, latent, q, pre, suf, [0, 3], plen, slen, kv, 0.1)


@pytest.mark.parametrize("width", WIDTHS[:3], ids=str)
def test_attention_many_query_rows(width):
    """More query rows per group than one tile holds, and a last tile that is ragged."""
    torch, latent = mods()
    kv, rope, H = width
    g = torch.Generator(device="cuda").manual_seed(6)
    groups, plen = [37, 1, 20], [140, 64, 300]
    B, T = sum(groups), 4
    slen = [(7 * b) % 50 for b in range(B)]
    pre = make_cache(torch, g, plen, 300, kv, rope, torch.bfloat16, False)
    suf = make_cache(torch, g, slen, 50, kv, rope, torch.bfloat16, False)
    q = torch.randn(B, T, H, kv + rope, generator=g, device="cuda").bfloat16()
    check_attention(torch, latent, q, pre, suf, [0, 37, 38, 58], plen, slen, kv, 0.1)


@pytest.mark.parametrize("width", [WIDTHS[0], WIDTHS[1], WIDTHS[4]], ids=str)
def test_attention_without_prefix_or_suffix(width):
    torch, latent = mods()
    kv, rope, H = width
    g = torch.Generator(device="cuda").manual_seed(7)
    q = torch.randn(5, 1, H, kv + rope, generator=g, device="cuda").half()
    pre = make_cache(torch, g, [33, 70], 70, kv, rope, torch.float16, False)
    suf = make_cache(torch, g, [1, 0, 90, 17, 64], 90, kv, rope, torch.float16, False)
    check_attention(torch, latent, q, pre, (None, None), [0, 2, 5], [33, 70], [0] * 5, kv, 0.1)
    check_attention(torch, latent, q, (None, None), suf, [0], [], [1, 0, 90, 17, 64], kv, 0.1)
    # rows before the first and after the last group have no prefix
    check_attention(torch, latent, q, pre, suf, [1, 2, 4], [33, 70], [1, 0, 90, 17, 64], kv, 0.1)


@pytest.mark.parametrize("width", [WIDTHS[0], WIDTHS[1], WIDTHS[4]], ids=str)
@pytest.mark.parametrize("fp8", [False, True])
def test_attention_strides(width, fp8):
    """q with permuted strides, caches that are slices of larger ones, bounds below the capacity."""
    torch, latent = mods()
    kv, rope, H = width
    g = torch.Generator(device="cuda").manual_seed(8)
    plen, slen = [50, 129], [3, 80, 0, 9]
    T = 2
    q = torch.randn(H, 4, T, kv + rope + 8, generator=g, device="cuda").half().permute(1, 2, 0, 3)[..., :kv + rope]

    def sliced(lens, positions):
        c, v = make_cache(torch, g, [n for n in lens for _ in (0, 1)], 2 * positions, kv, rope, torch.float16, fp8)
        cut = lambda t: t[1::2, positions // 2:]  # noqa: E731
        # the slice starts inside the row: its own lengths, NaN past them
        if fp8:
            v = cut(v)
            c = tuple(cut(t) for t in c)
        else:
            c = v = cut(c)
        return c, v.double()

    # lengths inside a slice that begins at positions // 2
    pre, suf = sliced([50 + 65, 129 + 65], 130), sliced([3 + 40, 80 + 40, 40, 9 + 40], 80)
    check_attention(torch, latent, q, pre, suf, [0, 1, 4], plen, slen, kv, 0.1, max_prefix=129, max_suffix=80,
                    max_group=3)


@pytest.mark.parametrize("width", WIDTHS[:2], ids=str)
@pytest.mark.parametrize("which", ["q", "prefix", "suffix", "pos_stride", "rope", "codes"])
def test_attention_unaligned(width, which):
    """Bases and strides that no 16-byte load can take."""
    torch, latent = mods()
    kv, rope, H = width
    W = kv + rope
    g = torch.Generator(device="cuda").manual_seed(13)
    plen, slen = [150], [40, 66]

    def odd(t, pad=1, off=1):
        n = t.shape[-1]
        big = torch.zeros(*t.shape[:-1], n + pad, dtype=t.dtype, device="cuda")
        big[..., off:off + n] = t
        return big[..., off:off + n]

    fp8 = which in ("rope", "codes")
    pre = make_cache(torch, g, plen, 150, kv, rope, torch.float16, fp8)
    suf = make_cache(torch, g, slen, 66, kv, rope, torch.float16, fp8)
    q = torch.randn(2, 2, H, W, generator=g, device="cuda").half()
    if which == "q":
        q = odd(q)
    elif which == "prefix":
        pre = (odd(pre[0], 8, 3), pre[1])
    elif which == "suffix":
        suf = (odd(suf[0], 8, 3), suf[1])
    elif which == "pos_stride":
        pre = (odd(pre[0], 3, 0), pre[1])
    elif which == "rope":
        suf = ((suf[0][0], odd(suf[0][1]), suf[0][2]), suf[1])
    else:
        codes = odd(pre[0][0].view(torch.uint8), 5, 2).view(torch.float8_e4m3fn)
        pre = ((codes, pre[0][1], pre[0][2]), pre[1])
    check_attention(torch, latent, q, pre, suf, [0, 2], plen, slen, kv, 0.1)


def test_attention_lengths_are_clamped_and_groups_bounded():
    torch, latent = mods()
    kv, rope, H = 128, 16, 8
    g = torch.Generator(device="cuda").manual_seed(9)
    q = torch.randn(4, 1, H, kv + rope, generator=g, device="cuda").half()
    pre = make_cache(torch, g, [64], 64, kv, rope, torch.float16, False)
    suf = make_cache(torch, g, [32] * 4, 32, kv, rope, torch.float16, False)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    got = latent.shared_prefix_attention(q, pre[0], suf[0], i32([0, 4]), i32([2 ** 30]), i32([2 ** 30, -5, 7, 32]),
                                         0.1, kv_rank=kv, max_prefix=48, max_suffix=20)
    want = latent.shared_prefix_attention(q, pre[0], suf[0], i32([0, 4]), i32([48]), i32([20, 0, 7, 20]), 0.1,
                                          kv_rank=kv)
    assert torch.allclose(got.float(), want.float(), atol=4e-3)


@pytest.mark.parametrize("width", WIDTHS[:2], ids=str)
def test_attention_offsets_beyond_32_bits(width):
    """Cache rows more than 2^31 elements from the base."""
    torch, latent = mods()
    kv, rope, H = width
    W = kv + rope
    g = torch.Generator(device="cuda").manual_seed(10)
    stride = 2 ** 31 // 16 * 16 + 16 * W
    base = torch.empty(stride + 128 * W, dtype=torch.float16, device="cuda")
    pre = base.as_strided((2, 128, W), (stride, W, 1))
    pre.copy_(torch.randn(2, 128, W, generator=g, device="cuda"))
    q = torch.randn(4, 1, H, W, generator=g, device="cuda").half()
    check_attention(torch, latent, q, (pre, pre.double()), (None, None), [0, 2, 4], [128, 77], [0] * 4, kv, 0.1)
    # the same storage as the rows' own suffixes
    check_attention(torch, latent, q[:2], (None, None), (pre, pre.double()), [0], [], [128, 77], kv, 0.1)


@pytest.mark.parametrize("width", WIDTHS[:2], ids=str)
def test_attention_extreme_scores(width):
    """Scores that rise steeply along the keys (the running maximum keeps moving), scores of large
    magnitude, and keys equal to each other."""
    torch, latent = mods()
    kv, rope, H = width
    W = kv + rope
    g = torch.Generator(device="cuda").manual_seed(11)
    n, m = 400, 150
    q = torch.zeros(2, 1, H, W, device="cuda").half()
    q[..., kv:] = 1.0
    pre = torch.randn(1, n, W, generator=g, device="cuda").half()
    suf = torch.randn(2, m, W, generator=g, device="cuda").half()
    pre[0, :, kv:] = torch.linspace(-60, 60, n, device="cuda")[:, None].half()
    suf[:, :, kv:] = torch.linspace(60, 75, m, device="cuda")[None, :, None].half()
    suf[1, :, kv:] = -60.0
    for scale in (0.25, 1.0, -0.5):
        check_attention(torch, latent, q, (pre, pre.double()), (suf, suf.double()), [0, 2], [n], [m, m], kv, scale)


@pytest.mark.parametrize("width", [WIDTHS[0], WIDTHS[1], WIDTHS[4]], ids=str)
def test_attention_is_deterministic_and_runs_on_the_callers_stream(width):
    torch, latent = mods()
    kv, rope, H = width
    g = torch.Generator(device="cuda").manual_seed(12)
    plen, slen = [700, 90], [300, 4, 55, 128, 17, 0]
    pre = make_cache(torch, g, plen, 700, kv, rope, torch.float16, True)[0]
    suf = make_cache(torch, g, slen, 300, kv, rope, torch.float16, True)[0]
    q = torch.randn(6, 1, H, kv + rope, generator=g, device="cuda").half()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    args = (i32([0, 4, 6]), i32(plen), i32(slen), 0.1)
    first = latent.shared_prefix_attention(q, pre, suf, *args, kv_rank=kv, return_lse=True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    big = torch.randn(4096, 4096, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = torch.zeros_like(q)
        for _ in range(8):
            big = big @ big * 1e-4
        late.copy_(q)  # behind a long product on the same stream
        again = latent.shared_prefix_attention(late, pre, suf, *args, kv_rank=kv, return_lse=True)
    side.synchronize()
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    # the call can be captured and replayed
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = latent.shared_prefix_attention(q, pre, suf, *args, kv_rank=kv)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first[0])


# ------------------------------------------------------------------ 8-bit cache
def e4m3_nearest(torch, v):
    """Nearest e4m3 value of |v| <= 448 in 64 bits, ties to even."""
    e = torch.frexp(v)[1].clamp_min(-5)
    step = torch.ldexp(torch.ones_like(v), e - 4)
    return (v / step).round() * step


@pytest.mark.parametrize("width", [(128, 16), (512, 32), (8, 4), (40, 6), (1, 0), (130, 10), (1024, 64)], ids=str)
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rope_dtype", ["float16", "bfloat16"])
def test_cache_write_and_read(width, dtype, rope_dtype):
    torch, latent = mods()
    kv, rope = width
    dtype, rope_dtype = getattr(torch, dtype), getattr(torch, rope_dtype)
    g = torch.Generator(device="cuda").manual_seed(kv)
    R, P, n = 3, 50, 77
    cache = latent.alloc_cache(R, P, kv, rope, rope_dtype)
    x = torch.randn(n, kv, generator=g, device="cuda") * torch.logspace(-6, 4, n, device="cuda")[:, None]
    x = x.to(dtype)
    x[5] = 0
    r = torch.randn(n, rope, generator=g, device="cuda").to(dtype)
    slots = torch.randperm(R * P, generator=g, device="cuda")[:n]
    slots[7], slots[8], slots[9] = -1, R * P, -(2 ** 40)  # skipped
    latent.cache_write(cache, x, r, slots)
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[7:10] = False
    s = (x.float().abs().amax(1) / torch.tensor(448.0, device="cuda")).clamp_min(2.0 ** -100)
    assert torch.equal(cache.scale.view(-1)[slots[keep]], s[keep])
    codes = cache.latent.float().view(-1, kv)[slots[keep]].double()
    v = x[keep].double() / s[keep].double()[:, None]
    # IEEE division in fp32 (relative 2^-24) can move a value across the middle of two codes only
    # when it lies that close to it
    near = e4m3_nearest(torch, v)
    off = codes != near
    assert torch.all((codes - v)[off].abs() <= (near - v)[off].abs() + 2.0 ** -22 * v[off].abs())
    assert torch.equal(cache.rope.view(R * P, rope)[slots[keep]], r[keep].float().to(rope_dtype))
    # every other position is untouched
    rest = torch.ones(R * P, dtype=torch.bool, device="cuda")
    rest[slots[keep]] = False
    assert torch.all(cache.latent.float().view(-1, kv)[rest] == 0) and torch.all(cache.scale.view(-1)[rest] == 0)
    for out_dtype in (torch.float32, torch.float16, torch.bfloat16):
        y = latent.cache_read(cache, slots, out_dtype)
        want = torch.cat([codes.float() * s[keep][:, None], cache.rope.view(R * P, rope)[slots[keep]].float()], 1)
        assert torch.equal(y[keep], want.to(out_dtype))
        assert torch.all(y[~keep] == 0)
    # what 8 bits lose: half a unit of 3 stored bits, or of the smallest subnormal's
    y = latent.cache_read(cache, slots[keep], torch.float32)[:, :kv].double()
    assert torch.all((y - x[keep].double()).abs() <= x[keep].double().abs() * (2.0 ** -4 + 2.0 ** -20) +
                     s[keep].double()[:, None] * 2.0 ** -10)


def test_cache_write_nonfinite_rows_stay_their_own():
    torch, latent = mods()
    cache = latent.alloc_cache(1, 8, 128, 16)
    x = torch.ones(4, 128, device="cuda")
    x[1, 3], x[2, 5] = NAN, float("inf")
    latent.cache_write(cache, x, torch.ones(4, 16, device="cuda"), torch.arange(4, device="cuda"))
    y = latent.cache_read(cache, torch.arange(4, device="cuda"), torch.float32)
    assert torch.all(y[0] == 1) and torch.all(y[3] == 1)
    assert torch.isnan(y[1, 3]) and torch.all(y[1, :3] == 1) and torch.all(y[1, 4:] == 1)
    assert torch.isnan(y[2, :128]).any() and torch.all(y[2, 128:] == 1)


def test_cache_strides_and_empty_calls():
    torch, latent = mods()
    big = latent.alloc_cache(4, 40, 512, 32, torch.bfloat16)
    cut = latent.LatentCache(big.latent[1::2, 3:20], big.rope[1::2, 3:20], big.scale[1::2, 3:20])
    wide = torch.randn(6, 700, device="cuda").bfloat16()
    slots = torch.tensor([0, 16, 17, 33, 5, 20], device="cuda")
    latent.cache_write(cut, wide[:, 100:612], wide[:, 650:682], slots)
    y = latent.cache_read(cut, slots)
    assert y.dtype == torch.bfloat16
    assert (y[:, :512].float() - wide[:, 100:612].float()).abs().max() < 0.3
    assert torch.equal(y[:, 512:], wide[:, 650:682])
    touched = torch.zeros(4, 40, dtype=torch.bool, device="cuda")
    for s in slots.tolist():
        touched[1 + 2 * (s // 17), 3 + s % 17] = True
    assert torch.equal(big.scale != 0, touched)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    latent.cache_write(cut, wide[:0, :512], wide[:0, :32], none)
    assert latent.cache_read(cut, none).shape == (0, 544)


# ------------------------------------------------------------------ draft verification
def verify_reference(torch, p, q, x, lens, ua, us):
    """The definition with Python integers."""
    B, K1, V = p.shape
    K = K1 - 1
    tokens, counts = [], []
    f32 = lambda t: t.float().cpu()  # noqa: E731
    p, ua, us, x, lens = f32(p), ua.cpu(), us.cpu(), x.cpu().tolist(), lens.cpu().tolist()
    q = None if q is None else f32(q)
    for b in range(B):
        n, L = 0, min(max(lens[b], 0), K)
        while n < L:
            t = x[b][n]
            if not 0 <= t < V:
                break
            qx = q[b, n, t] if q is not None else torch.tensor(1.0)
            if not bool(ua[b, n] * qx < p[b, n, t]):
                break
            n += 1

        def weigh(r):
            return [int(v) for v in (torch.nan_to_num(r, nan=0.0).clamp(0, 1).double() * 2.0 ** 38).floor().tolist()]
        w = weigh(p[b, n])
        if n < L:
            qn = q[b, n] if q is not None else torch.zeros(V)
            if q is None and 0 <= x[b][n] < V:
                qn[x[b][n]] = 1.0
            r = weigh((p[b, n] - qn))
            w = r if sum(r) > 0 else w
        total = sum(w)
        y = -1
        if total > 0:
            k = min(max(int(float(us[b]) * 2 ** 24), 0), 2 ** 24 - 1)
            t, run = total * k // 2 ** 24, 0
            for y, v in enumerate(w):
                run += v
                if run > t:
                    break
        tokens.append(x[b][:n] + [y] + [-1] * (K - n))
        counts.append(n)
    return tokens, counts


@pytest.mark.parametrize("V", [1, 3, 31, 512, 513, 4096, 16384, 20001])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("drawn", [True, False])
def test_verify_drafts(V, dtype, drawn):
    torch, latent = mods()
    dtype = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(V)
    B, K = 9, 5
    z = torch.randn(B, K + 1, V, generator=g, device="cuda") * 2
    p = torch.softmax(z, -1)
    d = torch.softmax(z[:, :K] + 0.5 * torch.randn(B, K, V, generator=g, device="cuda"), -1)
    x = torch.multinomial(d.view(-1, V), 1, generator=g).view(B, K).int()
    p, d = p.to(dtype), d.to(dtype)
    lens = torch.tensor([5, 0, 1, 4, 5, 9, -3, 2, 5], dtype=torch.int32, device="cuda")
    ua = torch.rand(B, K, generator=g, device="cuda") * (0.2 if not drawn else 1.0)
    us = torch.rand(B, generator=g, device="cuda")
    us[0], us[1], us[2] = 0.0, 1.0 - 2.0 ** -24, 1.5
    x[4, 1], x[7, 0] = V + 3, -2  # outside the vocabulary: rejected
    d[8] = p[8, :K]  # no residual after a rejection: the target itself
    ua[8] = 1.0 if drawn else 0.0
    tokens, n = latent.verify_drafts(p, x, lens, ua, us, draft_probs=d if drawn else None)
    want, wn = verify_reference(torch, p, d if drawn else None, x, lens, ua, us)
    assert n.tolist() == wn
    assert tokens.tolist() == want


def test_verify_drafts_many_drafts_and_degenerate_rows():
    torch, latent = mods()
    g = torch.Generator(device="cuda").manual_seed(3)
    B, K, V = 4, 70, 97
    p = torch.softmax(torch.randn(B, K + 1, V, generator=g, device="cuda"), -1)
    x = torch.randint(0, V, (B, K), generator=g, device="cuda").int()
    lens = torch.tensor([70, 33, 64, 32], dtype=torch.int32, device="cuda")
    ua = torch.zeros(B, K, device="cuda")
    ua[2, 40] = 1.0
    us = torch.rand(B, generator=g, device="cuda")
    us[3] = NAN
    p[1, 33] = NAN   # no weight at all: no token
    p[0, 70, :50] = NAN
    p[3, 32, 7] = 5.0  # clamped to 1
    got = latent.verify_drafts(p, x, lens, ua, us)
    us[3] = 0.0
    want = verify_reference(torch, p, None, x, lens, ua, us)
    assert got[0].tolist() == want[0] and got[1].tolist() == want[1]
    assert got[0][1, 33].item() == -1
    # no drafts at all: one token per row from its only distribution
    t, n = latent.verify_drafts(p[:, :1].contiguous(), x[:, :0].contiguous(), lens, ua[:, :0].contiguous(), us)
    want = verify_reference(torch, p[:, :1], None, x[:, :0], lens, ua[:, :0], us)
    assert t.tolist() == want[0] and n.tolist() == want[1] == [0] * B


def test_verify_drafts_follows_the_target_distribution():
    """Over many draws, token 0 (the draft or its replacement) is distributed as the target."""
    torch, latent = mods()
    g = torch.Generator(device="cuda").manual_seed(4)
    V, N = 5, 200000
    p = torch.tensor([0.5, 0.2, 0.15, 0.1, 0.05], device="cuda")
    q = torch.tensor([0.1, 0.3, 0.2, 0.3, 0.1], device="cuda")
    x = torch.multinomial(q, N, replacement=True, generator=g).int()[:, None]
    tokens, _ = latent.verify_drafts(p.expand(N, 2, V).contiguous(), x, torch.ones(N, dtype=torch.int32, device="cuda"),
                                     torch.rand(N, 1, generator=g, device="cuda"), torch.rand(N, generator=g, device="cuda"),
                                     draft_probs=q.expand(N, 1, V).contiguous())
    freq = torch.bincount(tokens[:, 0].long(), minlength=V).double() / N
    # five standard deviations of a binomial share
    assert torch.all((freq - p.double()).abs() < 5 * (p.double() * (1 - p.double()) / N).sqrt())


# ------------------------------------------------------------------ refusals
def test_refusals():
    torch, latent = mods()
    from cpp_inference_train_engine_b200 import EngineError
    half = dict(dtype=torch.float16, device="cuda")
    q = torch.zeros(2, 1, 8, 144, **half)
    pre, suf = torch.zeros(1, 16, 144, **half), torch.zeros(2, 16, 144, **half)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    gs, pl, sl = i32([0, 2]), i32([4]), i32([1, 2])

    def bad(match, f, *a, **k):
        with pytest.raises(EngineError, match=match) as e:
            f(*a, **k)
        assert e.value.name in ("invalid_argument", "unsupported")

    att = latent.shared_prefix_attention
    bad("fp16 or bf16", att, q.float(), pre, suf, gs, pl, sl, 0.1, kv_rank=128)
    bad("type must be", att, q, pre.bfloat16(), suf, gs, pl, sl, 0.1, kv_rank=128)
    bad("width", att, q, pre[..., :140].contiguous(), suf, gs, pl, sl, 0.1, kv_rank=128)
    bad("kv_rank", att, q, pre, suf, gs, pl, sl, 0.1, kv_rank=145)
    bad("prefix row per group", att, q, pre, suf, i32([0, 1, 2]), i32([4, 4]), sl, 0.1, kv_rank=128)
    bad("suffix row per row", att, q, pre, suf[:1], gs, pl, sl, 0.1, kv_rank=128)
    bad("prefix_len", att, q, pre, suf, gs, i32([4, 4]), sl, 0.1, kv_rank=128)
    bad("int32", att, q, pre, suf, gs, pl, sl.long(), 0.1, kv_rank=128)
    bad("exceed", att, q, pre, suf, gs, pl, sl, 0.1, kv_rank=128, max_prefix=17)
    bad("exceed", att, q, pre, suf, gs, pl, sl, 0.1, kv_rank=128, max_suffix=-1)
    bad("a prefix or a suffix", att, q, None, None, None, None, None, 0.1, kv_rank=128)
    bad("adjacent", att, q.transpose(2, 3), pre, suf, gs, pl, sl, 0.1, kv_rank=128)
    bad("one CUDA device", att, q, pre.cpu(), suf, gs, pl, sl, 0.1, kv_rank=128)
    bad("CUDA tensor", att, q.cpu(), pre, suf, gs, pl, sl, 0.1, kv_rank=128)
    empty = att(q[:0], pre, suf[:0], i32([0, 0]), pl, sl[:0], 0.1, kv_rank=128)
    assert empty.shape == (0, 1, 8, 128)

    c = latent.alloc_cache(2, 16, 128, 16)
    x, r, s = torch.zeros(3, 128, **half), torch.zeros(3, 16, **half), torch.arange(3, device="cuda")
    bad("8-bit cache", latent.cache_write, pre, x, r, s)
    bad("match", latent.cache_write, c, x[:, :64].contiguous(), r, s)
    bad("one floating type", latent.cache_write, c, x, r.float(), s)
    bad("int64", latent.cache_write, c, x, r, s.int())
    bad("float8", latent.cache_read, (c.latent.float(), c.rope, c.scale), s)
    bad("fp32, fp16 or bf16", latent.cache_read, c, s, torch.float64)

    p, xt, ua, us = torch.ones(2, 3, 8, device="cuda") / 8, i32([[0, 0], [0, 0]]), torch.zeros(2, 2, device="cuda"), \
        torch.zeros(2, device="cuda")
    bad("draft_tokens", latent.verify_drafts, p, xt.long(), sl, ua, us)
    bad("draft_probs", latent.verify_drafts, p, xt, sl, ua, us, draft_probs=p)
    bad("u_accept", latent.verify_drafts, p, xt, sl, ua[:1], us)
    bad("262,144", latent.verify_drafts, torch.zeros(1, 1, 262145, device="cuda"), xt[:1, :0].contiguous(), sl[:1],
        ua[:1, :0].contiguous(), us[:1])


@pytest.mark.parametrize("width", WIDTHS[:2], ids=str)
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_attention_reads_every_code(width, dtype):
    """All 254 finite e4m3 codes as latent values, and a NaN that stays with the queries that see it."""
    torch, latent = mods()
    kv, rope, H = width
    dtype = getattr(torch, dtype)
    codes = [c for c in range(256) if c & 0x7F != 0x7F]
    raw = torch.tensor([codes[i % 254] for i in range(2 * kv)], dtype=torch.uint8, device="cuda").view(2, 1, kv)
    lat = raw.view(torch.float8_e4m3fn)
    rk = torch.zeros(2, 1, rope, dtype=dtype, device="cuda")
    for scale in (1.0, 2.0 ** -7):
        cache = (lat, rk, torch.full((2, 1), scale, device="cuda"))
        q = torch.zeros(2, 1, H, kv + rope, dtype=dtype, device="cuda")
        one = torch.ones(2, dtype=torch.int32, device="cuda")
        out = latent.shared_prefix_attention(q, None, cache, None, None, one, 1.0, kv_rank=kv)
        # one key: its probability is 1, so the output is the value itself, exactly
        assert torch.equal(out.float(), (lat.float() * scale).view(2, 1, 1, kv).expand(2, 1, H, kv).to(dtype).float())
    bad = raw.clone()
    bad[1, 0, 5] = 0x7F
    out = latent.shared_prefix_attention(q, None, (bad.view(torch.float8_e4m3fn), rk, cache[2]), None, None, one, 1.0,
                                         kv_rank=kv)
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1, 0, :, 5]).all()


@pytest.mark.parametrize("width", WIDTHS[:2], ids=str)
@pytest.mark.parametrize("prefix", [40, 1100])
def test_attention_thousands_of_groups(width, prefix):
    """More groups than the work list has entries, most of them of one row or none, with no bound on
    their sizes given; short prefixes (one range each) and long ones (several)."""
    torch, latent = mods()
    kv, rope, H = width
    g = torch.Generator(device="cuda").manual_seed(16)
    groups = [(i * 7919) % 5 % 3 for i in range(1300)]
    groups[700] = 41
    starts = [sum(groups[:i]) for i in range(len(groups) + 1)]
    plen = [0 if i % 3 == 0 else 1 + i % 33 for i in range(len(groups))]
    for i in (0, 511, 512, 513, 700, 1299):
        plen[i] = prefix
    slen = [i % 4 for i in range(starts[-1])]
    pre = make_cache(torch, g, plen, prefix, kv, rope, torch.float16, False)
    suf = make_cache(torch, g, slen, 4, kv, rope, torch.float16, False)
    q = torch.randn(starts[-1], 1, H, kv + rope, generator=g, device="cuda").half()
    check_attention(torch, latent, q, pre, suf, starts, plen, slen, kv, 0.1)


@pytest.mark.parametrize("vocab", [1024, 1027])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_verify_many_rows(vocab, dtype):
    """A batch of several blocks per multiprocessor gives each row what it gets in a small batch."""
    torch, latent = mods()
    dtype = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(21)
    B, K = 900, 3
    p = torch.softmax(2 * torch.randn(B, K + 1, vocab, generator=g, device="cuda"), -1).to(dtype)
    q = torch.softmax(2 * torch.randn(B, K, vocab, generator=g, device="cuda"), -1).to(dtype)
    x = torch.randint(0, vocab, (B, K), generator=g, device="cuda", dtype=torch.int32)
    n = torch.randint(0, K + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    ua, us = torch.rand(B, K, generator=g, device="cuda"), torch.rand(B, generator=g, device="cuda")
    for d in (q, None):
        tokens, accepted = latent.verify_drafts(p, x, n, ua, us, draft_probs=d)
        for b in range(0, B, 90):
            r = slice(b, b + 90)
            t, a = latent.verify_drafts(p[r], x[r], n[r], ua[r], us[r], draft_probs=None if d is None else d[r])
            assert torch.equal(t, tokens[r]) and torch.equal(a, accepted[r])


@pytest.mark.parametrize("kind", ["fp16", "bf16", "fp8/fp16", "mixed"])
@pytest.mark.parametrize("shape", ["ragged", "one long", "alike", "many"])
def test_attention_rows_divided_by_their_lengths(kind, shape):
    """Suffixes of very different lengths over as many rows as there are CTAs, with short prefixes: rows
    are cut where a CTA's share ends."""
    torch, latent = mods()
    kv, rope, H = 512, 32, 5
    dtype = torch.bfloat16 if "bf16" in kind else torch.float16
    g = torch.Generator(device="cuda").manual_seed(23)
    T = 2 if shape == "ragged" else 1
    B = 700 if shape == "many" else 141
    slen = {"ragged": [(b * 211) % 601 for b in range(B)], "one long": [b % 3 for b in range(B - 1)] + [1500],
            "alike": [520 + b % 3 for b in range(B)], "many": [0 if b % 5 else (b * 37) % 700 for b in range(B)]}[shape]
    groups = [B // 3, 0, B - B // 3 - 4]  # the last rows have no prefix
    starts = [0, groups[0], groups[0], groups[0] + groups[2]]
    plen = [130, 5, 0 if shape == "many" else 64]
    pre = make_cache(torch, g, plen, 131, kv, rope, dtype, "fp8" in kind or kind == "mixed")
    suf = make_cache(torch, g, slen, max(slen), kv, rope, dtype, "fp8" in kind)
    q = torch.randn(B, T, H, kv + rope, generator=g, device="cuda").to(dtype)
    a = check_attention(torch, latent, q, pre, suf, starts, plen, slen, kv, 0.08)
    b = check_attention(torch, latent, q, pre, suf, starts, plen, slen, kv, 0.08)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
