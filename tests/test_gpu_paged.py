"""Paged-cache decode and beam-search operators (paged.py / include/mm_paged.h) against their definitions
in 64 bits: appending through a page table, attention of one token over pages, beam selection and
reordering."""
import math
import random

import pytest

from tests.gpu_util import require_gpu

pytestmark = pytest.mark.gpu

# (latent width, rope width, heads); the last two have no tensor-core form
WIDTHS = [(128, 16, 8), (512, 32, 16), (128, 16, 19), (512, 32, 5), (512, 32, 33), (8, 4, 2), (40, 6, 3)]
NAN = float("nan")
UNIT = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def mods():
    require_gpu()
    import torch

    from cpp_inference_train_engine_b200 import paged
    return torch, paged


def i32(torch, v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ attention
def seen_positions(n, window, sinks):
    first = max(n - window, 0) if window else 0
    return sorted(set(range(min(sinks, n) if window else 0)) | set(range(first, n)))


def make_pages(torch, g, lens, page, kv, rope, dtype, fp8, window=0, sinks=0, spread=1.0):
    """A pool whose seen positions hold values and everything else NaN, its table (pages that no row sees: -1)
    and the seen values of every row in 64 bits."""
    seen = [seen_positions(n, window, sinks) for n in lens]
    columns = max(1, (max(lens) + page - 1) // page) + 1
    used = [(b, j) for b, s in enumerate(seen) for j in sorted({t // page for t in s})]
    pages = len(used) + 2
    order = torch.randperm(pages, generator=g, device="cuda")[:len(used)].tolist()
    table = torch.full((len(lens), columns), -1, dtype=torch.int32)
    for (b, j), p in zip(used, order):
        table[b, j] = p
    x = torch.full((pages, page, kv + rope), NAN, device="cuda", dtype=dtype)
    codes = torch.full((pages, page, kv), 0x7F, dtype=torch.uint8, device="cuda")
    scale = torch.full((pages, page), NAN, device="cuda")
    values = []
    for b, s in enumerate(seen):
        v = spread * torch.randn(len(s), kv + rope, generator=g, device="cuda").to(dtype)
        at = torch.tensor(s, dtype=torch.int64)
        p, e = table[b, at // page].long().cuda(), (at % page).cuda()
        x[p, e] = v
        if fp8 and s:
            sc = (v[:, :kv].float().abs().amax(-1) / 448).clamp_min(2.0 ** -100)
            c = (v[:, :kv].float() / sc[:, None]).to(torch.float8_e4m3fn)
            codes[p, e], scale[p, e] = c.view(torch.uint8), sc
            v = torch.cat([c.float().double() * sc.double()[:, None], v[:, kv:].double()], -1)
        values.append(v.double())
    from cpp_inference_train_engine_b200.latent import LatentCache
    cache = LatentCache(codes.view(torch.float8_e4m3fn), x[..., kv:].contiguous(), scale) if fp8 else x
    return cache, table.cuda(), values


def check_attention(torch, paged, q, cache, table, lens, values, kv, scale, **kw):
    """Against the definition in 64 bits. The tolerance of a result counts three roundings to 16 bits
    (weight, result; with an 8-bit value's scale folded into the weight), the scores' fp32 sums of W products
    in steps of 16 (2^-23 of their magnitude each) as a change of the weights, above and below the line, and
    weights below fp16's normal range (2^-25 of the largest each at most)."""
    out, lse = paged.attention(q, cache, table, i32(torch, lens), scale, kv_rank=kv, return_lse=True, **kw)
    assert out.shape == (len(lens), q.shape[1], kv) and out.dtype == q.dtype and lse.dtype == torch.float32
    u, W = UNIT[str(q.dtype).split(".")[1]], q.shape[-1]
    for b, k in enumerate(values):
        if k.shape[0] == 0:
            assert torch.all(out[b] == 0) and torch.all(lse[b] == float("-inf"))
            continue
        qd = q[b].double()
        z = qd @ k.T * scale
        p = torch.softmax(z, -1)
        want, size = p @ k[:, :kv], p @ k[:, :kv].abs()
        es = (W / 16 + 2) * 2.0 ** -23 * (qd.abs() @ k.abs().T * abs(scale)).amax(-1)
        tol = size * (3 * u + 2 * es[:, None]) + k.shape[0] * 2.0 ** -25 * k[:, :kv].abs().max() + 1e-7
        err = (out[b].double() - want).abs()
        assert torch.all(err <= tol), (b, float((err / tol).max()))
        wl = torch.logsumexp(z, -1)
        assert torch.all((lse[b].double() - wl).abs() <= es + k.shape[0] * 2.0 ** -24 + 2.0 ** -20 * (1 + wl.abs())), b
    return out, lse


CASES = [  # page size, lengths, window, sinks
    (16, [1], 0, 0),
    (64, [197, 0, 64, 65], 0, 0),
    (32, [31, 32, 33, 1000, 0, 17, 512], 0, 0),
    (16, [4097, 3, 260], 0, 0),
    (128, [129, 2500, 7, 640, 5000] + list(range(0, 300, 7)), 0, 0),
    (16, [500, 20, 0, 33, 1], 32, 4),
    (64, [1000, 129, 40, 700, 70], 100, 1),
    (32, [777, 36, 37, 38, 2000], 1, 37),
    (16, [300, 64, 10], 1000, 5),
    (48, [300, 64, 10, 2000], 555, 0),
    (24, [100, 24, 7, 0], 0, 0),  # no tensor-core form
    (1, [3, 0, 40], 0, 0),
]


@pytest.mark.parametrize("width", WIDTHS, ids=str)
@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("kind", ["fp16", "bf16", "fp8/fp16", "fp8/bf16"])
def test_attention(width, case, kind):
    torch, paged = mods()
    kv, rope, H = width
    page, lens, window, sinks = CASES[case]
    dtype = torch.bfloat16 if "bf16" in kind else torch.float16
    g = torch.Generator(device="cuda").manual_seed(case * 100 + kv)
    cache, table, values = make_pages(torch, g, lens, page, kv, rope, dtype, "fp8" in kind, window, sinks)
    q = torch.randn(len(lens), H, kv + rope, generator=g, device="cuda").to(dtype)
    check_attention(torch, paged, q, cache, table, lens, values, kv, 1 / math.sqrt(96), window=window or None, sinks=sinks)
    paged.check_status()


@pytest.mark.parametrize("width", [(128, 16, 8), (512, 32, 16), (40, 6, 3)], ids=str)
@pytest.mark.parametrize("kind", ["bf16", "fp8/fp16"])
def test_attention_over_long_rows(width, kind):
    """Rows cut between many blocks, and ragged ones beside them."""
    torch, paged = mods()
    kv, rope, H = width
    dtype = torch.bfloat16 if "bf16" in kind else torch.float16
    for lens in ([40001], [1, 30000, 0, 17, 9000], [700 + 13 * i for i in range(40)]):
        g = torch.Generator(device="cuda").manual_seed(len(lens))
        cache, table, values = make_pages(torch, g, lens, 64, kv, rope, dtype, "fp8" in kind)
        q = torch.randn(len(lens), H, kv + rope, generator=g, device="cuda").to(dtype)
        one = check_attention(torch, paged, q, cache, table, lens, values, kv, 0.09)
        two = paged.attention(q, cache, table, i32(torch, lens), 0.09, kv_rank=kv, return_lse=True)
        assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])  # equal inputs, equal bits
        tight = paged.attention(q, cache, table, i32(torch, lens), 0.09, kv_rank=kv, max_length=max(lens))
        assert (tight.float() - one[0].float()).abs().max() <= 4 * UNIT[str(dtype).split(".")[1]] * one[0].float().abs().max()


@pytest.mark.parametrize("width", [(128, 16, 8), (512, 32, 16), (40, 6, 3)], ids=str)
@pytest.mark.parametrize("fp8", [False, True])
def test_strides_alignment_and_shared_pages(width, fp8):
    """q and pool with strides of their own (some without a tensor-core form), rows that share a page, a table
    that is part of a wider one."""
    torch, paged = mods()
    from cpp_inference_train_engine_b200.latent import LatentCache
    kv, rope, H = width
    g = torch.Generator(device="cuda").manual_seed(5)
    lens, page = [200, 37, 64], 32
    cache, table, values = make_pages(torch, g, lens, page, kv, rope, torch.float16, fp8)
    table[1, 0] = table[0, 0]  # rows 0 and 1 share their first page
    values[1] = torch.cat([values[0][:32], values[1][32:]])
    wide = torch.full((3, table.shape[1] + 5), 10 ** 6, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + table.shape[1]] = table
    table = wide[:, 2:2 + table.shape[1]]
    for pad in (1, 4, 8):
        q = torch.randn(3, H, kv + rope + pad, generator=g, device="cuda").half()[..., pad // 2:pad // 2 + kv + rope]
        check_attention(torch, paged, q, cache, table, lens, values, kv, 0.1)

        def padded(t):
            w = torch.zeros(*t.shape[:-1], t.shape[-1] + 8 * pad, dtype=t.dtype, device="cuda")
            w = w.view(torch.uint8).fill_(0xFF).view(t.dtype) if t.element_size() == 1 else w.fill_(NAN)
            w = w[..., 3 * pad:3 * pad + t.shape[-1]]
            w.view(w.dtype).copy_(t)
            return w
        other = LatentCache(*(padded(t) for t in cache)) if fp8 else padded(cache)
        check_attention(torch, paged, q, other, table, lens, values, kv, 0.1)


@pytest.mark.parametrize("width", [(128, 16, 8), (512, 32, 16), (40, 6, 3)], ids=str)
@pytest.mark.parametrize("kind", ["fp16", "bf16", "fp8/fp16", "fp8/bf16"])
def test_scores_and_values_of_any_size(width, kind):
    """Scores far from zero, keys masked by the lowest score beside others, small and large values."""
    torch, paged = mods()
    kv, rope, H = width
    dtype = torch.bfloat16 if "bf16" in kind else torch.float16
    for spread, scale in ((1e-3, 50.0), (1e-2, 1.0), (30.0, 0.02), (1.0, 3.0), (1.0, -0.5), (1.0, 0.0)):
        g = torch.Generator(device="cuda").manual_seed(int(spread * 1000) + H)
        lens = [300, 5, 129]
        cache, table, values = make_pages(torch, g, lens, 16, kv, rope, dtype, "fp8" in kind, spread=spread)
        q = torch.randn(3, H, kv + rope, generator=g, device="cuda").to(dtype)
        check_attention(torch, paged, q, cache, table, lens, values, kv, scale)


@pytest.mark.parametrize("width", [(128, 16, 8), (512, 32, 16), (40, 6, 3)], ids=str)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("low", ["lowest", "-inf"])
def test_positions_masked_by_their_rope_key(width, fp8, low):
    """Positions whose rope key makes them score the type's lowest value or minus infinity weigh nothing,
    wherever they stand."""
    torch, paged = mods()
    kv, rope, H = width
    g = torch.Generator(device="cuda").manual_seed(2)
    lens = [333, 70]
    cache, table, values = make_pages(torch, g, lens, 16, kv, rope, torch.bfloat16, fp8)
    q = torch.randn(2, H, kv + rope, generator=g, device="cuda").bfloat16()
    q[..., kv] = 1.0
    rk = cache[1] if fp8 else cache[..., kv:]
    bad = torch.finfo(torch.bfloat16).min if low == "lowest" else float("-inf")
    kept = []
    for b, n in enumerate(lens):
        hide = [t for t in range(n) if t < 40 or t % 3 == 0 or t == n - 1]
        at = torch.tensor(hide)
        rk[table[b, (at // 16).cuda()].long(), (at % 16).cuda(), 0] = bad
        kept.append(values[b][[t for t in range(n) if t not in set(hide)]])
    check_attention(torch, paged, q, cache, table, lens, kept, kv, 0.1)


@pytest.mark.parametrize("width", [(128, 16, 8), (512, 32, 16), (40, 6, 3)], ids=str)
@pytest.mark.parametrize("what", ["latent", "rope", "scale", "query"])
@pytest.mark.parametrize("bad", [NAN, float("inf")])
def test_a_bad_value_stays_in_its_row(width, what, bad):
    torch, paged = mods()
    kv, rope, H = width
    for fp8 in (False, True):
        if what == "scale" and not fp8 or what == "latent" and fp8 and bad == bad:
            continue  # (codes have no infinity)
        g = torch.Generator(device="cuda").manual_seed(3)
        lens = [100, 300, 50, 4000]
        cache, table, values = make_pages(torch, g, lens, 32, kv, rope, torch.float16, fp8)
        q = torch.randn(4, H, kv + rope, generator=g, device="cuda").half()
        clean = paged.attention(q, cache, table, i32(torch, lens), 0.1, kv_rank=kv)
        page, at = int(table[1, 77 // 32]), 77 % 32
        if what == "query":
            q[1, H - 1, 3] = bad
        elif what == "scale":
            cache.scale[page, at] = bad
        elif what == "rope":
            (cache.rope[page, at] if fp8 else cache[page, at, kv:])[1] = bad
        elif fp8:
            cache.latent.view(torch.uint8)[page, at, 5] = 0x7F
        else:
            cache[page, at, 5] = bad
        out = paged.attention(q, cache, table, i32(torch, lens), 0.1, kv_rank=kv)
        if what == "query":
            assert torch.equal(out[1, :H - 1], clean[1, :H - 1]) and not torch.isfinite(out[1, H - 1]).any()
        elif what != "rope" or bad != bad:
            assert not torch.isfinite(out[1]).all(-1).any()  # every head's result
        for b in (0, 2, 3):
            assert torch.equal(out[b], clean[b])


def test_entries_outside_the_pool_and_lengths_outside_the_table():
    """Pages that are not there are not seen; lengths end at the table and at max_length."""
    torch, paged = mods()
    for kv, rope, H, page in ((128, 16, 8, 16), (512, 32, 16, 32), (40, 6, 3, 5)):
        for fp8 in (False, True):
            g = torch.Generator(device="cuda").manual_seed(1)
            lens = [10 * page, 10 * page, 7 * page, 3]
            cache, table, values = make_pages(torch, g, lens, page, kv, rope, torch.float16, fp8)
            table = table[:, :10]
            q = torch.randn(4, H, kv + rope, generator=g, device="cuda").half()
            table[0, 3], table[0, 9], table[1, 0], table[2, :] = -1, 10 ** 6, -2 ** 31, 2 ** 31 - 1
            rows = [[t for t in range(n) if t // page not in gone] for n, gone in zip(lens, ((3, 9), (0,), range(10), ()))]
            left = [v[r] for v, r in zip(values, rows)]
            check_attention(torch, paged, q, cache, table, [10 * page, 2 ** 31 - 1, 7 * page, 3], left, kv, 0.1)
            check_attention(torch, paged, q, cache, table, [10 * page, -5, 7 * page, 3], [left[0], left[0][:0], left[2], left[3]], kv, 0.1)
            cut = [v[[i for i, t in enumerate(r) if t < 2 * page + 1]] for v, r in zip(left, rows)]
            check_attention(torch, paged, q, cache, table, lens, cut, kv, 0.1, max_length=2 * page + 1)


def test_attention_of_nothing():
    torch, paged = mods()
    for kv, rope, H in ((128, 16, 8), (40, 6, 3)):
        cache = paged.alloc_pages(1, 4, 16, kv, rope)[0]
        q = torch.ones(3, H, kv + rope, dtype=torch.float16, device="cuda")
        for lens, columns in (([0, 0, -3], 2), ([5, 9, 1], 0)):
            out, lse = paged.attention(q, cache, torch.zeros(3, columns, dtype=torch.int32, device="cuda"), i32(torch, lens), 0.1,
                                       kv_rank=kv, return_lse=True)
            assert torch.all(out == 0) and torch.all(lse == float("-inf"))
        empty = paged.attention(q[:0], cache, torch.zeros(0, 2, dtype=torch.int32, device="cuda"), i32(torch, []), 0.1, kv_rank=kv)
        assert empty.shape == (0, H, kv)
        none = paged.attention(q, cache[:0], torch.zeros(3, 2, dtype=torch.int32, device="cuda"), i32(torch, [5, 9, 1]), 0.1, kv_rank=kv)
        assert torch.all(none == 0)


def test_offsets_past_32_bits():
    """A pool of more than 2^31 values: its last pages."""
    torch, paged = mods()
    pages, page, kv, rope, H = 123400, 64, 512, 32, 16  # 4.3e9 values, 8.6 GB
    pool = torch.empty(pages, page, kv + rope, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    used = [pages - 1, 3, pages - 2, pages // 2 + 1]
    rows = []
    for p in used:
        pool[p] = torch.randn(page, kv + rope, generator=g, device="cuda")
        rows.append(pool[p].double())
    table = i32(torch, [used])
    q = torch.randn(1, H, kv + rope, generator=g, device="cuda").bfloat16()
    check_attention(torch, paged, q, pool, table, [250], [torch.cat(rows)[:250]], kv, 0.1)
    values = torch.randn(1, kv + rope, generator=g, device="cuda")
    paged.append(pool, values, i32(torch, [[3, pages - 1]]), i32(torch, [64 + 9]), kv_rank=kv)
    assert torch.equal(pool[-1, 9, :kv], values[0, :kv].bfloat16())


@pytest.mark.parametrize("width", [(128, 16, 8), (512, 32, 16), (40, 6, 3)], ids=str)
@pytest.mark.parametrize("window,sinks", [(50, 3), (1, 0), (33, 70)])
def test_rows_of_2_31_positions_through_a_window(width, window, sinks):
    """The last positions that 32 bits hold: every column of the table is one of two pages."""
    torch, paged = mods()
    kv, rope, H = width
    g = torch.Generator(device="cuda").manual_seed(0)
    pool = torch.randn(2, 16, kv + rope, generator=g, device="cuda").half()
    table = torch.zeros(1, 2 ** 27 - 1, dtype=torch.int32, device="cuda")
    table[0, -3:] = 1
    q = torch.randn(1, H, kv + rope, generator=g, device="cuda").half()
    for n in (2 ** 31 - 16, 2 ** 31 - 17, 2 ** 31 - 40):
        at = list(range(sinks)) + list(range(n - window, n))
        keys = torch.stack([pool[int(table[0, t // 16]), t % 16] for t in at]).double()
        check_attention(torch, paged, q, pool, table, [n], [keys], kv, 0.1, window=window, sinks=sinks)


# ------------------------------------------------------------------ append
def entry_bits(torch, cache):
    return [t.view(torch.uint8).clone() for t in (cache if isinstance(cache, tuple) else (cache,))]


def check_append(torch, paged, cache, values, table, rows, positions, kv, norm, theta=10000.0, eps=1e-5):
    """Stored values against 64 bits, and everything else left as it was. Tolerances: one rounding to the stored
    type, the normalisation's fp32 sum of kv squares in steps of 16 and four more roundings, the rotation's
    fp32 sine and cosine of an angle known to 2^-21."""
    fp8 = isinstance(cache, tuple)
    before = entry_bits(torch, cache)
    paged.append(cache, values, table, i32(torch, positions), kv_rank=kv, rows=None if rows is None else i32(torch, rows),
                 theta=theta, norm=norm, eps=eps)
    pages, page = (cache[0] if fp8 else cache).shape[:2]
    rope = values.shape[1] - kv
    touched = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    for i, t in enumerate(positions):
        r = i if rows is None else rows[i]
        if not (0 <= r < table.shape[0] and 0 <= t < table.shape[1] * page):
            continue
        p, e = int(table[r, t // page]), t % page
        if not 0 <= p < pages:
            continue
        touched[p, e] = True
        x = values[i].double()
        lat = x[:kv]
        if norm is not None:
            lat = lat / math.sqrt(float((lat * lat).mean()) + eps) * norm.double()
        angle = t * theta ** (-torch.arange(0, rope, 2, dtype=torch.float64, device="cuda") / rope)
        a, b = x[kv::2], x[kv + 1::2]
        key = torch.stack([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], -1).flatten()
        size = torch.stack([a.abs() + b.abs()] * 2, -1).flatten()
        rel = (kv / 16 + 4) * 2.0 ** -24 if norm is not None else 0.0
        got_key = cache[1][p, e] if fp8 else cache[p, e, kv:]
        u = UNIT[str(got_key.dtype).split(".")[1]]
        tiny = 2.0 ** -25 if got_key.dtype == torch.float16 else 0.0  # half a step below the normal range
        assert torch.all((got_key.double() - key).abs() <= u * key.abs() + 2.0 ** -20 * size + tiny), (i, t)
        if not fp8:
            assert torch.all((cache[p, e, :kv].double() - lat).abs() <= (u + 2 * rel) * lat.abs() + tiny), (i, t)
            continue
        s = max(float(lat.abs().max()) / 448, 2.0 ** -100)
        got = float(cache[2][p, e])
        assert abs(got - s) <= (2 * rel + 2.0 ** -23) * s
        code = cache[0][p, e].float().double()
        ratio = lat / s
        # half a step: 2^-4 of the value, 2^-10 below the smallest normal code
        assert torch.all((code - ratio).abs() <= (2.0 ** -4 + 4 * rel + 2.0 ** -22) * ratio.abs() + 2.0 ** -10)
    for t, old in zip(cache if fp8 else (cache,), before):
        now = t.view(torch.uint8).reshape(pages, page, -1)
        assert torch.equal(now[~touched], old.reshape(pages, page, -1)[~touched])


@pytest.mark.parametrize("width", [(128, 16), (512, 32), (40, 6), (7, 0), (128, 32)], ids=str)
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("kind", ["float16", "bfloat16", "fp8/float16", "fp8/bfloat16"])
@pytest.mark.parametrize("normed", [False, True])
def test_append(width, dtype, kind, normed):
    torch, paged = mods()
    kv, rope = width
    g = torch.Generator(device="cuda").manual_seed(kv)
    for page, n, far in ((16, 1, 0), (64, 13, 900), (3, 70, 10 ** 6)):
        cache = paged.layer(paged.alloc_pages(2, 140, page, kv, rope, getattr(torch, kind.split("/")[-1]), 8 if "fp8" in kind else 16), 1)
        columns = far // page + 20
        table = torch.full((5, columns), -1, dtype=torch.int32, device="cuda")
        table[:, far // page:] = torch.randperm(100, generator=g, device="cuda").view(5, -1)[:, :columns - far // page].int()
        rows = [i % 5 for i in range(n)]
        positions = [far // page * page + i // 5 for i in range(n)]
        if n > 8:  # a free row, a position without a page, one past the table, rows outside it
            positions[2], positions[4], positions[6], rows[7], rows[8] = -1, 0 if far else 10 ** 6, columns * page, 5, -1
        values = (2 * torch.randn(n, kv + rope + 3, generator=g, device="cuda")).to(getattr(torch, dtype))[:, 3:] \
            if n == 13 else (2 * torch.randn(n, kv + rope, generator=g, device="cuda")).to(getattr(torch, dtype))
        norm = 1 + 0.2 * torch.randn(kv, generator=g, device="cuda") if normed else None
        check_append(torch, paged, cache, values, table, rows, positions, kv, norm)


@pytest.mark.parametrize("width", [(128, 16), (512, 32), (8, 4)], ids=str)
@pytest.mark.parametrize("bits", [8, 16])
def test_append_of_a_step(width, bits):
    """One token per row without row numbers, rows of all sizes: zeros, tiny and large values, a NaN."""
    torch, paged = mods()
    kv, rope = width
    g = torch.Generator(device="cuda").manual_seed(1)
    cache = paged.layer(paged.alloc_pages(1, 64, 32, kv, rope, bits=bits), 0)
    table = torch.randperm(64, generator=g, device="cuda").view(32, 2).int()
    values = torch.randn(32, kv + rope, generator=g, device="cuda") * (2.0 ** torch.arange(-20, 12, device="cuda"))[:, None] / 16
    values[3] = 0
    positions = [(7 * i) % 64 for i in range(32)]
    check_append(torch, paged, cache, values, table, None, positions, kv, None)
    check_append(torch, paged, cache, values, table, None, positions, kv, torch.ones(kv, device="cuda"))
    values[5, 2] = NAN
    paged.append(cache, values, table, i32(torch, positions), kv_rank=kv, norm=torch.ones(kv, device="cuda"))
    p, e = int(table[5, positions[5] // 32]), positions[5] % 32
    stored = (cache[0] if bits == 8 else cache)[p, e, :kv].float()
    assert torch.isnan(stored).all()


@pytest.mark.parametrize("width", [(128, 16), (512, 32)], ids=str)
@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("bits", [8, 16])
def test_append_of_many_tokens(width, dtype, bits):
    """More tokens than the blocks of one launch look up at a time: the same bits as in small calls."""
    torch, paged = mods()
    kv, rope = width
    n, page, columns, group = 160001, 64, 4, 9973
    g = torch.Generator(device="cuda").manual_seed(kv + bits)
    count = -(-n // (page * columns))
    values = torch.randn(n, kv + rope, generator=g, device="cuda").to(getattr(torch, dtype))
    place = torch.randperm(count * page * columns, generator=g, device="cuda")[:n].int()
    rows, positions = place // (page * columns), place % (page * columns)
    positions[::1013] = -1
    table = torch.randperm(count * columns, generator=g, device="cuda").int().view(count, columns)
    table[3, 2], table[5, 0] = -1, count * columns
    norm = torch.rand(kv, generator=g, device="cuda") + 0.5
    a, b = (paged.layer(paged.alloc_pages(1, count * columns, page, kv, rope, torch.float16, bits=bits), 0) for _ in range(2))
    paged.append(a, values, table, positions, kv_rank=kv, rows=rows, norm=norm)
    for i in range(0, n, group):
        at = slice(i, i + group)
        paged.append(b, values[at], table, positions[at], kv_rank=kv, rows=rows[at], norm=norm)
    for x, y in zip(*((t if bits == 8 else [t]) for t in (a, b))):
        assert x.float().any() and torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_far_positions_keep_their_angle():
    """Angles of positions up to the last 32-bit one: fp32 products would lose them."""
    torch, paged = mods()
    for kv, rope in ((128, 16), (512, 32), (8, 6)):
        cache = paged.layer(paged.alloc_pages(1, 3, 16, kv, rope, torch.bfloat16), 0)
        x = torch.zeros(1, kv + rope, device="cuda")
        x[0, kv::2] = 1
        wide = torch.full((1, 2 ** 27 - 1), 2, dtype=torch.int32, device="cuda")
        for t in (0, 1, 12345, 1000003, 2 ** 24 + 1, 2 ** 31 - 17):
            check_append(torch, paged, cache, x, wide, [0], [t], kv, None)


# ------------------------------------------------------------------ beam selection
def select_reference(torch, x, scores, count, finished, eos, equal=False):
    B, K, V = x.shape
    # (of equal beams once: a sum's rounding may depend on where a row begins)
    lse = torch.logsumexp(x[:, :1 if equal else K].double(), -1, keepdim=True)
    cand = scores.double()[..., None] + (x.double() - lse)
    live = torch.isfinite(scores)[..., None]
    if finished is not None:
        only = torch.arange(V, device="cuda") == eos
        cand = torch.where(finished[..., None], torch.where(only, scores.double()[..., None], float("-inf")), cand)
    cand = torch.where(live & torch.isfinite(cand.float()), cand, float("-inf")).view(B, K * V)
    best, at = torch.sort(cand, dim=1, descending=True, stable=True)
    if best.shape[1] < count:
        best = torch.nn.functional.pad(best, (0, count - best.shape[1]), value=float("-inf"))
        at = torch.nn.functional.pad(at, (0, count - at.shape[1]))
    best, at = best[:, :count], at[:, :count]
    none = best == float("-inf")
    slot = torch.arange(count, device="cuda").clamp_max(K - 1)[None]
    return best, torch.where(none, slot, at // V).int(), torch.where(none, -1, at % V).int()


def check_select(torch, paged, x, scores, count=None, finished=None, eos=None, equal=False):
    got = paged.beam_select(x, scores, beams=count, finished=finished, eos=eos)
    want = select_reference(torch, x, scores, count or x.shape[1], finished, eos, equal)
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    fine = torch.isfinite(want[0])
    assert torch.equal(torch.isfinite(got[0]), fine) and torch.all(got[0][~fine] == float("-inf"))
    # one rounding to fp32, and the log-sum-exp's exponentials (2^-22 each)
    err = (got[0].double() - want[0])[fine].abs()
    assert torch.all(err <= 2.0 ** -24 * want[0][fine].abs() + 2.0 ** -21), float(err.max())
    return got


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 3, 5), (1, 4, 16384), (5, 8, 1001), (3, 16, 32768), (40, 2, 257), (2, 32, 50001)], ids=str)
def test_beam_select(shape, dtype):
    torch, paged = mods()
    B, K, V = shape
    g = torch.Generator(device="cuda").manual_seed(V)
    x = (2 * torch.randn(B, K, V, generator=g, device="cuda")).to(getattr(torch, dtype))
    scores = -torch.rand(B, K, generator=g, device="cuda").cumsum(1) * 3
    check_select(torch, paged, x, scores)
    check_select(torch, paged, x, scores, count=min(32, 2 * K))
    finished = torch.rand(B, K, generator=g, device="cuda") < 0.4
    check_select(torch, paged, x, scores, finished=finished, eos=V // 2)
    first = torch.full_like(scores, float("-inf"))
    first[:, 0] = 0
    check_select(torch, paged, x, first)
    wide = torch.full((B, K + 2, V + 5), NAN, dtype=x.dtype, device="cuda")[:, 1:K + 1, 2:V + 2]
    wide.copy_(x)
    check_select(torch, paged, wide, scores)


def test_beam_select_takes_the_lowest_of_equal_candidates():
    torch, paged = mods()
    for V in (3, 1000, 20000):
        x = torch.zeros(2, 4, V, device="cuda")
        s = torch.zeros(2, 4, device="cuda")
        got = check_select(torch, paged, x, s, count=16)
        assert got[2][0].tolist() == ([0, 1, 2] * 4 + [-1] * 4 if V == 3 else list(range(16)))
        x[:, :, V // 2] = 1.0
        x[:, :, V - 1] = 1.0
        check_select(torch, paged, x, s, count=7)
        check_select(torch, paged, x.half(), s, count=32)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("shape", [(3, 4, 257), (2, 8, 1003), (1, 7, 50001), (70, 8, 3001), (1, 3, 16387)], ids=str)
def test_equal_beams_tie(shape, dtype):
    """Beams with the same logits and scores have the same candidates, wherever their rows begin: the lowest beam's
    come first, each token as often as there are beams."""
    torch, paged = mods()
    B, K, V = shape
    g = torch.Generator(device="cuda").manual_seed(V)
    x = (2 * torch.randn(B, 1, V, generator=g, device="cuda")).to(getattr(torch, dtype)).expand(B, K, V).contiguous()
    s = torch.full((B, K), -3.25, device="cuda")
    check_select(torch, paged, x, s, count=min(32, 2 * K + 1), equal=True)


def test_beam_select_of_dead_beams_and_banned_tokens():
    torch, paged = mods()
    g = torch.Generator(device="cuda").manual_seed(0)
    for V in (6, 700, 16384):
        inf = float("inf")
        x = torch.randn(6, 4, V, generator=g, device="cuda")
        s = torch.randn(6, 4, generator=g, device="cuda")
        x[0, :, 2:] = -inf  # two tokens are allowed
        s[0, 1:] = -inf     # in one beam: two candidates for four entries
        x[1, 2] = -inf      # a beam without a token
        x[2, 1, 3] = NAN
        x[3, 0, 5] = inf
        s[4] = torch.tensor([NAN, inf, -inf, -1.0], device="cuda")
        s[5] = -inf
        got = check_select(torch, paged, x, s)
        assert got[2][5].tolist() == [-1] * 4 and got[1][5].tolist() == [0, 1, 2, 3]
        check_select(torch, paged, x, s, finished=torch.ones(6, 4, dtype=torch.bool, device="cuda"), eos=0)
        x.fill_(-inf)
        check_select(torch, paged, x, s)
    big = torch.tensor([[[3e38, -3e38, 0.0]], [[-3e38, -3.4e38, -3e38]]], device="cuda")
    check_select(torch, paged, big, torch.zeros(2, 1, device="cuda"), count=3)


# ------------------------------------------------------------------ reorder
def reorder_reference(torch, cache, table, spare, lengths, parents, page):
    rows, columns = table.shape
    tensors = list(cache) if isinstance(cache, tuple) else [cache]
    old, new = [t.clone() for t in tensors], [t.clone() for t in tensors]
    t2, s2, n2 = table.clone(), spare.clone(), lengths.clone()
    for i in range(rows):
        p = int(parents[i])
        p = p if 0 <= p < rows else i
        n = min(max(int(lengths[p]), 0), columns * page)
        full, part = n // page, n % page
        t2[i, :full] = table[p, :full]
        n2[i] = n
        own = min(max(int(lengths[i]), 0), columns * page)
        if p != i and full < columns and (part or n != own):
            source, target = int(table[p, full]), int(spare[i])
            t2[i, full] = target
            s2[i] = table[i, own // page] if own < columns * page else -1
            pages = tensors[0].shape[1]
            if 0 <= source < pages and 0 <= target < pages:
                for o, t in zip(old, new):
                    t[:, target, :part] = o[:, source, :part]
    return new, t2, s2, n2


def check_reorder(torch, paged, cache, table, spare, lengths, parents, page):
    fp8 = isinstance(cache, tuple)
    bits = tuple(t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in cache) if fp8 else cache
    new, t2, s2, n2 = reorder_reference(torch, bits, table, spare, lengths, parents, page)
    got = paged.beam_reorder(cache, table, spare, lengths, parents)
    assert torch.equal(got[0], t2) and torch.equal(got[1], s2) and torch.equal(got[2], n2)
    for a, b in zip(bits if fp8 else (bits,), new):
        assert torch.equal(a, b)
    return got


@pytest.mark.parametrize("width", [(128, 16), (512, 32), (5, 2), (40, 6)], ids=str)
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("page", [1, 16, 30, 64])
def test_beam_reorder(width, bits, page):
    torch, paged = mods()
    kv, rope = width
    g = torch.Generator(device="cuda").manual_seed(page)
    for batch, k, layers, n in ((1, 1, 1, 5), (1, 4, 3, 2 * page), (3, 5, 2, 2 * page + page // 2 + 1), (2, 8, 1, 1)):
        rows, columns = batch * k, 4
        cache = paged.alloc_pages(layers, rows * (columns + 1), page, kv, rope, torch.bfloat16, bits)
        for t in cache if bits == 8 else (cache,):
            b = t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
            b.copy_(torch.randint(0, 100, b.shape, generator=g, device="cuda"))
        own = torch.randperm(rows * (columns + 1), generator=g, device="cuda").int()
        table, spare = own[:rows * columns].view(rows, columns).clone(), own[rows * columns:].clone()
        lengths = torch.full((rows,), min(n, columns * page), dtype=torch.int32, device="cuda")
        for step in range(3):
            parents = torch.randint(0, k, (rows,), generator=g, device="cuda") + torch.arange(rows, device="cuda") // k * k
            table, spare, lengths = check_reorder(torch, paged, cache, table, spare, lengths, parents.int(), page)
            # what a step may write to, a row's own: its last page, the spare one and those to come
            mine = torch.cat([spare, torch.cat([table[i, int(lengths[i]) // page:] for i in range(rows)])])
            assert mine.unique().numel() == mine.numel()
            lengths = (lengths + 1).clamp_max(columns * page).int()


def test_reorder_of_rows_of_all_lengths_and_bad_entries():
    """Finished beams keep their length; parents, pages and lengths outside their ranges touch nothing else."""
    torch, paged = mods()
    g = torch.Generator(device="cuda").manual_seed(4)
    for bits in (8, 16):
        cache = paged.alloc_pages(2, 60, 16, 128, 16, torch.float16, bits)
        for t in cache if bits == 8 else (cache,):
            b = t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
            b.copy_(torch.randint(0, 100, b.shape, generator=g, device="cuda"))
        own = torch.randperm(60, generator=g, device="cuda").int()
        table, spare = own[:40].view(8, 5).clone(), own[40:48].clone()
        lengths = i32(torch, [0, 80, 16, 17, 33, 79, 1, 64])
        for parents in ([1, 0, 3, 3, 5, 4, 7, 6], [-1, 8, 5, 5, 5, 2 ** 31 - 1, 5, 5], [3] * 8):
            check_reorder(torch, paged, cache, table, spare, lengths, i32(torch, parents), 16)
        table[3, 1], spare[2] = 10 ** 6, -1
        check_reorder(torch, paged, cache, table, spare, i32(torch, [-4, 10 ** 9, 16, 17, 33, 79, 1, 64]), i32(torch, [3, 3, 4, 4, 4, 3, 0, 1]), 16)
        wide = torch.full((8, 9), -7, dtype=torch.int32, device="cuda")[:, 1:6]
        wide.copy_(table)
        check_reorder(torch, paged, cache, wide, spare, lengths, i32(torch, [1, 0, 3, 3, 5, 4, 7, 6]), 16)


@pytest.mark.parametrize("page", [1, 4, 16])
@pytest.mark.parametrize("seed", [0, 1, 2])
def test_a_long_search_never_mixes_rows(page, seed):
    """Rows that finish (and stop growing), are dropped, copied and taken over again for many steps: every row's
    positions hold what its hypothesis stored, whatever pages they share."""
    torch, paged = mods()
    rng = random.Random(seed)
    rows, columns = 6, 64 // page
    cache = paged.alloc_pages(1, rows * (columns + 1), page, 8, 0, torch.bfloat16)
    own = list(range(rows * (columns + 1)))
    rng.shuffle(own)
    table = i32(torch, own[:rows * columns]).view(rows, columns)
    spare, lengths = i32(torch, own[rows * columns:]), i32(torch, [0] * rows)
    held, done, mark = [[] for _ in range(rows)], [False] * rows, 0
    for _ in range(55):
        values = torch.zeros(rows, 8, device="cuda")
        positions = []
        for r in range(rows):  # rows that are not done store a number of their own
            positions.append(-1 if done[r] else len(held[r]))
            if not done[r]:
                mark += 1
                held[r] = held[r] + [mark]
                values[r, 0], values[r, 1] = mark // 128, mark % 128  # (bf16 holds both)
        paged.append(cache[0], values, table, i32(torch, positions), kv_rank=8)
        lengths = i32(torch, [len(h) for h in held])
        parents = [rng.choice([r, r, rng.randrange(rows)]) for r in range(rows)]
        if all(done[p] for p in parents):  # some hypothesis goes on
            parents[0] = next((r for r in range(rows) if not done[r]), parents[0])
        table, spare, lengths = paged.beam_reorder(cache, table, spare, lengths, i32(torch, parents))
        held = [held[p] for p in parents]
        done = [done[p] or rng.random() < 0.08 for p in parents]
        if all(done):
            done[rng.randrange(rows)] = False if len(set(map(len, held))) == 1 else True
        assert lengths.tolist() == [len(h) for h in held]
        stored, pages = cache[0].float().cpu(), table.cpu()
        for r, h in enumerate(held):
            got = [int(stored[pages[r, t // page], t % page, 0] * 128 + stored[pages[r, t // page], t % page, 1]) for t in range(len(h))]
            assert got == h, (r, parents)
        if all(done):
            break


# ------------------------------------------------------------------ together
def step(torch, paged, cache, table, spare, lengths, values, logits, scores, q, kv, k):
    """One step of a beam search over one layer: store, attend, select, follow the parents."""
    paged.append(paged.layer(cache, 0), values, table, lengths, kv_rank=kv)
    out = paged.attention(q, paged.layer(cache, 0), table, lengths + 1, 0.1, kv_rank=kv)
    rows = table.shape[0]
    scores, parents, tokens = paged.beam_select(logits, scores)
    parent_rows = (parents + torch.arange(0, rows, k, device="cuda", dtype=torch.int32)[:, None]).view(-1)
    return out, scores, tokens, paged.beam_reorder(cache, table, spare, lengths + 1, parent_rows)


@pytest.mark.parametrize("bits", [8, 16])
def test_a_step_on_another_stream_and_in_a_graph(bits):
    """The four operators of a step together give the same bits eagerly, on a stream of their own and replayed
    from a graph whose inputs change between replays."""
    torch, paged = mods()
    kv, rope, H, k, batch = 128, 16, 8, 4, 3
    rows, page, columns = batch * k, 16, 6
    g = torch.Generator(device="cuda").manual_seed(0)
    n = torch.full((rows,), 39, dtype=torch.int32, device="cuda")
    own = torch.randperm(rows * (columns + 1), generator=g, device="cuda").int()
    table, spare = own[:rows * columns].view(rows, columns).clone(), own[rows * columns:].clone()
    start = torch.randn(1, rows * (columns + 1), page, kv + rope, generator=g, device="cuda").half()

    def inputs(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        return [r(rows, kv + rope), r(batch, k, 999), -r(batch, k).abs(), r(rows, H, kv + rope).half()]

    def fresh():
        if bits == 16:
            return start.clone()
        from cpp_inference_train_engine_b200.latent import LatentCache
        return LatentCache((start[..., :kv].float() * 40).to(torch.float8_e4m3fn), start[..., kv:].contiguous(),
                           torch.full(start.shape[:3], 1 / 40, device="cuda"))

    def flat(x):
        return [t for v in x for t in (flat(v) if isinstance(v, (tuple, list)) else [v])]

    want = []
    for seed in (1, 2):
        cache = fresh()
        v, x, s, q = inputs(seed)
        want.append(flat([step(torch, paged, cache, table, spare, n, v, x, s, q, kv, k), cache if bits == 8 else [cache]]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache = fresh()
        v, x, s, q = inputs(1)
        got = flat([step(torch, paged, cache, table, spare, n, v, x, s, q, kv, k), cache if bits == 8 else [cache]])
    side.synchronize()
    same = lambda a, b: torch.equal(a.view(torch.uint8), b.view(torch.uint8))  # noqa: E731
    assert all(same(a, b) for a, b in zip(got, want[0]))
    static = inputs(1)
    cache = fresh()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        v, x, s, q = static
        got = flat([step(torch, paged, cache, table, spare, n, v, x, s, q, kv, k), cache if bits == 8 else [cache]])
    for seed, w in zip((1, 2), want):
        for dst, src in zip(static, inputs(seed)):
            dst.copy_(src)
        for dst, src in zip(cache if bits == 8 else [cache], fresh() if bits == 8 else [fresh()]):
            dst.view(torch.uint8).copy_(src.view(torch.uint8))
        graph.replay()
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(got, w))


@pytest.mark.parametrize("width", [(128, 16, 8), (512, 32, 16)], ids=str)
@pytest.mark.parametrize("fp8", [False, True])
def test_cut_rows_in_graphs_and_on_two_streams_at_once(width, fp8):
    """Calls whose rows are cut between blocks (partial results in a workspace of the call's own) give the same bits
    eagerly, side by side on two streams, and from two graphs replayed in turn."""
    torch, paged = mods()
    kv, rope, H = width
    g = torch.Generator(device="cuda").manual_seed(0)
    sets = []
    for lens in ([9000, 5, 4000], [300 * i for i in range(40)]):
        cache, table, _ = make_pages(torch, g, lens, 32, kv, rope, torch.float16, fp8)
        q = torch.randn(len(lens), H, kv + rope, generator=g, device="cuda").half()
        sets.append((q, cache, table, i32(torch, lens)))
    call = lambda s: paged.attention(*s, 0.1, kv_rank=kv, return_lse=True)  # noqa: E731
    want = [call(s) for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(call(sets[i]))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call(s))
    for _ in range(3):
        for gr in graphs:
            gr.replay()
    torch.cuda.synchronize()
    for w, many, out in zip(want, got, outs):
        for r in many + [out]:
            assert torch.equal(w[0], r[0]) and torch.equal(w[1], r[1])


@pytest.mark.parametrize("shape", [(1, 4, 16384), (60, 6, 3001), (2, 20, 40000)], ids=str)
def test_beam_select_in_graphs_and_on_two_streams_at_once(shape):
    torch, paged = mods()
    g = torch.Generator(device="cuda").manual_seed(0)
    sets = [(torch.randn(*shape, generator=g, device="cuda"), -torch.rand(shape[:2], generator=g, device="cuda")) for _ in range(2)]
    want = [paged.beam_select(*s) for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(paged.beam_select(*sets[i]))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    x, s = sets[0][0].clone(), sets[0][1].clone()
    with torch.cuda.graph(graph):
        out = paged.beam_select(x, s)
    for i in (0, 1):
        x.copy_(sets[i][0])
        s.copy_(sets[i][1])
        graph.replay()
        torch.cuda.synchronize()
        for r in got[i] + [out]:
            assert all(torch.equal(a, b) for a, b in zip(want[i], r))


def test_writes_count_as_in_place():
    torch, paged = mods()
    cache = paged.alloc_pages(1, 4, 16, 128, 16)
    version = cache._version
    paged.append(cache[0], torch.zeros(1, 144, device="cuda"), i32(torch, [[0]]), i32(torch, [0]), kv_rank=128)
    assert cache._version > version
    version = cache._version
    paged.beam_reorder(cache, i32(torch, [[0]]), i32(torch, [1]), i32(torch, [3]), i32(torch, [0]))
    assert cache._version > version


# ------------------------------------------------------------------ refusals
# Every pointer is a tensor's and every entry of a table, length or parent is 0, so that a call that were not refused
# would stay in bounds.
@pytest.mark.parametrize("kv, rope", [(128, 16), (512, 32)])
@pytest.mark.parametrize("page_stride", [None, 1 << 45])  # one page: of no meaning, but one that no tensor map takes
def test_attention_wants_the_workspace_that_it_reports(kv, rope, page_stride):
    torch, paged = mods()
    from tests.test_paged_cpu import CACHE, F16, TABLE, desc, entries, message
    L, w, page, columns = entries(), kv + rope, 64, 1000
    pool, q = (torch.zeros(*s, dtype=torch.float16, device="cuda") for s in ((1, page, w), (2, 8, w)))
    out, table, lengths = torch.zeros(2, 8, kv, dtype=torch.float16, device="cuda"), i32(torch, [[0] * columns] * 2), i32(torch, [0, 0])
    p = pool.data_ptr()
    c = CACHE.pack(p, p, p, page_stride or page * w, w, page * rope, rope, page, 1, page, kv, rope, F16, F16) + \
        TABLE.pack(table.data_ptr(), columns, 2, columns)
    d = desc(q=q.data_ptr(), q_row=8 * w, q_head=w, lengths=lengths.data_ptr(), max_length=columns * page, out=out.data_ptr())
    need = L.mm_paged_attention_workspace(d, c)
    assert need > 0
    room = torch.zeros(need + 16, dtype=torch.uint8, device="cuda")
    for work, n in ((room.data_ptr(), need - 1), (room.data_ptr(), 0), (room.data_ptr() + 8, need)):
        assert L.mm_paged_attention(d, c, work, n, None) == 1 and "workspace" in message()
    torch.cuda.synchronize()
    assert L.mm_paged_attention(d, c, room.data_ptr(), need, None) == 0
    torch.cuda.synchronize()
    assert not out.any()


def test_beam_select_wants_the_workspace_that_it_reports():
    torch, paged = mods()
    from tests.test_paged_cpu import F32, entries, message
    L, B, K, V = entries(), 200, 4, 30000
    x, s = torch.zeros(B, K, V, device="cuda"), torch.zeros(B, K, device="cuda")
    out = [torch.zeros(B, K, dtype=torch.int32, device="cuda") for _ in range(3)]
    need = L.mm_beam_select_workspace(B, K, V, K)
    assert need > 0
    room = torch.zeros(need + 16, dtype=torch.uint8, device="cuda")
    for work, n in ((room.data_ptr(), need - 1), (room.data_ptr(), 0), (room.data_ptr() + 8, need)):
        rc = L.mm_beam_select(x.data_ptr(), K * V, V, F32, s.data_ptr(), None, 0, B, K, V, K, *(t.data_ptr() for t in out), work, n, None)
        assert rc == 1 and "workspace" in message()
    torch.cuda.synchronize()


def attention_refusals(torch, paged, d):
    pool = paged.alloc_pages(2, 4, 16, 128, 16, device=d)
    q = torch.zeros(2, 8, 144, dtype=torch.float16, device=d)
    table, ints = torch.zeros(2, 3, dtype=torch.int32, device=d), torch.zeros(2, dtype=torch.int32, device=d)
    att = lambda *a, **k: paged.attention(*a, **{"kv_rank": 128, **k})  # noqa: E731
    return [
        (lambda: att(q[0], pool[0], table, ints, 0.1), "q is"), (lambda: att(q.float(), pool[0], table, ints, 0.1), "q is"),
        (lambda: att(q.bfloat16(), pool[0], table, ints, 0.1), "type"), (lambda: att(q, pool, table, ints, 0.1), "16-bit cache"),
        (lambda: att(q, pool[0], table.long(), ints, 0.1), "table"), (lambda: att(q, pool[0], table[:1], ints, 0.1), "table row"),
        (lambda: att(q, pool[0], table, ints[:1], 0.1), "lengths"), (lambda: att(q, pool[0], table, ints.long(), 0.1), "lengths"),
        (lambda: att(q, pool[0], table, ints, None), "scale"), (lambda: att(q, pool[0], table, ints, 0.1, kv_rank=0), "kv_rank"),
        (lambda: att(q, pool[0], table, ints, 0.1, kv_rank=145), "kv_rank"), (lambda: att(q, pool[0], table, ints, 0.1, window=0), "window"),
        (lambda: att(q, pool[0], table, ints, 0.1, window=-3), "window"), (lambda: att(q, pool[0], table, ints, 0.1, sinks=-1), "sinks"),
        (lambda: att(q, pool[0], table, ints, 0.1, max_length=49), "max_length"), (lambda: att(q[..., :140], pool[0], table, ints, 0.1), "width"),
        (lambda: paged.append(pool[0], q[:, 0, :100], table, ints, kv_rank=128), "values"),
        (lambda: paged.append(pool[0], q[:, 0], table, ints[:1], kv_rank=128), "positions"),
        (lambda: paged.append(pool[0], q[:1, 0], table, ints[:1], kv_rank=128), "per table row"),
        (lambda: paged.append(pool[0], q[:, 0], table, ints, kv_rank=128, rows=ints[:1]), "rows"),
        (lambda: paged.append(pool[0], q[:, 0], table, ints, kv_rank=128, norm=torch.ones(127, device=d)), "norm"),
        (lambda: paged.append(pool[0], q[:, 0], table, ints, kv_rank=128, theta=0.0), "theta"),
        (lambda: paged.append(pool[0], q[:, 0], table, ints, kv_rank=128, theta="x"), "theta"),
        (lambda: paged.append(pool[0], q[:, 0], table, ints, kv_rank=128, norm=torch.ones(128, device=d), eps=-1.0), "eps"),
        (lambda: paged.append(pool[0], q[:, 0], table, ints, kv_rank=129), "even")]


def beam_refusals(torch, paged, d):
    pool = paged.alloc_pages(2, 4, 16, 128, 16, device=d)
    table, ints = torch.zeros(2, 3, dtype=torch.int32, device=d), torch.zeros(2, dtype=torch.int32, device=d)
    x, s = torch.zeros(2, 4, 10, device=d), torch.zeros(2, 4, device=d)
    return [
        (lambda: paged.beam_select(x[0], s), "logits"), (lambda: paged.beam_select(x, s[:, :3]), "scores"),
        (lambda: paged.beam_select(x, s.double()), "scores"), (lambda: paged.beam_select(x, s, beams=0), "beams"),
        (lambda: paged.beam_select(x, s, beams=33), "32 beams"), (lambda: paged.beam_select(x, s, finished=s > 0), "eos"),
        (lambda: paged.beam_select(x, s, finished=s, eos=1), "finished"), (lambda: paged.beam_select(x, s, finished=s > 0, eos=10), "eos"),
        (lambda: paged.beam_reorder(pool[0], table, ints, ints, ints), "layers"),
        (lambda: paged.beam_reorder(pool, table, ints[:1], ints, ints), "spare"),
        (lambda: paged.beam_reorder(pool, table, ints, ints, ints.long()), "parents"),
        (lambda: paged.beam_reorder(pool.float(), table, ints, ints, ints), "16-bit"),
        (lambda: paged.beam_reorder((pool, pool), table, ints, ints, ints), "cache is"),
        (lambda: paged.beam_reorder(pool, table[:, :0], ints, ints, ints), "no pages")]


@pytest.mark.parametrize("calls", [attention_refusals, beam_refusals])
def test_calls_refuse_what_they_can_see(calls):
    torch, paged = mods()
    from cpp_inference_train_engine_b200 import EngineError
    for call, what in calls(torch, paged, "cuda"):
        with pytest.raises(EngineError, match=what):
            call()
    torch.cuda.synchronize()
