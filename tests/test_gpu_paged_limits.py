"""Paged-cache operators at the limits of what their documentation allows."""
import pytest

from tests.gpu_util import require_gpu

pytestmark = pytest.mark.gpu


def mods():
    require_gpu()
    import torch

    from cpp_inference_train_engine_b200 import paged
    return torch, paged


def i32(torch, v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("kv, rope", [(1024, 64), (1024, 256), (1000, 200), (1, 1)])
@pytest.mark.parametrize("bits", [8, 16])
def test_reorder_of_every_width_that_is_appended(kv, rope, bits):
    """Positions of up to 1,024 + 256 values are stored, and move when their row's parent changes."""
    torch, paged = mods()
    g = torch.Generator(device="cuda").manual_seed(kv + rope)
    cache = paged.alloc_pages(2, 8, 4, kv, rope & ~1, torch.bfloat16, bits)
    rope &= ~1
    table, spare, lengths = i32(torch, [[0, 1], [2, 3]]), i32(torch, [4, 5]), i32(torch, [6, 6])
    for l in range(2):
        for t in range(6):
            paged.append(paged.layer(cache, l), torch.randn(2, kv + rope, generator=g, device="cuda"), table, i32(torch, [t, t]), kv_rank=kv)
    held = [x[:, 3, :2].clone() for x in (cache if bits == 8 else (cache,))]  # row 1's positions 4 and 5
    table, spare, lengths = paged.beam_reorder(cache, table, spare, lengths, i32(torch, [1, 1]))
    assert table.tolist() == [[2, 4], [2, 3]] and spare.tolist() == [1, 5] and lengths.tolist() == [6, 6]
    for x, want in zip(cache if bits == 8 else (cache,), held):
        assert want.float().any() or want.numel() == 0
        assert torch.equal(x[:, 4, :2].float(), want.float())


def marks(torch, cache, table, held, page):
    """Of every row the numbers that stand at its positions (0 where it has no page)."""
    stored, pages = cache[0].float().cpu(), table.cpu()
    at = lambda r, t: int(pages[r, t // page])  # noqa: E731
    return [[int(stored[at(r, t), t % page, 0] * 128 + stored[at(r, t), t % page, 1]) if at(r, t) >= 0 else 0 for t in range(len(h))]
            for r, h in enumerate(held)]


def store(torch, paged, cache, table, positions, numbers):
    values = torch.zeros(len(positions), 8, device="cuda")
    for r, m in enumerate(numbers):
        values[r, 0], values[r, 1] = m // 128, m % 128  # (bf16 holds both)
    paged.append(cache[0], values, table, i32(torch, positions), kv_rank=8)


def test_a_row_that_takes_over_a_shorter_one_leaves_the_others_alone():
    """Rows 0 and 1 share five pages of four positions; row 0 takes over row 2, which is half as long, and grows on: what it
    has no page for is not stored, and nothing changes under row 1. With pages of its own there it stores again."""
    torch, paged = mods()
    page = 4
    for refill in (False, True):
        cache = paged.alloc_pages(1, 80, page, 8, 0, torch.bfloat16)
        table = i32(torch, [[0, 1, 2, 3, 4, 10, 11, 12], [0, 1, 2, 3, 4, 20, 21, 22], [30, 31, 32, 33, 34, 35, 36, 37]])
        spare, lengths = i32(torch, [50, 51, 52]), i32(torch, [22, 22, 11])
        held = [list(range(1, 23)), list(range(1, 21)) + [201, 202], list(range(301, 312))]
        for t in range(22):
            store(torch, paged, cache, table, [t, t if t > 19 else -1, t if t < 11 else -1], [h[t] if t < len(h) else 0 for h in held])
        table, spare, lengths = paged.beam_reorder(cache, table, spare, lengths, i32(torch, [2, 1, 2]))
        held[0] = held[2][:]
        assert table[0, :5].tolist() == [30, 31, 50, -1, -1] and table[1:].tolist() == [[0, 1, 2, 3, 4, 20, 21, 22], list(range(30, 38))]
        free = iter((70, 71, 72, 73, 74))
        for step in range(20):
            n = len(held[0])
            if table[0, n // page] < 0 and refill:
                table[0, n // page] = next(free)
            there = int(table[0, n // page]) >= 0
            store(torch, paged, cache, table, [n, -1, -1], [1000 + step, 0, 0])
            held[0] = held[0] + [1000 + step if there else 0]
            assert there or not refill
            lengths = i32(torch, [len(h) for h in held])
            table, spare, lengths = paged.beam_reorder(cache, table, spare, lengths, i32(torch, [0, 1, 2]))
            assert marks(torch, cache, table, held, page) == held, step


@pytest.mark.parametrize("page", [1, 2, 4, 16])
@pytest.mark.parametrize("seed", range(4))
def test_rows_that_grow_at_different_paces_never_write_into_each_others_pages(page, seed):
    """Rows grow or not, and take over any other row, longer or shorter, for many steps. What a row stored under a page
    stays for all that descend from it, and the page that a row writes next and its spare one are no other row's. A position
    is lost only where the table has no page for it, or the row lacks the pages to take over its parent's tail."""
    import random
    torch, paged = mods()
    rng = random.Random(seed)
    rows, most = 6, 64
    columns = most // page
    own = list(range(rows * (columns + 1)))
    rng.shuffle(own)
    cache = paged.alloc_pages(1, len(own), page, 8, 0, torch.bfloat16)
    table, spare = i32(torch, own[:rows * columns]).view(rows, columns), i32(torch, own[rows * columns:])
    held, mark, kept = [[] for _ in range(rows)], 0, 0
    for _ in range(100):
        positions, numbers, pages = [], [], table.cpu()
        for r in range(rows):
            grows = len(held[r]) < most and rng.random() < 0.75
            positions.append(len(held[r]) if grows else -1)
            mark += 1
            numbers.append(mark)
            if grows:
                held[r] = held[r] + [mark if pages[r, len(held[r]) // page] >= 0 else 0]
        store(torch, paged, cache, table, positions, numbers)
        parents = [rng.choice([r, r, r, rng.randrange(rows)]) for r in range(rows)]
        before, aside = table.cpu(), spare.cpu()
        table, spare, lengths = paged.beam_reorder(cache, table, spare, i32(torch, [len(h) for h in held]), i32(torch, parents))
        held = [list(held[p]) for p in parents]
        for r, p in enumerate(parents):
            n, full = len(held[r]), len(held[r]) // page
            if p != r and n % page and (before[p, full] < 0 or aside[r] < 0):
                held[r][full * page:] = [0] * (n % page)  # (a parent's tail without a page, or no page to copy it into)
        got = marks(torch, cache, table, held, page)
        assert all(h in (0, m) for row, want in zip(got, held) for m, h in zip(row, want)) and lengths.tolist() == [len(h) for h in held]
        kept += sum(m > 0 for h in held for m in h)
        pages = table.cpu()
        mine = [int(pages[r, len(h) // page]) for r, h in enumerate(held) if len(h) < most] + spare.tolist()
        mine = [p for p in mine if p >= 0]
        used = {int(pages[r, j]) for r, h in enumerate(held) for j in range(len(h) // page)}
        assert len(set(mine)) == len(mine) and not used & set(mine)
    assert kept > 1000


# rows, heads, latent width, rope width, longest row, 8-bit pages, steps until the loads end: whole rows a CTA, several in turn;
# few rows that many CTAs share; more rows than CTAs; heads of two blocks; a row that no CTA has for itself
GIVE_UP = [(700, 8, 128, 16, 197, False, 1), (700, 8, 128, 16, 197, False, 0), (5, 16, 512, 32, 4000, False, 2), (400, 16, 512, 32, 700, False, 4),
           (90, 19, 128, 16, 2500, True, 2), (300, 16, 512, 32, 900, True, 9), (1, 16, 512, 32, 30000, True, 0)]


@pytest.mark.parametrize("case", GIVE_UP, ids=str)
def test_a_wait_that_runs_out_makes_its_rows_nan_and_is_reported(case):
    """The loads of every other CTA end early, so that the waits for them run out. A row that one of these CTAs has a part of
    is NaN, every other one is as ever, and none is what the memory held before; the host is told once, and the next
    call is as ever. (The workspace holds zeros: a cut that the join were not told of would leave the outputs' mark.)"""
    import ctypes
    torch, paged = mods()
    import cpp_inference_train_engine_b200 as E
    from cpp_inference_train_engine_b200 import EngineError
    from tests.test_latent_cpu import E4M3, F16
    from tests.test_paged_cpu import cache as describe, desc, entries
    rows, heads, kv, rope, longest, fp8, steps = case
    g = torch.Generator(device="cuda").manual_seed(rows)
    page, columns = 32, -(-longest // 32)
    pools = paged.layer(paged.alloc_pages(1, 600, page, kv, rope, torch.float16, 8 if fp8 else 16), 0)
    for t in pools if fp8 else (pools,):
        t.copy_(torch.randn(t.shape, generator=g, device="cuda").abs() + 0.5 if t.dim() == 2 else torch.randn(t.shape, generator=g, device="cuda"))
    table = torch.randint(0, 600, (rows, columns), generator=g, device="cuda", dtype=torch.int32)
    lengths = torch.randint(1, longest + 1, (rows,), generator=g, device="cuda", dtype=torch.int32)
    lengths[-1] = longest
    if rows > 2:
        lengths[1] = 0
    q = torch.randn(rows, heads, kv + rope, generator=g, device="cuda").half()
    want, want_lse = paged.attention(q, pools, table, lengths, 0.05, kv_rank=kv, return_lse=True)
    out, lse = torch.full_like(want, 777.0), torch.full_like(want_lse, 777.0)
    latent, rk, scale = (t.data_ptr() for t in pools) if fp8 else (pools.data_ptr(), 0, 0)
    c = describe(kind=E4M3 if fp8 else F16, pages=600, page=page, kv=kv, rope=rope, table=table.data_ptr(), rows=rows, columns=columns,
                 latent=latent, rk=rk, scale=scale)
    d = desc(q=q.data_ptr(), q_row=heads * (kv + rope), q_head=kv + rope, lengths=lengths.data_ptr(), rows=rows, heads=heads,
             max_length=columns * page, scale=0.05, out=out.data_ptr(), lse=lse.data_ptr())
    L = entries()
    f = L.mm_paged_selftest_wait_timeout
    f.restype, f.argtypes = ctypes.c_int, [ctypes.c_char_p, ctypes.c_char_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_void_p]
    n = L.mm_paged_attention_workspace(d, c)
    work = torch.zeros(max(n, 16), dtype=torch.uint8, device="cuda")
    paged.check_status()
    assert f(d, c, work.data_ptr(), n, steps, torch.cuda.current_stream().cuda_stream) == 0
    with pytest.raises(EngineError, match="gave up"):
        paged.check_status()
    paged.check_status()
    lost = torch.isnan(lse)
    assert torch.equal(torch.isnan(out), lost[..., None].expand_as(out))
    assert torch.equal(torch.where(lost[..., None], 0, out), torch.where(lost[..., None], 0, want))
    assert torch.equal(torch.where(lost, 0, lse), torch.where(lost, 0, want_lse))
    assert lost.any() and (rows < 100 or not lost.all())
    again = paged.attention(q, pools, table, lengths, 0.05, kv_rank=kv, return_lse=True)
    assert torch.equal(again[0], want) and torch.equal(again[1], want_lse)
    assert f(d, c, work.data_ptr(), n, -1, None) == 1 and E.lib() is not None


@pytest.mark.parametrize("kv, rope", [(128, 16), (512, 32), (40, 8)])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_codes_are_those_of_the_quotients(kv, rope, dtype):
    """Latents that are a scale times the middle of two e4m3 codes: the quotient is that middle and goes to the even code,
    where a product with the scale's reciprocal may come out on either side of it. The codes are the same in pools that
    take 16 bytes at a time and in those that do not."""
    torch, paged = mods()
    g = torch.Generator(device="cuda").manual_seed(kv)
    n, bits = 600, {"float32": 18, "float16": 6, "bfloat16": 3}[dtype]  # (of a scale: its products with a middle's 5 bits are exact)
    scales = (torch.randint(0, 2 ** (bits - 2), (n,), generator=g, device="cuda") * 2 + 2 ** (bits - 1) + 1).float() * 2.0 ** -(bits - 1)
    middles = (2 * torch.randint(8, 16, (n, kv), generator=g, device="cuda") + 1).float() / 16
    size = torch.randint(-6, 8, (n, kv), generator=g, device="cuda").float()
    sign = torch.randint(0, 2, (n, kv), generator=g, device="cuda").float() * 2 - 1
    lat = middles * 2.0 ** size * sign * scales[:, None]
    lat[:, 5] = 448 * scales
    values = torch.cat([lat, torch.randn(n, rope, generator=g, device="cuda")], 1).to(getattr(torch, dtype))
    assert torch.equal(values[:, :kv].float(), lat)
    by_quotient = (lat / scales[:, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    by_product = (lat * (1 / scales)[:, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    assert dtype != "float32" or (by_quotient != by_product).sum() > 100  # (the inputs tell the two apart)
    table = torch.arange(n, dtype=torch.int32, device="cuda")[:, None]
    positions = torch.arange(n, dtype=torch.int32, device="cuda") % 16
    for aligned in (True, False):
        pools = paged.layer(paged.alloc_pages(1, n, 16, kv, rope, bits=8), 0)
        if not aligned:  # rows of an odd stride
            wide = torch.zeros(n, 16, kv + 1, dtype=torch.uint8, device="cuda")[..., 1:].view(torch.float8_e4m3fn)
            pools = pools._replace(latent=wide)
        paged.append(pools, values, table, positions, kv_rank=kv)
        at = torch.arange(n, device="cuda"), positions.long()
        assert torch.equal(pools.scale[at], scales)
        assert torch.equal(pools.latent.view(torch.uint8)[at], by_quotient), aligned


def test_normalised_codes_where_the_weights_are_zero():
    """Tiny latents without eps have a large reciprocal norm: what the weights make zero stays zero."""
    torch, paged = mods()
    for kv, rope in ((128, 16), (512, 32), (40, 8)):
        pools = paged.layer(paged.alloc_pages(1, 2, 16, kv, rope, bits=8), 0)
        pools.latent.view(torch.uint8).fill_(0x7F)
        norm = torch.zeros(kv, device="cuda")
        paged.append(pools, torch.full((1, kv + rope), 1e-12, device="cuda"), i32(torch, [[1]]), i32(torch, [3]), kv_rank=kv, norm=norm, eps=0.0)
        assert not pools.latent[1, 3].float().any() and float(pools.scale[1, 3]) == 2.0 ** -100


def test_a_flag_without_a_truth_value_is_refused():
    torch, paged = mods()
    from cpp_inference_train_engine_b200 import EngineError, latent
    pool = torch.zeros(2, 16, 144, dtype=torch.float16, device="cuda")
    q, table, ints = torch.zeros(2, 8, 144, dtype=torch.float16, device="cuda"), i32(torch, [[0], [1]]), i32(torch, [3, 4])
    for call in (lambda flag: paged.attention(q, pool, table, ints, 0.1, kv_rank=128, return_lse=flag),
                 lambda flag: latent.shared_prefix_attention(q[:, None], None, pool, None, None, ints, 0.1, kv_rank=128, return_lse=flag)):
        with pytest.raises(EngineError, match="return_lse"):
            call(torch.zeros(2))
        assert len(call(1)) == 2 and torch.is_tensor(call(0))
