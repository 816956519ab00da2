"""The paged operators' C entries and calls refuse what they can see on the host, without a GPU."""
import ctypes
import struct

import pytest

torch = pytest.importorskip("torch")

import cpp_inference_train_engine_b200 as E
from cpp_inference_train_engine_b200 import EngineError, paged
from tests.test_latent_cpu import BF16, CACHE, E4M3, F16, F32, message

P = 1 << 20  # an address that is never read: these calls are refused first
# what mm_paged_cache has behind its pool, and mm_paged_attention_desc
TABLE = struct.Struct("=Qq2i")
DESC = struct.Struct("=Q2qQ6ifi2Q")


def entries():
    L = E.lib()
    vp, i64, i32, f32, text = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_char_p
    for name, res, args in (
            ("mm_paged_append", i32, [text, vp, i64, i32, vp, vp, i64, ctypes.c_double, vp, f32, vp]),
            ("mm_paged_attention_workspace", i64, [text, text]),
            ("mm_paged_attention", i32, [text, text, vp, ctypes.c_size_t, vp]),
            ("mm_beam_select_workspace", i64, [i32] * 4),
            ("mm_beam_select", i32, [vp, i64, i64, i32, vp, vp] + [i32] * 5 + [vp] * 4 + [ctypes.c_size_t, vp]),
            ("mm_beam_reorder", i32, [text, i32, ctypes.POINTER(i64)] + [vp] * 7)):
        f = getattr(L, name)
        f.restype, f.argtypes = res, args
    return L


def cache(kind=F16, pages=4, page=16, kv=128, rope=16, rope_kind=F16, table=P, rows=2, columns=3, latent=P, rk=P, scale=P):
    w = kv + (rope if kind != E4M3 else 0)
    return CACHE.pack(latent, rk, scale, page * w, w, page * rope, rope, page, pages, page, kv, rope, kind, rope_kind) + \
        TABLE.pack(table, columns, rows, columns)


def desc(**over):
    d = dict(q=P, q_row=8 * 144, q_head=144, lengths=P, dtype=F16, rows=2, heads=8, max_length=48, window=0, sinks=0, scale=0.1,
             reserved=0, out=P, lse=0)
    d.update(over)
    return DESC.pack(*d.values())


@pytest.mark.parametrize("over, what", [
    (dict(rows=-1), "sizes"), (dict(heads=0), "sizes"), (dict(heads=2 ** 30, rows=3), "sizes"), (dict(dtype=F32), "fp16 or bf16"),
    (dict(dtype=BF16), "type"), (dict(rows=3), "table row"), (dict(window=-1), "window"), (dict(sinks=-1), "window"),
    (dict(max_length=49), "exceeds"), (dict(max_length=-1), "exceeds"), (dict(q=0), "null"), (dict(out=0), "null"),
    (dict(lengths=0), "null"), (dict(q=P + 1), "aligned"), (dict(out=P + 1), "aligned"), (dict(lse=P + 2), "aligned"),
    (dict(lengths=P + 1), "aligned")])
def test_attention_refuses(over, what):
    L = entries()
    assert L.mm_paged_attention_workspace(desc(**over), cache()) == -1 and what in message()
    assert L.mm_paged_attention(desc(**over), cache(), P, 1 << 40, None) == 1 and what in message()


BAD_CACHES = [
    (dict(pages=-1), "negative"), (dict(page=0), "page"), (dict(kv=0), "kv"), (dict(kv=1025), "kv"), (dict(rope=257), "kv"),
    (dict(kind=F32), "kind"), (dict(kind=E4M3, rope_kind=F32), "rope"), (dict(latent=0), "null"), (dict(latent=P + 1), "aligned"),
    (dict(kind=E4M3, scale=0), "null"), (dict(kind=E4M3, scale=P + 2), "aligned"), (dict(rows=-1), "negative"),
    (dict(columns=-1), "negative"), (dict(table=0), "table"), (dict(table=P + 2), "table"), (dict(columns=2 ** 27), "32 bits")]


@pytest.mark.parametrize("over, what", BAD_CACHES)
def test_every_entry_refuses_bad_caches(over, what):
    L, c, strides = entries(), cache(**over), (ctypes.c_int64 * 3)()
    assert L.mm_paged_attention_workspace(desc(), c) == -1 and what in message()
    assert L.mm_paged_append(c, P, 144, F32, P, P, 1, 1e4, None, 0.0, None) == 1 and what in message()
    assert L.mm_beam_reorder(c, 1, strides, P, P, P, P, P, P, None) == 1 and what in message()


@pytest.mark.parametrize("at, value, code, what", [
    (1, 0, 1, "null"), (1, P + 2, 1, "aligned"), (3, 7, 1, "type"), (4, P + 1, 1, "aligned"), (5, 0, 1, "null"), (5, P + 2, 1, "aligned"),
    (6, -1, 1, "count"), (7, 0.0, 1, "theta"), (7, float("nan"), 1, "theta"), (7, float("inf"), 1, "theta"), (8, P + 2, 1, "aligned"),
    (9, -1.0, 1, "eps")])
def test_append_refuses(at, value, code, what):
    args = [cache(), P, 144, F32, P, P, 1, 1e4, P, 1e-5, None]
    args[at] = value
    assert entries().mm_paged_append(*args) == code and what in message()


def test_append_refuses_an_odd_rope():
    assert entries().mm_paged_append(cache(rope=15), P, 143, F32, P, P, 1, 1e4, None, 0.0, None) == 1 and "even" in message()


@pytest.mark.parametrize("at, value, code, what", [
    (0, 0, 1, "null"), (0, P + 2, 1, "aligned"), (3, 9, 1, "type"), (4, 0, 1, "null"), (4, P + 1, 1, "aligned"), (6, -1, 1, "eos"),
    (6, 100, 1, "eos"), (7, -1, 1, "sizes"), (8, 0, 1, "sizes"), (8, 33, 3, "32 beams"), (9, 0, 1, "sizes"), (9, 2 ** 20 + 1, 3, "1,048,576"),
    (10, 0, 1, "sizes"), (10, 33, 3, "32 beams"), (11, 0, 1, "null"), (12, P + 2, 1, "aligned"), (13, 0, 1, "null")])
def test_beam_select_refuses(at, value, code, what):
    args = [P, 400, 100, F32, P, P, 5, 2, 4, 100, 4, P, P, P, P, 1 << 40, None]
    args[at] = value
    L = entries()
    assert L.mm_beam_select(*args) == code and what in message()
    if what in ("sizes", "32 beams", "1,048,576"):
        assert L.mm_beam_select_workspace(*args[7:11]) == -code


@pytest.mark.parametrize("at, value, what", [(1, -1, "layers"), (2, None, "layers")] + [(i, 0, "null") for i in range(3, 9)] +
                         [(i, P + 2, "aligned") for i in range(3, 9)])
def test_beam_reorder_refuses(at, value, what):
    args = [cache(), 2, (ctypes.c_int64 * 3)(0, 0, 0), P, P, P, P, P, P, None]
    args[at] = value
    assert entries().mm_beam_reorder(*args) == 1 and what in message()
    assert entries().mm_beam_reorder(cache(columns=0), *args[1:3], P, P, P, P, P, P, None) == 1


def test_calls_of_nothing_return():
    """Sizes of zero launch nothing, whatever the pointers."""
    L, strides = entries(), (ctypes.c_int64 * 3)()
    assert L.mm_paged_append(cache(), None, 144, F32, None, None, 0, 1e4, None, 0.0, None) == 0
    assert L.mm_paged_attention(desc(rows=0, q=0, out=0, lengths=0), cache(), None, 0, None) == 0
    assert L.mm_beam_select(None, 0, 0, F32, None, None, 0, 0, 4, 100, 4, None, None, None, None, 0, None) == 0
    assert L.mm_beam_reorder(cache(rows=0, table=0), 1, strides, None, None, None, None, None, None, None) == 0


def test_status_is_reported():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert E.lib().mm_paged_status(None) == 5 and "status" in message()


def test_tensors_that_require_a_gradient_or_are_not_on_a_gpu_are_refused():
    q = torch.zeros(2, 8, 144, dtype=torch.float16, requires_grad=True)
    x = torch.zeros(2, 4, 10, requires_grad=True)
    table, ints = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    pool = torch.zeros(4, 16, 144, dtype=torch.float16)
    for call in (lambda: paged.attention(q, pool, table, ints, 0.1, kv_rank=128),
                 lambda: paged.append(pool, q[:, 0], table, ints, kv_rank=128),
                 lambda: paged.beam_select(x, x[..., 0])):
        with pytest.raises(EngineError, match="gradient"):
            call()
        with torch.no_grad(), pytest.raises(EngineError, match="CUDA tensor"):
            call()
    with pytest.raises(EngineError, match="CUDA tensor"):
        paged.beam_reorder(pool[None], table, ints, ints, ints)


def test_alloc_pages():
    c = paged.alloc_pages(2, 3, 16, 128, 16, torch.bfloat16, device="cpu")
    assert c.shape == (2, 3, 16, 144) and c.dtype == torch.bfloat16 and paged.layer(c, 1).data_ptr() == c[1].data_ptr()
    c = paged.alloc_pages(2, 3, 16, 128, 16, bits=8, device="cpu")
    assert [t.shape for t in paged.layer(c, 1)] == [(3, 16, 128), (3, 16, 16), (3, 16)] and c.latent.dtype == torch.float8_e4m3fn
    for kw in (dict(dtype=torch.float32), dict(bits=4)):
        with pytest.raises(EngineError):
            paged.alloc_pages(1, 1, 16, 128, 16, device="cpu", **kw)


@pytest.mark.parametrize("over, what", [
    (dict(cache_bits=4), "cache_bits"), (dict(new=0), "new_tokens"), (dict(prompts=[]), "new_tokens"), (dict(prompts=[[1], []]), "new_tokens"),
    (dict(beams=0), "beams"), (dict(beams=33), "beams"), (dict(page_size=0), "positive"), (dict(window=0), "positive"),
    (dict(sinks=-1), "negative"), (dict(new=64), "exceeds context"), (dict(prompts=[[1, 264]]), "vocabulary"), (dict(prompts=[[-1]]), "vocabulary"),
    (dict(extra=1), "parameters")])
def test_beam_decoder_refuses(over, what):
    import numpy as np

    from cpp_inference_train_engine_b200 import TINY
    from cpp_inference_train_engine_b200.beam_decode import BeamDecoder
    d = dict(prompts=[[1, 2]], beams=2, new=4, page_size=4, cache_bits=16, window=None, sinks=0, extra=0)
    d.update(over)
    with pytest.raises(EngineError, match=what):
        BeamDecoder(TINY, np.zeros(TINY.parameter_count() + d["extra"], np.float32), d["prompts"], d["beams"], d["new"], d["page_size"],
                    d["cache_bits"], d["window"], d["sinks"], device="cpu")
