"""The latent operators' C entries refuse what they can see on the host, without a GPU."""
import ctypes
import struct

import pytest

torch = pytest.importorskip("torch")

import cpp_inference_train_engine_b200 as E
from cpp_inference_train_engine_b200 import latent

F32, F16, BF16, E4M3 = range(4)
# mm_latent_cache and mm_shared_prefix_desc, field by field
CACHE = struct.Struct("=3Q5q6i")
DESC = struct.Struct("=Q3q4i3Q4ifi2Q")


def entries():
    L = E.lib()
    vp, i64, i32, text = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_char_p
    for name, res, args in (
            ("mm_latent_last_error", ctypes.c_size_t, [text, ctypes.c_size_t]),
            ("mm_latent_cache_write", i32, [text, vp, i64, vp, i64, i32, vp, i64, vp]),
            ("mm_latent_cache_read", i32, [text, vp, i64, vp, i64, i32, vp]),
            ("mm_shared_prefix_attention_workspace", i64, [text, text, text]),
            ("mm_shared_prefix_attention", i32, [text, text, text, vp, ctypes.c_size_t, vp]),
            ("mm_verify_drafts", i32, [vp, vp, i32, vp, vp, vp, vp, i32, i32, i32, vp, vp, vp])):
        f = getattr(L, name)
        f.restype, f.argtypes = res, args
    return L


def message():
    buf = ctypes.create_string_buffer(256)
    entries().mm_latent_last_error(buf, 256)
    return buf.value.decode()


def cache(kind=F16, rows=2, positions=16, kv=128, rope=16, rope_kind=F16):
    p = 1 << 20  # never read: these calls are refused first
    return CACHE.pack(p, p, p, positions * (kv + rope), kv + rope, positions * rope, rope, positions, rows,
                              positions, kv, rope, kind, rope_kind)


def desc(**over):
    d = dict(q=1 << 20, q_row_stride=8 * 144, q_token_stride=8 * 144, q_head_stride=144, dtype=F16, rows=2,
             tokens=1, heads=8, group_start=1 << 20, prefix_len=1 << 20, suffix_len=1 << 20, groups=1, max_group=2,
             max_prefix=16, max_suffix=16, scale=0.1, reserved=0, out=1 << 20, lse=0)
    pre, suf = over.pop("prefix", cache(rows=1)), over.pop("suffix", cache())
    d.update({k: v or 0 for k, v in over.items()})
    return DESC.pack(*d.values()), pre, suf


@pytest.mark.parametrize("over, what", [
    (dict(rows=-1), "sizes"), (dict(tokens=0), "sizes"), (dict(heads=0), "sizes"), (dict(groups=-1), "sizes"),
    (dict(dtype=F32), "fp16 or bf16"), (dict(prefix=None, suffix=None), "is needed"),
    (dict(prefix=cache(kind=BF16)), "type"), (dict(prefix=cache(E4M3, rope_kind=BF16)), "type"),
    (dict(prefix=cache(kv=64)), "widths"), (dict(groups=3), "per group"), (dict(suffix=cache(rows=1)), "per row"),
    (dict(max_prefix=17), "exceed"), (dict(max_suffix=17), "exceed"), (dict(max_prefix=-1), "exceed"),
    (dict(q=None), "null q"), (dict(out=None), "null q"), (dict(group_start=None), "group_start"),
    (dict(suffix_len=None), "suffix_len"), (dict(prefix=cache(kv=2000)), "kv must be"), (dict(suffix=cache(kind=7)), "kind"),
    (dict(tokens=2 ** 20, heads=2 ** 12), "too many"),
])
def test_attention_refusals(over, what):
    d = desc(**over)
    assert entries().mm_shared_prefix_attention_workspace(*d) == -1
    assert what in message()
    assert entries().mm_shared_prefix_attention(*d, None, 0, None) == 1
    assert what in message()


def test_null_arguments_are_refused():
    L = entries()
    assert L.mm_shared_prefix_attention(None, None, None, None, 0, None) == 1
    assert L.mm_latent_cache_write(None, None, 0, None, 0, 0, None, 1, None) == 1
    assert L.mm_latent_cache_read(None, None, 1, None, 0, 0, None) == 1
    c = cache(E4M3)
    assert L.mm_latent_cache_write(c, None, 0, None, 0, 0, None, 1, None) == 1 and "null" in message()
    assert L.mm_latent_cache_write(c, None, 0, None, 0, 0, None, -1, None) == 1
    assert L.mm_latent_cache_write(c, None, 0, None, 0, 0, None, 0, None) == 0  # nothing to do
    f16 = cache()
    assert L.mm_latent_cache_read(f16, 1 << 20, 1, 1 << 20, 144, 1, None) == 1 and "e4m3" in message()
    assert L.mm_verify_drafts(None, None, 0, None, None, None, None, 1, 1, 8, None, None, None) == 1
    assert L.mm_verify_drafts(None, None, 0, None, None, None, None, 1, 1, 0, None, None, None) == 1
    assert L.mm_verify_drafts(None, None, 0, None, None, None, None, 1, 1, 2 ** 19, None, None, None) == 3
    assert L.mm_verify_drafts(None, None, 0, None, None, None, None, 0, 1, 8, None, None, None) == 0


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 1, 8, 144, dtype=torch.float16)
    with pytest.raises(E.EngineError, match="CUDA tensor"):
        latent.shared_prefix_attention(q, None, None, None, None, None, 0.1, kv_rank=128)


@pytest.mark.parametrize("kwargs,message", [
    (dict(cache_bits=4), "cache_bits"), (dict(drafts=-1), "drafts"), (dict(new_tokens=0), "new_tokens"),
    (dict(new_tokens=64), "context"), (dict(prompts=[]), "prompts"), (dict(prompts=[[1], []]), "prompts"),
    (dict(rows=[1, 2]), "rows"), (dict(rows=0), "rows"),
])
def test_group_decoder_refuses_bad_arguments(kwargs, message):
    import numpy as np

    from cpp_inference_train_engine_b200 import TINY, EngineError
    from cpp_inference_train_engine_b200.group_decode import GroupDecoder
    args = dict(prompts=[[1, 2]], rows=1, new_tokens=4, drafts=0)
    args.update(kwargs)
    with pytest.raises(EngineError, match=message):
        GroupDecoder(TINY, np.zeros(1, np.float32), **args)
