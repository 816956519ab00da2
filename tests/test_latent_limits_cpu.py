"""What the latent operators' entries decide on the host, without a GPU: alignment, the choice of the form,
and refusals that keep bad values from the kernels."""
import pytest

torch = pytest.importorskip("torch")

from tests.test_latent_cpu import BF16, E4M3, F16, F32, cache, desc, entries, message

P = 1 << 20  # an address that is never read: these calls are refused first


@pytest.mark.parametrize("kind", [F16, E4M3])
@pytest.mark.parametrize("offset", [2, 4, 6])
def test_results_at_any_element_address_need_no_wider_stores(offset, kind):
    """The join kernel of the tensor-core form stores 8 bytes at a time: results that do not start at a
    multiple of 8 take the any-width form, which needs no workspace."""
    d = desc(out=P + offset, prefix=cache(kind, rows=1), suffix=cache(kind))
    assert entries().mm_shared_prefix_attention_workspace(*d) == 0


@pytest.mark.parametrize("over", [dict(q=P + 1), dict(out=P + 1), dict(lse=P + 2)])
def test_attention_refuses_pointers_inside_an_element(over):
    d = desc(**over)
    assert entries().mm_shared_prefix_attention_workspace(*d) == -1 and "aligned" in message()
    assert entries().mm_shared_prefix_attention(*d, P, 1 << 30, None) == 1 and "aligned" in message()


def test_caches_refuse_pointers_inside_an_element():
    import struct
    L = entries()
    for field, off in ((0, 1), (8, 1), (16, 2)):  # latent, rope, scale
        for kind in (F16, E4M3):
            raw = bytearray(cache(kind))
            struct.pack_into("=Q", raw, field, P + off)
            d = desc(suffix=bytes(raw))
            if (kind == F16) == (field == 0):  # codes are bytes; a 16-bit cache has nothing else
                assert L.mm_shared_prefix_attention_workspace(*d) == -1 and "aligned" in message()
            if kind == E4M3 and field > 0:
                assert L.mm_latent_cache_write(bytes(raw), P, 128, P, 16, F32, P, 1, None) == 1 and "aligned" in message()
                assert L.mm_latent_cache_read(bytes(raw), P, 1, P, 144, F32, None) == 1 and "aligned" in message()


@pytest.mark.parametrize("dtype,off", [(F32, 2), (F16, 1), (BF16, 1)])
def test_inputs_inside_an_element_are_refused(dtype, off):
    L, c = entries(), cache(E4M3)
    assert L.mm_latent_cache_write(c, P + off, 128, P, 16, dtype, P, 1, None) == 1 and "aligned" in message()
    assert L.mm_latent_cache_write(c, P, 128, P + off, 16, dtype, P, 1, None) == 1 and "aligned" in message()
    assert L.mm_latent_cache_read(c, P, 1, P + off, 144, dtype, None) == 1 and "aligned" in message()
    assert L.mm_verify_drafts(P + off, None, dtype, P, P, P, P, 1, 1, 8, P, P, None) == 1 and "aligned" in message()
    assert L.mm_verify_drafts(P, P + off, dtype, P, P, P, P, 1, 1, 8, P, P, None) == 1 and "aligned" in message()


@pytest.mark.parametrize("prompts", [[[1, 264]], [[1], [-1, 3]], [[1, 2 ** 40]]])
def test_group_decoder_refuses_tokens_outside_the_vocabulary(prompts):
    import numpy as np

    from cpp_inference_train_engine_b200 import TINY, EngineError
    from cpp_inference_train_engine_b200.group_decode import GroupDecoder
    with pytest.raises(EngineError, match="vocabulary"):
        GroupDecoder(TINY, np.zeros(TINY.parameter_count(), np.float32), prompts, 1, 4, device="cpu")


@pytest.mark.parametrize("by", [-1, 1])
def test_group_decoder_refuses_parameters_of_another_model(by):
    import numpy as np

    from cpp_inference_train_engine_b200 import TINY, EngineError
    from cpp_inference_train_engine_b200.group_decode import GroupDecoder
    with pytest.raises(EngineError, match="parameters"):
        GroupDecoder(TINY, np.zeros(TINY.parameter_count() + by, np.float32), [[1]], 1, 4, device="cpu")


def test_status_of_the_waits_is_reported():
    """mm_latent_status tells the host of waits that ran out; without a device it fails loudly."""
    import cpp_inference_train_engine_b200 as E
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert E.lib().mm_latent_status(None) == 5 and "status" in message()


@pytest.mark.parametrize("field,value", [(3, 2 ** 39), (3, -2304), (4, 0), (4, -144), (4, 2 ** 39)])
def test_strides_that_no_tensor_map_takes_use_the_other_form(field, value):
    """Row strides (field 3) and position strides (field 4) of 16-bit caches outside a tensor map's range."""
    import struct
    raw = bytearray(cache())
    struct.pack_into("=q", raw, 8 * field, value)
    assert entries().mm_shared_prefix_attention_workspace(*desc(suffix=bytes(raw))) == 0


def test_tensors_that_require_a_gradient_are_refused():
    """No gradient flows through the operators; without recording, or detached, the tensors are taken (and
    refused here for not being on a GPU)."""
    from cpp_inference_train_engine_b200 import EngineError, latent
    q = torch.zeros(1, 1, 8, 144, dtype=torch.float16, requires_grad=True)
    p = torch.ones(1, 2, 8, requires_grad=True)
    ints, one = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1)
    calls = [lambda: latent.shared_prefix_attention(q, None, None, None, None, None, 0.1, kv_rank=128),
             lambda: latent.cache_write(None, q[0, 0, :, :128], q[0, 0, :, 128:], torch.zeros(8, dtype=torch.int64)),
             lambda: latent.verify_drafts(p, ints, ints[0], one[None], one)]
    for call in calls:
        with pytest.raises(EngineError, match="gradient"):
            call()
        with torch.no_grad(), pytest.raises(EngineError, match="CUDA tensor"):
            call()
