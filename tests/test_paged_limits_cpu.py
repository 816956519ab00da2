"""What the latent and paged operators refuse without a GPU: tensors that are more than the values in their storage."""
import pytest

torch = pytest.importorskip("torch")

from cpp_inference_train_engine_b200 import EngineError, latent, paged


def calls(q, values, logits, pool):
    """A call of every operator that reads floating tensors, with these."""
    table, ints = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    return {
        "attention": lambda: paged.attention(q, pool, table, ints, 0.1, kv_rank=128),
        "append": lambda: paged.append(pool, values, table, ints, kv_rank=128),
        "beam_select": lambda: paged.beam_select(logits, torch.zeros(2, 4)),
        "verify_drafts": lambda: latent.verify_drafts(logits, ints[:, None], ints, logits[:, 0, :1], logits[:, 0, 0]),
        "shared_prefix_attention": lambda: latent.shared_prefix_attention(q[:, None], None, pool, None, None, ints, 0.1, kv_rank=128),
    }


def plain():
    return (torch.randn(2, 8, 144).half(), torch.randn(2, 144), torch.randn(2, 4, 10), torch.zeros(2, 16, 144).half())


@pytest.mark.parametrize("name", calls(*plain()))
def test_tangents_are_refused(name):
    """A dual tensor of forward-mode differentiation does not require a gradient, but carries one."""
    import torch.autograd.forward_ad as fw
    q, values, logits, pool = plain()
    with fw.dual_level():
        duals = [fw.make_dual(t, torch.ones_like(t)) for t in (q, values, logits)]
        call = calls(*duals, pool)[name]
        with torch.no_grad(), pytest.raises(EngineError, match="tangent"):  # no_grad is of backward mode alone
            call()
        with fw._set_fwd_grad_enabled(False), pytest.raises(EngineError, match="CUDA tensor"):
            call()
        with pytest.raises(EngineError, match="CUDA tensor"):
            calls(*(fw.unpack_dual(t).primal for t in duals), pool)[name]()


@pytest.mark.parametrize("name", calls(*plain()))
def test_views_that_stand_for_other_values_are_refused(name):
    """The imaginary part of a conjugate is a view whose storage has the other sign."""
    def negated(t):
        twin = torch.complex(torch.zeros_like(t, dtype=torch.float32), -t.float())
        v = (twin.to(torch.complex32) if t.dtype == torch.float16 else twin).conj().imag
        assert v.is_neg() and torch.equal(v, t)
        return v
    q, values, logits, pool = plain()
    views = [torch._neg_view(t) if t.dtype == torch.float16 else negated(t) for t in (q, values, logits)]
    with pytest.raises(EngineError, match="storage"):
        calls(*views, pool)[name]()
    with pytest.raises(EngineError, match="CUDA tensor"):
        calls(*(t.resolve_neg() for t in views), pool)[name]()


def test_the_self_test_of_waits_refuses_what_has_none():
    """The slower form of attention waits for nothing; a negative number of steps is no number of steps."""
    import ctypes

    from tests.test_paged_cpu import P, cache, desc, entries, message
    f = entries().mm_paged_selftest_wait_timeout
    f.restype, f.argtypes = ctypes.c_int, [ctypes.c_char_p, ctypes.c_char_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_void_p]
    narrow = (desc(heads=2, q_row=24, q_head=12), cache(kv=8, rope=4))
    assert f(*narrow, P, 1 << 40, 0, None) == 3 and "waits for nothing" in message()
    for steps in (-1, 2 ** 24 + 1, 2 ** 31 - 1):
        assert f(*narrow, P, 1 << 40, steps, None) == 1 and "steps" in message()
    assert f(desc(rows=-1), cache(), P, 1 << 40, 0, None) == 1 and "sizes" in message()
