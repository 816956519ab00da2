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


def run(torch, latent, q, pre, suf, starts, plen, slen, kv, scale):
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return latent.shared_prefix_attention(
        q, pre, suf, i32(starts) if pre is not None else None, i32(plen) if pre is not None else None,
        i32(slen) if suf is not None else None, scale, kv_rank=kv, return_lse=True)


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
