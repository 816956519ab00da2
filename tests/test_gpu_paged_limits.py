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
