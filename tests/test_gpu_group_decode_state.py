"""What a GroupDecoder keeps between calls and how it fails; long prompts and the scaled model's widths."""
import numpy as np
import pytest

import cpp_inference_train_engine_b200 as E
from cpp_inference_train_engine_b200.config import MLA36M, TINY, ModelConfig
from tests.gpu_util import require_gpu
from tests.test_gpu_group_decode import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("drafts", [0, 3])
@pytest.mark.parametrize("bits", [8, 16])
def test_a_second_generation_starts_from_the_prompts(drafts, bits):
    d = make("tiny", bits, drafts=drafts)[3]
    for temperature in (0.0, 1.0):
        first = d.generate(temperature, 5)
        assert d.generate(temperature, 5) == first
        assert make("tiny", bits, drafts=drafts)[3].generate(temperature, 5) == first


def test_logits_without_a_token_are_an_error():
    import torch
    for where in ("prompt", "step"):
        d = make("tiny", 8)[3]
        if where == "prompt":
            d.prompt_logits[1] = float("nan")
        else:
            d.final_norm = torch.full_like(d.final_norm, float("nan"))
        for temperature in (1.0,):
            with pytest.raises(E.EngineError, match="no token") as e:
                d.generate(temperature)
            assert e.value.name == "numerical_error"


@pytest.mark.parametrize("where", ["prompt", "step"])
def test_greedy_logits_with_a_nan_are_an_error(where):
    import torch
    d = make("tiny", 8)[3]
    if where == "prompt":
        d.prompt_logits[1, 7] = float("nan")
    else:
        d.final_norm = torch.full_like(d.final_norm, float("nan"))
    with pytest.raises(E.EngineError, match="no token"):
        d.generate(0.0)


def test_more_tokens_than_a_completion_has_room_for_are_refused():
    import torch
    d = make("tiny", 8, new=5, drafts=2)[3]
    rows = d.row_group.numel()
    tokens = torch.ones(rows, 8, dtype=torch.int32, device="cuda")
    with pytest.raises(E.EngineError, match="room"):
        d.step_logits(tokens)
    assert torch.isfinite(d.step_logits(tokens[:, :7])).all()
    d._append(tokens[:, :4], torch.full_like(d.count, 4))
    with pytest.raises(E.EngineError, match="room"):
        d.step_logits(tokens[:, :5])
    assert torch.isfinite(d.step_logits(tokens[:, :4])).all()


# 512 latent and 32 rope columns as the scaled model's, 16 heads, small elsewhere
WIDE = ModelConfig(vocab_size=512, max_sequence_length=512, n_layers=2, d_model=256, n_heads=16, head_dim_nope=96,
                   head_dim_rope=32, head_dim_value=128, q_lora_rank=128, kv_lora_rank=512, d_ff=512)


@pytest.mark.parametrize("name", ["mla36m", "wide"])
def test_long_prompts_match_the_context_forward(name):
    """Prompts of several key tiles, shared, then steps of several tokens and of one."""
    import torch
    require_gpu()
    from cpp_inference_train_engine_b200.group_decode import GroupDecoder
    cfg = {"mla36m": MLA36M, "wide": WIDE}[name]
    tol = 2 * 2e-2  # both sides' fp16 logits, as for the short prompts
    params = E.init_params(cfg, 3)
    rng = np.random.default_rng(6)
    prompts = [rng.integers(0, 256, n).tolist() for n in (333, 65, 200)]
    rows = [2, 1, 3]
    d = GroupDecoder(cfg, params, prompts, rows, 12, 3, 16)
    ex = E.make_execution(cfg, params)
    for i, p in enumerate(prompts):
        want = ex.forward(np.array(p), 1, len(p))[-1]
        assert np.abs(d.prompt_logits[i].cpu().numpy() - want).max() < tol
    groups = d.row_group.tolist()
    chosen = rng.integers(0, 256, (len(groups), 5))
    at = 0
    for T in (4, 1):
        tokens = torch.tensor(chosen[:, at:at + T], dtype=torch.int32, device="cuda")
        d._append(tokens[:, :1], torch.ones_like(d.count))
        got = d.step_logits(tokens).cpu().numpy()
        for b, g in enumerate(groups):
            ids = np.array(prompts[g] + chosen[b, :at + T].tolist())
            want = ex.forward(ids, 1, len(ids))[-T:]
            assert np.abs(got[b] - want).max() < tol, (T, b)
        d._append(tokens[:, 1:], torch.full_like(d.count, T - 1))
        at += T


def test_wide_completions_with_8_bit_caches_follow_their_own_logits():
    """Greedy tokens with drafts are the argmax (to the tolerance) of a replay of one token a step."""
    import torch
    require_gpu()
    from cpp_inference_train_engine_b200.group_decode import GroupDecoder
    params = E.init_params(WIDE, 4)
    rng = np.random.default_rng(7)
    prompts = [rng.integers(0, 256, n).tolist() for n in (150, 70)]
    out, stats = GroupDecoder(WIDE, params, prompts, [3, 2], 10, 3, 8).generate()
    r = GroupDecoder(WIDE, params, prompts, [3, 2], 10, 0, 8)
    logits = r.prompt_logits[r.row_group]
    for i in range(10):
        forced = torch.tensor([[o[i]] if i < len(o) else [0] for o in out], dtype=torch.int32, device="cuda")
        for b, o in enumerate(out):
            if i < len(o):
                assert logits[b, o[i]] >= logits[b].max() - 2 * 2 * 2e-2, (b, i)
        r._append(forced, torch.ones_like(r.count))
        logits = r.step_logits(forced)[:, 0]
