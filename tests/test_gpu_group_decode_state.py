"""What a GroupDecoder keeps between calls and how it fails."""
import pytest

import cpp_inference_train_engine_b200 as E
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
