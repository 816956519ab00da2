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
