"""Beam search where kernels fail, hypotheses end early, and the prompt is seen through a window."""
import numpy as np
import pytest

import cpp_inference_train_engine_b200 as E
from tests.gpu_util import require_gpu
from tests.test_gpu_beam_decode import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("module", ["latent", "paged"])
def test_a_kernel_that_gave_up_is_reported_as_such(module, monkeypatch):
    """The status that the device keeps is asked for after the prompts, at a search's end, and before a missing
    continuation is blamed on the logits: here a fake one that says yes."""
    require_gpu()
    from cpp_inference_train_engine_b200 import latent, paged
    asked = []

    def gave_up(device=None):
        asked.append(device)
        raise E.EngineError(5, "a kernel gave up")

    d = make("tiny")[3]
    with monkeypatch.context() as m:
        m.setattr({"latent": latent, "paged": paged}[module], "check_status", gave_up)
        with pytest.raises(E.EngineError, match="gave up"):
            make("tiny")
        with pytest.raises(E.EngineError, match="gave up"):
            d.search()
        kept = d.prompt_logits.clone()
        d.prompt_logits.fill_(float("nan"))
        with pytest.raises(E.EngineError, match="gave up"):
            d.search()
        d.prompt_logits.copy_(kept)
    assert asked == [d.device] * 3
    assert len(d.search()) == 3
