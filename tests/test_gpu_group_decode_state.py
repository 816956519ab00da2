"""What a GroupDecoder keeps between calls and how it fails."""
import pytest

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
