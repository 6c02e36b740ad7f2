"""The attention layer of comp_amd/examples/cached_attention.py: quantized projections, cache and attention together."""

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("prompt", [1, 2, 70])
def test_cached_attention_layer(fmt, prompt):
    """The attention of f32 queries is within 1e-5 (their 22 bits and the softmax's f32) of plain attention over the cache."""
    from comp_amd.examples import cached_attention

    assert cached_attention.run(prompt, 3, fmt) <= 1e-5
