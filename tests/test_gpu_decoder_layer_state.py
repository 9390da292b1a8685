"""A decoder layer's call that is refused leaves the residual stream, the cache and the lengths as they were."""
import pytest
import torch

from test_gpu_decoder_layer import E, HIDDEN, R, layer_of, weights_of_norms

pytestmark = pytest.mark.gpu


def test_refused_calls_change_nothing(w4a8, oracle, cuda):
    tables, layer = layer_of(w4a8, oracle, cuda, weights_of_norms(cuda))
    tables.step(torch.ones(R, dtype=torch.int32, device=cuda), R)
    h, y = torch.randn(R + 1, HIDDEN, device=cuda), torch.randn(R + 1, HIDDEN, device=cuda)
    before = h.clone()
    with pytest.raises(ValueError, match="planned for 3"):
        layer(h, y)
    assert torch.equal(h, before)
    with pytest.raises((ValueError, w4a8.W4A8Error), match="max_q"):
        layer(h[:R], y[:R], max_q=-1)
    assert torch.equal(h, before) and all((t == 0).all() for t in layer.attention.cache._tensors)
    layer(h[:R], y[:R])
    assert not torch.equal(h[:R], before[:R]) and torch.equal(h[R], before[R]) and E == layer.router.experts
