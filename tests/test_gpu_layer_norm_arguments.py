"""Arguments of layer norm that are no numbers, or numbers that no dimension has: errors that say so."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_shapes_and_eps_that_are_no_numbers_or_too_large():
    import float8_experimental_amd as f8

    x = torch.randn(4, 64, device="cuda")
    for shape in (2**70, (2**70,), -(2**70), (2**40, 2**40)):
        with pytest.raises(ValueError, match="normalized_shape"):
            f8.layer_norm(x, shape)
    for eps in (None, "1e-5"):
        with pytest.raises(TypeError):
            f8.layer_norm(x, 64, eps=eps)
    want = f8.layer_norm(x, 64, eps=0.5)
    assert torch.equal(f8.layer_norm(x, 64, eps=torch.tensor(0.5)), want)
    with pytest.raises(TypeError):
        f8.grad_norm([x], None)
    with pytest.raises(TypeError):
        f8.clip_grads([x], None)
