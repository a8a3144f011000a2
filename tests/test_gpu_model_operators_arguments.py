"""Arguments of RMS norm that are wrong in two ways at once: one exception, of a kind that says what is wrong."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eps", ["1e-6", [1e-6], object()])
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("shape", [64, (4, 64)])
def test_an_eps_that_is_no_number(eps, grad, shape):
    import float8_experimental_amd as f8

    x = torch.ones(4, 64, device="cuda", requires_grad=grad)
    for call in (f8.rms_norm, f8.rms_norm_blockwise):
        with pytest.raises((TypeError, ValueError)):
            call(x, shape, None, eps)
    with torch.no_grad():
        assert torch.isfinite(f8.rms_norm(x, 64, None, 1e-6)).all()
