"""Gradients that share memory, clipped in place: tied parameters that are listed more than once, and views of one buffer that overlap."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def f8():
    import float8_experimental_amd

    return float8_experimental_amd


def factor_of(norm, max_norm):
    return torch.clamp(torch.tensor(max_norm) / (norm.cpu() + torch.tensor(1e-6)), max=1.0).cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [5, 1000, 300000])
def test_a_parameter_that_is_listed_twice_is_scaled_once(f8, n, dtype):
    made = [torch.randn(n, generator=torch.Generator().manual_seed(i)).to(dtype).cuda() for i in range(3)]
    params = [torch.nn.Parameter(torch.zeros_like(g)) for g in made]
    for p, g in zip(params, made):
        p.grad = g.clone()
    listed = [params[0], params[1], params[0], params[2], params[0]]
    norm = f8.clip_grad_norm_(listed, 0.5)
    exact = sum(made[i].double().square().sum() for i in (0, 1, 0, 2, 0)).sqrt()  # the norm is that of what is listed
    assert abs(norm.double() - exact) <= 2.0**-23 * exact
    for p, g in zip(params, made):
        assert torch.equal(p.grad, (g.float() * factor_of(norm, 0.5)).to(dtype))


def test_gradients_that_overlap_are_scaled_once(f8):
    flat = torch.randn(5000, generator=torch.Generator().manual_seed(0)).cuda()
    want, params = flat.clone(), []
    for begin, end in ((0, 3000), (2000, 5000), (100, 200)):
        params.append(torch.nn.Parameter(torch.zeros(end - begin, device="cuda")))
        params[-1].grad = flat[begin:end]
    norm = f8.clip_grad_norm_(params, 0.5)
    assert torch.equal(flat, want * factor_of(norm, 0.5))


def test_neighbours_in_one_buffer_are_clipped_where_they_lie(f8):
    """As buckets of gradients are laid out: next to each other, in any order, at any alignment."""
    flat = torch.randn(5003, generator=torch.Generator().manual_seed(0)).bfloat16().cuda()
    want, params = flat.clone(), []
    for begin, end in ((3001, 5003), (0, 1), (1, 3001), (77, 77)):
        params.append(torch.nn.Parameter(torch.zeros(end - begin, device="cuda", dtype=torch.bfloat16)))
        params[-1].grad = flat[begin:end]
    norm = f8.clip_grad_norm_(params, 0.5)
    assert torch.equal(flat, (want.float() * factor_of(norm, 0.5)).bfloat16())
    assert abs(norm.double() - want.double().norm()) <= 2.0**-23 * norm
