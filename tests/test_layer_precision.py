"""The error bounds that the dense operators' GPU tests use, against models of the kernels'
arithmetic on the CPU: the right one is within them, mistakes that lose digits are not."""

import pytest
import torch

from oracle import dense_torch

# ----------------------------------------------------- float32 products ---


def planes(x, count):
    """x as the sum of ``count`` bfloat16 numbers, the largest first, each in float32."""
    out = []
    for _ in range(count):
        out.append(x.bfloat16().float())
        x = x - out[-1]
    return out


def product_model(x, w, count=3, most=2):
    """x w^T from the products of planes i and j (from 0) with i + j <= most."""
    total = torch.zeros(x.shape[0], w.shape[0])
    for i, a in enumerate(planes(x, count)):
        for j, b in enumerate(planes(w, count)):
            if i + j <= most:
                total = total + a @ b.t()
    return total


def relative_rms(got, exact):
    return float((got.double() - exact).square().mean().sqrt() / exact.square().mean().sqrt())


@pytest.mark.parametrize("inner", [32, 256, 1024])
def test_product_bound_holds_for_three_planes_and_rejects_two(inner):
    gen = torch.Generator().manual_seed(2)
    x, w = torch.randn((400, inner), generator=gen), torch.randn((300, inner), generator=gen)
    exact = x.double() @ w.double().t()
    limit = dense_torch.product_rms(inner)
    assert relative_rms(product_model(x, w), exact) <= limit
    # two planes, all four of their products; the third planes without their products with
    # the first; one operand in two planes
    assert relative_rms(product_model(x, w, count=2), exact) > limit
    assert relative_rms(product_model(x, w, most=1), exact) > limit
    assert relative_rms(product_model(sum(planes(x, 2)), w), exact) > limit


# ------------------------------------------------------------- layer norm ---


def norm_model(x, eps, mistake=None):
    """The normalised values in float32 as the kernels compute them. ``mistake``: "shift"
    subtracts the row's first value from every value and keeps what that rounds to,
    "uncorrected" leaves the first sum's error in the mean."""
    n = x.shape[-1]
    x0 = x[:, :1]
    from_x0 = (x - x0).sum(-1, keepdim=True) / n
    if mistake == "shift":
        c = (x - x0) - from_x0
        return c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    mean = x0 + from_x0
    near = from_x0.abs() < mean.abs()
    base, offset = torch.where(near, x0, 0.0), torch.where(near, from_x0, mean)
    c = (x - base) - offset
    rest = c.sum(-1, keepdim=True) / n
    var = (c * c).mean(-1, keepdim=True) - rest * rest
    if mistake != "uncorrected":
        offset = offset + rest
    return ((x - base) - offset) / torch.sqrt(var.clamp_min(0.0) + eps)


def rows_with_a_channel(cols, size, far=0.0):
    gen = torch.Generator().manual_seed(1)
    x = torch.randn((200, cols), generator=gen) + far
    x[:, 0] = size * (1.0 + 0.1 * torch.randn(200, generator=gen))
    return x


def outside(x, model):
    results, bounds = dense_torch.layer_norm(x, None, None, 1e-5)
    return ((model.double() - results[0]).abs() > bounds[0])[:, 1:]


@pytest.mark.parametrize("far", [0.0, 1e4])
@pytest.mark.parametrize("size", [1.0, 1e3, 1e5])
@pytest.mark.parametrize("cols", [64, 256, 4096])
def test_norm_bound_holds_for_the_kernels_arithmetic(cols, size, far):
    x = rows_with_a_channel(cols, size, far)
    assert not outside(x, norm_model(x, 1e-5)).any()


@pytest.mark.parametrize("mistake", ["shift", "uncorrected"])
def test_norm_bound_rejects_a_mean_of_the_first_values_size(mistake):
    for cols, size in ((4096, 1e4), (20000, 1e5)):
        x = rows_with_a_channel(cols, size)
        assert outside(x, norm_model(x, 1e-5, mistake)).any()
