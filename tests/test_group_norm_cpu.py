"""Group norm + residual + activation on the CPU primitives: the formulas and gradients in fp64
against differences, argument checks, and empty inputs."""
import pytest
import torch

from pytorch_multiprocessing_distributed_amd.ops import functional as OF


def _gn(groups, c, dtype=torch.float64, seed=0):
    g = torch.Generator().manual_seed(seed)
    m = torch.nn.GroupNorm(groups, c, eps=1e-5).to(dtype)
    with torch.no_grad():
        m.weight.copy_(torch.rand(c, generator=g) + 0.5)
        m.bias.copy_(torch.randn(c, generator=g))
    return m


@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("res", [False, True])
@pytest.mark.parametrize("shape,groups", [((2, 3, 5, 6), 3), ((1, 1, 1, 4), 2), ((3, 4), 1), ((2, 7, 5), 5)])
def test_gradients_against_differences(act, res, shape, groups):
    g = torch.Generator().manual_seed(1)
    gn = _gn(groups, shape[-1])
    x = torch.randn(shape, generator=g, dtype=torch.float64, requires_grad=True)
    r = torch.randn(shape, generator=g, dtype=torch.float64, requires_grad=True) if res else None

    def f(x, w, b, *r):
        m = torch.nn.GroupNorm(groups, shape[-1], eps=1e-5).double()
        m.weight, m.bias = torch.nn.Parameter(w), torch.nn.Parameter(b)
        return OF._GroupNormActFn.apply(x, w, b, r[0] if r else None, groups, 1e-5, act)
    args = [x, gn.weight, gn.bias] + ([r] if res else [])
    # central differences of step 1e-6 in fp64: truncation ~1e-12, rounding ~1e-10; a group of one or
    # two elements has derivatives up to 1/sqrt(eps) = 316 and second ones up to 1e5
    assert torch.autograd.gradcheck(f, args, eps=1e-6, atol=1e-4, rtol=1e-4)


@pytest.mark.parametrize("shape,groups", [((2, 4, 4, 12), 4), ((5, 9), 3)])
def test_forward_matches_torch(shape, groups):
    x = torch.randn(shape, dtype=torch.float64, generator=torch.Generator().manual_seed(2))
    gn = _gn(groups, shape[-1])
    ref = gn(x.movedim(-1, 1)).movedim(1, -1)
    # the same fp64 formula in another order: some tens of 2^-53 roundings of values below 10
    torch.testing.assert_close(OF.group_norm_act(x, gn, act="none"), ref, rtol=0, atol=1e-13)
    torch.testing.assert_close(OF.group_norm_act(x, gn, residual=x, act="relu"), torch.relu(ref + x), rtol=0, atol=1e-13)


def test_strided_input_is_laid_out():
    gn = _gn(2, 4)
    x = torch.randn(2, 4, 5, 3, dtype=torch.float64).movedim(1, -1)      # a channels-first tensor's view
    assert not x.is_contiguous()
    torch.testing.assert_close(OF.group_norm_act(x, gn), OF.group_norm_act(x.contiguous(), gn), rtol=0, atol=0)


@pytest.mark.parametrize("shape", [(0, 3, 3, 4), (2, 0, 3, 4)])
def test_empty(shape):
    gn = _gn(2, 4, torch.float32)
    x = torch.randn(shape, requires_grad=True)
    out = OF.group_norm_act(x, gn)
    assert out.shape == x.shape
    gx, gw, gb = torch.autograd.grad(out.sum(), [x, gn.weight, gn.bias])
    assert gx.shape == x.shape and not gw.any() and not gb.any()


def test_refusals():
    gn = _gn(2, 4, torch.float32)
    x = torch.randn(2, 3, 3, 4)
    with pytest.raises(ValueError, match="activation"):
        OF.group_norm_act(x, gn, act="tanh")
    with pytest.raises(ValueError, match="must be"):
        OF.group_norm_act(x[..., :3], gn)
    with pytest.raises(ValueError, match="residual"):
        OF.group_norm_act(x, gn, residual=x[:1])
    with pytest.raises(ValueError, match="residual"):
        OF.group_norm_act(x, gn, residual=x.double())
    with pytest.raises(ValueError, match="weight and bias"):
        OF.group_norm_act(x, torch.nn.GroupNorm(2, 4, affine=False))
    with pytest.raises(ValueError, match="must be"):
        OF.group_norm_act(torch.randn(4), gn)


def test_no_second_derivative():
    gn = _gn(2, 4)
    x = torch.randn(2, 3, 4, dtype=torch.float64, requires_grad=True)
    (gx,) = torch.autograd.grad(OF.group_norm_act(x, gn).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gx.sum(), x)
