"""Newton-Schulz orthogonalisation on the CPU primitives: against the singular values, shapes, checks."""
import pytest
import torch

from pytorch_multiprocessing_distributed_amd.ops import functional as OF


def _poly(s, steps, coeffs):
    a, b, c = coeffs
    for _ in range(steps):
        s = s * (a + b * s ** 2 + c * s ** 4)
    return s


@pytest.mark.parametrize("m,n", [(5, 9), (9, 5), (4, 4), (1, 7), (6, 1), (1, 1)])
def test_acts_on_the_singular_values(m, n):
    u = torch.randn(m, n, dtype=torch.float64, generator=torch.Generator().manual_seed(0))
    out = OF.newton_schulz(u, steps=5, eps=1e-7)
    U, S, V = torch.linalg.svd(u, full_matrices=False)
    ref = U @ torch.diag(_poly(S / (S.square().sum().sqrt() + 1e-7), 5, OF.NS_COEFFS)) @ V
    # fp64 roundings of 2^-53, multiplied by at most 3.4445^5 = 485 on the way, a few dozen of them
    torch.testing.assert_close(out, ref, rtol=0, atol=485 * 100 * 2.0 ** -53)


def test_structures():
    g = torch.Generator().manual_seed(1)
    a, b = torch.randn(3, 4, 6, generator=g), torch.randn(5, 2, generator=g).bfloat16()
    out = OF.newton_schulz([a, b, a[:0]])
    assert isinstance(out, list) and [o.shape for o in out] == [a.shape, b.shape, (0, 4, 6)]
    assert out[1].dtype == torch.bfloat16
    for i in range(3):
        assert torch.equal(out[0][i], OF.newton_schulz(a[i]))
    assert torch.equal(OF.newton_schulz(a.transpose(1, 2)), OF.newton_schulz(a.transpose(1, 2).contiguous()))
    assert OF.newton_schulz([]) == []
    assert not OF.newton_schulz(torch.zeros(3, 4)).any()
    assert not OF.newton_schulz(torch.randn(2, 3, requires_grad=True)).requires_grad


def test_refusals():
    with pytest.raises(ValueError, match="matrices"):
        OF.newton_schulz(torch.randn(4))
    with pytest.raises(ValueError, match="step"):
        OF.newton_schulz(torch.randn(4, 4), steps=0)
    with pytest.raises(ValueError, match="three"):
        OF.newton_schulz(torch.randn(4, 4), coeffs=(1.5, -0.5))
