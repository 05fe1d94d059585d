"""Cross-entropy of a linear classifier on the CPU primitives: against the separate operators, against
differences, rows to ignore, argument checks."""
import pytest
import torch

from pytorch_multiprocessing_distributed_amd.ops import functional as OF


def _case(n, d, v, dtype=torch.float64, seed=0, bias=True):
    g = torch.Generator().manual_seed(seed)
    lin = torch.nn.Linear(d, v, bias=bias).to(dtype)
    with torch.no_grad():
        lin.weight.copy_(torch.randn(v, d, generator=g))
        if bias:
            lin.bias.copy_(torch.randn(v, generator=g))
    x = torch.randn(n, d, generator=g, dtype=torch.float64).to(dtype)
    return x.requires_grad_(True), lin, torch.randint(0, v, (n,), generator=g)


@pytest.mark.parametrize("bias", [True, False])
def test_matches_torch(bias):
    x, lin, t = _case(9, 5, 13, bias=bias)
    t[[2, 7]] = -100
    loss, correct = OF.linear_cross_entropy(x, lin, t)
    logits = torch.nn.functional.linear(x, lin.weight, lin.bias)
    ref = torch.nn.functional.cross_entropy(logits, t)
    leaves = [x, lin.weight] + ([lin.bias] if bias else [])
    # one fp64 formula in two orders: values below 30, some tens of roundings of 2^-53
    torch.testing.assert_close(loss, ref, rtol=0, atol=1e-13)
    for a, b in zip(torch.autograd.grad(loss * 3, leaves), torch.autograd.grad(ref * 3, leaves)):
        torch.testing.assert_close(a, b, rtol=0, atol=1e-13)
    assert correct.item() == ((logits.argmax(1) == t) & (t != -100)).sum().item()


def test_gradients_against_differences():
    x, lin, t = _case(4, 3, 5, seed=1)
    t[1] = 99

    def f(x, w, b):
        return OF._LinearXentFn.apply(x, w, b, t, 99, False)[0]
    # central differences of step 1e-6: truncation 1e-12, rounding 1e-10
    assert torch.autograd.gradcheck(f, (x, lin.weight, lin.bias), eps=1e-6, atol=1e-8, rtol=1e-6)


def test_ignored_rows_may_hold_anything():
    x, lin, t = _case(6, 4, 7, seed=2)
    t[[0, 3]] = -1
    with torch.no_grad():
        ref, _ = OF.linear_cross_entropy(x[[1, 2, 4, 5]], lin, t[[1, 2, 4, 5]], ignore_index=-1)
        x[0], x[3] = float("nan"), float("inf")
    loss, _ = OF.linear_cross_entropy(x, lin, t, ignore_index=-1)
    gx, gw = torch.autograd.grad(loss, [x, lin.weight])
    torch.testing.assert_close(loss, ref, rtol=0, atol=1e-13)
    assert not gx[[0, 3]].any() and gw.isfinite().all()


def test_no_row_left_and_no_rows():
    x, lin, t = _case(3, 4, 5, torch.float32)
    for xx, tt in ((x, torch.full_like(t, -100)), (x[:0], t[:0])):
        loss, correct = OF.linear_cross_entropy(xx, lin, tt)
        grads = torch.autograd.grad(loss, [x, lin.weight, lin.bias])
        assert loss.item() == 0 and correct.item() == 0 and not any(g.any() for g in grads)


def test_target_outside_the_classes_is_nan():
    x, lin, t = _case(3, 4, 5)
    for bad in (5, -7):
        t[1] = bad
        assert OF.linear_cross_entropy(x, lin, t)[0].isnan()


def test_leading_dimensions():
    x, lin, t = _case(6, 4, 5)
    a, ca = OF.linear_cross_entropy(x, lin, t)
    b, cb = OF.linear_cross_entropy(x.reshape(2, 3, 4), lin, t.reshape(2, 3))
    assert torch.equal(a, b) and torch.equal(ca, cb)


def test_compute_dtype_rounds_the_operands():
    x, lin, t = _case(6, 8, 5, torch.float32)
    a, _ = OF.linear_cross_entropy(x, lin, t, compute_dtype=torch.bfloat16)
    lr = torch.nn.Linear(8, 5)
    with torch.no_grad():
        lr.weight.copy_(lin.weight.bfloat16())
        lr.bias.copy_(lin.bias)
    b, _ = OF.linear_cross_entropy(x.bfloat16().float(), lr, t)
    assert torch.equal(a, b)


def test_refusals():
    x, lin, t = _case(3, 4, 5, torch.float32)
    with pytest.raises(ValueError, match="x must be"):
        OF.linear_cross_entropy(x[:, :3], lin, t)
    with pytest.raises(ValueError, match="target must be"):
        OF.linear_cross_entropy(x, lin, t[:2])
    with pytest.raises(ValueError, match="int64"):
        OF.linear_cross_entropy(x, lin, t.int())
    with pytest.raises(ValueError, match="compute_dtype"):
        OF.linear_cross_entropy(x, lin, t, compute_dtype=torch.float16)
