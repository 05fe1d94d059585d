"""Cross-entropy of a linear classifier without its logits (kernels/linear_xent.hip) against fp64."""
import pytest
import torch

from pytorch_multiprocessing_distributed_amd.ops import functional as OF

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24
UB = 2.0 ** -8          # half a bf16 step, relative
SIZES = [(1, 8, 2), (1, 1, 1), (5, 17, 3), (32, 512, 10), (64, 64, 64), (65, 72, 129), (197, 300, 1007),
         (256, 512, 1000), (3, 2048, 5003), (300, 40, 20011), (1030, 136, 4100)]


def _case(n, d, v, dtype, seed=0, bias=True, ignored=None, bias_dtype=None):
    g = torch.Generator().manual_seed(seed)
    lin = torch.nn.Linear(d, v, bias=bias)
    t = torch.randint(0, v, (n,), generator=g)
    with torch.no_grad():
        lin.weight.copy_(torch.randn(v, d, generator=g) / d ** 0.5)
        if bias:
            lin.bias.copy_(torch.randn(v, generator=g) * 0.3)
    x = torch.randn(n, d, generator=g) + 6.0 * (torch.arange(n) % 2)[:, None] * lin.weight.detach()[t]
    if ignored if ignored is not None else n > 4:
        t[torch.randperm(n, generator=g)[:max(1, n // 5)]] = -100
    lin = lin.to(dtype).cuda()
    if bias and bias_dtype is not None:
        lin.bias.data = lin.bias.data.to(bias_dtype)
    return x.to(dtype).cuda().requires_grad_(True), lin, t.cuda()


def _ref(x, w, b, t, gloss=1.0):
    x, w = x.detach().double(), w.detach().double()
    b = torch.zeros(w.shape[0], dtype=torch.float64, device=x.device) if b is None else b.detach().double()
    keep = t != -100
    xk, tk = x[keep], t[keep]
    n = max(1, xk.shape[0])
    logits = xk @ w.t() + b
    lse = torch.logsumexp(logits, 1)
    ar = torch.arange(xk.shape[0], device=x.device)
    loss = (lse - logits[ar, tk]).sum() / n
    p = torch.exp(logits - lse[:, None])
    p[ar, tk] -= 1
    p *= gloss / n
    dx = torch.zeros_like(x)
    dx[keep] = p @ w
    # |.| sums: what roundings of the factors scale with
    ax = torch.zeros_like(x)
    ax[keep] = p.abs() @ w.abs()
    mag = (xk.abs() @ w.abs().t()).amax() + b.abs().amax() + 1 if xk.numel() else torch.tensor(1.0)
    correct = ((logits.argmax(1) == tk).sum() if xk.numel() else torch.tensor(0)).item()
    return loss, correct, dx, p.t() @ xk, p.sum(0), ax, p.abs().t() @ xk.abs(), p.abs().sum(0), mag


def _check(x, lin, t, gloss=1.0, bf16=False, **kw):
    dt = x.dtype
    loss, correct = OF.linear_cross_entropy(x, lin, t, **kw)
    leaves = [x, lin.weight] + ([lin.bias] if lin.bias is not None else [])
    got = torch.autograd.grad(loss, leaves, torch.tensor(gloss, device="cuda"))
    xr, wr = (x.bfloat16(), lin.weight.bfloat16()) if bf16 else (x, lin.weight)
    loss_r, correct_r, dx_r, dw_r, db_r, ax, aw, ab, mag = _ref(xr, wr, lin.bias, t, gloss)
    d = x.shape[1]
    # a logit: exact products (fp32 operands: to 2^-22), d + 2 fp32 additions of partial sums up to mag;
    # then exp and log at a few steps each
    l_err = (d / 4 + 40) * U32 * mag
    assert abs(loss.item() - loss_r.item()) <= 2 * l_err + 16 * U32 * (1 + abs(loss_r.item())) + len(t) * U32 * 4
    assert correct.item() == correct_r
    # p: exp of a logit off by 2 l_err and its own steps; bf16 products round softmax - onehot once
    two = bf16 or dt == torch.bfloat16
    # and take exponentials that were kept in fp16, half a step each
    kept = 2.0 ** -11 if two else 0.0
    p_rel = 2 * l_err + 32 * U32 + kept + (UB if two else 2.0 ** -22)
    n = x.shape[0]
    # onehot - softmax near 1 cancels: an absolute 2 l_err of the softmax, relative to |p - 1|'s ab share
    out = UB if dt == torch.bfloat16 else 0.0
    extra = (2 * l_err + 32 * U32)
    keep = max(1, int((t != -100).sum()))
    same = int(torch.bincount(t[t != -100]).max()) if (t != -100).any() else 1    # rows of one class
    sum_rel = (len(t) / 4 + 64) * U32
    vsum = (lin.weight.shape[0] / 4 + 64) * U32
    wmax, xmax = wr.double().abs().max(), xr.double().masked_fill((t == -100)[:, None], 0).abs().max()
    g = abs(gloss) / keep
    assert ((got[0].double() - dx_r).abs() <= out * dx_r.abs() + (p_rel + vsum) * ax + extra * g * wmax).all()
    wout = UB if lin.weight.dtype == torch.bfloat16 else 0.0
    assert ((got[1].double() - dw_r).abs() <= wout * dw_r.abs() + (p_rel + sum_rel) * aw + extra * g * xmax * same).all()
    if lin.bias is not None:
        bout = UB if lin.bias.dtype == torch.bfloat16 else 0.0
        assert ((got[2].double() - db_r).abs() <= bout * db_r.abs() + (2 * l_err + 32 * U32 + kept + sum_rel) * ab
                + extra * g * same).all()
    assert not got[0][t == -100].any()
    return loss, got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,d,v", SIZES)
def test_against_fp64(n, d, v, dtype):
    x, lin, t = _case(n, d, v, dtype)
    _check(x, lin, t)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_no_bias_and_upstream_gradient(dtype):
    x, lin, t = _case(70, 96, 333, dtype, seed=1, bias=False)
    _check(x, lin, t, gloss=-2.5)


def test_fp32_bias_of_a_bf16_classifier():
    x, lin, t = _case(70, 96, 333, torch.bfloat16, seed=2, bias_dtype=torch.float32)
    _, got = _check(x, lin, t)
    assert got[2].dtype == torch.float32


def test_bf16_products_of_fp32_operands():
    x, lin, t = _case(130, 200, 777, torch.float32, seed=3)
    _check(x, lin, t, bf16=True, compute_dtype=torch.bfloat16)


@pytest.mark.parametrize("xd,wd", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
def test_mixed_operands_keep_fp32(xd, wd):
    x, lin, t = _case(40, 56, 130, torch.float32, seed=4)
    lin = lin.to(wd)
    _check(x.detach().to(xd).requires_grad_(True), lin, t)


def test_large_tiles_and_pieces():
    # enough tiles for the 256-wide kernels, a last column and row tile that are not full
    x, lin, t = _case(2300, 264, 9001, torch.bfloat16, seed=5)
    _check(x, lin, t)


def test_vocabulary_in_pieces(monkeypatch):
    # 2^24 rows never fit a test; 98,304 rows leave a piece of 1,024 classes: three pieces, the last ragged
    x, lin, t = _case(98304, 16, 2100, torch.bfloat16, seed=6)
    _check(x, lin, t)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,d,v", [(1, 8, 2), (65, 72, 129), (300, 40, 20011), (2300, 264, 9001), (70000, 16, 2100)])
def test_with_and_without_kept_exponentials(n, d, v, dtype):
    """The backward that computes the logits again agrees with the one that has their exponentials."""
    x, lin, t = _case(n, d, v, dtype, seed=19)
    P = OF.prims_for(x)
    args = (lin.weight.detach(), lin.bias.detach(), t, -100, False)
    x = x.detach()
    loss, _, lse, inv, xp, kept = P.linear_xent_fwd(x, *args, True)
    loss2, _, lse2, _, _, none = P.linear_xent_fwd(x, *args, False)
    assert none.numel() == 0 < kept.numel() and torch.equal(loss, loss2) and torch.equal(lse, lse2)
    one = torch.ones(1, device="cuda")
    r = []
    for k in (kept, none):
        dw, db = torch.empty_like(lin.weight), torch.empty_like(lin.bias)
        dx = P.linear_xent_bwd(one, xp, dtype, *args, lse, inv, True, dw, db, False, k)
        r.append((dx.double(), dw.double(), db.double()))
    _, _, _, _, _, ax, aw, ab, mag = _ref(x, lin.weight, lin.bias, t)
    # what _check allows a side, twice: a logit's error in the exponential, the roundings of it, the sums;
    # at the target, where the onehot cancels it, the absolute error of the exponential
    e = 2 * (d / 4 + 40) * U32 * mag + 32 * U32
    two = dtype == torch.bfloat16
    rel = 2 * (e + (2.0 ** -11 + UB if two else 2.0 ** -22) + (max(n, v) / 4 + 64) * U32)
    out = 2 * UB if two else 0.0
    g = 1.0 / max(1, int((t != -100).sum()))
    same = int(torch.bincount(t[t != -100]).max())
    wmax, xmax = lin.weight.double().abs().max(), x.double().masked_fill((t == -100)[:, None], 0).abs().max()
    for a, b, m, f in zip(r[0], r[1], (ax, aw, ab), (wmax, xmax * same, same)):
        assert ((a - b).abs() <= out * b.abs() + rel * m + 2 * e * g * f).all()


def test_unaligned_weight_and_features():
    x, lin, t = _case(33, 64, 200, torch.bfloat16, seed=7)
    wbuf = torch.empty(200 * 64 + 8, dtype=torch.bfloat16, device="cuda")
    w = wbuf[1:1 + 200 * 64].view(200, 64)
    w.copy_(lin.weight.detach())
    lin2 = torch.nn.Linear(64, 200).cuda().bfloat16()
    lin2.weight = torch.nn.Parameter(w)
    lin2.bias = lin.bias
    a, ga = _check(x, lin, t)
    b, gb = _check(x, lin2, t)
    assert torch.equal(a, b) and all(torch.equal(p, q) for p, q in zip(ga, gb))
    xt = x.detach().t().contiguous().t().requires_grad_(True)      # features with other strides
    c, _ = OF.linear_cross_entropy(xt, lin, t)
    assert torch.equal(a, c)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_rows_and_classes(dtype):
    x, lin, t = _case(40, 24, 90, dtype, seed=8)
    keep = t != -100
    with torch.no_grad():
        ref = OF.linear_cross_entropy(x, lin, t)[0]
        x[~keep] = float("nan")
    loss, _ = _check_finite(x, lin, t)
    assert torch.equal(loss, ref)
    # classes that are masked by a bias of -inf or the type's lowest value get no probability
    with torch.no_grad():
        lin.bias[::3] = float("-inf")
        lin.bias[1] = torch.finfo(dtype).min
    t[keep] = (t[keep] // 3) * 3 + 2
    _, got = _check_finite(x, lin, t)
    assert not got[1][::3].any() and not got[1][1].any() and not got[2][::3].any()


def _check_finite(x, lin, t):
    loss, _ = OF.linear_cross_entropy(x, lin, t)
    got = torch.autograd.grad(loss, [x, lin.weight, lin.bias])
    assert loss.isfinite() and all(g.isfinite().all() for g in got)
    return loss, got


def test_everything_masked_target_masked_and_nan():
    x, lin, t = _case(8, 16, 12, torch.float32, seed=9, ignored=False)
    loss, correct = OF.linear_cross_entropy(x, lin, torch.full_like(t, -100))
    assert loss.item() == 0 and correct.item() == 0
    assert not any(g.any() for g in torch.autograd.grad(loss, [x, lin.weight, lin.bias]))
    t2 = t.clone()
    t2[3] = 12
    loss, _ = OF.linear_cross_entropy(x, lin, t2)
    assert loss.isnan() and torch.autograd.grad(loss, x)[0][3].isnan().all()
    with torch.no_grad():
        lin.bias[t[0]] = float("-inf")
    assert OF.linear_cross_entropy(x, lin, t)[0].item() == float("inf")
    with torch.no_grad():
        lin.bias.fill_(float("-inf"))
    assert OF.linear_cross_entropy(x, lin, t)[0].isnan()


def test_extreme_logits():
    # logits up to +-3e4: the running maximum keeps every exponential in range
    x, lin, t = _case(16, 32, 300, torch.float32, seed=10, ignored=False)
    with torch.no_grad():
        lin.weight.mul_(3e3)
        ref = torch.nn.functional.cross_entropy(x.double() @ lin.weight.double().t() + lin.bias.double(), t)
    loss, _ = OF.linear_cross_entropy(x, lin, t)
    # two logits of up to ~1e5, each 32/4 + 40 roundings off
    assert abs(loss.item() - ref.item()) <= 2 * 48 * U32 * 2e5


def test_ties_go_to_the_lowest_class():
    lin = torch.nn.Linear(8, 600).cuda()
    with torch.no_grad():
        lin.weight.zero_()
        lin.bias.zero_()
    x = torch.randn(3, 8, device="cuda")
    _, c = OF.linear_cross_entropy(x, lin, torch.tensor([0, 1, 599], device="cuda"))
    assert c.item() == 1


def test_no_rows():
    x, lin, t = _case(4, 8, 6, torch.float32, ignored=False)
    loss, c = OF.linear_cross_entropy(x[:0], lin, t[:0])
    gx, gw, gb = torch.autograd.grad(loss, [x, lin.weight, lin.bias])
    assert loss.item() == 0 and c.item() == 0 and not gx.any() and not gw.any() and not gb.any()


def test_repeatable_other_stream_and_two_at_once():
    x, lin, t = _case(257, 128, 3001, torch.bfloat16, seed=11)

    def step():
        loss, c = OF.linear_cross_entropy(x, lin, t)
        return [loss.detach(), c, *torch.autograd.grad(loss, [x, lin.weight, lin.bias])]
    a = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append(step())
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(p, q) for p, q in zip(a, o))


def test_graph_capture_and_replay():
    x, lin, t = _case(96, 64, 500, torch.bfloat16, seed=12)
    x = x.detach()
    with torch.no_grad():
        OF.linear_cross_entropy(x, lin, t)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loss, correct = OF.linear_cross_entropy(x, lin, t)
        for i in range(4):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(i)).to(x.dtype))
            graph.replay()
            torch.cuda.synchronize()
            l2, c2 = OF.linear_cross_entropy(x, lin, t)
            assert torch.equal(loss, l2) and torch.equal(correct, c2)


def test_arena_gradients_accumulate():
    from pytorch_multiprocessing_distributed_amd.parallel.flat import flatten_module
    x, lin, t = _case(50, 48, 70, torch.float32, seed=13)
    loss, _ = OF.linear_cross_entropy(x, lin, t, compute_dtype=torch.bfloat16)
    gw, gb = torch.autograd.grad(loss, [lin.weight, lin.bias])
    flat = flatten_module(lin)
    for k in (1, 2):
        loss, _ = OF.linear_cross_entropy(x, lin, t, compute_dtype=torch.bfloat16)
        loss.backward()
        assert torch.equal(lin.weight.grad, gw * k) and torch.equal(lin.bias.grad, gb * k)
    flat.zero_grad()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_backward_twice_over_a_retained_graph(dtype):
    x, lin, t = _case(130, 72, 900, dtype, seed=23)
    loss, _ = OF.linear_cross_entropy(x, lin, t)
    a = torch.autograd.grad(loss, [x, lin.weight, lin.bias], retain_graph=True)
    b = torch.autograd.grad(loss, [x, lin.weight, lin.bias])
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_too_many_logits_are_refused():
    x = torch.zeros(2 ** 24, 1, device="cuda", dtype=torch.bfloat16)
    lin = torch.nn.Linear(1, 2 ** 14 + 1, bias=False, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="2\\^38 logits"):
        OF.linear_cross_entropy(x, lin, torch.zeros(2 ** 24, dtype=torch.int64, device="cuda"))


@pytest.mark.parametrize("want", [False, True])
def test_captured_step_beside_an_eager_one(want):
    """A forward and backward captured on its own leaves, replayed between eager calls of other sizes."""
    x, lin, t = _case(96, 64, 500, torch.bfloat16, seed=24)
    leaves = [x, lin.weight] + ([lin.bias] if want else [])
    lin.bias.requires_grad_(want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            torch.autograd.grad(OF.linear_cross_entropy(x, lin, t)[0], leaves)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        loss, correct = OF.linear_cross_entropy(x, lin, t)
        got = torch.autograd.grad(loss, leaves)
    x2, lin2, t2 = _case(70, 48, 1300, torch.bfloat16, seed=25)
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(i)).to(x.dtype))
        graph.replay()
        torch.autograd.grad(OF.linear_cross_entropy(x2, lin2, t2)[0], [x2])
        torch.cuda.synchronize()
        l2, c2 = OF.linear_cross_entropy(x, lin, t)
        ref = torch.autograd.grad(l2, leaves)
        assert torch.equal(loss, l2) and torch.equal(correct, c2)
        assert all(torch.equal(p, q) for p, q in zip(got, ref))


def test_refusals_gpu():
    x, lin, t = _case(4, 8, 6, torch.float32, ignored=False)
    with pytest.raises(RuntimeError, match="bf16 or fp32"):
        OF.linear_cross_entropy(x.half(), lin, t)
    with pytest.raises(RuntimeError, match="one device"):
        OF.linear_cross_entropy(x, lin, t.cpu())
    with pytest.raises(RuntimeError, match="one device"):
        OF.linear_cross_entropy(x, torch.nn.Linear(8, 6), t)


def test_native_and_python_nodes_agree():
    x, lin, t = _case(70, 96, 333, torch.bfloat16, seed=14)

    def grads(fn):
        loss, c = fn()
        return [loss.detach(), c, *torch.autograd.grad(loss, [x, lin.weight, lin.bias], torch.tensor(0.5, device="cuda"))]
    a = grads(lambda: OF.linear_cross_entropy(x, lin, t))
    b = grads(lambda: OF._LinearXentFn.apply(x, lin.weight, lin.bias, t, -100, False))
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_frozen_inputs_and_no_second_derivative():
    x, lin, t = _case(70, 96, 333, torch.bfloat16, seed=15)
    loss, _ = OF.linear_cross_entropy(x, lin, t)
    all_of = torch.autograd.grad(loss, [x, lin.weight, lin.bias])
    lin.weight.requires_grad_(False)
    loss, _ = OF.linear_cross_entropy(x, lin, t)
    gx, gb = torch.autograd.grad(loss, [x, lin.bias])
    assert torch.equal(gx, all_of[0]) and torch.equal(gb, all_of[2])
    lin.weight.requires_grad_(True)
    loss, _ = OF.linear_cross_entropy(x.detach(), lin, t)
    (gw,) = torch.autograd.grad(loss, [lin.weight])
    assert torch.equal(gw, all_of[1])
    (gx,) = torch.autograd.grad(OF.linear_cross_entropy(x, lin, t)[0], x, create_graph=True)
    with pytest.raises(RuntimeError):                # nothing leads from the gradient back to the input
        torch.autograd.grad(gx.sum(), x, retain_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        gx.sum().backward()


def test_two_products_that_fill_the_device_alone():
    # dx and dW of 256 blocks and more each take a grid of their own
    x, lin, t = _case(1100, 2064, 9001, torch.bfloat16, seed=16)
    _check(x, lin, t)
