"""Group norm + residual + activation kernels (kernels/group_norm.hip) against the formulas in fp64."""
import pytest
import torch

from pytorch_multiprocessing_distributed_amd.ops import functional as OF

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24                 # half a step of fp32
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: U32}

SHAPES = [  # N, spatial, C, groups
    (2, (8, 8), 64, 32), (1, (4, 4), 512, 32), (3, (5, 7), 24, 3), (2, (3, 3), 120, 10), (2, (1, 1), 32, 32),
    (5, (), 48, 6), (2, (9, 9), 3, 1), (2, (6, 5), 7, 7), (1, (33, 41), 10, 5), (2, (2, 2), 2056, 8),
    (1, (3,), 4100, 1), (70, (2, 2), 16, 2), (1, (130, 130), 16, 4), (4, (56, 56), 64, 32), (2, (28, 28), 512, 32),
]


def _ref(x, res, w, b, dy, groups, eps, act):
    """fp64: out, dx, dw, db, dres, z and the [N, pixels, G, cg] view's (mean, rstd)."""
    n, c = x.shape[0], x.shape[-1]
    v = x.double().reshape(n, -1, groups, c // groups)
    mu = v.mean((1, 3), keepdim=True)
    rstd = ((v - mu).square().mean((1, 3), keepdim=True) + eps).rsqrt()
    xh = (v - mu) * rstd
    ga, be = w.double().reshape(groups, -1), b.double().reshape(groups, -1)
    z = xh * ga + be
    if res is not None:
        z = z + res.double().reshape(z.shape)
    s = torch.sigmoid(z)
    out = {"none": z, "relu": z.clamp_min(0), "silu": z * s}[act]
    g = dy.double().reshape(z.shape)
    dz = {"none": g, "relu": g * (z > 0), "silu": g * (s + z * s * (1 - s))}[act]
    dh = dz * ga
    dx = rstd * (dh - dh.mean((1, 3), keepdim=True) - xh * (dh * xh).mean((1, 3), keepdim=True))
    sh = x.shape
    return (out.reshape(sh), dx.reshape(sh), (dz * xh).sum((0, 1)).reshape(-1), dz.sum((0, 1)).reshape(-1),
            dz.reshape(sh), z.reshape(sh), mu, rstd, (dz * xh).abs().sum((0, 1)).reshape(-1),
            dz.abs().sum((0, 1)).reshape(-1))


def _case(n, sp, c, groups, dtype, seed=0, shift=2.0):
    g = torch.Generator().manual_seed(seed)
    shape = (n, *sp, c)
    x = (torch.randn(shape, generator=g) * (torch.rand(c, generator=g) + 0.5) + shift * torch.randn(c, generator=g))
    gn = torch.nn.GroupNorm(groups, c)
    with torch.no_grad():
        gn.weight.copy_(torch.rand(c, generator=g) + 0.5)
        gn.bias.copy_(torch.randn(c, generator=g) * 0.5)
    res = torch.randn(shape, generator=g)
    dy = torch.randn(shape, generator=g)
    return x.to(dtype).cuda(), gn.cuda(), res.to(dtype).cuda(), dy.to(dtype).cuda()


def _check(x, gn, res, dy, act):
    groups, eps = gn.num_groups, gn.eps
    w, b = gn.weight.detach(), gn.bias.detach()
    z = _ref(x, res, w, b, dy, groups, eps, act)[5]
    # at the ReLU's corner either slope is right: no gradient goes in there
    dy = dy.masked_fill((z.abs() < 1e-3), 0.0)
    out_r, dx_r, dw_r, db_r, dz_r, _, mu, rstd, dw_a, db_a = _ref(x, res, w, b, dy, groups, eps, act)
    xg = x.clone().requires_grad_(True)
    rg = res.clone().requires_grad_(True) if res is not None else None
    out = OF.group_norm_act(xg, gn, residual=rg, act=act)
    leaves = [xg, gn.weight, gn.bias] + ([rg] if res is not None else [])
    got = torch.autograd.grad(out, leaves, dy)
    h = HALF[x.dtype]
    # fp32 roundings on the way to z: the mean and rstd come through at most ~64 dependent fp32 sums
    # of values up to max|x|, then a handful of operations
    n = x.shape[0]
    xh_err = 64 * U32 * (x.double().abs().amax() * rstd.amax() + 1)
    z_err = xh_err * w.abs().max().double() + 8 * U32 * (z.abs().amax() + 1)
    slope = 1.1 if act == "silu" else 1.0
    assert ((out.double() - out_r).abs() <= h * out_r.abs() + slope * z_err).all()
    # dz: silu's slope moves by at most 0.5 per unit of z
    gmax = dy.double().abs().amax()
    dz_err = gmax * (0.5 * z_err if act == "silu" else 0.0) + 8 * U32 * gmax
    if res is not None:
        assert ((got[3].double() - dz_r).abs() <= h * dz_r.abs() + dz_err).all()
    # dx = rstd (dh - m1 - xh m2): every term's error, the means' sums among them
    xh_max = (x.double().abs().amax() * 2 * rstd.amax()).clamp_max(rstd.amax() * 1e4)
    xh_max = torch.minimum(xh_max, torch.tensor(float(x[0].numel() // groups) ** 0.5, dtype=torch.float64, device=x.device) + 1)
    wm = w.abs().max().double()
    term = wm * (dz_err + gmax * 64 * U32) * (1 + xh_max * xh_max) + wm * gmax * (xh_err * xh_max * 2)
    dx_err = rstd.amax() * term + 64 * U32 * dx_r.abs().amax()
    assert ((got[0].double() - dx_r).abs() <= h * dx_r.abs() + dx_err).all()
    # parameter gradients: fp32 sums down a thread's pixels (a few hundred terms at most here), then fp64
    dw_err = 512 * U32 * dw_a + (db_a * xh_err) + dz_err * xh_max * (x.numel() // x.shape[-1])
    db_err = 512 * U32 * db_a + dz_err * (x.numel() // x.shape[-1])
    assert ((got[1].double() - dw_r).abs() <= dw_err).all()
    assert ((got[2].double() - db_r).abs() <= db_err).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,sp,c,groups", SHAPES)
def test_against_fp64(n, sp, c, groups, dtype):
    x, gn, res, dy = _case(n, sp, c, groups, dtype)
    for act, r in (("relu", res), ("none", None)):
        _check(x, gn, r, dy, act)


@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("with_res", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_activations(act, with_res, dtype):
    x, gn, res, dy = _case(3, (7, 9), 40, 5, dtype, seed=3)
    _check(x, gn, res if with_res else None, dy, act)


# samples whose groups fit a block's registers: a few and many pixels a thread, threads without any, groups of
# 2 channels to all of a block's, one pixel
ONE = [(64, (28, 28), 32, 4), (40, (27, 29), 64, 8), (300, (40, 43), 32, 16), (2, (14, 14), 256, 1), (3, (13,), 512, 8),
       (260, (1,), 64, 32), (257, (56, 57), 32, 4), (9, (10, 11), 40, 8), (5, (6, 7), 56, 8), (6, (20, 21), 120, 10),
       (3, (9, 5), 24, 2), (4, (12, 11), 160, 16), (2, (7, 7), 224, 2)]


@pytest.mark.parametrize("act,with_res", [("none", True), ("relu", False), ("relu", True), ("silu", False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,sp,c,groups", ONE)
def test_in_registers(n, sp, c, groups, dtype, act, with_res):
    x, gn, res, dy = _case(n, sp, c, groups, dtype, seed=20)
    _check(x, gn, res if with_res else None, dy, act)


@pytest.mark.parametrize("n,sp,c,groups", ONE + [(1, (130, 130), 16, 4), (4, (56, 56), 64, 32), (5, (31, 33), 10, 5)])
def test_large_mean_everywhere(n, sp, c, groups):
    g = torch.Generator().manual_seed(21)
    x = (torch.randn(n, *sp, c, generator=g) + 1000.0).cuda()
    x.view(n, -1, c)[:, 0] += 300.0                        # the first pixel is no guide to the mean
    gn = torch.nn.GroupNorm(groups, c).cuda()
    out = OF.group_norm_act(x, gn, act="none")
    ref = _ref(x, None, gn.weight.detach(), gn.bias.detach(), x, groups, gn.eps, "none")[0]
    # x - mean carries the mean's rounding and the last sums', each up to 1300 * 2^-24 for a few of them; a thread's
    # sums about a shift 300 off lose up to 64 of their steps
    rstd = _ref(x, None, gn.weight.detach(), gn.bias.detach(), x, groups, gn.eps, "none")[7].amax()
    assert (out.double() - ref).abs().max() <= 128 * U32 * 1300 * rstd * (1 + ref.abs().max())


@pytest.mark.parametrize("offset", [1, 2, 4])
def test_unaligned_storage(offset):
    # a view that starts 2, 4 or 8 bytes into its storage: narrower loads, same values
    x, gn, res, dy = _case(2, (6, 6), 64, 8, torch.bfloat16, seed=4)
    buf = torch.empty(x.numel() + 8, dtype=x.dtype, device="cuda")
    xo = buf[offset:offset + x.numel()].view(x.shape)
    xo.copy_(x)
    _check(xo, gn, res, dy, "relu")
    a = OF.group_norm_act(x, gn, residual=res)
    b = OF.group_norm_act(xo, gn, residual=res)
    assert (a.double() - b.double()).abs().max() <= 2.0 ** -7 * a.abs().max()


def test_large_mean():
    # mean 1000 at a width of 1 in fp32: sums of squares would leave 1000^2 * 2^-24 = 6% of the variance
    g = torch.Generator().manual_seed(5)
    x = (torch.randn(4, 16, 16, 32, generator=g) + 1000.0).cuda()
    gn = torch.nn.GroupNorm(4, 32).cuda()
    out = OF.group_norm_act(x, gn, act="none")
    ref = _ref(x, None, gn.weight.detach(), gn.bias.detach(), x, 4, gn.eps, "none")[0]
    # x - mean is exact to the mean's own rounding: 1000 * a few 2^-24
    assert (out.double() - ref).abs().max() <= 64 * U32 * 1010


def test_constant_group_and_nan():
    x = torch.full((2, 4, 4, 8), 3.0, device="cuda")
    gn = torch.nn.GroupNorm(2, 8).cuda()
    with torch.no_grad():
        gn.bias.fill_(0.25)
    assert torch.equal(OF.group_norm_act(x, gn), torch.full_like(x, 0.25))
    x[1, 0, 0, 0] = float("nan")
    out = OF.group_norm_act(x, gn)
    assert out[1, ..., :4].isnan().all() and not out[0].isnan().any() and not out[1, ..., 4:].isnan().any()


def test_bitwise_repeatable_and_other_stream():
    x, gn, res, dy = _case(8, (32, 32), 64, 32, torch.bfloat16, seed=6)

    def step():
        xg = x.clone().requires_grad_(True)
        out = OF.group_norm_act(xg, gn, residual=res)
        return [out.detach(), *torch.autograd.grad(out, [xg, gn.weight, gn.bias], dy)]
    a = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = step()
    torch.cuda.current_stream().wait_stream(s)
    for p, q in zip(a, b):
        assert torch.equal(p, q)


def test_graph_capture_and_replay():
    x, gn, res, dy = _case(4, (16, 16), 32, 8, torch.bfloat16, seed=7)
    with torch.no_grad():
        OF.group_norm_act(x, gn, residual=res)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = OF.group_norm_act(x, gn, residual=res)
    for i in range(4):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(i)).to(x.dtype))
        graph.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            assert torch.equal(out, OF.group_norm_act(x, gn, residual=res))


def test_broadcast_gradient_and_strides():
    x, gn, _, _ = _case(2, (4, 4), 16, 4, torch.float32, seed=8)
    xt = x.movedim(-1, 1).contiguous().movedim(1, -1).requires_grad_(True)   # channels-first storage
    out = OF.group_norm_act(xt, gn, act="silu")
    (g,) = torch.autograd.grad(out.sum(), xt)                                # an expanded gradient of ones
    xr = x.double().requires_grad_(True)
    z = torch.nn.functional.group_norm(xr.movedim(-1, 1), 4, gn.weight.double(), gn.bias.double()).movedim(1, -1)
    (gr,) = torch.autograd.grad((z * torch.sigmoid(z)).sum(), xr)
    # the terms of dx (rstd * slope * gamma, below 4 each) through ~64 fp32 roundings
    assert (g.double() - gr).abs().max() <= 64 * U32 * 16


def test_arena_gradients_accumulate():
    from pytorch_multiprocessing_distributed_amd.parallel.flat import flatten_module
    x, gn, res, dy = _case(2, (8, 8), 32, 8, torch.bfloat16, seed=9)
    ref = torch.nn.GroupNorm(8, 32).cuda()
    ref.load_state_dict(gn.state_dict())
    out = OF.group_norm_act(x, ref, residual=res)
    gw, gb = torch.autograd.grad(out, [ref.weight, ref.bias], dy)
    flat = flatten_module(gn)
    for k in (1, 2):
        OF.group_norm_act(x, gn, residual=res).backward(dy)
        assert torch.equal(gn.weight.grad, gw * k) and torch.equal(gn.bias.grad, gb * k)
    flat.zero_grad()


def test_refusals_gpu():
    x, gn, res, _ = _case(2, (4, 4), 16, 4, torch.float32)
    with pytest.raises(RuntimeError, match="bf16 or fp32"):
        OF.group_norm_act(x.half(), gn)
    with pytest.raises(RuntimeError, match="device"):
        OF.group_norm_act(x, torch.nn.GroupNorm(4, 16))
    with pytest.raises(RuntimeError, match="residual"):
        OF.group_norm_act(x, gn, residual=res.cpu())
    big = torch.nn.GroupNorm(1, 16392).cuda()
    with pytest.raises(RuntimeError, match="channels"):
        OF.group_norm_act(torch.zeros(1, 16392, device="cuda"), big)
    with pytest.raises(RuntimeError, match="samples"):
        OF.group_norm_act(torch.zeros(2 ** 23 + 1, 4, device="cuda"), torch.nn.GroupNorm(2, 4).cuda())


@pytest.mark.parametrize("n,c", [(2 ** 23, 8), (2 ** 20, 64)])
def test_many_samples(n, c):
    # a pixel a sample: more samples than one grid's threads would allow at 512 a block
    x = torch.randn(n, c, device="cuda", dtype=torch.bfloat16)
    gn = torch.nn.GroupNorm(2, c).cuda()
    with torch.no_grad():
        out = OF.group_norm_act(x, gn, act="none")
    rows = torch.tensor([0, 1, n // 2, n - 2, n - 1], device="cuda")
    ref = _ref(x[rows], None, gn.weight.detach(), gn.bias.detach(), x[rows], 2, gn.eps, "none")[0]
    # outputs of up to 2^3: half a bf16 step, and fp32 errors far below one
    assert ((out[rows].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -14).all()


@pytest.mark.parametrize("n,hw,c,groups", [(700, 3136, 1024, 32), (720, 3136, 1000, 8)])
def test_offsets_past_32_bits(n, hw, c, groups):
    # more than 2^31 elements (4.5 GB): the last sample, in registers and split
    x = torch.randn(n, hw, c, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    gn = torch.nn.GroupNorm(groups, c).cuda()
    out = OF.group_norm_act(x, gn, act="none")
    dy = torch.zeros_like(out)
    dy[-1] = torch.randn(hw, c, device="cuda").to(torch.bfloat16)
    dx, dw = torch.autograd.grad(out, [x, gn.weight], dy)
    r = _ref(x.detach()[-1:], None, gn.weight.detach(), gn.bias.detach(), dy[-1:], groups, gn.eps, "none")
    # values of at most 2^3: half a bf16 step, and fp32 errors far below one
    assert ((out[-1:].double() - r[0]).abs() <= 2.0 ** -8 * r[0].abs() + 2.0 ** -14).all()
    assert ((dx[-1:].double() - r[1]).abs() <= 2.0 ** -8 * r[1].abs() + 2.0 ** -14).all()
    assert not dx[-2].any()
    # fp32 sums of a few thousand terms
    assert ((dw.double() - r[2]).abs() <= 512 * U32 * r[8] + 2.0 ** -14 * r[9]).all()


@pytest.mark.parametrize("act,with_res", [("relu", True), ("silu", True), ("relu", False)])
def test_backward_twice_over_a_retained_graph(act, with_res):
    for shape in ((4, (56, 56), 64, 32), (6, (14, 14), 64, 32)):
        x, gn, res, dy = _case(*shape, torch.bfloat16, seed=22)
        xg = x.clone().requires_grad_(True)
        out = OF.group_norm_act(xg, gn, residual=res if with_res else None, act=act)
        a = torch.autograd.grad(out, [xg, gn.weight, gn.bias], dy, retain_graph=True)
        b = torch.autograd.grad(out, [xg, gn.weight, gn.bias], dy)
        assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("act", ["none", "relu", "silu"])
def test_native_and_python_nodes_agree(act):
    x, gn, res, dy = _case(2, (6, 6), 32, 8, torch.bfloat16, seed=10)

    def grads(fn):
        xg, rg = x.clone().requires_grad_(True), res.clone().requires_grad_(True)
        out = fn(xg, rg)
        return [out.detach(), *torch.autograd.grad(out, [xg, rg, gn.weight, gn.bias], dy)]
    a = grads(lambda xg, rg: OF.group_norm_act(xg, gn, residual=rg, act=act))
    b = grads(lambda xg, rg: OF._GroupNormActFn.apply(xg, gn.weight, gn.bias, rg, 8, gn.eps, act))
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_frozen_inputs_and_no_second_derivative():
    x, gn, res, dy = _case(2, (6, 6), 32, 8, torch.float32, seed=11)
    gn.weight.requires_grad_(False)
    out = OF.group_norm_act(x, gn, residual=res)                    # only the bias wants a gradient
    (gb,) = torch.autograd.grad(out, gn.bias, dy)
    assert (gb.double() - (dy.double() * (out > 0)).sum((0, 1, 2))).abs().max() <= 512 * U32 * dy.abs().sum((0, 1, 2)).max()
    assert not OF.group_norm_act(x, gn.requires_grad_(False), residual=res).requires_grad
    xg = x.clone().requires_grad_(True)
    (gx,) = torch.autograd.grad(OF.group_norm_act(xg, gn).sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):                # nothing leads from the gradient back to the input
        torch.autograd.grad(gx.sum(), xg, retain_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        gx.sum().backward()


def test_misaligned_gradient_with_the_mask():
    x, gn, res, dy = _case(2, (6, 6), 64, 8, torch.bfloat16, seed=12)
    buf = torch.empty(dy.numel() + 8, dtype=dy.dtype, device="cuda")
    off = buf[1:1 + dy.numel()].view(dy.shape)
    off.copy_(dy)
    xg = x.clone().requires_grad_(True)
    out = OF.group_norm_act(xg, gn, residual=res)
    a, b = torch.autograd.grad(out, xg, dy, retain_graph=True), torch.autograd.grad(out, xg, off)
    assert torch.equal(a[0], b[0])
