"""Newton-Schulz orthogonalisation kernels (kernels/newton_schulz.hip) against fp64."""
import pytest
import torch

from pytorch_multiprocessing_distributed_amd.ops import functional as OF

pytestmark = pytest.mark.gpu
UB = 2.0 ** -8      # half a bf16 step, relative


def _ref(u, steps=5, coeffs=OF.NS_COEFFS, eps=1e-7):
    a, b, c = coeffs
    x = u.double()
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    x = x / (x.norm() + eps)
    for _ in range(steps):
        s = x @ x.t()
        x = a * x + (b * s + c * s @ s) @ x
    return x.t() if tall else x


def _mat(m, n, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    r = max(1, min(m, n) // 8)
    u = torch.randn(m, r, generator=g) @ torch.randn(r, n, generator=g) / r ** 0.5 + torch.randn(m, n, generator=g)
    return (u * scale).to(dtype).cuda()


def _tol(ref, dtype, growth=485.0):
    """Entrywise.  A step makes about ten roundings (the planes of X, S and P, the fp32 sums of three
    products), each a matrix of spectral norm at most 2^-22 of its operands' (below 1.5); what a step
    leaves grows with the smallest singular values, 485 times from the first step and 3.4445 times less
    from each later one (together 1.41 times 485).  No entry exceeds the spectral norm."""
    return 10 * 1.41 * growth * 2.0 ** -22 + (UB * ref.abs() if dtype == torch.bfloat16 else 0.0)


def _check(u, out, full_rank=True, **kw):
    ref = _ref(u, **kw)
    assert out.shape == u.shape and out.dtype == u.dtype
    assert ((out.double() - ref).abs() <= _tol(ref, u.dtype)).all()
    if u.dtype == torch.float32 and full_rank:
        # as a whole, where no singular value is zero: an error grows no faster than the smallest singular
        # values themselves, so relative to the matrix the roundings only add up: 5 steps x 10, twice
        assert (out.double() - ref).norm() <= 100 * 2.0 ** -22 * ref.norm()


SIZES = [(1, 1), (1, 9), (7, 1), (2, 3), (64, 27), (64, 147), (63, 65), (128, 64), (65, 576), (200, 130),
         (512, 128), (257, 1031), (512, 4608), (1000, 2048),
         # at and past the limits of the one-block kernel
         (96, 96), (97, 97), (96, 113), (96, 114), (101, 96), (32, 1024), (1025, 32), (8, 4096), (4097, 8), (1, 32768),
         (1, 32769), (17, 1900), (33, 962), (3, 10923)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n", SIZES)
def test_against_fp64(m, n, dtype):
    u = _mat(m, n, dtype=dtype)
    _check(u, OF.newton_schulz(u))


# the last two: symmetric products on 192-wide tiles, the last row of tiles short and full
@pytest.mark.parametrize("m,n", [(2048, 2048), (1500, 5000), (3990, 4100), (4224, 4224)])
def test_large_tiles(m, n):
    u = _mat(m, n, seed=1)
    _check(u, OF.newton_schulz(u))


@pytest.mark.parametrize("steps", [1, 3])
@pytest.mark.parametrize("m,n", [(200, 130), (512, 128), (257, 1031), (600, 4608), (3990, 4100)])
def test_planes_hold_22_bits(m, n, steps):
    """X <- X leaves the normalised matrix: what the two planes hold, entry by entry."""
    u = _mat(m, n, seed=9)
    out = OF.newton_schulz(u, steps=steps, coeffs=(1.0, 0.0, 0.0))
    ref = u.double() / (u.double().norm() + 1e-7)
    # a split leaves half a step of the lower plane, 2^-22 of the entry (2^-40 where that plane is subnormal), at
    # the start and after every step but the last; a handful of fp32 operations around each
    assert ((out.double() - ref).abs() <= steps * (2.0 ** -22 + 6 * 2.0 ** -24) * ref.abs() + steps * 2.0 ** -39).all()


def test_a_models_matrices_in_one_call():
    shapes = [(64, 27)] + [(64, 576), (256, 64), (128, 1152), (30, 7), (5, 300)] * 11 + [(512, 512)]
    us = [_mat(m, n, seed=i) for i, (m, n) in enumerate(shapes)]     # more than one group
    keep = [u.clone() for u in us]
    outs = OF.newton_schulz(us)
    for u, k, o in zip(us, keep, outs):
        assert torch.equal(u, k)
        _check(u, o)


def test_stack_and_strides():
    u = torch.stack([_mat(40, 72, seed=i) for i in range(3)]).transpose(1, 2)
    out = OF.newton_schulz(u)
    for i in range(3):
        _check(u[i], out[i])


@pytest.mark.parametrize("steps,coeffs", [(1, OF.NS_COEFFS), (3, (1.5, -0.5, 0.0)), (12, (1.875, -1.25, 0.375)),
                                          (2, (8.2, -23.0, 17.0))])
def test_other_coefficients(steps, coeffs):
    u = _mat(96, 160, seed=2)
    growth = max(485.0, abs(coeffs[0]) ** steps)
    ref = _ref(u, steps=steps, coeffs=coeffs)
    out = OF.newton_schulz(u, steps=steps, coeffs=coeffs)
    assert ((out.double() - ref).abs() <= _tol(ref, u.dtype, min(growth, 1e5)) * max(1.0, ref.abs().max().item())).all()


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e12, 1e30])
def test_scale_of_the_update_does_not_matter(scale):
    u = _mat(70, 90, seed=3, scale=scale)
    _check(u, OF.newton_schulz(u, eps=0.0), eps=0.0)


def test_zero_nan_and_inf():
    z = torch.zeros(33, 50, device="cuda")
    assert not OF.newton_schulz(z).any()
    u = _mat(33, 50, seed=4)
    u[3, 4] = float("nan")
    assert OF.newton_schulz(u).isnan().any()
    u[3, 4] = float("inf")
    assert OF.newton_schulz(u).isnan().any()


def test_rank_one():
    # all singular values but one are zero: they stay zero to rounding
    u = (_mat(60, 1) @ _mat(1, 80, seed=1))
    _check(u, OF.newton_schulz(u), full_rank=False)


def test_in_place_update_with_device_rate():
    from pytorch_multiprocessing_distributed_amd.ops.hip_prims import newton_schulz_
    us = [_mat(30, 40, seed=5), _mat(50, 20, seed=6)]
    ps = [_mat(30, 40, seed=7), _mat(50, 20, seed=8)]
    lr = torch.tensor([0.25], device="cuda")
    refs = [0.5 * p.double() + a * 0.25 * _ref(u) for p, u, a in zip(ps, us, (2.0, -1.0))]
    newton_schulz_(us, ps, 5, OF.NS_COEFFS, 1e-7, [2.0, -1.0], 0.5, lr)
    for p, r in zip(ps, refs):
        assert ((p.double() - r).abs() <= _tol(r, torch.float32) + 4 * 2.0 ** -24 * r.abs().max()).all()


def test_repeatable_other_stream_and_two_at_once():
    us = [_mat(300, 700, seed=9), _mat(64, 64, seed=10)]
    a = OF.newton_schulz(us)
    torch.cuda.synchronize()
    outs = []
    for s in [torch.cuda.Stream() for _ in range(2)]:
        with torch.cuda.stream(s):
            outs.append(OF.newton_schulz(us))
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(p, q) for p, q in zip(a, o))


def test_graph_capture_and_replay():
    u = _mat(128, 300, seed=11)
    OF.newton_schulz(u)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = OF.newton_schulz(u)
    for i in range(4):
        u.copy_(_mat(128, 300, seed=20 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, OF.newton_schulz(u))


def test_refusals_gpu():
    u = _mat(4, 4)
    with pytest.raises(RuntimeError, match="bf16 or fp32"):
        OF.newton_schulz(u.half())
    with pytest.raises(RuntimeError, match="singular values"):
        OF.newton_schulz(u, steps=20, coeffs=(3.0, 1.0, 1.0))
    with pytest.raises(RuntimeError, match="singular values"):
        OF.newton_schulz(u, coeffs=(float("nan"), 0.0, 0.0))
    with pytest.raises(RuntimeError, match="steps"):
        OF.newton_schulz(u, steps=65)
    with pytest.raises(RuntimeError, match="eps"):
        OF.newton_schulz(u, eps=-1.0)
