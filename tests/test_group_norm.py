"""Group normalisation with an activation on channels-last maps (vit_amd.group_norm): forward and gradients against the
formula in 64 bits, gradients against differences, refusals.

eps32 = 2^-24 below is half a unit in the last place of 1 in f32; the bounds count the roundings of the kernels' f32
arithmetic with room (means and deviations are merged in trees of at most a few hundred steps)."""
import math

import pytest
import torch

import vit_amd
from vit_amd import VitkError, lib

EPS32 = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}      # the final rounding, relative
ACTS = ["none", "relu", "gelu", "silu"]
gpu = pytest.mark.gpu


def _rnd(*shape, seed, scale=1.0, shift=0.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * scale + shift


def formula(x, G, w, b, eps, act, dy=None):
    """(y, dx, dw, db, z, h, rstd) in 64 bits."""
    C = x.shape[-1]
    g = x.reshape(x.shape[0], -1, G, C // G)
    mean = g.mean((1, 3), keepdim=True)
    var = ((g - mean) ** 2).mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    h = ((g - mean) * rstd).reshape(x.shape)
    z = h * w + b
    if act == "relu":
        y, slope = z.clamp(min=0), (z > 0).double()
    elif act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        y, slope = z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    elif act == "silu":
        s = torch.sigmoid(z)
        y, slope = z * s, s * (1 + z * (1 - s))
    else:
        y, slope = z, torch.ones_like(z)
    if dy is None:
        return y, None, None, None, z, h, rstd
    dz = dy * slope
    gz, gh = (dz * w).reshape(g.shape), h.reshape(g.shape)
    dx = rstd * (gz - gz.mean((1, 3), keepdim=True) - gh * (gz * gh).mean((1, 3), keepdim=True))
    dims = tuple(range(x.dim() - 1))
    return y, dx.reshape(x.shape), (dz * h).sum(dims), dz.sum(dims), z, h, rstd


# one value; odd widths and groups (the scalar path); groups of 3 channels (a vector spans groups); groups of one value;
# more channels than one workgroup's lanes, with a group across both; long maps (many chunks); tokens
SHAPES = [((1, 1, 8), 1), ((2, 7, 5, 30), 3), ((3, 14, 14, 96), 32), ((2, 9, 64), 64), ((2, 50, 2056), 1),
          ((2, 3000, 24), 4), ((4, 33, 1024), 2), ((1, 61, 97, 90), 9), ((5, 197, 768), 32), ((2, 28, 28, 512), 32)]


def _inputs(shape, dtype, shift=0.4):
    C = shape[-1]
    x = _rnd(*shape, seed=sum(shape), scale=1.5, shift=shift).to(dtype)
    w, b = _rnd(C, seed=1, scale=0.3, shift=1.0).float(), _rnd(C, seed=2, scale=0.3).float()
    return x, w, b, _rnd(*shape, seed=3).to(dtype)


def _y_bound(x, w, b, rstd, y, dtype, act):
    # mean within 8 eps of the largest |x|, rstd within 16 eps: (|x| + |mean|) 8 eps rstd |w| + 16 eps |z|, and the
    # activation's own 8 eps of |z| (silu: exp2, rcp) or 1.5e-7 |z| / 2 (gelu's erf)
    z_abs = 2 * x.abs().max() * rstd.max() * w.abs().max() + b.abs().max()
    return HALF[dtype] * y.abs() + 48 * EPS32 * z_abs


@gpu
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,G", SHAPES)
def test_forward(shape, G, dtype, act):
    x, w, b, _ = _inputs(shape, dtype)
    y, _, _, _, z, h, rstd = formula(x.double(), G, w.double(), b.double(), 1e-5, act)
    got = vit_amd.group_norm(x.cuda(), G, w.cuda(), b.cuda(), 1e-5, act)
    assert got.dtype == dtype and got.shape == x.shape
    err = (got.double().cpu() - y).abs()
    assert (err <= _y_bound(x.double(), w, b, rstd, y, dtype, act)).all(), err.max()


@gpu
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,G", [s for s in SHAPES if s[0] != (1, 1, 8)])
def test_gradients(shape, G, dtype, act):
    x, w, b, dy = _inputs(shape, dtype)
    X, W, Bi, DY = x.double(), w.double(), b.double(), dy.double()
    y, dx, dw, db, z, h, rstd = formula(X, G, W, Bi, 1e-5, act, DY)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    out = vit_amd.group_norm(leaves[0], G, leaves[1], leaves[2], 1e-5, act)
    got = [g.double().cpu() for g in torch.autograd.grad(out, leaves, dy.cuda())]
    n = X[0].numel() // G
    # terms whose slope may land on the other side of relu's corner: |z| within the forward's error
    near = (z.abs() < 1e-4).double() if act == "relu" else torch.zeros_like(z)
    grp = lambda t: t.reshape(X.shape[0], -1, G, X.shape[-1] // G)              # noqa: E731
    flip = (grp(near * (DY * W).abs() * (1 + h * h)).sum((1, 3), keepdim=True) / n * rstd).expand_as(grp(X)).reshape(X.shape) * (1 + h.abs())
    # dz within 64 eps (|z| from the forward's bound enters through act', whose slope is below 1.2), the means within
    # 256 eps of the largest term; the three terms of dx are each at most rstd |dz w| max (1 + h^2)
    zb = 48 * EPS32 * (2 * X.abs().max() * rstd.max() * W.abs().max() + Bi.abs().max())
    big = DY.abs().max() * W.abs().max() * rstd.max() * (1 + h.abs().max()) ** 2
    tol = HALF[dtype] * dx.abs() + (256 * EPS32 + (0.0 if act in ("none", "relu") else 2 * zb)) * big + 2 * flip
    err = (got[0] - dx).abs()
    assert ((err <= tol) | (near > 0)).all(), (err - tol).max()
    dims = tuple(range(X.dim() - 1))
    # f32 sums of at most 512 steps in a row
    for g, want, terms in ((got[1], dw, (DY * h).abs()), (got[2], db, DY.abs())):
        bound = (512 * EPS32 + 2 * zb) * 1.2 * terms.sum(dims) + (near * terms).sum(dims)
        assert ((g - want).abs() <= bound).all(), ((g - want).abs() / bound).max()


# The one-pass form's other cuts.  3136 pixels: 1,024 threads and rows of 64 bytes in the forward, the two of a 128-byte line
# on one XCD where batch * slabs is a multiple of 16 (f32: 4 x 4, bf16: 4 x 2), the backward in two passes.  1536 pixels:
# 512 threads and paired rows of 64 bytes in both directions (8 x 4, 8 x 2), 2000 with samples that are no multiple of the
# pairs (3 x 4, 3 x 2: unpaired), 1600 with one pair a sample (f32: 16 x 2) and with none (bf16: 16 x 1).
CUTS = [((4, 56, 56, 64), 8), ((8, 32, 48, 64), 8), ((3, 2000, 64), 8), ((16, 1600, 32), 4)]


@gpu
@pytest.mark.parametrize("act", ["none", "gelu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,G", CUTS)
def test_cuts_of_the_one_pass_form(shape, G, dtype, act):
    test_forward(shape, G, dtype, act)
    test_gradients(shape, G, dtype, act)


@gpu
@pytest.mark.parametrize("act", ACTS)
def test_gradients_against_differences(act):
    x, w, b, dy = _inputs((2, 11, 13, 24), torch.float32)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    out = vit_amd.group_norm(leaves[0], 4, leaves[1], leaves[2], 1e-5, act)
    got = torch.autograd.grad(out, leaves, dy.cuda())
    for i, t in enumerate((x, w, b)):
        v = _rnd(*t.shape, seed=9 + i)
        step = 1e-5

        def loss(s):
            a = [u.double() for u in (x, w, b)]
            a[i] = a[i] + s * v
            return float((formula(a[0], 4, a[1], a[2], 1e-5, act)[0] * dy.double()).sum())
        want = (loss(step) - loss(-step)) / (2 * step)
        have = float((got[i].double().cpu() * v).sum())
        # second-order error of the difference, a corner of relu inside the step, f32 gradients
        assert abs(have - want) <= 1e-3 * (1 + abs(want)), (have, want)


@gpu
@pytest.mark.parametrize("shape", [(1, 4, 2048), (3, 3000, 64)])                # one pass, two passes
def test_gelu_in_f32_is_accurate_relative_to_small_results(shape):
    """A weight of 0 makes z the bias: the activation and its derivative alone, over both tails."""
    C = shape[-1]
    z = torch.linspace(-12.0, 6.0, C, dtype=torch.float32)
    Z = z.double()
    cdf, den = 0.5 * torch.special.erfc(-Z / math.sqrt(2)), torch.exp(-Z * Z / 2) / math.sqrt(2 * math.pi)
    x = _rnd(*shape, seed=8).float().cuda()
    w, b = torch.zeros(C, device="cuda"), z.cuda().requires_grad_(True)
    y = vit_amd.group_norm(x, 2, w, b, 1e-5, "gelu")
    # erfc's argument is off by 2 eps (the constant, the product), which erfc turns into at most (z^2 + 1) times as much;
    # erfc itself within 16 units in the last place (32 eps), two products
    ecdf = (2 * (Z * Z + 1) + 32 + 4) * EPS32
    err = ((y.detach().double().cpu() - Z * cdf).abs() / (Z * cdf).abs().clamp(min=1e-300)).amax(tuple(range(y.dim() - 1)))
    assert (err <= ecdf)[Z != 0].all(), (err / ecdf).max()
    dy = torch.zeros(shape, device="cuda")
    dy[0, 1] = 1.0                                                              # one term of each channel's sum
    slope = torch.autograd.grad(y, b, dy)[0].double().cpu()
    # the exponent off by eps of z^2 / 2 twice, exp within 4 units, the constant and two products; their sum rounded once
    bound = ecdf * cdf + (Z * Z + 8 + 4) * EPS32 * Z.abs() * den + EPS32 * (cdf + Z * den).abs()
    assert ((slope - (cdf + Z * den)).abs() <= bound).all(), ((slope - (cdf + Z * den)).abs() / bound).max()


@gpu
def test_large_mean_against_small_deviation():
    # values of 1000 +- 1: sums of squares in f32 would leave no digit of the variance
    x = _rnd(2, 500, 32, seed=5, scale=1.0, shift=1000.0).float()
    y, _, _, _, _, _, rstd = formula(x.double(), 4, torch.ones(32).double(), torch.zeros(32).double(), 1e-5, "none")
    got = vit_amd.group_norm(x.cuda(), 4).double().cpu()
    # x itself carries 1000 * 2^-24; the mean is within 8 eps of 1000
    assert ((got - y).abs() <= 32 * EPS32 * 1000 * rstd.max()).all()


@gpu
def test_constant_group_and_non_finite_values_stay_in_their_group():
    x = torch.randn(2, 40, 16, device="cuda")
    x[0, :, :4] = 3.0                                                  # a group without deviation: 0 behind the norm
    x[1, 7, 5] = float("nan")
    x[1, 9, 9] = float("inf")
    y = vit_amd.group_norm(x, 4)
    assert (y[0, :, :4] == 0).all()
    assert y[1, :, 4:8].isnan().all() and y[1, :, 8:12].isnan().all()
    for g in (0, 3):
        alone = vit_amd.group_norm(x[1:2, :, 4 * g:4 * g + 4].contiguous(), 1)
        assert torch.allclose(y[1:2, :, 4 * g:4 * g + 4], alone, atol=1e-5)
    assert y[0].isfinite().all()


@gpu
def test_optional_parameters_views_and_empty_batches():
    x = torch.randn(3, 10, 10, 24, device="cuda", dtype=torch.bfloat16)
    w, b = torch.rand(24, device="cuda") + 0.5, torch.randn(24, device="cuda")
    one, zero = torch.ones_like(w), torch.zeros_like(b)
    assert torch.equal(vit_amd.group_norm(x, 3), vit_amd.group_norm(x, 3, one, zero))
    assert torch.equal(vit_amd.group_norm(x, 3, w), vit_amd.group_norm(x, 3, w, zero))
    assert torch.equal(vit_amd.group_norm(x, 3, None, b), vit_amd.group_norm(x, 3, one, b))
    # a view that is 2-byte aligned only takes the scalar path
    flat = torch.empty(x.numel() + 1, device="cuda", dtype=torch.bfloat16)
    flat[1:] = x.reshape(-1)
    odd = flat[1:].view(x.shape)
    assert torch.allclose(vit_amd.group_norm(odd, 3, w, b).float(), vit_amd.group_norm(x, 3, w, b).float(), rtol=2 ** -7, atol=1e-5)
    # only the bias wants a gradient
    bias = b.clone().requires_grad_(True)
    g, = torch.autograd.grad(vit_amd.group_norm(x, 3, w, bias).float().sum(), bias)
    assert torch.allclose(g, torch.full_like(g, 300.0))
    # a channels_last feature map goes in as a view
    nchw = torch.randn(2, 24, 6, 7, device="cuda").to(memory_format=torch.channels_last)
    y = vit_amd.group_norm(nchw.permute(0, 2, 3, 1), 3, w, b).permute(0, 3, 1, 2)
    assert torch.allclose(y, torch.nn.functional.group_norm(nchw, 3, w, b), atol=1e-5)
    for shape in ((0, 5, 24), (2, 0, 24)):
        e = torch.empty(shape, device="cuda", requires_grad=True)
        ww = w.clone().requires_grad_(True)
        out = vit_amd.group_norm(e, 3, ww, b)
        assert out.shape == shape
        ge, gw = torch.autograd.grad(out.sum(), (e, ww))
        assert ge.shape == shape and (gw == 0).all()


@gpu
def test_results_do_not_change_from_run_to_run_or_by_stream():
    x = torch.randn(4, 56, 56, 64, device="cuda", requires_grad=True)
    w, b = torch.rand(64, device="cuda").requires_grad_(True), torch.randn(64, device="cuda").requires_grad_(True)

    def step():
        y = vit_amd.group_norm(x, 8, w, b, 1e-5, "silu")
        return [y] + list(torch.autograd.grad(y, (x, w, b), torch.ones_like(y)))
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    again = step()
    torch.cuda.synchronize()
    for a, c, d in zip(first, other, again):
        assert torch.equal(a, c) and torch.equal(a, d)


@gpu
def test_captured_step_replays():
    x = torch.randn(2, 30, 30, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w, b = torch.rand(64, device="cuda").requires_grad_(True), torch.randn(64, device="cuda").requires_grad_(True)
    dy = torch.randn(2, 30, 30, 64, device="cuda").to(torch.bfloat16)

    def step():
        y = vit_amd.group_norm(x, 8, w, b, 1e-5, "gelu")
        return [y.detach()] + list(torch.autograd.grad(y, (x, w, b), dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(held, step()):
            assert torch.equal(a, c)


@gpu
def test_second_derivatives_are_refused():
    x = torch.randn(1, 4, 8, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(vit_amd.group_norm(x, 2, activation="gelu").square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


# ---- refusals --------------------------------------------------------------------------------------

def test_forward_mode_tangents_are_found_without_a_gpu():
    from torch.autograd import forward_ad
    from vit_amd.functional import _needs_grad
    x = torch.ones(2, 4)
    with forward_ad.dual_level():
        assert not _needs_grad(x, None)
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(VitkError, match="forward-mode"):
                _needs_grad(None, forward_ad.make_dual(x, x))
    assert not _needs_grad(x, None) and _needs_grad(x.clone().requires_grad_(True))


@gpu
def test_forward_mode_is_refused():
    """A tangent would come back as none at all, which reads as a derivative of zero."""
    from torch.autograd import forward_ad
    x = torch.ones(2, 3, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    with forward_ad.dual_level():
        for args in ((forward_ad.make_dual(x, x), 2, w, w), (x, 2, forward_ad.make_dual(w, w), w)):
            with pytest.raises(VitkError, match="forward-mode"):
                vit_amd.group_norm(*args)
        assert vit_amd.group_norm(x, 2, w, w).isfinite().all()


def test_refusals_without_a_gpu():
    with pytest.raises(VitkError, match="no CPU fallback"):
        vit_amd.group_norm(torch.randn(2, 5, 8), 2)
    L = lib.load()
    p = 4096                                          # never dereferenced: every call below is refused first
    ok = dict(batch=2, pixels=5, channels=8, groups=2)

    def call(act=0, dtype=0, ws=p, floats=1 << 20, mean=p, rstd=p, x=p, **kw):
        s = {**ok, **kw}
        return L.vitk_group_norm(x, None, None, p, mean, rstd, ws, floats, s["batch"], s["pixels"], s["channels"], s["groups"],
                                 1e-5, act, dtype, None)
    assert call(x=None) == 1 and call(ws=None) == 1
    assert call(groups=3) == 1 and b"divide" in L.vitk_last_error()
    assert call(batch=0) == 1 and call(groups=0) == 1 and call(channels=-8) == 1
    assert call(act=4) == 1 and call(act=-1) == 1
    assert call(dtype=7) == 2
    assert call(batch=70000) == 2
    assert call(rstd=None) == 1
    assert call(floats=3) == 1 and b"needed" in L.vitk_last_error()
    assert L.vitk_group_norm_workspace(2, 5, 9, 2, 0, 0) == -1
    assert L.vitk_group_norm_backward(p, None, None, p, None, p, p, None, None, p, 1 << 20, 2, 5, 8, 2, 0, 0, None) == 1
    assert L.vitk_group_norm_backward(p, None, None, p, p, p, p, None, None, p, 2, 2, 5, 8, 2, 0, 0, None) == 1


@gpu
def test_refusals():
    x = torch.randn(2, 6, 6, 8, device="cuda")
    for bad in (dict(num_groups=3), dict(num_groups=0), dict(num_groups=2, activation="tanh"),
                dict(num_groups=2, weight=torch.ones(4, device="cuda")), dict(num_groups=2, bias=torch.ones(8)),
                dict(num_groups=2, weight=torch.ones(8, device="cuda", dtype=torch.bfloat16))):
        with pytest.raises(VitkError):
            vit_amd.group_norm(x, **bad)
    for t in (x.half(), x.double(), x.permute(0, 3, 1, 2), x[..., ::2], torch.ones(8, device="cuda")):
        with pytest.raises(VitkError):
            vit_amd.group_norm(t, 2)


@gpu
def test_sizes_beyond_the_counters_are_refused():
    x = torch.empty(1, 2 ** 32 + 8, 1, device="cuda", dtype=torch.bfloat16)    # 8 GiB, not read
    with pytest.raises(VitkError, match="too large"):
        vit_amd.group_norm(x, 1)
    with pytest.raises(VitkError):
        vit_amd.group_norm(x[:, :2 ** 30 + 1], 1)
